"""CPU restatement, in 64 bits and plain loops, of the decoding-loop operators beside tree verification
(test infrastructure only: imported by tests/, never by the product path).  The reference has no such
operators; the rules restated are those include/fta.h states."""
from __future__ import annotations

import math

import torch


def sequence_rows(cache, block_table, b, n):
    """Rows [0, n) of sequence b of a dense or paged cache, [Hkv, n, D]."""
    if block_table is None:
        return cache[b, :, :n]
    page = cache.size(2)
    parts = [cache[int(block_table[b, s])] for s in range(-(-n // page))]
    return torch.cat(parts, 1)[:, :n] if parts else cache[0][:, :0]


def decode_attention_oracle(q, k_cache, v_cache, kv_seq_len, block_table=None, kv_group_num=1, sm_scale=None, softcap=None,
                            alibi_slopes=None, window=None):
    """out, lse, the weights of every row [B, Hkv, longest], sum_r p_r |v_r| (the scale of out's
    rounding errors) and sum_i |q_i k_i| * scale at its largest (the scale of a score's)."""
    q, k_cache, v_cache = (t.detach().cpu() for t in (q, k_cache, v_cache))
    table = None if block_table is None else block_table.cpu()
    B, H, _, D = q.shape
    G = kv_group_num
    Hkv = H // G
    lens = [int(x) for x in kv_seq_len]
    scale = 1.0 / math.sqrt(D) if sm_scale is None else sm_scale
    out = torch.zeros(B, H, 1, D, dtype=torch.float64)
    size = torch.zeros_like(out)
    lse = torch.full((B, H, 1), float("-inf"), dtype=torch.float64)
    weights = torch.zeros(B, Hkv, max(lens + [1]), dtype=torch.float64)
    most = 0.0
    for b, L in enumerate(lens):
        lo = max(0, L - window) if window else 0
        if L == 0:
            continue
        k = sequence_rows(k_cache, table, b, L)[:, lo:].double()
        v = sequence_rows(v_cache, table, b, L)[:, lo:].double()
        for h in range(H):
            kk, vv, x = k[h // G], v[h // G], q[b, h, 0].double()
            s = kk @ x * scale
            most = max(most, float((kk.abs() @ x.abs()).max()) * scale)
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            if alibi_slopes is not None:
                s = s + float(alibi_slopes[h]) * torch.arange(lo - (L - 1), 1, dtype=torch.float64)
            lse[b, h, 0] = torch.logsumexp(s, 0)
            p = torch.exp(s - lse[b, h, 0])
            out[b, h, 0], size[b, h, 0] = p @ vv, p @ vv.abs()
            weights[b, h // G, lo:L] += p
    return {"out": out, "lse": lse, "weights": weights, "size": size, "score": most}


def rotary_oracle(x, positions, inv_freq, layout="half", amplitude=1.0, inverse=False):
    """x [B, heads, Q, D] turned to positions [B][Q] (Python integers), in 64 bits."""
    y = x.detach().cpu().double().clone()
    f = [float(v) for v in inv_freq]
    n = len(f)
    for b in range(x.size(0)):
        for i in range(x.size(2)):
            for j in range(n):
                a = math.fmod(int(positions[b][i]) * f[j], 2.0 * math.pi)
                c, s = amplitude * math.cos(a), amplitude * math.sin(a) * (-1.0 if inverse else 1.0)
                u, w = (j, n + j) if layout == "half" else (2 * j, 2 * j + 1)
                x1, x2 = y[b, :, i, u].clone(), y[b, :, i, w].clone()
                y[b, :, i, u], y[b, :, i, w] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


def write_rows(cache, block_table, b, row, values):
    """cache row `row` of sequence b becomes values [Hkv, D]."""
    if block_table is None:
        cache[b, :, row] = values
    else:
        page = cache.size(2)
        cache[int(block_table[b, row // page]), :, row % page] = values


def evict_oracle(k_cache, v_cache, kv_seq_len, row_weights, budget, recent, block_table=None):
    """New CPU tensors (k, v, lengths, weights, kept)."""
    k, v, w = (t.detach().cpu().clone() for t in (k_cache, v_cache, row_weights))
    table = None if block_table is None else block_table.cpu()
    lens = kv_seq_len.detach().cpu().clone()
    B, Hkv = w.shape[:2]
    kept = torch.full((B, Hkv, budget), -1, dtype=torch.int32)
    for b in range(B):
        L = int(lens[b])
        new_k, new_v = (sequence_rows(t, table, b, L).clone() for t in (k, v))
        for h in range(Hkv):
            rows = list(range(L))
            if L > budget:
                x = w[b, h].tolist()
                size = [math.inf if math.isnan(t) else t for t in x]
                nan = [math.isnan(t) for t in x]
                old = sorted(range(L - recent), key=lambda r: (not nan[r], -size[r], r))[: budget - recent]
                rows = sorted(old) + list(range(L - recent, L))
                moved = w[b, h, rows].clone()
                w[b, h, :L] = 0
                w[b, h, : len(rows)] = moved
                new_k[h, : len(rows)], new_v[h, : len(rows)] = new_k[h, rows].clone(), new_v[h, rows].clone()
            kept[b, h, : len(rows)] = torch.tensor(rows, dtype=torch.int32)
        if L > budget:
            for r in range(budget):
                write_rows(k, table, b, r, new_k[:, r])
                write_rows(v, table, b, r, new_v[:, r])
            lens[b] = budget
    return k, v, lens, w, kept


def logprobs_oracle(logits, tokens, top_k):
    """(logprobs, entropy, lse, top_logprobs, top_ids) of [rows, vocab], in 64 bits."""
    x = logits.detach().cpu().double()
    rows, V = x.shape
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isneginf(m), torch.zeros_like(m), m)
    e = torch.exp(x - m)
    s = e.sum(-1, keepdim=True)
    lse = (m + torch.log(s))[:, 0]
    lp = x - m - torch.log(s)
    entropy = -torch.where(e == 0, torch.zeros_like(e), e / s * lp).sum(-1)
    dead = s[:, 0] == 0
    lp[dead], lse[dead], entropy[dead] = -math.inf, -math.inf, 0.0
    lp[torch.isnan(s[:, 0])] = math.nan
    given = torch.full(tokens.shape, -math.inf, dtype=torch.float64)
    inside = (tokens >= 0) & (tokens < V)
    given[inside] = lp.gather(-1, tokens.long().clamp(0, V - 1))[inside]
    order = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x + 0.0)
    rank = torch.argsort(order, dim=-1, descending=True, stable=True)
    for r in range(rows):  # NaN before inf
        if torch.isnan(x[r]).any():
            at = rank[r].tolist()
            rank[r] = torch.tensor([i for i in at if math.isnan(x[r, i])] + [i for i in at if not math.isnan(x[r, i])])
    ids = rank[:, :top_k]
    return given, entropy, lse, lp.gather(-1, ids), ids
