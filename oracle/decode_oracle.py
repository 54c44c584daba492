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
