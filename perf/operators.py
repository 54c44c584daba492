"""The decoding-loop operators beside tree verification, as measured workloads: attention of one new
token over the cache, rotary positions with the cache append, eviction of cache rows by accumulated
attention weight, and log probabilities of given tokens.

`own` chooses between this package's operators and a plain form of the same mathematics in elementary
torch operations.  `exact` states each operator once more in 64 bits.  Lengths are a function of the
case alone; values come from the seed.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------


def attend(name, B, H, Hkv, D, lo, hi, dtype="bf16", page=0, softcap=0.0, alibi=False, window=0, weights=False):
    return {"name": name, "op": "attend", "B": B, "H": H, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "dtype": dtype, "page": page,
            "softcap": softcap, "alibi": alibi, "window": window, "weights": weights}


def append(name, B, H, Hkv, D, Q, lo, hi, rot, layout="half", scaling="none", base=10000.0, dtype="bf16", page=0):
    return {"name": name, "op": "append", "B": B, "H": H, "Hkv": Hkv, "D": D, "Q": Q, "lo": lo, "hi": hi, "rot": rot, "layout": layout,
            "scaling": scaling, "base": base, "dtype": dtype, "page": page}


def rotate(name, B, H, Hkv, D, Q, lo, hi, rot, layout="half", scaling="none", base=10000.0, dtype="bf16", inverse=False):
    return {"name": name, "op": "rotate", "B": B, "H": H, "Hkv": Hkv, "D": D, "Q": Q, "lo": lo, "hi": hi, "rot": rot, "layout": layout,
            "scaling": scaling, "base": base, "dtype": dtype, "inverse": inverse}


def evict(name, B, Hkv, D, lo, hi, budget, recent, dtype="bf16", page=0):
    return {"name": name, "op": "evict", "B": B, "Hkv": Hkv, "D": D, "lo": lo, "hi": hi, "budget": budget, "recent": recent, "dtype": dtype,
            "page": page}


def logprobs(name, rows, V, n, k, dtype="bf16", pad=0):
    return {"name": name, "op": "logprobs", "rows": rows, "V": V, "n": n, "k": k, "dtype": dtype, "pad": pad}


def listed():
    return [
        # a single chat just after its prompt: latency is all that counts
        attend("attend one chat", 1, 32, 8, 128, 1000, 1000),
        # a serving batch over a paged cache, lengths as ragged as requests are
        attend("attend paged batch", 64, 32, 8, 128, 16, 8192, page=64),
        # one document of 128k tokens: the cache's length has to be split over the machine; weights kept for eviction
        attend("attend long weights", 1, 64, 8, 128, 131072, 131072, page=64, weights=True),
        # a model with capped scores and a sliding window, wide heads
        attend("attend capped window", 16, 16, 8, 256, 500, 16384, dtype="fp16", softcap=50.0, window=4096),
        # plain multi-head attention with a distance bias, odd lengths
        attend("attend distance bias", 8, 32, 32, 128, 777, 3001, dtype="fp16", alibi=True),
        # the decode step of one chat: rotate q and k, append k and v
        append("append one token", 1, 32, 8, 128, 1, 1000, 1000, 128),
        # a chunk of a long prompt at far positions, interleaved pairs in half of the head, paged cache
        append("append prompt chunk", 8, 32, 8, 128, 2048, 5000, 30000, 64, layout="interleaved", scaling="ramp", page=64),
        # the 26 nodes of a draft tree for a batch of 32: positions follow the nodes' depths
        rotate("rotate draft trees", 32, 32, 8, 128, 26, 2048, 8192, 128, scaling="bands", base=500000.0),
        # one long chat is brought back to half of its cache
        evict("evict one chat", 1, 8, 128, 4100, 4100, 2048, 256),
        # a batch over its budget, paged
        evict("evict paged batch", 32, 8, 128, 4500, 8192, 4096, 512, page=64),
        # the next token's distribution for one row, five alternatives shown
        logprobs("logprobs one row", 1, 128256, 1, 5),
        # every node of 32 draft trees scored against its children, odd vocabulary
        logprobs("logprobs draft trees", 832, 50257, 4, 20, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "rotate", "evict", "logprobs"])
    dtype = rng.choice(["bf16", "fp16"])
    D, Hkv, G = rng.choice([32, 64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16])
    page = rng.choice([0, 64, 128])
    if op == "attend":
        B = _log(rng, 1, 64)
        hi = _log(rng, 1, max(2, min(131072, 64 * 8192 * 8 * 128 // (B * Hkv * D * max(1, G // 4)))))
        return attend("", B, Hkv * G, Hkv, D, _log(rng, 1, hi), hi, dtype, page, rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.3,
                      rng.choice([0, 0, _log(rng, 1, hi)]), rng.random() < 0.3)
    rot = rng.choice([r for r in (16, 32, 48, 64, 96, 128, 256) if r <= D])
    layout, scaling = rng.choice(["half", "interleaved"]), rng.choice(["none", "linear", "base", "bands", "ramp"])
    if op == "append":
        B = _log(rng, 1, 64)
        Q = _log(rng, 1, max(2, 8 * 2048 * 48 * 128 // (B * (G + 2) * Hkv * D * 2)))
        hi = max(1, min(_log(rng, 64, 65536), 4_000_000 // (B * Hkv)))
        return append("", B, Hkv * G, Hkv, D, min(Q, 4096), _log(rng, 1, hi), hi, rot, layout, scaling, rng.choice([10000.0, 1e6]), dtype, page)
    if op == "rotate":
        B = _log(rng, 1, 64)
        Q = _log(rng, 1, max(2, 8 * 2048 * 40 * 128 // (B * (G + 1) * Hkv * D)))
        hi = _log(rng, 64, 1_000_000)
        return rotate("", B, Hkv * G, Hkv, D, min(Q, 4096), _log(rng, 1, hi), hi, rot, layout, scaling, rng.choice([10000.0, 1e6]), dtype,
                      rng.random() < 0.5)
    if op == "evict":
        B = _log(rng, 1, 32)
        hi = _log(rng, 64, max(65, min(65536, 32 * 8 * 8192 * 128 // (B * Hkv * D))))
        budget = rng.randint(1, hi)
        return evict("", B, Hkv, D, _log(rng, 1, hi), hi, budget, rng.randint(0, budget), dtype, page)
    V = _log(rng, 100, 262144)
    rows = _log(rng, 1, max(2, 832 * 50257 // V))
    return logprobs("", rows, V, rng.randint(1, 8), rng.choice([0, 1, 5, 20, 64]), rng.choice(["bf16", "fp16", "fp32"]), rng.choice([0, 8, 3]))


# ---- inputs -------------------------------------------------------------------------------------


def lengths(c):
    """Cache lengths of the case: spread over [lo, hi] by the golden ratio, the last one at hi."""
    frac = [(b * 0.6180339887498949) % 1.0 for b in range(1, c["B"])] + [1.0]
    return [c["lo"] + int(round((c["hi"] - c["lo"]) * f)) for f in frac]


def frequencies(rot, base, scaling):
    """Radians per position of the rot / 2 pairs, as Python floats (64 bits), and the factor on cosine and sine."""
    dims = [2.0 * i / rot for i in range(rot // 2)]
    factor, original, amplitude = 8.0, 8192.0, 1.0
    if scaling == "base":
        base = base * factor ** (rot / (rot - 2.0))
    f = [base ** -d for d in dims]
    if scaling == "linear":
        f = [x / factor for x in f]
    if scaling == "bands":  # long wavelengths are stretched, short ones kept, a blend between
        lo, hi, g = 1.0, 4.0, []
        for x in f:
            turns = original * x / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - lo) / (hi - lo)))
            g.append(x * keep + x / factor * (1.0 - keep))
        f = g
    if scaling == "ramp":  # the blend runs over the pair's index between two numbers of rotations
        def at(rotations):
            return rot * math.log(original / (rotations * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        g = []
        for i, x in enumerate(f):
            keep = 1.0 - min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            g.append(x * keep + x / factor * (1.0 - keep))
        f, amplitude = g, 0.1 * math.log(factor) + 1.0
    return f, amplitude


def tree_depths(Q):
    """Depths of a draft tree's nodes: node i > 0 hangs below node (i - 1) // 3."""
    depth = [0] * Q
    for i in range(1, Q):
        depth[i] = depth[(i - 1) // 3] + 1
    return depth


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, dtype):
        t = torch.empty(shape, dtype=dtype, device="cuda")
        return t.normal_(generator=g)

    dt = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "logprobs":
        wide = randn(c["rows"], c["V"] + c["pad"], dtype=dt).mul_(3.0)
        s["logits"] = wide[:, : c["V"]]
        s["tokens"] = torch.randint(0, c["V"], (c["rows"], c["n"]), generator=g, device="cuda")
        return s
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    lens = lengths(c)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    room = c["hi"] + c.get("Q", 0)
    if c["op"] != "rotate":
        if c["page"]:
            per = -(-room // c["page"])
            order = torch.randperm(B * per, generator=g, device="cuda").to(torch.int32)
            s["table"] = order.view(B, per)
            s["k"], s["v"] = (randn(B * per, Hkv, c["page"], D, dtype=dt) for _ in "kv")
            s["ctx"] = per * c["page"]
        else:
            s["table"] = None
            s["k"], s["v"] = (randn(B, Hkv, room, D, dtype=dt) for _ in "kv")
            s["ctx"] = room
    if c["op"] == "attend":
        s["q"] = randn(B, c["H"], 1, D, dtype=dt)
        s["slopes"] = None
        if c["alibi"]:
            s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / c["H"]) for h in range(c["H"])], device="cuda")
        s["weights"] = torch.zeros(B, Hkv, s["ctx"], device="cuda") if c["weights"] else None
    if c["op"] in ("append", "rotate"):
        s["q"] = randn(B, c["H"], c["Q"], D, dtype=dt)
        s["new_k"] = randn(B, Hkv, c["Q"], D, dtype=dt)
        f, s["amplitude"] = frequencies(c["rot"], c["base"], c["scaling"])
        s["inv_freq"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        s["offsets"] = torch.tensor(tree_depths(c["Q"]), dtype=torch.int32, device="cuda")
    if c["op"] == "append":
        s["new_v"] = randn(B, Hkv, c["Q"], D, dtype=dt)
        s["lens_now"] = s["lens"].clone()
    if c["op"] == "evict":
        # accumulated weights span orders of magnitude; a tenth of the rows was never looked at (ties at 0)
        w = torch.exp(2.5 * torch.randn(B, Hkv, s["ctx"], generator=g, device="cuda"))
        w = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.1, 0.0, w)
        rows = torch.arange(s["ctx"], device="cuda")
        s["weights"] = torch.where(rows < s["lens"][:, None, None], w, 0.0)
        s["weights_now"], s["lens_now"] = s["weights"].clone(), s["lens"].clone()
    return s


# ---- one pass -----------------------------------------------------------------------------------


def run(s):
    return RUN[s["case"]["op"]](s)


def run_attend(s):
    c = s["case"]
    G = c["H"] // c["Hkv"]
    if own:
        import flash_tree_attn_b200 as fta

        opts = dict(kv_group_num=G, softcap=c["softcap"] or None, alibi_slopes=s["slopes"], window=c["window"] or None,
                    row_weights=s["weights"])
        if c["page"]:
            out = fta.decode_attention_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], **opts)
        else:
            out = fta.decode_attention(s["q"], s["k"], s["v"], s["lens"], **opts)
        return {"out": out, "weights": s["weights"]} if c["weights"] else {"out": out}
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    k, v = s["k"], s["v"]
    if c["page"]:
        k, v = (t[s["table"].long()].transpose(1, 2).reshape(B, Hkv, s["ctx"], D) for t in (k, v))
    scores = s["q"].float().view(B, Hkv, G, D) @ k.float().transpose(-1, -2) * (1.0 / math.sqrt(D))
    rows = torch.arange(s["ctx"], device=k.device)
    L = s["lens"][:, None, None, None]
    if c["softcap"]:
        scores = c["softcap"] * torch.tanh(scores / c["softcap"])
    if c["alibi"]:
        scores = scores + s["slopes"].view(1, Hkv, G, 1) * (rows - (L - 1)).float()
    seen = rows < L
    if c["window"]:
        seen = seen & (rows >= L - c["window"])
    scores = scores.masked_fill(~seen, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = (p @ v.float()).view(B, H, 1, D).to(s["q"].dtype)
    if c["weights"]:
        s["weights"].add_(p.sum(2))
        return {"out": out, "weights": s["weights"]}
    return {"out": out}


def turn(x, cos, sin, layout):
    """x [B, heads, Q, D] in 32 bits, cos and sin [B, 1, Q, rot / 2]."""
    half = cos.shape[-1]
    a, rest = x[..., : 2 * half], x[..., 2 * half:]
    if layout == "half":
        x1, x2 = a[..., :half], a[..., half:]
        y = torch.cat((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1)
    else:
        x1, x2 = a[..., 0::2], a[..., 1::2]
        y = torch.stack((x1 * cos - x2 * sin, x2 * cos + x1 * sin), -1).flatten(-2)
    return torch.cat((y, rest), -1)


def cos_sin(positions, s, sign=1.0):
    angle = positions.double()[..., None] * s["inv_freq"]  # far positions need 64 bits
    return (torch.cos(angle) * s["amplitude"]).float()[:, None], (torch.sin(angle) * (sign * s["amplitude"])).float()[:, None]


def run_append(s):
    c = s["case"]
    lens = s["lens_now"]
    lens.copy_(s["lens"])  # the same step again: the operator lets the lengths grow
    if own:
        import flash_tree_attn_b200 as fta

        q = fta.append_tokens(s["k"], s["v"], s["q"], s["new_k"], s["new_v"], lens, inv_freq=s["inv_freq"], layout=c["layout"],
                              amplitude=s["amplitude"], block_table=s["table"])
        return {"q": q, "k": s["k"], "v": s["v"], "lens": lens}
    rows = lens.long()[:, None] + torch.arange(c["Q"], device=lens.device)
    cos, sin = cos_sin(rows, s)
    q = turn(s["q"].float(), cos, sin, c["layout"]).to(s["q"].dtype)
    k = turn(s["new_k"].float(), cos, sin, c["layout"]).to(s["q"].dtype)
    at = torch.arange(c["B"], device=lens.device)[:, None]
    if c["page"]:
        at, rows = s["table"].long().gather(1, rows // c["page"]), rows % c["page"]
    s["k"][at, :, rows] = k.transpose(1, 2)
    s["v"][at, :, rows] = s["new_v"].transpose(1, 2)
    lens.add_(c["Q"])
    return {"q": q, "k": s["k"], "v": s["v"], "lens": lens}


def run_rotate(s):
    c = s["case"]
    if own:
        import flash_tree_attn_b200 as fta

        q, k = fta.apply_rotary(s["q"], s["new_k"], s["lens"], s["inv_freq"], offsets=s["offsets"], layout=c["layout"],
                                amplitude=s["amplitude"], inverse=c["inverse"])
        return {"q": q, "k": k}
    cos, sin = cos_sin(s["lens"].long()[:, None] + s["offsets"], s, -1.0 if c["inverse"] else 1.0)
    return {"q": turn(s["q"].float(), cos, sin, c["layout"]).to(s["q"].dtype), "k": turn(s["new_k"].float(), cos, sin, c["layout"]).to(s["q"].dtype)}


def run_evict(s):
    c = s["case"]
    weights, lens = s["weights_now"], s["lens_now"]
    weights.copy_(s["weights"])  # the same step again: eviction works in place
    lens.copy_(s["lens"])
    if own:
        import flash_tree_attn_b200 as fta

        kept = fta.evict_rows(s["k"], s["v"], lens, weights, c["budget"], c["recent"], block_table=s["table"])
        return {"k": s["k"], "v": s["v"], "weights": weights, "lens": lens, "kept": kept}
    n = c["budget"]
    rows = torch.arange(s["ctx"], device=lens.device)
    L = lens.long()[:, None, None]
    # one whole number orders the rows: the weight (not negative, so its bits are ordered), then the lower row first
    order = ((weights + 0.0).view(torch.int32).long() << 24) | (0xFFFFFF - rows)
    order = torch.where(rows >= L - c["recent"], order | (1 << 60), order)
    order = torch.where(rows >= L, -1 - rows, order)
    kept = torch.topk(order, min(n, s["ctx"]), dim=-1).indices.sort(-1).values
    kept = torch.nn.functional.pad(kept, (0, n - kept.shape[-1]))
    new = torch.arange(n, device=lens.device)
    live = new < L
    B, Hkv, D = c["B"], c["Hkv"], c["D"]
    b = torch.arange(B, device=lens.device)[:, None, None]
    h = torch.arange(Hkv, device=lens.device)[None, :, None]
    src, dst = kept, torch.where(live, new, 0).expand(B, Hkv, n)
    src = torch.where(live, src, src[..., :1])  # places past a short sequence's end repeat its first row
    w = torch.where(live, weights.gather(-1, src), 0.0)
    if c["page"]:
        table = s["table"].long()
        from_at, from_row = table[b, src // c["page"]], src % c["page"]
        to_at, to_row = table[b, dst // c["page"]], dst % c["page"]
    else:
        from_at, from_row, to_at, to_row = b, src, b, dst
    k, v = s["k"][from_at, h, from_row], s["v"][from_at, h, from_row]
    s["k"][to_at, h, to_row] = k
    s["v"][to_at, h, to_row] = v
    weights.masked_fill_((rows >= n) & (rows < L), 0.0)
    weights[..., : min(n, s["ctx"])] = torch.where(live, w, 0.0)[..., : s["ctx"]]
    lens.clamp_(max=n)
    return {"k": s["k"], "v": s["v"], "weights": weights, "lens": lens, "kept": torch.where(live, kept, -1).int()}


def run_logprobs(s):
    c = s["case"]
    if own:
        import flash_tree_attn_b200 as fta

        r = fta.token_logprobs(s["logits"], s["tokens"], top_k=c["k"])
        out = {"logprobs": r.logprobs, "entropy": r.entropy, "lse": r.lse}
        return {**out, "top_logprobs": r.top_logprobs, "top_ids": r.top_ids} if c["k"] else out
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    out = {"logprobs": x.gather(-1, s["tokens"]) - lse, "entropy": (torch.log(total) - (e * d).sum(-1, keepdim=True) / total)[:, 0],
           "lse": lse[:, 0]}
    if c["k"]:
        # ties go to the lowest token: the value's ordered bits and the token make one whole number
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
        key = (bits << 20) | (0xFFFFF - torch.arange(c["V"], device=x.device))
        ids = 0xFFFFF - (torch.topk(key, c["k"], dim=-1).values & 0xFFFFF)
        out["top_logprobs"], out["top_ids"] = x.gather(-1, ids) - lse, ids
    return out


RUN = {"attend": run_attend, "append": run_append, "rotate": run_rotate, "evict": run_evict, "logprobs": run_logprobs}


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "logprobs":
        n = c["rows"] * c["V"]
        return {"bytes": n * size + c["rows"] * (8 + c["n"] * 12 + c["k"] * 12), "flops": 5 * n}
    lens = lengths(c)
    row = c["Hkv"] * c["D"] * size
    if c["op"] == "attend":
        seen = sum(min(L, c["window"]) if c["window"] else L for L in lens)
        return {"bytes": 2 * row * seen + 2 * c["B"] * c["H"] * c["D"] * size + (8 * c["Hkv"] * seen if c["weights"] else 0),
                "flops": 4 * c["H"] * c["D"] * seen}
    if c["op"] in ("append", "rotate"):
        heads = c["H"] + (2 if c["op"] == "append" else 1) * c["Hkv"]
        n = c["B"] * c["Q"] * heads * c["D"]
        return {"bytes": 2 * n * size, "flops": 3 * n}
    kept = sum(min(L, c["budget"]) for L in lens if L > c["budget"])
    # the weights are read, written and cleared; of K and V the kept rows are read and written
    return {"bytes": 4 * row * kept + c["Hkv"] * (8 * sum(lens) + 4 * c["B"] * c["budget"]) + 1, "flops": c["Hkv"] * sum(lens)}


# ---- the same in 64 bits ------------------------------------------------------------------------


def exact(case, seed):
    c = dict(case)
    s = prepare(c, seed)
    return {"attend": exact_attend, "append": exact_append, "rotate": exact_rotate, "evict": exact_evict, "logprobs": exact_logprobs}[c["op"]](c, s)


def sequence_rows(s, c, cache, b, n):
    """The first n rows of sequence b, [Hkv, n, D]."""
    if not c["page"]:
        return cache[b, :, :n]
    pages = cache[s["table"][b, : -(-n // c["page"])].long()]
    return pages.permute(1, 0, 2, 3).flatten(1, 2)[:, :n]


def exact_attend(c, s):
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    G = H // Hkv
    out = torch.zeros(B, H, 1, D, dtype=torch.float64, device="cuda")
    weights = torch.zeros(B, Hkv, s["ctx"], dtype=torch.float64, device="cuda") if c["weights"] else None
    for b, L in enumerate(lengths(c)):
        first = max(0, L - c["window"]) if c["window"] else 0
        k, v = (sequence_rows(s, c, s[t], b, L)[:, first:].double() for t in "kv")
        for h in range(Hkv):
            x = torch.mv(k[h], s["q"][b, h * G, 0].double())[None] if G == 1 else s["q"][b, h * G:(h + 1) * G, 0].double() @ k[h].T
            x = x / D ** 0.5
            if c["softcap"]:
                x = torch.tanh(x / c["softcap"]) * c["softcap"]
            if c["alibi"]:
                back = torch.arange(L - first - 1, -1, -1, dtype=torch.float64, device="cuda")
                x = x - s["slopes"][h * G:(h + 1) * G, None].double() * back
            p = torch.softmax(x, -1)
            out[b, h * G:(h + 1) * G, 0] = p @ v[h]
            if c["weights"]:
                weights[b, h, first:L] = p.sum(0)
    return {"out": out, "weights": weights} if c["weights"] else {"out": out}


def exact_turn(x, positions, s, c, inverse):
    """x [B, heads, Q, D]; pair i of a head is the complex number that turns by position * frequency."""
    f = s["inv_freq"]
    angle = positions.double()[:, :, None] * f
    by = torch.polar(torch.full_like(angle, s["amplitude"]), -angle if inverse else angle)[:, None]
    y = x.double().clone()
    n = f.numel()
    first, second = (slice(0, n), slice(n, 2 * n)) if c["layout"] == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    z = torch.complex(y[..., first], y[..., second]) * by
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact_append(c, s):
    lens = lengths(c)
    at = torch.tensor(lens, device="cuda")[:, None] + torch.arange(c["Q"], device="cuda")
    k = exact_turn(s["new_k"], at, s, c, False)
    cache_k, cache_v = s["k"].double(), s["v"].double()
    for b, L in enumerate(lens):
        if not c["page"]:
            cache_k[b, :, L:L + c["Q"]], cache_v[b, :, L:L + c["Q"]] = k[b], s["new_v"][b].double()
            continue
        i = 0
        while i < c["Q"]:
            page, r = divmod(L + i, c["page"])
            n = min(c["page"] - r, c["Q"] - i)
            page = int(s["table"][b, page])
            cache_k[page, :, r:r + n], cache_v[page, :, r:r + n] = k[b, :, i:i + n], s["new_v"][b, :, i:i + n].double()
            i += n
    return {"q": exact_turn(s["q"], at, s, c, False), "k": cache_k, "v": cache_v, "lens": None}


def exact_rotate(c, s):
    at = torch.tensor(lengths(c), device="cuda")[:, None] + torch.tensor(tree_depths(c["Q"]), device="cuda")
    return {"q": exact_turn(s["q"], at, s, c, c["inverse"]), "k": exact_turn(s["new_k"], at, s, c, c["inverse"])}


def exact_evict(c, s):
    """K and V are copies and not computed numbers; the weights that move with them say where each row went."""
    if sum(lengths(c)) * c["Hkv"] > 1 << 22:
        return None
    weights = s["weights"].cpu().double()
    for b, L in enumerate(lengths(c)):
        if L <= c["budget"]:
            continue
        for h in range(c["Hkv"]):
            w = weights[b, h].tolist()
            old = sorted(range(max(0, L - c["recent"])), key=lambda r: (-w[r], r))[: c["budget"] - c["recent"]]
            rows = sorted(old) + list(range(L - c["recent"], L))
            weights[b, h, :L] = torch.tensor([w[r] for r in rows] + [0.0] * (L - len(rows)), dtype=torch.float64)
    return {"k": None, "v": None, "weights": weights, "lens": None, "kept": None}


def exact_logprobs(c, s):
    out = {"logprobs": [], "entropy": [], "lse": [], "top_logprobs": []}
    for x, tokens in zip(s["logits"].split(64), s["tokens"].split(64)):
        x = x.double()
        lp = torch.log_softmax(x, -1)
        out["logprobs"].append(lp.gather(-1, tokens))
        out["entropy"].append(-(lp.exp() * lp).sum(-1))
        out["lse"].append(torch.logsumexp(x, -1))
        if c["k"]:
            out["top_logprobs"].append(torch.topk(lp, c["k"], dim=-1).values)
    out = {name: torch.cat(v) for name, v in out.items() if v}
    return {**out, "top_ids": None} if c["k"] else out
