"""The forms that the decoding loop's kernels take at a serving batch's sizes: the launch rules go by the number of
tokens, of (sequence, KV head) pairs, of rows, so small cases do not reach them.  Formulas, bit comparisons and
tolerances are those of the operators' own tests."""
import random

import pytest
import torch


def _turned(x, at, f, layout, amplitude=1.0):
    """x [B, heads, Q, D] turned to positions [B, Q] in 64 bits; positions small enough for a plain product."""
    y = x.double().clone()
    n = f.numel()
    a = at.double()[:, None, :, None] * f
    c, s = amplitude * torch.cos(a), amplitude * torch.sin(a)
    u, w = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    x1, x2 = y[..., u].clone(), y[..., w].clone()
    y[..., u], y[..., w] = x1 * c - x2 * s, x2 * c + x1 * s
    return y


# four tokens a block: from 2368 tokens of sequences of at least 4 on
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,H,Hkv,Q,D,n", [(592, 2, 1, 4, 64, 16), (474, 3, 2, 5, 32, 16), (400, 1, 1, 6, 256, 128), (340, 5, 2, 7, 128, 40), (1, 4, 0, 2371, 64, 32)])
def test_rotation_of_many_tokens(dtype, layout, B, H, Hkv, Q, D, n):
    import flash_tree_attn_b200 as fta
    from test_rotary import _tolerance

    g = torch.Generator().manual_seed(Q)
    q, k = (torch.randn(B, h, Q, D, generator=g).to(dtype).cuda() for h in (H, max(Hkv, 1)))
    k = k if Hkv else None
    f, amplitude = fta.rotary_frequencies(2 * n, scaling="ramp", factor=4.0)
    start = torch.randint(0, 5000, (B,), generator=g).cuda()
    depth = torch.randint(0, 9, (Q,), generator=g).to(torch.int32).cuda()
    at = start[:, None] + depth
    for inverse in (False, True):
        got = fta.apply_rotary(q, k, start, f, offsets=depth, layout=layout, amplitude=amplitude, inverse=inverse)
        per_token = fta.apply_rotary(q, k, at, f, layout=layout, amplitude=amplitude, inverse=inverse)
        for x, y, z in zip((q, k), got, per_token):
            if x is None:
                continue
            assert torch.equal(y, z)
            ref = _turned(x, -at if inverse else at, f, layout, amplitude).cpu()
            assert ((y.double().cpu() - ref).abs() <= _tolerance(x, ref, dtype, n, layout, amplitude, 5009)).all()
            assert torch.equal(y[..., 2 * n:], x[..., 2 * n:])
            # few tokens a call take one token a block: the same bits
            few = min(B, max(1, 2000 // Q))
            part = fta.apply_rotary(x[:few, :, : min(Q, 2000)], None, at[:few, : min(Q, 2000)], f, layout=layout, amplitude=amplitude, inverse=inverse)[0]
            assert torch.equal(part, y[:few, :, : min(Q, 2000)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("page", [0, 64, 192])
@pytest.mark.parametrize("B,Q", [(40, 66), (48, 65), (37, 67), (37, 64)])
def test_append_of_a_chunk_is_that_of_its_tokens(dtype, layout, page, B, Q):
    """Chunks across page ends and past the cache's end, against one token a call, bit for bit."""
    import flash_tree_attn_b200 as fta

    H, Hkv, D, n, ctx = 3, 2, 64, 24, 384
    g = torch.Generator().manual_seed(B + Q + page)
    q, k, v = (torch.randn(B, h, Q, D, generator=g).to(dtype).cuda() for h in (H, Hkv, Hkv))
    lens = torch.randint(0, ctx + 1, (B,), generator=g)
    lens[:6] = torch.tensor([0, 63, ctx - Q, ctx - Q + 1, ctx - 1, ctx])
    pos = torch.randint(0, 10000, (B, Q), generator=g).cuda()
    f, _ = fta.rotary_frequencies(2 * n)
    table = None
    if page:
        per = ctx // page
        table = torch.randperm(B * per, generator=g).view(B, per).to(torch.int32).cuda()
        kc, vc = (torch.randn(B * per, Hkv, page, D, generator=g).to(dtype).cuda() for _ in "kv")
    else:
        kc, vc = (torch.randn(B, ctx, Hkv, D, generator=g).to(dtype).cuda().transpose(1, 2) for _ in "kv")
    k1, v1, n1 = kc.clone(), vc.clone(), lens.to(torch.int32).cuda()
    k2, v2, n2 = kc.clone(), vc.clone(), lens.cuda()
    whole = fta.append_tokens(k1, v1, q, k, v, n1, inv_freq=f, positions=pos, layout=layout, block_table=table)
    for i in range(Q):
        one = [t[:, :, i: i + 1] for t in (q, k, v)]
        part = fta.append_tokens(k2, v2, *one, n2, inv_freq=f, positions=pos[:, i: i + 1], layout=layout, block_table=table)
        assert torch.equal(whole[:, :, i: i + 1], part)
    assert torch.equal(k1, k2) and torch.equal(v1, v2)
    assert n1.tolist() == n2.tolist() == (lens + Q).clamp(max=ctx).tolist()
    # positions by default: the cache's rows
    k3, v3, n3 = kc.clone(), vc.clone(), lens.cuda()
    rows = lens.cuda()[:, None] + torch.arange(Q, device="cuda")
    by_default = fta.append_tokens(k3, v3, q, k, v, n3, inv_freq=f, layout=layout, block_table=table)
    given = fta.append_tokens(kc.clone(), vc.clone(), q, k, v, lens.cuda(), inv_freq=f, positions=rows, layout=layout, block_table=table)
    assert torch.equal(by_default, given)


# one block a KV head joins all of its heads: from 148 (sequence, KV head) pairs on
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,Hkv,G,D,ctx,page", [(80, 2, 1, 64, 4096, 64), (75, 2, 2, 128, 2100, 0), (50, 3, 4, 64, 3000, 0), (75, 2, 5, 128, 2112, 64), (75, 2, 3, 256, 1500, 0),
                                                (40, 4, 20, 32, 5000, 0), (150, 1, 9, 256, 1088, 64)])
def test_attention_of_a_batch(dtype, B, Hkv, G, D, ctx, page):
    from flash_tree_attn_b200 import decode
    from oracle.decode_oracle import decode_attention_oracle
    from test_decode_attention import _caches, _check

    rng = random.Random(ctx)
    lens = [rng.choice([0, 1, 64, rng.randint(1, 300)]) for _ in range(B)]
    lens[3], lens[-1], lens[B // 2] = ctx, ctx - 1, ctx // 2  # a few long ones, cut into many pieces
    k, v, table = _caches(B, Hkv, ctx, D, dtype, lens, page, ctx, "cuda")
    q = torch.randn(B, Hkv * G, 1, D, generator=torch.Generator().manual_seed(B)).to(dtype).cuda()
    n = torch.tensor(lens, device="cuda")
    ora = decode_attention_oracle(q, k, v, n, table, G)
    w = torch.zeros(B, Hkv, ctx, device="cuda")
    for weights in (None, w):
        out, lse = decode._decode(q, k, v, n, table, None, None, G, None, None, None, weights, True)
        _check(out, lse, weights, ora, dtype, D, None, None, ctx)
        again = decode._decode(q, k, v, n, table, None, None, G, None, None, None, None if weights is None else torch.zeros_like(w), True)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def _evict(B, Hkv, D, ctx, page, budget, recent, kind, lens, seed, dtype=torch.float16):
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import evict_oracle
    from test_evict import _weights

    g = torch.Generator().manual_seed(seed)
    table = None
    if page:
        per = ctx // page
        table = torch.randperm(B * per, generator=g).view(B, per).to(torch.int32).cuda()
        k, v = (torch.randn(B * per, Hkv, page, D, generator=g).to(dtype).cuda() for _ in "kv")
    else:
        k, v = (torch.randn(B, Hkv, ctx, D, generator=g).to(dtype).cuda() for _ in "kv")
    w = _weights(kind, B, Hkv, ctx, lens, g).cuda()
    n = torch.tensor(lens, device="cuda")
    want = evict_oracle(k, v, n, w, budget, recent, table)
    kept = fta.evict_rows(k, v, n, w, budget, recent, block_table=table)
    for got, ref in zip((k, v, n, w.view(torch.int32), kept), want):
        assert torch.equal(got.cpu(), ref.view(torch.int32) if ref.dtype is torch.float32 else ref)


# a block a (sequence, KV head) moves rows from 222 pairs on, clusters of two from 111, of four from 56
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "ties", "odd"])
@pytest.mark.parametrize("B,Hkv,D,ctx,page,budget,recent", [(37, 6, 32, 512, 0, 100, 7), (60, 4, 64, 384, 192, 130, 0), (30, 4, 32, 448, 64, 64, 64), (15, 4, 128, 320, 0, 111, 20),
                                                            (15, 4, 256, 576, 192, 300, 31), (3, 2, 64, 1152, 192, 500, 1)])
def test_eviction_of_a_batch(kind, B, Hkv, D, ctx, page, budget, recent):
    rng = random.Random(B + D)
    lens = [rng.choice([0, 1, budget, budget + 1, ctx, rng.randint(0, ctx), rng.randint(0, ctx)]) for _ in range(B)]
    lens[0] = ctx
    _evict(B, Hkv, D, ctx, page, budget, recent, kind, lens, B * D)


# weights of more than 24576 old rows are read again in every pass
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("ctx,page,budget,recent,lens", [
    (24641, 0, 4096, 64, [24576 + 64, 24576 + 65, 24641]), (30016, 64, 20000, 0, [24576, 24577, 30000]), (52992, 192, 8191, 5000, [52992, 100, 29577]),
    (40000, 0, 39999, 0, [40000, 39999, 0]), (70000, 0, 3, 2, [70000, 24579])])
def test_eviction_of_long_caches(kind, ctx, page, budget, recent, lens):
    _evict(len(lens), 2, 32, ctx, page, budget, recent, kind, lens, ctx, torch.bfloat16)


# a block a row and several rounds: many rows of a whole vocabulary
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,k", [(600, 40000, 20), (593, 33001, 64), (650, 50257, 1), (600, 20000, 0)])
def test_logits_of_many_rows(dtype, rows, V, k):
    import flash_tree_attn_b200 as fta
    from test_logprobs import _check, _tokens

    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn(rows, V, generator=g)).to(dtype)
    x[5] = 1.5                                   # equals
    x[6, : V - 30] = float("-inf")               # what is left stands at the end
    x[7] = torch.arange(V).float() * 1e-3        # every round passes the one before
    x[8] = -x[7]
    x[9, V // 3] = float("nan")
    x[10] = torch.finfo(dtype).min
    x = x.cuda()
    t = _tokens(rows, V, 3, g)
    _check(x, t, k, fta.token_logprobs(x, t, k))
