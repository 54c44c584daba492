"""Rotary positions (apply_rotary, rotary_frequencies) and the cache append (append_tokens) against a plain
statement in 64 bits, and their refusals.

Tolerance of a turned element: one rounding to the type (u = eps / 2), and in 32 bits the angle's rounding
(2^-25 of pi), the cosine's and sine's (2^-23) and three roundings of the products (2^-24 each), together
below 2^-21 of |x1| + |x2|, plus what one rounding of inv_freq / 2 pi in 64 bits and one of the
oracle's product make at a far position: position * inv_freq * 2^-51.  fp16 results below 2^-14 are off by up to 2^-25."""
import ctypes as C
import math

import pytest
import torch

from flash_tree_attn_b200 import _lib


def _tolerance(x, ref, dtype, n, layout, amplitude, far):
    t = torch.finfo(dtype).eps / 2 * ref.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    a = x.detach().cpu().double().abs()
    size = torch.zeros_like(a)
    if layout == "half":
        both = a[..., :n] + a[..., n: 2 * n]
        size[..., :n], size[..., n: 2 * n] = both, both
    else:
        both = a[..., 0: 2 * n: 2] + a[..., 1: 2 * n: 2]
        size[..., 0: 2 * n: 2], size[..., 1: 2 * n: 2] = both, both
    return t + size * abs(amplitude) * (2.0 ** -21 + far * 2.0 ** -51)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("B,H,Hkv,Q,D,n,first", [
    (1, 1, 1, 1, 32, 8, 0), (3, 5, 1, 7, 64, 8, 131071), (2, 4, 2, 26, 128, 64, 1 << 20), (2, 3, 0, 5, 128, 16, 2 ** 31 - 3), (1, 2, 2, 3, 256, 128, 99),
    (2, 33, 3, 2, 96 + 160, 48, 5000)])
def test_matches_the_formula(dtype, layout, B, H, Hkv, Q, D, n, first):
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import rotary_oracle

    g = torch.Generator().manual_seed(n + Q)
    q, k = (torch.randn(B, h, Q, D, generator=g).to(dtype).cuda() for h in (H, max(Hkv, 1)))
    k = k if Hkv else None
    f, amplitude = fta.rotary_frequencies(2 * n, 10000.0, "ramp", 4.0)
    start = torch.tensor([first - 17 * b for b in range(B)], dtype=torch.int64, device="cuda")
    depth = torch.randint(0, 9, (Q,), generator=g).to(torch.int32)
    each = [[int(start[b]) + i for i in range(Q)] for b in range(B)]
    tree = [[int(start[b]) + int(depth[i]) for i in range(Q)] for b in range(B)]
    for inverse in (False, True):
        for offsets, at, positions in ((None, each, start), (depth.cuda(), tree, start), (None, tree, torch.tensor(tree, device="cuda")),
                                       (depth.cuda(), [[2 * t - s for t, s in zip(a, [int(start[b])] * Q)] for b, a in enumerate(tree)],
                                        torch.tensor(tree, device="cuda"))):
            got = fta.apply_rotary(q, k, positions, f, offsets=offsets, layout=layout, amplitude=amplitude, inverse=inverse)
            for x, y in zip((q, k), got):
                if x is None:
                    assert y is None
                    continue
                ref = rotary_oracle(x, at, f, layout, amplitude, inverse)
                tol = _tolerance(x, ref, dtype, n, layout, amplitude, max(map(max, at)))
                assert ((y.double().cpu() - ref).abs() <= tol).all()
                assert torch.equal(y[..., 2 * n:], x[..., 2 * n:])


@pytest.mark.gpu
def test_inverse_is_the_gradient():
    """<R x, g> = <x, R' g>, and R' g is what differences of <R x, g> along single elements give."""
    import flash_tree_attn_b200 as fta

    torch.manual_seed(0)
    B, H, Q, D = 2, 2, 3, 32
    f, _ = fta.rotary_frequencies(32)
    pos = torch.tensor([7, 1000], device="cuda")
    x, g = (torch.randn(B, H, Q, D, device="cuda").half() for _ in "xg")
    y, _ = fta.apply_rotary(x, None, pos, f, amplitude=1.25)
    back, _ = fta.apply_rotary(g, None, pos, f, amplitude=1.25, inverse=True)
    n = x.numel()
    # every output is off by at most u of itself (below |x1| + |x2| times the amplitude)
    bound = 2 * 2.0 ** -10 * 1.25 * float((x.double().abs().sum() * g.double().abs().max()))
    assert abs(float((y.double() * g.double()).sum() - (x.double() * back.double()).sum())) <= bound
    grad = torch.empty(n, dtype=torch.float64)
    step = 4.0  # the map is linear: a large step only makes the roundings small against the difference
    for e in range(n):
        d = torch.zeros(n, device="cuda", dtype=torch.float16)
        d[e] = step
        plus, _ = fta.apply_rotary(d.view_as(x), None, pos, f, amplitude=1.25)
        minus, _ = fta.apply_rotary(-d.view_as(x), None, pos, f, amplitude=1.25)
        grad[e] = float(((plus.double() - minus.double()) * g.double()).sum()) / (2 * step)
    # two outputs see an element, each off by u of at most 1.25; and `back` itself is rounded
    assert ((grad.view_as(back) - back.double().cpu()).abs() <= 2.0 ** -11 * (2 * 1.25 * 4 + back.double().cpu().abs()) + 2.0 ** -18).all()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, 64, 128])
@pytest.mark.parametrize("Q", [1, 5, 130])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_append_writes_the_rows_and_grows_the_lengths(page, Q, layout):
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import rotary_oracle, write_rows

    B, H, Hkv, D, n, ctx = 4, 6, 2, 64, 16, 256
    g = torch.Generator().manual_seed(Q)
    q, k, v = (torch.randn(B, h, Q, D, generator=g).bfloat16().cuda() for h in (H, Hkv, Hkv))
    lens = [0, 63, 250, 256]  # the third overflows for Q > 6, the fourth is full
    table = None
    if page:
        per = ctx // page
        table = torch.randperm(B * per, generator=g).view(B, per).to(torch.int32).cuda()
        kc, vc = (torch.randn(B * per, Hkv, page, D, generator=g).bfloat16().cuda() for _ in "kv")
    else:
        kc, vc = (torch.randn(B, ctx, Hkv, D, generator=g).bfloat16().cuda().transpose(1, 2) for _ in "kv")
    f, _ = fta.rotary_frequencies(2 * n)
    pos = torch.tensor([[100 * b + 3 * i for i in range(Q)] for b in range(B)], device="cuda", dtype=torch.int32)
    for dtype, positions in ((torch.int32, None), (torch.int64, pos), (torch.int64, pos[:, 0].contiguous())):
        at = [[lens[b] + i for i in range(Q)] for b in range(B)] if positions is None else \
            pos.tolist() if positions.dim() == 2 else [[100 * b + i for i in range(Q)] for b in range(B)]
        want_k, want_v = kc.cpu().clone(), vc.cpu().clone()
        k2, v2, n2 = kc.clone(), vc.clone(), torch.tensor(lens, dtype=dtype, device="cuda")
        qo = fta.append_tokens(k2, v2, q, k, v, n2, inv_freq=f, positions=positions, layout=layout, block_table=table)
        kr, _ = fta.apply_rotary(k, None, torch.tensor(at, device="cuda"), f, layout=layout)  # held to the formula above
        qr, _ = fta.apply_rotary(q, None, torch.tensor(at, device="cuda"), f, layout=layout)
        assert torch.equal(qo, qr)
        for b in range(B):
            for i in range(Q):
                if lens[b] + i < ctx:
                    write_rows(want_k, table, b, lens[b] + i, kr[b, :, i].cpu())
                    write_rows(want_v, table, b, lens[b] + i, v[b, :, i].cpu())
        assert torch.equal(k2.cpu(), want_k) and torch.equal(v2.cpu(), want_v)
        assert n2.tolist() == [min(L + Q, ctx) for L in lens]
    ref = rotary_oracle(k, at, f, layout)
    assert ((kr.double().cpu() - ref).abs() <= _tolerance(k, ref, torch.bfloat16, n, layout, 1.0, 1000)).all()
    # without frequencies nothing turns and q comes back itself
    k2, v2, n2 = kc.clone(), vc.clone(), torch.tensor(lens, device="cuda")
    assert fta.append_tokens(k2, v2, q, k, v, n2, block_table=table) is q
    from oracle.decode_oracle import sequence_rows
    got = sequence_rows(k2.cpu(), None if table is None else table.cpu(), 1, 63 + Q)
    assert torch.equal(got[:, 63:], k[1].cpu())


@pytest.mark.gpu
def test_append_drops_rows_of_a_page_outside_the_pool():
    import flash_tree_attn_b200 as fta

    kc, vc = (torch.zeros(2, 1, 64, 64, device="cuda", dtype=torch.float16) for _ in "kv")
    k = torch.ones(1, 1, 70, 64, device="cuda", dtype=torch.float16)
    n = torch.tensor([0], device="cuda")
    fta.append_tokens(kc, vc, k, k, k, n, block_table=torch.tensor([[7, 1]], dtype=torch.int32, device="cuda"))
    assert (kc[0] == 0).all() and (kc[1, :, :6] == 1).all() and (vc[1, :, 6:] == 0).all() and n.item() == 70


@pytest.mark.gpu
def test_strides_capture_and_streams():
    import flash_tree_attn_b200 as fta

    torch.manual_seed(0)
    f, _ = fta.rotary_frequencies(64)
    wide = torch.randn(2, 9, 8, 72, device="cuda").half()  # tokens before heads, rows of 72
    q, k = wide[..., 8:].transpose(1, 2)[:, ::2], wide[..., :64].transpose(1, 2)[:, 1:3]
    pos = torch.tensor([5, 6], device="cuda")
    want = fta.apply_rotary(q.contiguous(), k.contiguous(), pos, f)
    assert all(torch.equal(a, b) for a, b in zip(fta.apply_rotary(q, k, pos, f), want))
    same = torch.tensor([[4], [9]], device="cuda").expand(2, 9)
    want = fta.apply_rotary(q, k, same.contiguous(), f)
    assert all(torch.equal(a, b) for a, b in zip(fta.apply_rotary(q, k, same, f), want))
    kc, vc = (torch.zeros(2, 2, 64, 64, device="cuda").half() for _ in "kv")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    one_q, one_k = q[:, :, :1], k[:, :, :1]
    fta.append_tokens(kc, vc, one_q, one_k, one_k, n, inv_freq=f)
    n.zero_()
    kc.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fta.append_tokens(kc, vc, one_q, one_k, one_k, n, inv_freq=f)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(5):
            graph.replay()
    torch.cuda.synchronize()
    assert n.tolist() == [5, 5]
    for i in range(5):
        want, _ = fta.apply_rotary(one_k, None, torch.tensor([i, i], device="cuda"), f)
        assert torch.equal(kc[:, :, i], want[:, :, 0])
    assert not kc[:, :, 5:].any()


def test_frequencies():
    import flash_tree_attn_b200 as fta

    def freq(*a, **kw):
        f, amplitude = fta.rotary_frequencies(*a, device="cpu", **kw)
        assert f.dtype == torch.float64
        return f, amplitude

    plain, one = freq(64, 10000.0)
    assert one == 1.0 and plain[0] == 1.0 and math.isclose(plain[31], 10000.0 ** (-62 / 64), rel_tol=1e-15)
    assert torch.equal(freq(64, 10000.0, "linear", 4.0)[0], plain / 4)
    base, _ = freq(64, 10000.0, "base", 4.0)
    assert base[0] == 1.0 and math.isclose(base[31] * 4, plain[31], rel_tol=1e-12)
    bands, _ = freq(64, 10000.0, "bands", 8.0, 4096)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(bands[turns >= 4], plain[turns >= 4]) and torch.equal(bands[turns <= 1], plain[turns <= 1] / 8)
    between = (turns > 1) & (turns < 4)
    assert between.any() and ((bands < plain) & (bands > plain / 8))[between].all()
    ramp, amplitude = freq(64, 10000.0, "ramp", 8.0, 4096)
    assert math.isclose(amplitude, 0.1 * math.log(8) + 1) and ramp[0] == plain[0] and math.isclose(ramp[31], plain[31] / 8, rel_tol=1e-15)
    assert (ramp[1:] < ramp[:-1]).all()
    for bad in (dict(rotary_dim=3), dict(rotary_dim=16, scaling="other"), dict(rotary_dim=16, factor=0.5), dict(rotary_dim=2, scaling="base")):
        with pytest.raises(AssertionError):
            fta.rotary_frequencies(device="cpu", **bad)


def _fake(**kw):
    p = _lib.FtaRotaryParams()
    for name in ("q", "k", "v", "q_out", "k_out", "k_cache", "v_cache", "kv_seq_len", "positions", "inv_freq"):
        setattr(p, name, 4096)
    for name in ("q_sb", "q_sh", "q_sq", "k_sb", "k_sh", "k_sq", "v_sb", "v_sh", "v_sq", "kc_sb", "kc_sh", "kc_st", "vc_sb", "vc_sh", "vc_st"):
        setattr(p, name, 64)
    p.B, p.H, p.Hkv, p.Q, p.D, p.ctx, p.dtype, p.n_freq = 2, 4, 2, 3, 64, 256, _lib.DTYPE_F16, 32
    for name, value in kw.items():
        setattr(p, name, value)
    return p


BOTH = [dict(D=48), dict(B=0), dict(Q=0), dict(dtype=2), dict(n_freq=12), dict(n_freq=40), dict(layout=2), dict(inv_freq=None), dict(q=None), dict(q=4104),
        dict(q_sq=60), dict(k=None), dict(k_sh=4)]


@pytest.mark.parametrize("kw", BOTH + [dict(positions=None), dict(k_out=None), dict(n_freq=0)])
def test_apply_refuses(fta_lib, kw):
    assert fta_lib.fta_apply_rotary(C.byref(_fake(**kw)), None) == _lib.FTA_E_BADARG


@pytest.mark.parametrize("kw", BOTH + [dict(v=None), dict(k_cache=None), dict(kc_st=63), dict(kv_seq_len=None), dict(Hkv=0), dict(v_sb=1),
                                       dict(block_table=4096, page_size=64, n_pages=1, bt_sb=3), dict(block_table=4096, page_size=64, bt_sb=4)])
def test_append_refuses(fta_lib, kw):
    assert fta_lib.fta_append_tokens(C.byref(_fake(**kw)), None) == _lib.FTA_E_BADARG


def test_c_struct_and_null(fta_lib):
    assert C.sizeof(_lib.FtaRotaryParams) == 304  # as a C++ compile of include/fta.h prints
    assert fta_lib.fta_apply_rotary(None, None) == fta_lib.fta_append_tokens(None, None) == _lib.FTA_E_BADARG


@pytest.mark.gpu
def test_python_refusals():
    import flash_tree_attn_b200 as fta

    f, _ = fta.rotary_frequencies(64)
    x = torch.zeros(2, 2, 3, 64, device="cuda", dtype=torch.float16)
    pos, n = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    cache = torch.zeros(2, 2, 64, 64, device="cuda", dtype=torch.float16)
    fta.apply_rotary(x, x, pos, f)
    for a, kw in (((x.float(), x, pos, f), {}), ((x, x.bfloat16(), pos, f), {}), ((x, x, pos[:1], f), {}), ((x, x, pos.float(), f), {}),
                  ((x, x, pos, f.float()), {}), ((x, x, pos, f[:12]), {}), ((x, x, pos, f.cpu()), {}), ((x, x[:, :, :1], pos, f), {}),
                  ((x, x, pos, f), dict(layout="other")), ((x, x, pos, f), dict(offsets=n)), ((x[..., :48], None, pos, f), {})):
        with pytest.raises(AssertionError):
            fta.apply_rotary(*a, **kw)
    other = cache.clone()
    fta.append_tokens(cache, other, x, x, x, n)
    with pytest.raises(AssertionError, match="two tensors"):
        fta.append_tokens(cache, cache, x, x, x, n)
    for a, kw in (((cache[..., :32], other, x, x, x, n), {}), ((cache[:1], other[:1], x, x, x, n), {}), ((cache, other, x, x, x, n.float()), {}),
                  ((cache, other, x, x, x[:, :1], n), {}), ((cache[:1].expand(2, 2, 64, 64), other, x, x, x, n), {}),
                  ((cache.bfloat16(), other.bfloat16(), x, x, x, n), {}), ((cache, other, x, x, x, torch.zeros(4, dtype=torch.int32, device="cuda")[::2]), {}),
                  ((cache, other, x[:, :, :1], x, x, n), {}), ((cache, other, x, x, x, n), dict(block_table=torch.zeros(2, 1, device="cuda")))):
        with pytest.raises(AssertionError):
            fta.append_tokens(*a, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        fta.apply_rotary(x.cpu(), None, pos.cpu(), f.cpu())
    with pytest.raises(RuntimeError, match="CUDA"):
        fta.append_tokens(cache.cpu(), other.cpu(), x.cpu(), x.cpu(), x.cpu(), n.cpu())
