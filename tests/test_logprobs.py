"""Log probabilities of given tokens (token_logprobs) against a plain statement in 64 bits, and its refusals.

Tolerances.  A term e^(x - m) is off by 2^-22 (the exponential) and |x - m| 2^-23 of itself; a sum of
terms of one sign by at most the number of additions on one path (8 in a chunk, a chunk a time in a
thread, at most 8 rounds of 8 here, then 5 + 8 + 8 joins) times 2^-24, and each of at most 4 moves of the
reference by 2^-22: below 10^-5 together for the logarithm of the sum, and 10^-5 of t / s, which is at most
the entropy plus log s.  The result's own rounding is 2^-24 of it.  Tokens are exact."""
import ctypes as C

import pytest
import torch

from flash_tree_attn_b200 import _lib


def _check(logits, tokens, k, r):
    from oracle.decode_oracle import logprobs_oracle

    given, entropy, lse, top, ids = logprobs_oracle(logits, tokens.cpu(), k)

    def near(got, want, tol):
        got = got.double().cpu()
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        assert (same | ((got - want).abs() <= tol)).all(), float((got - want).abs().nan_to_num(0, 0, 0).max())

    big = 1e-5 + 2.0 ** -23 * lse.abs().nan_to_num(0, 0, 0)
    near(r.lse, lse, big)
    near(r.entropy, entropy, 2e-5 * (1 + entropy.abs().nan_to_num(0, 0, 0)) + 1e-5 * 12)
    near(r.logprobs, given, 1e-5 + 2.0 ** -23 * given.abs().nan_to_num(0, 0, 0))
    if k:
        assert torch.equal(r.top_ids.cpu(), ids)
        near(r.top_logprobs, top, 1e-5 + 2.0 ** -23 * top.abs().nan_to_num(0, 0, 0))


def _tokens(rows, V, n, g, dtype=torch.int64):
    t = torch.randint(0, V, (rows, n), generator=g)
    t[:, -1] = -1
    if rows > 1:
        t[1, 0] = V
    return t.to(dtype).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 64, 64), (3, 100, 64), (2, 255, 5), (2, 2049, 20), (3, 4097, 64), (2, 16384, 1),
                                      (2, 32768, 33), (2, 32769, 64), (300, 1000, 8), (3, 50257, 20), (2, 128256, 5), (1, 262144, 64), (2, 300001, 10), (4, 5000, 0),
                                      (700, 1000, 64), (601, 4095, 20), (601, 33, 5), (601, 1, 1), (601, 2047, 16), (601, 257, 33), (601, 300, 64), (601, 1023, 64), (601, 1040, 64), (601, 4000, 40), (2, 16500, 64), (20, 56697, 64)])
def test_matches_the_formula(dtype, rows, V, k):
    import flash_tree_attn_b200 as fta

    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn(rows, V, generator=g)).to(dtype).cuda()
    t = _tokens(rows, V, 3, g)
    _check(x, t, k, fta.token_logprobs(x, t, k))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("shift", range(8))
def test_rows_that_start_anywhere(dtype, shift):
    import flash_tree_attn_b200 as fta

    g = torch.Generator().manual_seed(shift)
    wide = (2 * torch.randn(6, 40013, generator=g)).to(dtype).cuda()
    wide[:, :shift] = float("nan")
    wide[:, shift + 33001:] = float("nan")
    x = wide[::2, shift: shift + 33001]
    t = _tokens(3, 33001, 4, g, torch.int32)
    _check(x, t, 10, fta.token_logprobs(x, t, 10))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["equal", "two values", "masked", "all masked", "nan", "inf", "rising", "one high", "far", "lowest", "lowest and masked", "blocks"])
@pytest.mark.parametrize("V,rows,k", [(50, 4, 40), (3000, 4, 40), (70001, 4, 40), (2999, 601, 40), (2999, 601, 41), (1999, 601, 16), (301, 601, 3)])
def test_rows_that_tie_or_are_masked(kind, V, rows, k):
    import flash_tree_attn_b200 as fta

    g = torch.Generator().manual_seed(V)
    x = torch.randn(rows, V, generator=g)
    if kind == "equal":
        x[:] = 1.5
    elif kind == "two values":
        x = (x > 1.0).float()
        x[0, ::2] = -0.0
    elif kind == "masked":
        keep = torch.rand(rows, V, generator=g) < 4.0 / V
        x = x.masked_fill(~keep, float("-inf"))
        x[:, V // 2] = 0.0
    elif kind == "all masked":
        x[1:3] = float("-inf")
    elif kind == "nan":
        x[1, 7] = float("nan")
        x[2, V - 1] = float("nan")
        x[2, 0] = float("nan")
    elif kind == "inf":
        x[1, 7] = float("inf")
    elif kind == "rising":
        x = torch.arange(V).float().expand(rows, V) * 1e-3
    elif kind == "one high":
        x[:, 3] = 300.0
    elif kind == "blocks":  # what is large sits together, in different places of each row
        for r in range(rows):
            x[r, (r * 977) % V: (r * 977) % V + 2500] += 50.0
    elif kind == "far":
        x = x - 20000.0
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        if kind.startswith("lowest"):  # masked with the type's lowest value, and two rows of nothing else
            x = torch.randn(rows, V, generator=g)
            x[:2] = torch.finfo(dtype).min
            x[2, 1:] = torch.finfo(dtype).min
            if kind.endswith("masked"):
                x[1:, ::3] = float("-inf")
        if dtype == torch.float16 and kind == "far":
            x = x / 4
        y = x.to(dtype).cuda()
        t = _tokens(rows, V, 2, g)
        _check(y, t, k, fta.token_logprobs(y, t, k))


@pytest.mark.gpu
def test_leading_sizes_strides_capture_and_repeat():
    import flash_tree_attn_b200 as fta

    torch.manual_seed(0)
    x = torch.randn(2, 3, 1001, device="cuda").bfloat16()
    t = torch.randint(0, 1001, (2, 3, 2), device="cuda")
    r = fta.token_logprobs(x, t, 4)
    assert r.logprobs.shape == (2, 3, 2) and r.entropy.shape == r.lse.shape == (2, 3) and r.top_ids.shape == r.top_logprobs.shape == (2, 3, 4)
    _check(x.view(6, -1), t.view(6, -1), 4, fta.TokenLogprobs(*(v.flatten(0, 1) for v in r)))
    turned = fta.token_logprobs(x.transpose(0, 1), t.transpose(0, 1), 4)
    _check(x.transpose(0, 1).reshape(6, -1), t.transpose(0, 1).reshape(6, -1), 4, fta.TokenLogprobs(*(v.flatten(0, 1) for v in turned)))
    column = fta.token_logprobs(x.transpose(1, 2).contiguous().transpose(1, 2), t, 4)
    assert all(torch.equal(a, b) for a, b in zip(r, column))
    flat = fta.token_logprobs(x[0, 0])
    assert flat.logprobs is None and flat.top_ids is None and flat.lse.shape == () and flat.lse == r.lse[0, 0]
    none = fta.token_logprobs(x[:0], t[:0], 4)
    assert none.top_ids.shape == (0, 3, 4) and none.lse.shape == (0, 3)
    same = fta.token_logprobs(x[:1].expand(5, 3, 1001), t[:1].expand(5, 3, 2), 4)
    _check(x[:1].expand(5, 3, 1001).reshape(15, -1), t[:1].expand(5, 3, 2).reshape(15, -1), 4, fta.TokenLogprobs(*(v.flatten(0, 1) for v in same)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = fta.token_logprobs(x, t, 4)
        b = fta.token_logprobs(x, a.top_ids, 1)
    x.normal_()
    graph.replay()
    torch.cuda.synchronize()
    want = fta.token_logprobs(x, t, 4)
    assert all(torch.equal(u, v) for u, v in zip(a, want)) and torch.equal(b.logprobs, want.top_logprobs)


def _fake(**kw):
    p = _lib.FtaLogprobParams()
    for name in ("logits", "tokens", "logprobs", "entropy", "lse", "top_logprobs", "top_ids"):
        setattr(p, name, 4096)
    p.l_sr, p.t_sr, p.rows, p.vocab, p.n_tokens, p.top_k, p.dtype = 100, 2, 3, 100, 2, 5, _lib.DTYPE_F16
    for name, value in kw.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(rows=0), 1), (dict(vocab=0), 1), (dict(top_k=-1), 1), (dict(top_k=101), 1), (dict(n_tokens=-1), 1), (dict(dtype=3), 1), (dict(logits=None), 1),
    (dict(logits=4097), 1), (dict(entropy=None), 1), (dict(lse=None), 1), (dict(tokens=None), 1), (dict(logprobs=None), 1), (dict(top_ids=None), 1),
    (dict(top_k=65), 2), (dict(vocab=(1 << 21) + 1), 2), (dict(rows=(1 << 27) + 1), 2)])
def test_c_entry_refuses(fta_lib, kw, code):
    assert fta_lib.fta_token_logprobs(C.byref(_fake(**kw)), None) == code


def test_c_struct_and_null(fta_lib):
    assert C.sizeof(_lib.FtaLogprobParams) == 96  # as a C++ compile of include/fta.h prints
    assert fta_lib.fta_token_logprobs(None, None) == _lib.FTA_E_BADARG


@pytest.mark.gpu
def test_python_refusals():
    import flash_tree_attn_b200 as fta

    x, t = torch.zeros(2, 10, device="cuda"), torch.zeros(2, 1, dtype=torch.int64, device="cuda")
    fta.token_logprobs(x, t, 10)
    for a in ((x.double(), t), (x, t.float()), (x, t[0]), (x, t[:1]), (x, t.cpu()), (x, t, 11), (x, t, -1), (x[:, :0], t)):
        with pytest.raises(AssertionError):
            fta.token_logprobs(*a)
    with pytest.raises(AssertionError):
        fta.token_logprobs(torch.zeros(1, 100, device="cuda"), None, 65)
    with pytest.raises(RuntimeError, match="CUDA"):
        fta.token_logprobs(x.cpu(), t.cpu())
