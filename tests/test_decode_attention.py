"""Attention of one new token over the cache (decode_attention, decode_attention_paged) against a plain
statement in 64 bits (oracle/decode_oracle.py), and its refusals.

Tolerances.  u = eps / 2 is the relative error of one rounding to the cache's type.  The weights P are
rounded once (u * sum p|v|), the result once (u * |out|); fp16 weights below 2^-14 are off by up to
2^-25 of the largest absolute value instead.  A score is a sum of D products in 32 bits: off by at most
(D + 8) * 2^-24 * sum|q k| * scale, which is `d` below (the cap adds 2^-21 of itself, a distance bias
three roundings of its own size), and moves a weight by that share."""
import ctypes as C

import pytest
import torch

from flash_tree_attn_b200 import _lib

SLOPES = "slopes"


def _caches(B, Hkv, ctx, D, dtype, lens, page, seed, device, layout="bhtd"):
    """Caches whose rows past each length, and pages that nobody owns, are NaN."""
    from flash_tree_attn_b200.workloads import to_paged

    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(B, Hkv, ctx, D, generator=g).to(dtype) for _ in "kv")
    for b, L in enumerate(lens):
        k[b, :, L:] = float("nan")
        v[b, :, L:] = float("nan")
    if page:
        k, v, table = to_paged(k, v, lens, page_size=page, seed=seed)
        return k.to(device), v.to(device), table.to(device)
    if layout == "bthd":  # rows of one head are Hkv * D apart
        k, v = (t.transpose(1, 2).contiguous().to(device).transpose(1, 2) for t in (k, v))
    return k.to(device), v.to(device), None


def _check(out, lse, weights, ora, dtype, D, softcap, slopes, longest):
    u = torch.finfo(dtype).eps / 2
    d = (D + 8) * 2.0 ** -24 * ora["score"] + (softcap or 0.0) * 2.0 ** -21 + 2.0 ** -20
    if slopes is not None:
        d += 3 * 2.0 ** -24 * float(slopes.abs().max()) * longest
    tiny = longest * 2.0 ** -25 * 6.0 if dtype == torch.float16 else 0.0  # |v| < 6
    ref = ora["out"]
    tol = (u + 2 * d) * ora["size"] + u * ref.abs() + tiny + 1e-30
    worst = ((out.double().cpu() - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"out is {worst:.3g} times its tolerance off"
    fin = torch.isfinite(ora["lse"])
    got = lse.double().cpu()
    assert torch.equal(torch.isfinite(got), fin) and torch.equal(got[~fin], ora["lse"][~fin])
    assert ((got - ora["lse"])[fin].abs() <= d + 2.0 ** -22 * ora["lse"][fin].abs() + 1e-6).all()
    if weights is not None:
        n = ora["weights"].size(2)
        w = weights.double().cpu()
        # the score, the LSE and one exponential, then a sum of at most 256 terms
        assert ((w[..., :n] - ora["weights"]).abs() <= ora["weights"] * (3 * d + 2.0 ** -15) + 2.0 ** -126).all()
        assert not w[..., n:].any()


CASES = [
    # B lens Hkv G D ctx page dtype, options
    (dict(lens=[1], Hkv=1, G=1, D=32, ctx=64, page=0), {}),
    (dict(lens=[0, 1, 15, 16, 17, 63, 64, 65, 130], Hkv=2, G=4, D=128, ctx=130, page=0), {}),
    (dict(lens=[0, 1, 64, 129, 300], Hkv=2, G=3, D=64, ctx=320, page=64), {}),
    (dict(lens=[0, 0], Hkv=2, G=2, D=64, ctx=64, page=0), {}),
    (dict(lens=[700, 5], Hkv=3, G=1, D=32, ctx=768, page=128), dict(window=100)),
    (dict(lens=[513, 64, 20], Hkv=1, G=8, D=256, ctx=576, page=64), dict(softcap=20.0)),
    (dict(lens=[257, 1000], Hkv=2, G=9, D=128, ctx=1000, page=0), dict(window=1)),
    (dict(lens=[333, 64], Hkv=1, G=16, D=64, ctx=384, page=64), dict(softcap=3.0, window=64)),
    (dict(lens=[400, 77], Hkv=1, G=37, D=128, ctx=448, page=64), {SLOPES: True}),
    (dict(lens=[90, 2], Hkv=2, G=20, D=256, ctx=128, page=0), dict(window=65)),
    (dict(lens=[1500, 1], Hkv=4, G=5, D=32, ctx=1536, page=64), {SLOPES: True, "softcap": 30.0, "window": 1000}),
    (dict(lens=[4097], Hkv=2, G=7, D=128, ctx=4160, page=64), {}),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("grid", [0, 1, 5])
def test_matches_the_formula(dtype, case, grid):
    from flash_tree_attn_b200 import decode
    from oracle.decode_oracle import decode_attention_oracle

    c, opt = CASES[case]
    opt = dict(opt)
    B, H = len(c["lens"]), c["Hkv"] * c["G"]
    k, v, table = _caches(B, c["Hkv"], c["ctx"], c["D"], dtype, c["lens"], c["page"], case, "cuda", "bthd" if case % 2 else "bhtd")
    g = torch.Generator().manual_seed(100 + case)
    q = torch.randn(B, H, 1, c["D"], generator=g).to(dtype).cuda()
    slopes = torch.rand(H, generator=g).cuda() if opt.pop(SLOPES, False) else None
    lens = torch.tensor(c["lens"], dtype=torch.int64 if case % 3 else torch.int32, device="cuda")
    ora = decode_attention_oracle(q, k, v, lens, table, c["G"], alibi_slopes=slopes, **opt)
    w = torch.zeros(B, c["Hkv"], c["ctx"], device="cuda")
    args = (q, k, v, lens, table, None, None, c["G"], opt.get("softcap"), slopes, opt.get("window"))
    out, lse = decode._decode(*args, w, True, grid=grid)
    _check(out, lse, w, ora, dtype, c["D"], opt.get("softcap"), slopes, max(c["lens"]))
    # without weights the rows may be split otherwise (one launch, clusters); a call repeats its bits
    out, lse = decode._decode(*args, None, True, grid=grid)
    _check(out, lse, None, ora, dtype, c["D"], opt.get("softcap"), slopes, max(c["lens"]))
    for keep in (None, w):
        first, again = (decode._decode(*args, keep, True, grid=grid) for _ in range(2))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
def test_weights_add_up_over_calls_and_stay_inside_the_window():
    import flash_tree_attn_b200 as fta

    B, Hkv, G, D = 2, 2, 4, 64
    lens = [200, 70]
    k, v, _ = _caches(B, Hkv, 256, D, torch.bfloat16, lens, 0, 3, "cuda")
    q = torch.randn(B, Hkv * G, 1, D, device="cuda").bfloat16()
    n = torch.tensor(lens, device="cuda")
    w = torch.full((B, Hkv, 256), 0.5, device="cuda")
    for _ in range(3):
        fta.decode_attention(q, k, v, n, kv_group_num=G, window=50, row_weights=w)
    seen = torch.zeros_like(w, dtype=torch.bool)
    for b, L in enumerate(lens):
        seen[b, :, L - 50: L] = True
    assert (w[~seen] == 0.5).all() and (w[seen] > 0.5).all()
    # three calls of G heads: every call's weights sum to G, in 32 bits (150 sums of terms below 4)
    assert torch.allclose((w - 0.5).sum(-1), torch.full((B, Hkv), 3.0 * G, device="cuda"), atol=150 * 2.0 ** -23 * 4)


@pytest.mark.gpu
def test_infinite_and_nan_scores():
    """A key of -inf takes its row out; nothing but such rows gives zeros; NaN in a seen row shows."""
    import flash_tree_attn_b200 as fta

    D = 64
    q = torch.ones(3, 1, 1, D, device="cuda").half()
    k = torch.zeros(3, 1, 64, D, device="cuda").half()
    v = torch.ones(3, 1, 64, D, device="cuda").half()
    k[0, 0, 3] = float("-inf")
    v[0, 0, 3] = 7.0
    k[1, 0, :5] = float("-inf")
    k[2, 0, 2] = float("nan")
    out, lse = fta.decode_attention(q, k, v, torch.tensor([10, 5, 10], device="cuda"), return_lse=True)
    assert (out[0] == 1.0).all() and (out[1] == 0.0).all() and torch.isneginf(lse[1]).all() and torch.isnan(out[2]).all()


@pytest.mark.gpu
def test_strides_streams_and_two_calls_at_once():
    import flash_tree_attn_b200 as fta

    torch.manual_seed(0)
    B, Hkv, G, D = 4, 2, 4, 128
    lens = torch.tensor([900, 3, 64, 511], device="cuda", dtype=torch.int32)
    k, v = (torch.randn(B, Hkv, 960, D, device="cuda").half() for _ in "kv")
    wide = torch.randn(B, 2 * Hkv * G, 3, D + 8, device="cuda").half()
    q = wide[:, ::2, 1:2, 8:]
    odd = torch.randn(B * Hkv * G * D + 1, device="cuda").half()[1:].view(B, Hkv * G, 1, D)
    want = fta.decode_attention(q.clone(memory_format=torch.contiguous_format), k, v, lens, kv_group_num=G)
    assert torch.equal(fta.decode_attention(q, k, v, lens, kv_group_num=G), want)
    want_odd = fta.decode_attention(odd.clone(), k, v, lens, kv_group_num=G)
    assert torch.equal(fta.decode_attention(odd, k, v, lens, kv_group_num=G), want_odd)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(50):
        with torch.cuda.stream(a):
            got.append((fta.decode_attention(q, k, v, lens, kv_group_num=G), want))
        with torch.cuda.stream(b):
            got.append((fta.decode_attention(odd, k, v, lens, kv_group_num=G), want_odd))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)


@pytest.mark.gpu
def test_captured_calls_follow_the_lengths():
    """Two calls in one graph, a second graph of the same sizes, replays in turn on two streams."""
    import flash_tree_attn_b200 as fta

    torch.manual_seed(1)
    B, Hkv, G, D = 3, 2, 4, 64
    k, v = (torch.randn(B, Hkv, 512, D, device="cuda").bfloat16() for _ in "kv")
    q = torch.randn(B, Hkv * G, 1, D, device="cuda").bfloat16()
    lens = torch.tensor([500, 1, 64], device="cuda", dtype=torch.int32)
    fta.decode_attention(q, k, v, lens, kv_group_num=G)
    w = torch.zeros(B, Hkv, 512, device="cuda")
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x = fta.decode_attention(q, k, v, lens, kv_group_num=G, row_weights=w)
            y = fta.decode_attention(x, k, v, lens, kv_group_num=G)
        graphs.append((graph, x, y))
    for n in ([500, 1, 64], [512, 0, 65], [7, 333, 128]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        want = fta.decode_attention(q, k, v, lens, kv_group_num=G)
        want2 = fta.decode_attention(want, k, v, lens, kv_group_num=G)
        torch.cuda.synchronize()
        for (graph, x, y), s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
            with torch.cuda.stream(s):
                graph.replay()
            torch.cuda.synchronize()  # the graphs add to the same row weights
            assert torch.equal(x, want) and torch.equal(y, want2)


@pytest.mark.gpu
def test_tables_and_lengths_of_other_kinds():
    """int64 and strided tables, strided lengths, caches longer than the batch, a bound on the lengths."""
    import flash_tree_attn_b200 as fta

    torch.manual_seed(4)
    k, v = (torch.randn(6, 2, 64, 64, device="cuda").half() for _ in "kv")
    q = torch.randn(2, 4, 1, 64, device="cuda").half()
    table = torch.tensor([[4, 1, 0], [2, 5, 3]], dtype=torch.int32, device="cuda")
    n = torch.tensor([150, 70], device="cuda")
    want = fta.decode_attention_paged(q, k, v, table, n, kv_group_num=2)
    strided = torch.zeros(2, 6, dtype=torch.int32, device="cuda")
    strided[:, ::2] = table
    two = torch.zeros(4, dtype=torch.int64, device="cuda")
    two[::2] = n
    for t, lens in ((table.long(), n), (strided[:, ::2], n), (table.cpu(), n), (table, two[::2])):
        assert torch.equal(fta.decode_attention_paged(q, k, v, t, lens, kv_group_num=2), want)
    dense = fta.decode_attention(q, k, v, torch.tensor([64, 3], device="cuda"), kv_group_num=2)
    assert torch.equal(fta.decode_attention(q, k, v, torch.tensor([200, 3], device="cuda"), kv_group_num=2), dense)  # never past the cache
    bound = fta.decode_attention(q, k, v, torch.tensor([20, 3], device="cuda"), kv_group_num=2)
    assert torch.equal(fta.decode_attention(q, k, v, torch.tensor([64, 3], device="cuda"), kv_group_num=2, max_seq_len_in_batch=20), bound)
    none = fta.decode_attention(q, k, v, torch.tensor([-5, 0], device="cuda"), kv_group_num=2)
    assert not none.any()


@pytest.mark.gpu
def test_page_outside_the_pool_takes_its_rows_out():
    import flash_tree_attn_b200 as fta

    torch.manual_seed(2)
    k, v = (torch.randn(4, 1, 64, 64, device="cuda").half() for _ in "kv")
    q = torch.randn(1, 1, 1, 64, device="cuda").half()
    n = torch.tensor([192], device="cuda")
    for bad in (-1, 4, 2 ** 31 - 1):
        got = fta.decode_attention_paged(q, k, v, torch.tensor([[2, bad, 0]], dtype=torch.int32, device="cuda"), n)
        want = fta.decode_attention_paged(q, k, v, torch.tensor([[2, 0]], dtype=torch.int32, device="cuda"),
                                          torch.tensor([128], device="cuda"))
        # the same rows in another split: two roundings of P apart
        assert torch.allclose(got.float(), want.float(), atol=4 * 2.0 ** -11 * 4)


@pytest.mark.gpu
def test_long_cache_offsets_pass_32_bits():
    """K and V of 2^31 elements and more each: the last sequence lies beyond a 32-bit offset."""
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import decode_attention_oracle

    B, Hkv, D, ctx = 17, 8, 128, 131072
    k, v = (torch.zeros(B, Hkv, ctx, D, device="cuda", dtype=torch.float16) for _ in "kv")
    assert k.numel() > 2 ** 31
    k[-1, :, -300:].normal_()
    v[-1, :, -300:].normal_()
    q = torch.randn(B, Hkv, 1, D, device="cuda").half()
    lens = torch.tensor([1] * (B - 1) + [ctx], device="cuda")
    out, lse = fta.decode_attention(q, k, v, lens, window=300, return_lse=True)
    ora = decode_attention_oracle(q[-1:], k[-1:, :, -300:], v[-1:, :, -300:], torch.tensor([300]))
    _check(out[-1:], lse[-1:], None, ora, torch.float16, D, None, None, 300)


def _fake(**kw):
    """Aligned pointers that nothing dereferences: validation ends before a launch."""
    p = _lib.FtaTokenParams()
    for name in ("q", "k_cache", "v_cache", "kv_seq_len", "out", "workspace"):
        setattr(p, name, 4096)
    for name in ("q_sb", "q_sh", "k_sb", "k_sh", "k_st", "v_sb", "v_sh", "v_st", "o_sb", "o_sh"):
        setattr(p, name, 64)
    p.B, p.H, p.Hkv, p.D, p.ctx, p.dtype, p.grid_override = 2, 8, 2, 64, 256, _lib.DTYPE_F16, 4
    p.sm_scale = 0.125
    for name, value in kw.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("kw,code", [
    (dict(D=48), _lib.FTA_E_BADARG), (dict(H=7), _lib.FTA_E_BADARG), (dict(B=0), _lib.FTA_E_BADARG), (dict(dtype=2), _lib.FTA_E_BADARG),
    (dict(B=8193), _lib.FTA_E_UNSUPPORTED), (dict(H=514), _lib.FTA_E_UNSUPPORTED), (dict(q=None), _lib.FTA_E_BADARG), (dict(k_cache=4104), _lib.FTA_E_BADARG),
    (dict(k_st=63), _lib.FTA_E_BADARG), (dict(o_sh=2), _lib.FTA_E_BADARG), (dict(softcap=-1.0), _lib.FTA_E_BADARG),
    (dict(softcap=float("nan")), _lib.FTA_E_BADARG), (dict(window=-1), _lib.FTA_E_BADARG), (dict(workspace=None), _lib.FTA_E_WORKSPACE),
    (dict(), _lib.FTA_E_WORKSPACE), (dict(block_table=4096, page_size=96, n_pages=4, bt_sb=8), _lib.FTA_E_BADARG),
    (dict(block_table=4096, page_size=64, n_pages=4, bt_sb=3), _lib.FTA_E_BADARG), (dict(block_table=4096, page_size=64, n_pages=0, bt_sb=4), _lib.FTA_E_BADARG),
])
def test_c_entry_refuses(fta_lib, kw, code):
    assert fta_lib.fta_decode_token(C.byref(_fake(**kw)), None) == code


def test_c_entry_sizes(fta_lib):
    assert C.sizeof(_lib.FtaTokenParams) == 256  # as a C++ compile of include/fta.h prints
    assert fta_lib.fta_decode_token(None, None) == _lib.FTA_E_BADARG
    plain, kept = _fake(), _fake(row_weights=4096)
    a, b = (fta_lib.fta_decode_token_workspace_bytes(C.byref(x)) for x in (plain, kept))
    assert a > 0 and 0 <= b - a - 4 * 2 * 8 * (1 + 256) < 16  # an LSE and ctx scores per head, aligned
    assert fta_lib.fta_decode_token_workspace_bytes(C.byref(_fake(D=48))) == -_lib.FTA_E_BADARG


def test_needs_cuda_tensors():
    import flash_tree_attn_b200 as fta

    k = torch.zeros(1, 1, 64, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        fta.decode_attention(torch.zeros(1, 1, 1, 64, dtype=torch.float16), k, k, torch.tensor([1]))


@pytest.mark.gpu
def test_refusals():
    import flash_tree_attn_b200 as fta

    k = torch.zeros(2, 2, 64, 64, dtype=torch.float16, device="cuda")
    q = torch.zeros(2, 4, 1, 64, dtype=torch.float16, device="cuda")
    n = torch.tensor([1, 1], device="cuda")

    def refused(*a, **kw):
        with pytest.raises((AssertionError, _lib.FtaError)):
            fta.decode_attention(*a, **{"kv_group_num": 2, **kw})

    fta.decode_attention(q, k, k, n, kv_group_num=2)
    refused(q.expand(2, 4, 2, 64), k, k, n)
    refused(q.float(), k, k, n)
    refused(q, k.bfloat16(), k, n)
    refused(q, k, k, n, kv_group_num=3)
    refused(q, k, k, n, kv_group_num=4)
    refused(q, k[:1], k[:1], n)
    refused(q, k[..., :32], k[..., :32], n)
    refused(q, k, k, n[:1])
    refused(q, k, k, n.float())
    refused(q, k, k, n.cpu())
    refused(q, k, k, n, softcap=0.0)
    refused(q, k, k, n, softcap=float("inf"))
    refused(q, k, k, n, window=0)
    refused(q, k, k, n, alibi_slopes=torch.ones(2, device="cuda"))
    refused(q, k, k, n, row_weights=torch.zeros(2, 2, 63, device="cuda"))
    refused(q, k, k, n, row_weights=torch.zeros(2, 2, 64, device="cuda").half())
    refused(q, torch.zeros(2, 2, 64, 65, dtype=torch.float16, device="cuda")[..., :64], k, n)
    with pytest.raises(AssertionError):
        fta.decode_attention_paged(q, k[:, :, :32], k[:, :, :32], torch.zeros(2, 1, dtype=torch.int32, device="cuda"), n, kv_group_num=2)
    with pytest.raises(AssertionError):
        fta.decode_attention_paged(q, k, k, torch.zeros(2, 1, device="cuda"), n, kv_group_num=2)
