"""Eviction by accumulated weight (evict_rows) against plain loops (oracle/decode_oracle.py), bit for bit,
and its refusals."""
import ctypes as C
import random

import pytest
import torch

from flash_tree_attn_b200 import _lib


def _weights(kind, B, Hkv, ctx, lens, g):
    w = torch.exp(2 * torch.randn(B, Hkv, ctx, generator=g))
    if kind == "ties":
        w = torch.randint(0, 4, (B, Hkv, ctx), generator=g).float()
    elif kind == "equal":
        w = torch.full((B, Hkv, ctx), 0.25)
    elif kind == "odd":
        pick = torch.randint(0, 8, (B, Hkv, ctx), generator=g)
        for i, x in enumerate((float("nan"), float("inf"), float("-inf"), -0.0, 0.0, -1.0, 1e-40)):
            w[pick == i] = x
    for b, L in enumerate(lens):
        w[b, :, L:] = 0
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("D,Hkv,ctx,page,budget,recent,dtype", [
    (32, 1, 64, 0, 1, 0, torch.float16), (64, 2, 128, 64, 7, 7, torch.bfloat16), (128, 2, 320, 64, 65, 1, torch.float16), (256, 1, 256, 128, 200, 100, torch.bfloat16),
    (128, 3, 2304, 0, 1100, 33, torch.bfloat16), (64, 1, 5120, 64, 5000, 0, torch.float16), (32, 2, 1024, 0, 1024, 5, torch.float16)])
def test_matches_the_loops(kind, D, Hkv, ctx, page, budget, recent, dtype):
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import evict_oracle

    rng = random.Random(D + budget)
    lens = [0, 1, budget, min(ctx, budget + 1), ctx, rng.randint(0, ctx)]
    lens = [min(L, ctx) for L in lens]
    B = len(lens)
    g = torch.Generator().manual_seed(D + ctx)
    table = None
    if page:
        per = ctx // page
        table = torch.randperm(B * per, generator=g).view(B, per).to(torch.int32).cuda()
        k, v = (torch.randn(B * per, Hkv, page, D, generator=g).to(dtype).cuda() for _ in "kv")
    else:
        k, v = (torch.randn(B, ctx, Hkv, D, generator=g).to(dtype).cuda().transpose(1, 2) for _ in "kv")
    room = torch.zeros(B, Hkv, ctx + 8, device="cuda")
    w = room[..., :ctx]
    w.copy_(_weights(kind, B, Hkv, ctx, lens, g))
    n = torch.tensor(lens, dtype=torch.int64 if page else torch.int32, device="cuda")
    want = evict_oracle(k, v, n, w, budget, recent, table)
    kept = fta.evict_rows(k, v, n, w, budget, recent, block_table=table)
    for got, ref in zip((k, v, n, w, kept), want):
        assert torch.equal(got.cpu().view(torch.int32) if got is w else got.cpu(), ref.view(torch.int32) if got is w else ref)
    assert not room[..., ctx:].any()


@pytest.mark.gpu
def test_page_outside_the_pool_is_left_alone():
    import flash_tree_attn_b200 as fta

    torch.manual_seed(0)
    k, v = (torch.randn(3, 1, 64, 64, device="cuda").half() for _ in "kv")
    before = k.clone()
    w = torch.zeros(1, 1, 192, device="cuda")
    w[..., 100:140] = 1.0
    n = torch.tensor([192], device="cuda")
    kept = fta.evict_rows(k, v, n, w, 40, 0, block_table=torch.tensor([[0, 9, 2]], dtype=torch.int32, device="cuda"))
    assert kept[0, 0].tolist() == list(range(100, 140)) and n.item() == 40
    assert torch.equal(k[0, 0, 28:40], before[2, 0, :12]) and torch.equal(k[0, 0, :28], before[0, 0, :28]) and torch.equal(k[1:], before[1:])


@pytest.mark.gpu
def test_captured_and_repeated():
    """A second eviction finds nothing to do; a captured one follows lengths and weights."""
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import evict_oracle

    torch.manual_seed(3)
    B, Hkv, ctx, D = 2, 2, 512, 64
    k0, v0 = (torch.randn(B, Hkv, ctx, D, device="cuda").half() for _ in "kv")
    k, v, w, n = k0.clone(), v0.clone(), torch.rand(B, Hkv, ctx, device="cuda"), torch.tensor([512, 30], device="cuda")
    fta.evict_rows(k, v, n, w, 100, 10)
    state = [t.clone() for t in (k, v, n, w)]
    kept = fta.evict_rows(k, v, n, w, 100, 10)
    assert all(torch.equal(a, b) for a, b in zip(state, (k, v, n, w)))
    assert torch.equal(kept[0, 0].cpu(), torch.arange(100, dtype=torch.int32)) and kept[1, 1, 30:].eq(-1).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = fta.evict_rows(k, v, n, w, 100, 10)
    for lens in ([400, 101], [90, 512]):
        k.copy_(k0); v.copy_(v0); w.uniform_(); n.copy_(torch.tensor(lens))
        want = evict_oracle(k, v, n, w, 100, 10)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.cpu(), b) for a, b in zip((k, v, n, w, kept), want))


def _fake(**kw):
    p = _lib.FtaEvictParams()
    for name in ("k_cache", "v_cache", "kv_seq_len", "row_weights", "kept"):
        setattr(p, name, 4096)
    for name in ("k_sb", "k_sh", "k_st", "v_sb", "v_sh", "v_st"):
        setattr(p, name, 64)
    p.B, p.Hkv, p.D, p.ctx, p.budget, p.recent = 2, 2, 64, 256, 10, 2
    for name, value in kw.items():
        setattr(p, name, value)
    return p


@pytest.mark.parametrize("kw", [dict(B=0), dict(D=48), dict(budget=0), dict(recent=-1), dict(recent=11), dict(k_cache=None), dict(v_cache=4104), dict(k_st=4),
                                dict(row_weights=None), dict(kept=None), dict(kv_seq_len=None),
                                dict(block_table=4096, page_size=64, n_pages=4, bt_sb=3), dict(block_table=4096, page_size=0, n_pages=4, bt_sb=4)])
def test_c_entry_refuses(fta_lib, kw):
    assert fta_lib.fta_evict_rows(C.byref(_fake(**kw)), None) == _lib.FTA_E_BADARG


def test_c_struct_and_null(fta_lib):
    assert C.sizeof(_lib.FtaEvictParams) == 160  # as a C++ compile of include/fta.h prints
    assert fta_lib.fta_evict_rows(None, None) == _lib.FTA_E_BADARG


@pytest.mark.gpu
def test_python_refusals():
    import flash_tree_attn_b200 as fta

    k = torch.zeros(2, 2, 64, 64, device="cuda", dtype=torch.float16)
    w, n = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    v = k.clone()
    fta.evict_rows(k, v, n, w, 4, 2)
    with pytest.raises(AssertionError, match="two tensors"):
        fta.evict_rows(k, k, n, w, 4, 2)
    for a in ((k, v, n, w, 0, 0), (k, v, n, w, 4, 5), (k, v, n, w, 4, -1), (k, v, n.float(), w, 4, 2), (k, v, n, w.half(), 4, 2), (k, v, n, w[..., :63], 4, 2),
              (k, v[..., :32], n, w, 4, 2), (k.float(), v.float(), n, w, 4, 2), (k, v, n, w[:, :1].expand(2, 2, 64), 4, 2),
              (k[:1].expand(2, 2, 64, 64), v, n, w, 4, 2), (k, v, torch.zeros(4, dtype=torch.int32, device="cuda")[::2], w, 4, 2)):
        with pytest.raises(AssertionError):
            fta.evict_rows(*a)
    with pytest.raises(RuntimeError, match="CUDA"):
        fta.evict_rows(k.cpu(), k.cpu(), n.cpu(), w.cpu(), 4, 2)
