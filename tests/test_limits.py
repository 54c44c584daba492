"""Sizes at the ends of what the decoding-loop entries take."""
import ctypes as C

import pytest
import torch

from flash_tree_attn_b200 import _lib

MOST = 0x7fff0000


@pytest.mark.parametrize("kw", [dict(budget=MOST + 1), dict(budget=2 ** 31 - 1), dict(ctx=MOST + 1), dict(ctx=2 ** 31 - 1)])
def test_eviction_refuses_sizes_whose_row_numbers_would_pass_32_bits(fta_lib, kw):
    from test_evict import _fake

    assert fta_lib.fta_evict_rows(C.byref(_fake(**kw)), None) == _lib.FTA_E_UNSUPPORTED


def test_attention_refuses_longer_caches(fta_lib):
    from test_decode_attention import _fake

    assert fta_lib.fta_decode_token(C.byref(_fake(ctx=MOST + 1)), None) == _lib.FTA_E_UNSUPPORTED
    # and batches whose 64-row tiles a 32-bit number does not count; a window keeps them few
    many = dict(B=8192, ctx=2 ** 24, bt_sb=2 ** 18)
    assert fta_lib.fta_decode_token(C.byref(_fake(**many)), None) == _lib.FTA_E_UNSUPPORTED
    assert fta_lib.fta_decode_token_workspace_bytes(C.byref(_fake(**many))) == -_lib.FTA_E_UNSUPPORTED
    assert fta_lib.fta_decode_token_workspace_bytes(C.byref(_fake(**many, window=4096))) > 0
    assert fta_lib.fta_decode_token_workspace_bytes(C.byref(_fake(B=8192, ctx=2 ** 23))) > 0


@pytest.mark.gpu
def test_eviction_without_a_limit_is_refused_before_anything_is_allocated():
    import flash_tree_attn_b200 as fta

    k, v = (torch.zeros(1, 1, 64, 32, device="cuda", dtype=torch.float16) for _ in "kv")
    n, w = torch.tensor([5], device="cuda"), torch.zeros(1, 1, 64, device="cuda")
    before = torch.cuda.memory_allocated()
    for budget in (2 ** 31 - 1, MOST + 1, 2 ** 40):
        with pytest.raises(AssertionError, match="budget"):
            fta.evict_rows(k, v, n, w, budget, 0)
    assert torch.cuda.memory_allocated() == before and n.item() == 5
    fta.evict_rows(k, v, n, w, 64, 64)
    assert n.item() == 5


@pytest.mark.gpu
def test_append_of_a_chunk_whose_row_numbers_pass_32_bits():
    """A table of 2^31 - 2^16 rows, all of one page; the chunk starts two rows before the end and is longer than
    what is left below 2^31.  Two rows are written, the others dropped."""
    import flash_tree_attn_b200 as fta

    Q, D = 70000, 32
    table = torch.zeros(1, MOST // 64 + 5, dtype=torch.int32, device="cuda")
    kc, vc = (torch.zeros(1, 1, 64, D, device="cuda", dtype=torch.float16) for _ in "kv")
    k = torch.randn(1, 1, Q, D, device="cuda").half()
    v = torch.randn(1, 1, Q, D, device="cuda").half()
    n = torch.tensor([MOST - 2], dtype=torch.int64, device="cuda")
    fta.append_tokens(kc, vc, k, k, v, n, block_table=table)
    assert n.item() == MOST
    for cache, x in ((kc, k), (vc, v)):
        assert torch.equal(cache[0, 0, 62:], x[0, 0, :2]) and not cache[0, 0, :62].any()


def _one_page(D, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(1, 1, 64, D, generator=g).half().cuda() for _ in "kv"] + [torch.randn(1, 2, 1, D, generator=g).half().cuda()]


@pytest.mark.gpu
@pytest.mark.parametrize("grid", [0, 3])
@pytest.mark.parametrize("L", [MOST, MOST - 37, 2 ** 30 + 1])
def test_attention_at_the_end_of_the_longest_cache(L, grid):
    """Every page is the same one; the window sees the last rows of a sequence of nearly 2^31."""
    from flash_tree_attn_b200 import decode
    from oracle.decode_oracle import decode_attention_oracle
    from test_decode_attention import _check

    k, v, q = _one_page(64, L % 97)
    table = torch.zeros(1, MOST // 64, dtype=torch.int32, device="cuda")
    n, slopes = torch.tensor([L], device="cuda"), torch.tensor([0.5, 0.01], device="cuda")
    out, lse = decode._decode(q, k, v, n, table, None, None, 2, None, slopes, 150, None, True, grid=grid)
    at = [(L - 150 + i) % 64 for i in range(150)]
    ora = decode_attention_oracle(q, k[:, :, at], v[:, :, at], torch.tensor([150]), None, 2, alibi_slopes=slopes)
    _check(out, lse, None, ora, torch.float16, 64, None, slopes, 150)


@pytest.mark.gpu
def test_row_weights_of_a_cache_of_many_chunks():
    """More rows than 65535 blocks of 1024: the weights of the last and of the first ones."""
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import decode_attention_oracle

    ctx = 65535 * 1024 + 64 * 1000
    k, v, q = _one_page(32, 1)
    table = torch.zeros(1, ctx // 64, dtype=torch.int32, device="cuda")
    w = torch.zeros(1, 1, ctx, device="cuda")
    for L in (ctx - 5, 700):
        w.zero_()
        fta.decode_attention_paged(q, k, v, table, torch.tensor([L], device="cuda"), kv_group_num=2, window=300, row_weights=w)
        at = [(L - 300 + i) % 64 for i in range(300)]
        ora = decode_attention_oracle(q, k[:, :, at], v[:, :, at], torch.tensor([300]), None, 2)
        # as test_decode_attention holds them: the score, the LSE, one exponential and a sum of two
        d = 40 * 2.0 ** -24 * ora["score"] + 2.0 ** -20
        assert ((w[..., L - 300: L].double().cpu() - ora["weights"]).abs() <= ora["weights"] * (3 * d + 2.0 ** -15)).all()
        assert not w[..., : L - 300].any() and not w[..., L:].any()


@pytest.mark.gpu
def test_the_smallest_row_weights_are_kept():
    """Rows that gain nothing (scores far below the largest) keep subnormal weights: eviction tells them apart."""
    import flash_tree_attn_b200 as fta

    k = torch.full((1, 1, 200, 64), -100.0, device="cuda").half()
    k[0, 0, 150] = 100.0
    q = torch.full((1, 1, 1, 64), 10.0, device="cuda").half()
    bits = torch.arange(1, 201, dtype=torch.int32, device="cuda")
    w = bits.view(torch.float32).clone().view(1, 1, 200)
    n = torch.tensor([200], device="cuda")
    fta.decode_attention(q, k, k, n, row_weights=w)
    got = w.view(torch.int32)[0, 0]
    assert w[0, 0, 150] == 1.0 and torch.equal(torch.cat([got[:150], got[151:]]), torch.cat([bits[:150], bits[151:]]))
    kept = fta.evict_rows(k, k.clone(), n, w, 5, 0)
    assert kept[0, 0].tolist() == [150, 196, 197, 198, 199]
