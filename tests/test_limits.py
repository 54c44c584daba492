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
