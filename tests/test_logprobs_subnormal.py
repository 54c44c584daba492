"""Logits below the smallest normal number: the likeliest tokens (token_logprobs) go by the values' bits, and so
does the bound that decides which elements are looked at.  fp32 and bf16 have such logits; fp16's smallest
are normal numbers in 32 bits."""
import pytest
import torch


def _bits(x):
    """fp32 values of the given multiples of the smallest subnormal, made by bits."""
    neg = x < 0
    return torch.where(neg, (-x).to(torch.int64) | (1 << 31), x.to(torch.int64)).to(torch.int64).sub(2 ** 32 * neg.to(torch.int64)).to(torch.int32).view(torch.float32)


def _rows(kind, rows, V, g):
    e = torch.arange(V).expand(rows, V)
    warp = (e // 4 % 256) // 32
    if kind == "one warp smaller":  # the first round's bound is that warp's: nearly all others are larger
        x = torch.where(warp == 7, torch.randint(1, 100, (rows, V), generator=g), torch.randint(1000, 2000, (rows, V), generator=g))
    elif kind == "negative":
        x = -torch.where(warp == 3, torch.randint(5000, 9000, (rows, V), generator=g), torch.randint(1, 4000, (rows, V), generator=g))
    elif kind == "both signs":
        x = torch.randint(-300, 300, (rows, V), generator=g)
    else:  # rising: every round's bound passes the one before's
        x = e + 1
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["one warp smaller", "negative", "both signs", "rising"])
@pytest.mark.parametrize("rows,V,k", [(2, 8192, 40), (2, 8193, 64), (3, 70001, 40), (700, 16384, 20), (601, 1000, 16), (601, 2000, 40), (601, 500, 64), (2, 20, 20)])
def test_subnormal_logits_rank_by_their_bits(dtype, kind, rows, V, k):
    import flash_tree_attn_b200 as fta
    from test_logprobs import _check, _tokens

    g = torch.Generator().manual_seed(V + k)
    x = _rows(kind, rows, V, g)
    if dtype == torch.bfloat16:
        # bf16 subnormals are 127 multiples of 2^-133; the patterns above are folded onto them
        x = (torch.where(x < 0, -((-x) % 127 + 1), x % 127 + 1) * 65536)
    y = _bits(x).to(dtype).cuda()
    assert torch.equal(y.cpu().float().view(torch.int32), _bits(x).view(torch.int32)), "the values are what was meant"
    t = _tokens(rows, V, 2, g)
    _check(y, t, k, fta.token_logprobs(y, t, k))


@pytest.mark.gpu
def test_subnormals_beside_zeros_and_ordinary_logits():
    import flash_tree_attn_b200 as fta
    from test_logprobs import _check, _tokens

    g = torch.Generator().manual_seed(3)
    x = _bits(torch.randint(-3, 4, (4, 30000), generator=g))
    x[0, ::2] = -0.0
    x[1] -= (torch.rand(30000, generator=g) < 0.5).float()
    x[2, 100:110] = torch.arange(10).float()
    x[3, ::3] = float("-inf")
    x[3, 7] = float("nan")
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype).cuda()
        t = _tokens(4, 30000, 2, g)
        _check(y, t, 33, fta.token_logprobs(y, t, 33))
