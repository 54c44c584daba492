"""Rows that a model is sure of (token_logprobs): the entropy is small and the likeliest token's log probability
lies just below 0.

Tolerance.  The largest logit's term is 1, and what the others add is summed beside it: an addition rounds by at
most 2^-24 (8 in a chunk, 8 chunks a round after the token was seen, 5 + 8 + 8 joins, a chunk's sum beside it
in each of the 8: 45 additions), in the sum and as much in t, the largest logit's term by two exponentials of
2^-22, and the other terms, which are the entropy's size, are off by 2^-20 of themselves.  Neither result may lie on the wrong side of 0 at all."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,V", [(600, 40000), (3, 128256), (64, 2000), (700, 1000)])
@pytest.mark.parametrize("where", ["last", "first", "middle"])
def test_a_token_far_above_the_others(dtype, rows, V, where):
    import flash_tree_attn_b200 as fta

    g = torch.Generator().manual_seed(V)
    x = torch.full((rows, V), -300.0)
    few = torch.rand(rows, V, generator=g) < 40.0 / V
    x[few] = (0.5 * torch.randn(rows, V, generator=g))[few].clamp(-1.5, 0.0)
    x[:, :: V // 7] = 0.0
    at = {"last": V - 3, "first": 1, "middle": V // 2 + 1}[where]
    x[:, at] = 4.0 + 10.0 * torch.rand(rows, generator=g)
    x = x.to(dtype)
    t = torch.full((rows, 1), at)
    r = fta.token_logprobs(x.cuda(), t.cuda(), 2)
    d = x.double()
    lp = torch.log_softmax(d, -1)
    entropy, given = -(lp.exp() * lp).sum(-1), lp[:, at]
    bound = 2 * (45 * 2.0 ** -24 + 2 * 2.0 ** -22)
    got, lg = r.entropy.double().cpu(), r.logprobs[:, 0].double().cpu()
    assert (got >= 0).all() and (r.logprobs <= 0).all() and (r.top_logprobs <= 0).all()
    assert ((got - entropy).abs() <= bound + 2.0 ** -20 * entropy).all(), float((got - entropy).abs().max())
    assert ((lg - given).abs() <= bound / 2 + 2.0 ** -20 * given.abs()).all(), float((lg - given).abs().max())
    assert (r.top_ids[:, 0] == at).all() and torch.equal(r.top_logprobs[:, 0], r.logprobs[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [2, 600])
def test_a_token_that_comes_late_above_one_that_came_early(dtype, rows):
    """Rows of nothing but two or three tokens, whole rounds apart: the entropy is near 10^-5 and less."""
    import flash_tree_attn_b200 as fta

    g = torch.Generator().manual_seed(rows)
    V, at = 40000, 39990
    x = torch.full((rows, V), float("-inf"))
    x[:, at - 32768], x[:, at - 16384] = 0.0, -1.0
    x[:, at] = 13.0 + 0.99 * torch.rand(rows, generator=g)
    x = x.to(dtype)
    r = fta.token_logprobs(x.cuda(), torch.full((rows, 1), at, device="cuda"))
    # exp(-13) and less beside 1, in 64 bits; -log1p keeps what a logarithm of their sum would lose
    d = x[:, at].double()
    a, b = torch.exp(-d), torch.exp(-1.0 - d)
    tail = a + b
    entropy = torch.log1p(tail) + (a * d + b * (1.0 + d)) / (1 + tail)
    got, lg = r.entropy.double().cpu(), r.logprobs[:, 0].double().cpu()
    assert (got >= 0).all() and (lg <= 0).all()
    # Three terms and additions of zeros: a sum is rounded twice beside 1.  The largest logit's own term is
    # 2^r 2^-r, r what the rounding of its product with log2 e left, by two exponentials that are off by 2^-22 each
    # (the instruction's documented bound).
    one = 2 * 2.0 ** -22 + 2 * 2.0 ** -24
    assert ((got - entropy).abs() <= one + 2 * 2.0 ** -24 + 2.0 ** -20 * entropy).all(), float((got - entropy).abs().max())
    assert ((lg + torch.log1p(tail)).abs() <= one + 2.0 ** -20 * tail).all(), float((lg + torch.log1p(tail)).abs().max())


@pytest.mark.gpu
def test_a_single_token_and_equal_ones():
    import flash_tree_attn_b200 as fta

    x = torch.full((4, 5000), float("-inf"))
    x[0, 17] = 5.0                   # nothing else: certain
    x[1, 4999] = -29000.0
    x[2, :2] = 123.25                # two equals: log 2
    x[3] = -3.0
    r = fta.token_logprobs(x.cuda(), torch.tensor([[17], [4999], [1], [0]], device="cuda"))
    # the exponent's reference, 29000 log2 e, is rounded by at most 2^-9; that is taken out of t again by a product and
    # a sum, each off by 2^-24 of it at most: 2^-32
    assert r.entropy[0] == 0.0 and 0.0 <= float(r.entropy[1]) <= 2.0 ** -32
    assert r.logprobs[:2, 0].tolist() == [0.0, 0.0] and r.lse[:2].tolist() == [5.0, -29000.0]
    want = torch.log(torch.tensor([2.0, 5000.0], dtype=torch.float64))
    assert ((r.entropy[2:].double().cpu() - want).abs() <= 2.0 ** -22 * want).all()
    assert ((r.logprobs[2:, 0].double().cpu() + want).abs() <= 2.0 ** -22 * want).all()
