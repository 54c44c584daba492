"""How near decode_attention comes to the formula where nothing but the softmax weights and the sums can be off.

Every query has a single element that is not zero, so a score is one product, exact in 32 bits, and a scale
(a power of two where head_dim is a power of four; one rounding otherwise).  What is left, u = eps / 2:

 * the result's own rounding, u * |out|;
 * the weights P, a sum of two values of the cache's type: the first, rounded down, leaves less than 2 u of P, and the
   second is that rounded, by u: 2 u^2 (fp16: the second is a multiple of 2^-31 of the largest weight and not 0,
   off by up to 2^-31 where that is more);
 * the exponential, the running sums and the joins in 32 bits: a score of at most 2^5 in log2 units is off by
   2^-18 (the product with log2 e and the difference to the reference, half a step of 2^-19 each), an
   exponential by 2^-22, a piece's sums by 2^-23 an addition: L / 16 of them and 32 for the joins.

Held to that is the difference from 64 bits, element by element, relative to sum p |v|; P rounded once would
be off by up to u = 2^-8 (bf16) or 2^-11 (fp16) of it."""
import pytest
import torch


def _case(dtype, D, G, lens, seed):
    Hkv, B = 2, len(lens)
    ctx = max(lens)
    g = torch.Generator().manual_seed(seed)
    q = torch.zeros(B, Hkv * G, 1, D)
    at = torch.randint(0, D, (B, Hkv * G), generator=g)
    q.scatter_(3, at[..., None, None], (D ** 0.5) * (0.5 + torch.rand(B, Hkv * G, 1, 1, generator=g)))
    k = torch.randn(B, Hkv, ctx, D, generator=g).clamp(-5, 5)
    v = torch.randn(B, Hkv, ctx, D, generator=g).clamp(-6, 6)
    return [t.to(dtype).cuda() for t in (q, k, v)] + [torch.tensor(lens, dtype=torch.int32, device="cuda")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("G,grid,weights", [(1, 0, False), (4, 0, False), (4, 5, False), (11, 0, False), (11, 7, True), (4, 0, True)])
def test_only_the_results_own_rounding_is_left(dtype, D, G, grid, weights):
    from flash_tree_attn_b200 import decode
    from oracle.decode_oracle import decode_attention_oracle

    lens = [1, 2, 17, 64, 129, 333, 1000]
    q, k, v, n = _case(dtype, D, G, lens, D + G)
    ora = decode_attention_oracle(q, k, v, n, None, G)
    w = torch.zeros(len(lens), 2, max(lens), device="cuda") if weights else None
    out, lse = decode._decode(q, k, v, n, None, None, None, G, None, None, None, w, True, grid=grid)
    u = torch.finfo(dtype).eps / 2
    length = torch.tensor(lens, dtype=torch.float64).view(-1, 1, 1, 1)
    rel = 2 * u * u + 2 * (2.0 ** -18 + 2.0 ** -22) + (length / 16 + 32) * 2.0 ** -23
    tiny = length * 6 * 2.0 ** -31 if dtype == torch.float16 else 0.0
    got, ref = out.double().cpu(), ora["out"]
    # u of the value that is rounded, which the other errors may have moved
    tol = u * ref.abs() + (1 + u) * (rel * ora["size"] + tiny)
    worst = ((got - ref).abs() / tol).max().item()
    assert worst <= 1.0, f"{worst:.3g} times its tolerance off"
    assert ((lse.double().cpu() - ora["lse"]).abs() <= rel[..., 0] + 2.0 ** -22 * ora["lse"].abs() + 2.0 ** -22).all()
    # a single row is the row itself
    assert torch.equal(out[0, :, 0], v[0, :, 0].repeat_interleave(G, 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("G,grid,weights", [(1, 0, False), (4, 5, False), (11, 0, True)])
def test_infinities_in_rows_that_are_seen(dtype, D, G, grid, weights):
    """A sum with an infinity is one, of the same sign, and nothing but its own element shows it; two of opposite signs
    make NaN.  A row's weight may be 1 (a single row), a power of two, or anything else."""
    from flash_tree_attn_b200 import decode
    from oracle.decode_oracle import decode_attention_oracle

    lens = [1, 2, 64, 129, 1000]
    q, k, v, n = _case(dtype, D, G, lens, D * G)
    k[1, :, 1] = k[1, :, 0]                       # two equal weights
    plain = v.clone()
    for b, L in enumerate(lens):
        v[b, :, L // 2, 3] = float("inf")
        v[b, :, L - 1, 5] = float("-inf")
        v[b, :, 0, 7], v[b, :, L - 1, 8] = float("inf"), float("nan")
        if L > 1:
            v[b, :, L - 1, 7] = float("-inf")
    w = torch.zeros(len(lens), 2, max(lens), device="cuda") if weights else None
    out = decode._decode(q, k, v, n, None, None, None, G, None, None, None, w, False, grid=grid)[:, :, 0].double().cpu()
    assert (out[..., 3] == float("inf")).all() and (out[..., 5] == float("-inf")).all()
    assert (out[0, :, 7] == float("inf")).all() and torch.isnan(out[1:, :, 7]).all() and torch.isnan(out[..., 8]).all()
    ora = decode_attention_oracle(q, k, plain, n, None, G)
    rest = [i for i in range(D) if i not in (3, 5, 7, 8)]
    u = torch.finfo(dtype).eps / 2
    # the tolerance of the test above at its loosest: 1000 rows
    rel = 2 * u * u + 2 * (2.0 ** -18 + 2.0 ** -22) + (1000 / 16 + 32) * 2.0 ** -23 + (1000 * 2.0 ** -31 if dtype == torch.float16 else 0.0) * 6
    tol = u * ora["out"].abs() + (1 + u) * rel * ora["size"].clamp(min=1.0)
    assert ((out - ora["out"][:, :, 0]).abs() <= tol[:, :, 0])[..., rest].all()
