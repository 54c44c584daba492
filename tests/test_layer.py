"""TreeVerifyAttention as a decoder's layer uses it: its cache's capacity, commits, casts of the module."""
import pytest
import torch

PARENTS = [-1, 0, 0, 1]


def _layer(page, max_seq_len, **kw):
    import flash_tree_attn_b200 as fta

    return fta.TreeVerifyAttention(4, 2, 64, 2, max_seq_len, torch.float16, page_size=page, **kw)


def _new(heads, count, g):
    return torch.randn(2, heads, count, 64, device="cuda", generator=g).half()


@pytest.mark.gpu
@pytest.mark.parametrize("page,max_seq_len,room", [(64, 100, 128), (128, 130, 256), (None, 100, 100), (64, 128, 128)])
def test_every_method_has_the_same_capacity(page, max_seq_len, room):
    """Steps over max_seq_len and over the cache's end: what is stored is attended to, the rest is dropped."""
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import decode_attention_oracle, sequence_rows
    from oracle.tree_attention_oracle import tree_attention_oracle
    from test_decode_attention import _check

    g = torch.Generator(device="cuda").manual_seed(max_seq_len)
    layer = _layer(page, max_seq_len, track_weights=True)
    tree = fta.DraftTree(PARENTS)
    lens = [max_seq_len - 1, 50]
    layer.load_prefix(*(torch.randn(2, 2, max_seq_len, 64, device="cuda", generator=g).half() for _ in "kv"), lens)
    table = None if page is None else layer.block_table.cpu()
    for step in range(room - max_seq_len + 4):
        q, k, v = _new(4, 1, g), _new(2, 1, g), _new(2, 1, g)
        before = layer.row_weights.clone()
        out = layer.decode(q, k, v)
        stored = lens[0] < room
        lens = [min(L + 1, room) for L in lens]
        assert layer.kv_seq_len.tolist() == lens
        ora = decode_attention_oracle(q, layer.k_cache, layer.v_cache, lens, layer.block_table, 2)
        _check(out, ora["lse"], None, ora, torch.float16, 64, None, None, room)
        gained = (layer.row_weights - before)[0, :, lens[0] - 1]
        assert (gained > 0).all()
        if stored:
            kb = sequence_rows(layer.k_cache.cpu(), table, 0, lens[0])
            assert torch.equal(kb[:, -1], k[0, :, 0].cpu())
    # the verification of a draft on the full cache sees all of it too
    q, k, v = _new(4, tree.Q, g), _new(2, tree.Q, g), _new(2, tree.Q, g)
    out = layer(q, k, v, tree.mask)
    kc, vc = (torch.zeros(2, 2, room, 64, device="cuda", dtype=torch.float16) for _ in "kv")
    for b, L in enumerate(lens):
        for full, t in ((kc, layer.k_cache), (vc, layer.v_cache)):
            full[b, :, :L] = sequence_rows(t.cpu(), table, b, L).cuda()
    ora = tree_attention_oracle(q, kc, vc, k, v, tree.mask, torch.tensor(lens, device="cuda"), None, 2)["out"]
    assert ((out.float() - ora).abs() <= 2e-3 + 2.0 ** -11 * ora.abs()).all()  # the tree operator's own tolerance


@pytest.mark.gpu
@pytest.mark.parametrize("page", [None, 64])
@pytest.mark.parametrize("kind", ["plain", "rotary", "weights"])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_accepted_lengths_of_any_shape(page, kind, dtype):
    """commit takes accept_len as commit_accepted does: as many elements as sequences.  Lengths past the path count
    as the path's, negative ones as none."""
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import sequence_rows

    g = torch.Generator(device="cuda").manual_seed(3)
    kw = {"rotary": dict(rotary=(fta.rotary_frequencies(64)[0], "half", 1.0)), "weights": dict(track_weights=True)}.get(kind, {})
    tree = fta.DraftTree(PARENTS)
    idx = torch.tensor([[0, 1, 3], [0, 2, 0]], dtype=torch.int32, device="cuda")
    for n, counts in (([[2], [1]], (2, 1)), ([[9], [-4]], (3, 0)), ([3, 2], (3, 2))):
        layer = _layer(page, 128, **kw)
        layer.load_prefix(*(torch.randn(2, 2, 50, 64, device="cuda", generator=g).half() for _ in "kv"), [50, 7])
        q, k, v = _new(4, tree.Q, g), _new(2, tree.Q, g), _new(2, tree.Q, g)
        layer(q, k, v, tree.mask, depth=tree.depth)
        layer.commit(idx, torch.tensor(n, dtype=dtype, device="cuda"))
        want = [50 + counts[0], 7 + counts[1]]
        assert layer.kv_seq_len.tolist() == want
        assert (layer.next_position is None) if kind == "plain" else (layer.next_position.tolist() == want)
        table = None if page is None else layer.block_table.cpu()
        for b, c in enumerate(counts):
            rows = sequence_rows(layer.v_cache.cpu(), table, b, want[b])
            assert torch.equal(rows[:, want[b] - c:], v[b][:, idx[b, :c].long()].cpu())
    out = layer.decode(_new(4, 1, g), _new(2, 1, g), _new(2, 1, g))
    assert out.shape == (2, 4, 1, 64) and layer.kv_seq_len.tolist() == [want[0] + 1, want[1] + 1]


def test_casts_leave_frequencies_and_weights_as_they_are():
    import flash_tree_attn_b200 as fta

    f, _ = fta.rotary_frequencies(64, device="cpu")
    for cast, dtype in ((lambda m: m.half(), torch.float16), (lambda m: m.to(torch.bfloat16), torch.bfloat16),
                        (lambda m: torch.nn.Sequential(m).to("cpu", torch.bfloat16)[0], torch.bfloat16), (lambda m: m.double().half(), torch.float16)):
        layer = fta.TreeVerifyAttention(4, 2, 64, 2, 100, torch.float16, device="cpu", rotary=(f, "half", 1.0), track_weights=True)
        layer.row_weights.normal_()
        weights = layer.row_weights.clone()
        got = cast(layer)
        assert got is layer and layer.k_cache.dtype is dtype and layer.v_cache.dtype is dtype
        assert layer.inv_freq.dtype is torch.float64 and torch.equal(layer.inv_freq, f)
        assert layer.row_weights.dtype is torch.float32 and torch.equal(layer.row_weights, weights)
        assert layer.kv_seq_len.dtype is torch.int32 and layer.next_position.dtype is torch.int64
    layer.to("meta")
    assert layer.inv_freq.is_meta and layer.row_weights.is_meta and layer.inv_freq.dtype is torch.float64
    layer.to_empty(device="cpu").half()
    assert layer.inv_freq.dtype is torch.float64 and layer.row_weights.shape == (2, 2, 100)
    plain = fta.TreeVerifyAttention(4, 2, 64, 2, 100, torch.float16, device="cpu").to(torch.bfloat16)
    assert plain.inv_freq is None and plain.row_weights is None and plain.k_cache.dtype is torch.bfloat16


@pytest.mark.gpu
def test_a_cast_layer_steps_on():
    import flash_tree_attn_b200 as fta

    g = torch.Generator(device="cuda").manual_seed(7)
    f, amplitude = fta.rotary_frequencies(64, scaling="ramp", factor=4.0)
    tree = fta.DraftTree(PARENTS)
    layers = [_layer(64, 128, rotary=(f, "half", amplitude), track_weights=True) for _ in range(2)]
    torch.nn.ModuleList(layers[1:]).half().cuda()
    prefix = [torch.randn(2, 2, 50, 64, device="cuda", generator=g).half() for _ in "kv"]
    for layer in layers:
        layer.load_prefix(*prefix, [50, 7])
    one, draft = [_new(h, 1, g) for h in (4, 2, 2)], [_new(h, tree.Q, g) for h in (4, 2, 2)]
    got = [(layer.decode(*one), layer(*draft, tree.mask, depth=tree.depth), layer.evict(20, 3), layer.row_weights) for layer in layers]
    assert all(torch.equal(a, b) for a, b in zip(*got))
