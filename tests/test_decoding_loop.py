"""The decoding loop's operators together, as a layer uses them: rotary positions, append, one-token
attention, tree verification, acceptance by the logits, commit and eviction, dense and paged, step after
step, against plain statements of each."""
import math

import pytest
import torch

PARENTS = [-1, 0, 0, 1, 1, 2, 3]


def _plain_node_ok(parents, logits, tokens, rule, epsilon=0.09, delta=0.3):
    x = logits.double().cpu()
    lp = torch.log_softmax(x, -1)
    H = -(lp.exp() * lp).sum(-1)
    ok = torch.ones(tokens.shape, dtype=torch.bool)
    margin = math.inf
    for b in range(tokens.size(0)):
        for i in range(1, len(parents)):
            p, t = parents[i], int(tokens[b, i])
            if rule == "greedy":
                best = min(j for j in range(x.size(-1)) if x[b, p, j] == x[b, p].max())
                ok[b, i] = t == best
            else:
                bar = min(math.log(epsilon), math.log(delta) - float(H[b, p]))
                ok[b, i] = float(lp[b, p, t]) > bar
                margin = min(margin, abs(float(lp[b, p, t]) - bar))
    return ok, margin


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_acceptance_rules(dtype):
    import flash_tree_attn_b200 as fta

    g = torch.Generator().manual_seed(5)
    tree = fta.DraftTree(PARENTS)
    B, Q, V = 5, len(PARENTS), 97
    logits = (2 * torch.randn(B, Q, V, generator=g)).to(dtype)
    logits[0, 1, 10] = logits[0, 1, 40] = 20.0  # two equals: the lower one is the choice
    tokens = torch.stack([torch.topk(logits.float(), 3, dim=-1).indices[:, p, i % 3] for i, p in enumerate([0] + PARENTS[1:])], 1)
    tokens[0, 3], tokens[0, 4] = 10, 40
    ok, _ = _plain_node_ok(PARENTS, logits, tokens, "greedy")
    assert torch.equal(fta.greedy_node_ok(tree, logits.cuda(), tokens.cuda()).cpu(), ok) and ok[0, 3] and not ok[0, 4]
    both = torch.zeros(2, dtype=torch.bool)
    for epsilon, delta in ((0.09, 0.3), (0.2, 0.9)):
        ok, margin = _plain_node_ok(PARENTS, logits, tokens, "typical", epsilon, delta)
        assert margin > 1e-4, "no value lies so near its bar that 32 bits could decide otherwise"
        assert torch.equal(fta.typical_node_ok(tree, logits.cuda(), tokens.to(torch.int32).cuda(), epsilon, delta).cpu(), ok)
        both |= torch.stack([ok[:, 1:].any(), ~ok[:, 1:].all()])
    assert both.all()
    one = fta.DraftTree([-1])
    assert fta.greedy_node_ok(one, logits[:, :1].cuda(), tokens[:, :1].cuda()).all()
    assert fta.typical_node_ok(one, logits[:, :1].cuda(), tokens[:, :1].cuda()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [None, 64])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_layer_step_after_step(page, layout):
    import flash_tree_attn_b200 as fta
    from oracle.decode_oracle import decode_attention_oracle, evict_oracle, rotary_oracle, sequence_rows
    from oracle.tree_attention_oracle import tree_attention_oracle
    from test_decode_attention import _check
    from test_rotary import _tolerance

    torch.manual_seed(11)
    B, H, Hkv, D, n, room = 3, 8, 2, 64, 24, 256
    G, dtype = H // Hkv, torch.bfloat16
    f, amplitude = fta.rotary_frequencies(2 * n, scaling="bands", factor=4.0, original_len=64)
    layer = fta.TreeVerifyAttention(H, Hkv, D, B, room, dtype, page_size=page, rotary=(f, layout, amplitude), track_weights=True)
    tree = fta.DraftTree(PARENTS)
    Q = tree.Q
    lens = [100, 0, 40]
    layer.load_prefix(*(torch.randn(B, Hkv, 128, D, device="cuda").to(dtype) for _ in "kv"), lens)
    pos = list(lens)
    table = None if page is None else layer.block_table.cpu()

    def rows_of(b, count):
        return tuple(sequence_rows(t.cpu(), table, b, count) for t in (layer.k_cache, layer.v_cache))

    def turned(x, at):
        ref = rotary_oracle(x, at, f, layout, amplitude)
        return ref, _tolerance(x, ref, dtype, n, layout, amplitude, 1000)

    for step in range(6):
        size = lambda h, k: torch.randn(B, h, k, D, device="cuda").to(dtype)  # noqa: E731
        if step in (2, 4):
            q, k, v = size(H, Q), size(Hkv, Q), size(Hkv, Q)
            before = [rows_of(b, L) for b, L in enumerate(lens)]
            out = layer(q, k, v, tree.mask, depth=tree.depth)
            at = [[pos[b] + int(d) for d in tree.depth] for b in range(B)]
            # what the layer turned is held to the formula, and what it attended with is that
            qr, kr = fta.apply_rotary(q, k, torch.tensor(pos, device="cuda"), f, offsets=tree.depth, layout=layout, amplitude=amplitude)
            for got, x in ((qr, q), (kr, k)):
                ref, tol = turned(x, at)
                assert ((got.double().cpu() - ref).abs() <= tol).all()
            kc, vc = (torch.zeros(B, Hkv, room, D, device="cuda", dtype=dtype) for _ in "kv")
            for b, (kb, vb) in enumerate(before):
                kc[b, :, : lens[b]], vc[b, :, : lens[b]] = kb.cuda(), vb.cuda()
            ora = tree_attention_oracle(qr, kc, vc, kr, v, tree.mask, torch.tensor(lens, device="cuda"), None, G)["out"]
            # the tree operator's own tolerance: 2e-3 and half a step of the result
            assert ((out.float() - ora).abs() <= 2e-3 + 2.0 ** -8 * ora.abs()).all()
            logits = torch.randn(B, Q, 50, device="cuda")
            tokens = torch.topk(logits, 2).indices[:, tree.parent, tree.slot % 2]
            ok = fta.greedy_node_ok(tree, logits, tokens)
            idx, count = fta.accept_longest_path(tree, ok)
            layer.commit(idx, count)
            for b in range(B):
                c = int(count[b])
                kb, vb = rows_of(b, lens[b] + c)
                nodes = idx[b, :c].long()
                assert c >= 1 and torch.equal(kb[:, lens[b]:], kr[b][:, nodes].cpu()) and torch.equal(vb[:, lens[b]:], v[b][:, nodes].cpu())
                assert torch.equal(kb[:, : lens[b]], before[b][0])
                lens[b] += c
                pos[b] += c
        else:
            q, k, v = size(H, 1), size(Hkv, 1), size(Hkv, 1)
            weights = layer.row_weights.clone()
            out = layer.decode(q, k, v)
            at = [[p] for p in pos]
            ref, tol = turned(k, at)
            for b in range(B):
                kb, vb = rows_of(b, lens[b] + 1)
                assert ((kb[:, -1].double() - ref[b, :, 0]).abs() <= tol[b, :, 0]).all() and torch.equal(vb[:, -1], v[b, :, 0].cpu())
                lens[b] += 1
                pos[b] += 1
            qr, _ = fta.apply_rotary(q, None, torch.tensor(at, device="cuda"), f, layout=layout, amplitude=amplitude)
            ora = decode_attention_oracle(qr, layer.k_cache, layer.v_cache, lens, layer.block_table, G)
            gained = layer.row_weights - weights if step == 0 else None  # later ones carry the sums' own roundings
            _check(out, ora["lse"], gained, ora, dtype, D, None, None, max(lens))
        assert layer.kv_seq_len.tolist() == lens and layer.next_position.tolist() == pos
        if step in (1, 3):
            want = evict_oracle(layer.k_cache, layer.v_cache, layer.kv_seq_len, layer.row_weights, 37, 9, table)
            kept = layer.evict(37, 9)
            for got, ref in zip((layer.k_cache, layer.v_cache, layer.kv_seq_len, layer.row_weights, kept), want):
                assert torch.equal(got.cpu(), ref)
            lens = [min(L, 37) for L in lens]


@pytest.mark.gpu
def test_whole_step_in_a_graph():
    """append, attention with weights, eviction and log probabilities in one captured graph, replayed."""
    import flash_tree_attn_b200 as fta

    torch.manual_seed(2)
    B, H, Hkv, D = 2, 8, 2, 64
    f, _ = fta.rotary_frequencies(D)
    head = torch.randn(D * H, 300, device="cuda").bfloat16()

    def make():
        layer = fta.TreeVerifyAttention(H, Hkv, D, B, 128, torch.bfloat16, page_size=64, rotary=(f, "half", 1.0), track_weights=True)
        g = torch.Generator(device="cuda").manual_seed(4)
        layer.load_prefix(*(torch.randn(B, Hkv, 60, D, device="cuda", generator=g).bfloat16() for _ in "kv"), [60, 17])
        return layer

    q, k, v = (torch.randn(B, h, 1, D, device="cuda").bfloat16() for h in (H, Hkv, Hkv))

    def step(layer):
        out = layer.decode(q, k, v)
        layer.evict(62, 8)
        return out, fta.token_logprobs(out.reshape(B, -1) @ head, top_k=3)

    a, b = make(), make()
    step(make())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, lp = step(a)
    for _ in range(5):
        q.normal_(), k.normal_(), v.normal_()
        graph.replay()
        want, want_lp = step(b)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(lp[1:], want_lp[1:]))
        assert torch.equal(a.kv_seq_len, b.kv_seq_len) and torch.equal(a.row_weights, b.row_weights) and torch.equal(a.k_cache, b.k_cache)
    assert a.kv_seq_len.tolist() == [62, 22] and a.next_position.tolist() == [65, 22]


def test_children_of_a_tree():
    import flash_tree_attn_b200 as fta

    tree = fta.DraftTree(PARENTS, device="cpu")
    assert tree.children.tolist() == [[1, 2], [3, 4], [5, -1], [6, -1], [-1, -1], [-1, -1], [-1, -1]]
    assert tree.parent.tolist() == [0, 0, 0, 1, 1, 2, 3] and tree.slot.tolist() == [0, 0, 1, 0, 1, 0, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("page", [None, 64])
def test_hundreds_of_steps_without_a_synchronisation(page):
    """Kernels are set up while the one before drains: steps queued without a pause, on two streams at once,
    give the bits of steps that wait for one another."""
    import flash_tree_attn_b200 as fta

    B, H, Hkv, D = 3, 8, 2, 128
    f, _ = fta.rotary_frequencies(64)
    tree = fta.DraftTree(PARENTS)
    g = torch.Generator(device="cuda").manual_seed(8)
    make = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()  # noqa: E731
    prompt, steps = (make(B, Hkv, 500, D), make(B, Hkv, 500, D)), [tuple(make(B, h, 1, D) for h in (H, Hkv, Hkv)) for _ in range(4)]
    draft = tuple(make(B, h, tree.Q, D) for h in (H, Hkv, Hkv))
    head = make(H * D, 5000)
    layers = [fta.TreeVerifyAttention(H, Hkv, D, B, 4096, torch.bfloat16, page_size=page, rotary=(f, "interleaved", 1.0), track_weights=True)
              for _ in range(3)]
    for layer in layers:
        layer.load_prefix(*prompt, [500, 3, 77])
    torch.cuda.synchronize()

    def run(layer, wait):
        seen = []
        for i in range(60):
            out = layer.decode(*steps[i % 4])
            wait()
            r = fta.token_logprobs(out.reshape(B, -1) @ head, top_k=5)
            wait()
            if i % 5 == 4:
                verified = layer(*draft, tree.mask, depth=tree.depth)
                wait()
                ok = fta.greedy_node_ok(tree, verified.transpose(1, 2).reshape(B, tree.Q, -1) @ head, r.top_ids[:, :1].expand(B, tree.Q))
                layer.commit(*fta.accept_longest_path(tree, ok))
                wait()
                seen.append(verified)
            if i % 7 == 6:
                seen.append(layer.evict(300, 40))
                wait()
            seen += [out, *r[1:]]
        return seen

    want = run(layers[0], torch.cuda.synchronize)
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for layer, s in zip(layers[1:], streams):
        with torch.cuda.stream(s):
            got.append(run(layer, lambda: None))
    torch.cuda.synchronize()
    for layer, seen in zip(layers[1:], got):
        assert all(torch.equal(a, b) for a, b in zip(seen, want))
        for name in ("k_cache", "v_cache", "kv_seq_len", "row_weights", "next_position"):
            assert torch.equal(getattr(layer, name), getattr(layers[0], name)), name
