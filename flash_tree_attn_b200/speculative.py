"""Caller-side pieces of a tree speculative-decoding loop around the operator: an attention layer
that owns its KV cache and runs verify -> accept -> commit, step after step.

The reference stops at the operator and lists "integration into transformers, medusa, glide" and
"kv cache management" as to do (README.md:60-64); its tree tokens stay outside the cache
(README.md:41-43).  This module is what a decoder's attention layer needs on top of
`flash_decoding_attention` to close that loop, written against plain torch interfaces only:

    layer = TreeVerifyAttention(num_heads, num_kv_heads, head_dim, max_batch, max_seq_len)
    layer.load_prefix(k_prompt, v_prompt, prompt_lens)          # after prefill
    for every decoding step:
        out = layer(q, k_new, v_new, mask)                      # verify: the tree's nodes attend to the
                                                                #   cache and, under the mask, to each other
        idx, n = accept_longest_path(tree, node_ok)             # caller's acceptance rule -> a root path
        layer.commit(idx, n)                                    # accepted nodes' K/V join the cache

A step without a draft is `layer.decode(q, k_new, v_new)`: the new token joins the cache and attends to
it.  With `rotary` the layer turns queries and keys to their positions itself; with `track_weights` it
adds up what every cache row was looked at, and `layer.evict(budget, recent)` keeps the cache within
a budget by it.  `greedy_node_ok` and `typical_node_ok` are acceptance rules over the model's logits.

Nothing here synchronises with the host: the lengths live on the device, the operator plans from
them on the device, and `commit` updates them in place, so a whole step can sit in a CUDA graph.
"""
from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch

from .decode import decode_attention, decode_attention_paged, evict_rows
from .logprobs import token_logprobs
from .op import commit_accepted, flash_decoding_attention, flash_decoding_attention_paged
from .rotary import append_tokens, apply_rotary


class DraftTree:
    """A fixed draft-tree topology: parents[i] < i, parents[0] = -1 (node 0 is the root).

    Precomputes what a step needs on the device: the additive ancestor-or-self mask the operator
    takes (flash_tree_attn.py:368 adds it to the scores), the ancestor matrix, node depths and, per
    node, the root-to-node path."""

    def __init__(self, parents: Sequence[int], device="cuda", allowed: float = 0.0):
        parents = [int(p) for p in parents]
        assert parents and parents[0] == -1 and all(0 <= p < i for i, p in enumerate(parents) if i > 0)
        self.parents = parents
        Q = self.Q = len(parents)
        depth = [0] * Q
        for i in range(1, Q):
            depth[i] = depth[parents[i]] + 1
        self.max_depth = max(depth) + 1
        anc = torch.zeros((Q, Q), dtype=torch.bool)
        paths = torch.zeros((Q, self.max_depth), dtype=torch.int32)
        for i in range(Q):
            j, chain = i, []
            while j >= 0:
                anc[i, j] = True
                chain.append(j)
                j = parents[j]
            chain.reverse()
            paths[i, :len(chain)] = torch.tensor(chain, dtype=torch.int32)
        dev = torch.device(device)
        self.ancestors = anc.to(dev)                                   # [Q, Q] j is i or an ancestor of i
        self.paths = paths.to(dev)                                     # [Q, max_depth] root ... node, zero padded
        self.depth = torch.tensor(depth, dtype=torch.int32, device=dev)
        children: List[List[int]] = [[] for _ in range(Q)]
        slot = [0] * Q                                                 # which of its parent's children a node is
        for i in range(1, Q):
            slot[i] = len(children[parents[i]])
            children[parents[i]].append(i)
        fan = max(1, max(len(c) for c in children))
        self.children = torch.tensor([c + [-1] * (fan - len(c)) for c in children], device=dev)  # [Q, fan], -1 padded
        self.parent = torch.tensor([max(p, 0) for p in parents], device=dev)                     # the root's: itself
        self.slot = torch.tensor(slot, device=dev)
        self.mask = torch.where(self.ancestors, float(allowed), float("-inf")).to(torch.float32)


def accept_longest_path(tree: DraftTree, node_ok: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """From per-node verdicts to the path to commit, on the device and without a host sync.

    node_ok [bsz, q_len] bool: whether the caller's rule accepts node i given its parent (for greedy
    verification: the token drafted at node i equals the model's choice at its parent).  A node can be
    committed only if it and all its ancestors are accepted; the deepest such node wins (lowest index
    among equals).  Returns (accept_idx [bsz, max_depth] int32: the path from the root in order,
    accept_len [bsz] int32: its length, 0 if even the root is rejected) as `commit` takes them."""
    ok = node_ok.to(torch.bool)
    Q = tree.Q
    assert ok.dim() == 2 and ok.size(1) == Q
    # rejected[b, i] = number of rejected nodes on the path to i
    rejected = (~ok).to(torch.float32) @ tree.ancestors.to(torch.float32).t()
    reach = rejected == 0
    score = torch.where(reach, tree.depth.to(torch.int64)[None] + 1, torch.zeros((), dtype=torch.int64, device=ok.device))
    best = torch.argmax(score * Q + (Q - 1 - torch.arange(Q, device=ok.device))[None], dim=1)
    n = score.gather(1, best[:, None])[:, 0].to(torch.int32)
    return tree.paths[best].contiguous(), n


def greedy_node_ok(tree: DraftTree, logits: torch.Tensor, tokens: torch.Tensor) -> torch.Tensor:
    """Greedy verification: a node is accepted if its token is the likeliest one at its parent (the lower
    token of equals); the root, whose token the model has chosen already, always is.

    logits [bsz, q_len, vocab] of the tree's nodes, tokens [bsz, q_len] int32/int64 drafted at them.
    Returns node_ok [bsz, q_len] bool as `accept_longest_path` takes it."""
    best = token_logprobs(logits, top_k=1).top_ids[..., 0]
    ok = tokens == best[:, tree.parent]
    ok[:, 0] = True
    return ok


def typical_node_ok(tree: DraftTree, logits: torch.Tensor, tokens: torch.Tensor, epsilon: float = 0.09, delta: float = 0.3) -> torch.Tensor:
    """Typical acceptance: a node is accepted if the model gives its token, at its parent, a probability
    above min(epsilon, delta * exp(-entropy)): an unlikely token passes where the model is unsure.

    Arguments and result as greedy_node_ok."""
    drafted = tokens[:, tree.children.clamp(min=0)]                    # [bsz, q_len, fan]
    drafted = torch.where(tree.children < 0, torch.full_like(drafted, -1), drafted)
    r = token_logprobs(logits, drafted)
    bar = torch.minimum(torch.full_like(r.entropy, math.log(epsilon)), math.log(delta) - r.entropy)
    ok = r.logprobs[:, tree.parent, tree.slot] > bar[:, tree.parent]
    ok[:, 0] = True
    return ok


class TreeVerifyAttention(torch.nn.Module):
    """The attention of one decoder layer during tree verification, with its KV cache.

    Dense cache: k_cache / v_cache [max_batch, num_kv_heads, max_seq_len, head_dim] right-padded per
    sequence, the layout the reference's operator reads (flash_tree_attn.py:238-239).  With
    `page_size` (a multiple of 64) the cache is a pool of pages and a block table, the layout the
    reference's docstring announces (:233); sequence b owns the pages block_table[b], handed out in a
    shuffled order at construction; a sequence then holds max_seq_len rows rounded up to whole pages, for
    every method alike.

    forward() is the verify step and leaves the cache untouched; commit() appends the accepted
    nodes' keys and values (as given to the last forward) and grows kv_seq_len in place.  decode() is
    the step of one token without a draft.  The row of a token that finds the cache full is dropped.

    rotary: (inv_freq, layout, amplitude) as apply_rotary takes them (`rotary_frequencies` makes the
    first and the last); queries and new keys are then turned to next_position and on.  Keys given to
    load_prefix are turned already.  next_position [max_batch] int64 counts every token of a sequence,
    evicted ones too; a layer with neither rotary nor track_weights has none (its rows are its positions).
    track_weights: keep row_weights [max_batch, num_kv_heads, rows] of decode(), which evict() goes by.
    Rows that verification looked at gain nothing; `recent` is there to keep new rows until decode()
    has looked at them."""

    def __init__(self, num_heads: int, num_kv_heads: int, head_dim: int, max_batch: int, max_seq_len: int,
                 dtype: torch.dtype = torch.float16, device="cuda", page_size: Optional[int] = None,
                 sm_scale: Optional[float] = None, seed: int = 0,
                 rotary: Optional[Tuple[torch.Tensor, str, float]] = None, track_weights: bool = False):
        super().__init__()
        assert num_heads % num_kv_heads == 0
        self.H, self.Hkv, self.D = num_heads, num_kv_heads, head_dim
        self.G = num_heads // num_kv_heads
        self.max_seq_len = int(max_seq_len)
        self.sm_scale = sm_scale
        dev = torch.device(device)
        self.page_size = page_size
        if page_size is None:
            k = torch.zeros((max_batch, num_kv_heads, max_seq_len, head_dim), dtype=dtype, device=dev)
            table = None
        else:
            assert page_size % 64 == 0
            per_seq = -(-max_seq_len // page_size)
            g = torch.Generator().manual_seed(seed)
            order = torch.randperm(max_batch * per_seq, generator=g).to(torch.int32)
            table = order.view(max_batch, per_seq).to(dev)
            k = torch.zeros((max_batch * per_seq, num_kv_heads, page_size, head_dim), dtype=dtype, device=dev)
        self.register_buffer("k_cache", k, persistent=False)
        self.register_buffer("v_cache", torch.zeros_like(k), persistent=False)
        self.register_buffer("kv_seq_len", torch.zeros(max_batch, dtype=torch.int32, device=dev), persistent=False)
        self.register_buffer("block_table", table, persistent=False)
        # the next token's position, where it can differ from kv_seq_len or is asked for; else None
        counted = rotary is not None or track_weights
        self.register_buffer("next_position", torch.zeros(max_batch, dtype=torch.int64, device=dev) if counted else None, persistent=False)
        self.register_buffer("inv_freq", None if rotary is None else rotary[0].to(dev), persistent=False)
        self.layout, self.amplitude = ("half", 1.0) if rotary is None else (rotary[1], float(rotary[2]))
        # what a sequence's cache holds: whole pages, where there are pages
        self.rows = self.max_seq_len if table is None else table.size(1) * page_size
        weights = torch.zeros((max_batch, num_kv_heads, self.rows), dtype=torch.float32, device=dev) if track_weights else None
        self.register_buffer("row_weights", weights, persistent=False)
        self._last_kv = None

    def _apply(self, fn, *args, **kwargs):
        """A cast of the module (`.half()`, `.to(dtype)`) is for the caches: frequencies stay in 64 bits and row
        weights in 32, as the operators take them.  As integers they only move."""
        kept = {name: self._buffers[name] for name in ("inv_freq", "row_weights") if self._buffers[name] is not None}
        super()._apply(fn, *args, **kwargs)
        for name, t in kept.items():
            if self._buffers[name].dtype is not t.dtype:
                as_int = torch.int64 if t.dtype is torch.float64 else torch.int32
                self._buffers[name] = fn(t.view(as_int)).view(t.dtype)
        return self

    @torch.no_grad()
    def load_prefix(self, k: torch.Tensor, v: torch.Tensor, lens: Sequence[int]) -> None:
        """Fill the cache after prefill: k, v [bsz, num_kv_heads, L, head_dim], lens[b] <= L rows count."""
        B = k.size(0)
        for b in range(B):
            n = int(lens[b])
            if self.block_table is None:
                self.k_cache[b, :, :n] = k[b, :, :n]
                self.v_cache[b, :, :n] = v[b, :, :n]
            else:
                ps = self.page_size
                for s in range(-(-n // ps)):
                    pg = int(self.block_table[b, s])
                    r0, r1 = s * ps, min((s + 1) * ps, n)
                    self.k_cache[pg, :, : r1 - r0] = k[b, :, r0:r1]
                    self.v_cache[pg, :, : r1 - r0] = v[b, :, r0:r1]
        self.kv_seq_len[:B] = torch.as_tensor(list(lens), dtype=torch.int32)
        if self.next_position is not None:
            self.next_position[:B] = torch.as_tensor(list(lens), dtype=torch.int64)
        if self.row_weights is not None:
            self.row_weights[:B] = 0.0

    @torch.no_grad()
    def forward(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, mask: torch.Tensor,
                depth: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Verify: q [bsz, num_heads, q_len, head_dim], k_new / v_new [bsz, num_kv_heads, q_len, head_dim]
        of the draft tree's nodes, additive mask over the nodes.  With rotary, depth [q_len] int32 says how
        far each node lies behind next_position (`DraftTree.depth`).  Returns [bsz, num_heads, q_len, head_dim]."""
        B = q.size(0)
        lens = self.kv_seq_len[:B]
        if self.inv_freq is not None:
            assert depth is not None, "a layer with rotary positions needs the nodes' depths"
            q, k_new = apply_rotary(q, k_new, self.next_position[:B], self.inv_freq, offsets=depth, layout=self.layout,
                                    amplitude=self.amplitude)
        self._last_kv = (k_new, v_new)
        if self.block_table is None:
            return flash_decoding_attention(q, self.k_cache[:B], self.v_cache[:B], k_new, v_new, mask, lens, 64,
                                            self.rows, sm_scale=self.sm_scale, kv_group_num=self.G)
        return flash_decoding_attention_paged(q, self.k_cache, self.v_cache, self.block_table[:B], k_new, v_new, mask, lens,
                                              self.rows, sm_scale=self.sm_scale, kv_group_num=self.G)

    @torch.no_grad()
    def commit(self, accept_idx: torch.Tensor, accept_len: torch.Tensor) -> None:
        """Append nodes accept_idx[b, :accept_len[b]] of the last forward's k_new / v_new to sequence
        b's cache rows kv_seq_len[b]..., and add accept_len to kv_seq_len, in place."""
        assert self._last_kv is not None, "commit() follows forward()"
        k_new, v_new = self._last_kv
        B = k_new.size(0)
        if self.block_table is None:
            commit_accepted(self.k_cache[:B], self.v_cache[:B], k_new, v_new, self.kv_seq_len[:B], accept_idx, accept_len,
                            kv_group_num=self.G)
        else:
            commit_accepted(self.k_cache, self.v_cache, k_new, v_new, self.kv_seq_len[:B], accept_idx, accept_len,
                            kv_group_num=self.G, block_table=self.block_table[:B])
        if self.next_position is not None:
            self.next_position[:B] += accept_len.to(self.next_position.device).reshape(-1).clamp(0, accept_idx.size(1))

    @torch.no_grad()
    def decode(self, q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor) -> torch.Tensor:
        """One token without a draft: q [bsz, num_heads, 1, head_dim], k_new / v_new [bsz, num_kv_heads, 1,
        head_dim].  The token joins the cache and attends to it, itself included.  Returns
        [bsz, num_heads, 1, head_dim]."""
        B = q.size(0)
        assert q.size(2) == 1 and k_new.size(2) == 1, "decode() takes one new token per sequence"
        lens, table = self.kv_seq_len[:B], None if self.block_table is None else self.block_table[:B]
        k, v = (self.k_cache[:B], self.v_cache[:B]) if table is None else (self.k_cache, self.v_cache)
        q = append_tokens(k, v, q, k_new, v_new, lens, inv_freq=self.inv_freq, layout=self.layout, amplitude=self.amplitude,
                          positions=None if self.inv_freq is None else self.next_position[:B], block_table=table)
        if self.next_position is not None:
            self.next_position[:B] += 1
        opts = dict(max_seq_len_in_batch=self.rows, sm_scale=self.sm_scale, kv_group_num=self.G,
                    row_weights=None if self.row_weights is None else self.row_weights[:B])
        if table is None:
            return decode_attention(q, k, v, lens, **opts)
        return decode_attention_paged(q, k, v, table, lens, **opts)

    @torch.no_grad()
    def evict(self, budget: int, recent: int, batch: Optional[int] = None) -> torch.Tensor:
        """Bring the first `batch` sequences (default: all) back to `budget` rows, the last `recent` of them
        kept in any case (see evict_rows).  Returns the old row of every row, [bsz, num_kv_heads, budget]."""
        assert self.row_weights is not None, "evict() needs a layer with track_weights"
        B = self.kv_seq_len.size(0) if batch is None else int(batch)
        table = None if self.block_table is None else self.block_table[:B]
        k, v = (self.k_cache[:B], self.v_cache[:B]) if table is None else (self.k_cache, self.v_cache)
        return evict_rows(k, v, self.kv_seq_len[:B], self.row_weights[:B], budget, recent, block_table=table)


def reference_path_walk(parents: Sequence[int], ok_row: Sequence[bool]) -> List[int]:
    """Plain-Python statement of accept_longest_path for one sequence (used by the tests)."""
    best: List[int] = []
    for i in range(len(parents)):
        chain, j, good = [], i, True
        while j >= 0:
            good = good and bool(ok_row[j])
            chain.append(j)
            j = parents[j]
        if good and len(chain) > len(best):
            best = chain[::-1]
    return best
