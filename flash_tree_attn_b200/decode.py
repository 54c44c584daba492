"""The decoding step without a draft tree: attention of one new token per sequence over the cache,
and the eviction of the rows that the attention looked at least.

Shapes, strides, lengths and page tables are those of `flash_decoding_attention` and
`flash_decoding_attention_paged` with q_len = 1; the new token's own key and value are already in
the cache (see `append_tokens`).  All arithmetic happens in libfta.so.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from ._lib import on_device, rows_ok

_DT = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_LEN = (torch.int32, torch.int64)


def _check_lengths(kv_seq_len: torch.Tensor, B: int, dev: torch.device) -> None:
    assert kv_seq_len.dtype in _LEN and kv_seq_len.dim() == 1 and kv_seq_len.size(0) == B and kv_seq_len.device == dev, \
        "kv_seq_len must be [bsz] int32 or int64 on q's device"


def _check_caches(k: torch.Tensor, v: torch.Tensor, B: int, Hkv: int, D: int, dtype, dev, block_table: Optional[torch.Tensor]) -> int:
    """The checks every entry makes of a dense or paged pair of caches; returns the rows that a sequence can hold."""
    assert k.dtype == dtype and v.dtype == dtype, "cache dtype must equal the new tokens' dtype"
    assert k.device == dev and v.device == dev, "caches must be on the new tokens' device"
    ks = k.shape
    assert len(ks) == 4 and v.shape == ks and ks[1] == Hkv and ks[3] == D, "caches must be [.., num_kv_heads, rows, head_dim], both alike"
    if block_table is None:
        assert ks[0] >= B, "dense caches must be [bsz, num_kv_heads, ctx, head_dim]"
        return ks[2]
    assert ks[2] % 64 == 0 and ks[2] > 0, "page_size must be a multiple of 64"
    assert block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.size(0) == B and block_table.device == dev \
        and block_table.stride(1) == 1, "block_table must be [bsz, max_pages] int32 on the caches' device, unit stride along a row"
    return block_table.size(1) * ks[2]


def _decode(q, k, v, kv_seq_len, block_table, max_seq_len_in_batch, sm_scale, kv_group_num, softcap, alibi_slopes, window, row_weights,
            return_lse, grid=0):
    lib = _lib.load()
    if not q.is_cuda:
        raise RuntimeError("decode_attention runs on CUDA tensors only (no CPU path exists)")
    B, H, one, D = q.shape
    dt = q.dtype
    dev = q.device
    assert one == 1, "q must be [bsz, num_heads, 1, head_dim]: one new token per sequence"
    assert D in (32, 64, 128, 256)
    assert dt in _DT, "q must be fp16 or bf16"
    G = int(kv_group_num)
    assert G >= 1 and H % G == 0, "num_heads must be a multiple of kv_group_num"
    Hkv = H // G
    ctx = _check_caches(k, v, B, Hkv, D, dt, dev, block_table)
    _check_lengths(kv_seq_len, B, dev)
    if max_seq_len_in_batch is not None:
        ctx = min(ctx, int(max_seq_len_in_batch))
    if not rows_ok(q):
        q = q.clone(memory_format=torch.contiguous_format)
    assert rows_ok(k) and rows_ok(v), "caches must have 16-byte rows: unit stride in head_dim, other strides multiples of 8 elements"
    if not kv_seq_len.is_contiguous():
        kv_seq_len = kv_seq_len.contiguous()
    cap = 0.0
    if softcap is not None:
        cap = float(softcap)
        assert cap > 0.0 and math.isfinite(cap), "softcap must be positive"
    if window is not None:
        assert int(window) > 0, "window must be positive"
    slopes = 0
    if alibi_slopes is not None:
        assert alibi_slopes.dtype == torch.float32 and alibi_slopes.shape == (H,) and alibi_slopes.device == dev \
            and alibi_slopes.is_contiguous(), "alibi_slopes must be [num_heads] fp32 on q's device"
        slopes = alibi_slopes.data_ptr()
    rw, rw_sb, rw_sh = 0, 0, 0
    if row_weights is not None:
        assert row_weights.dtype == torch.float32 and row_weights.dim() == 3 and row_weights.device == dev \
            and row_weights.size(0) == B and row_weights.size(1) == Hkv and row_weights.size(2) >= ctx and row_weights.stride(2) == 1 \
            and not _overlaps(row_weights), "row_weights must be [bsz, num_kv_heads, ctx] fp32 on q's device, unit stride along ctx"
        rw, rw_sb, rw_sh = row_weights.data_ptr(), row_weights.stride(0), row_weights.stride(1)
    out = torch.empty((B, H, 1, D), dtype=dt, device=dev)
    lse = torch.empty((B, H, 1), dtype=torch.float32, device=dev) if return_lse else None
    if B == 0:
        return (out, lse) if return_lse else out
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    paged = block_table is not None
    with on_device(dev) as stream:
        size = _workspace(lib, dev.index, B, H, Hkv, D, ctx, dt, row_weights is not None, grid)
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        p = _lib.pack_token(
            q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2],
            kv_seq_len.data_ptr(), block_table.data_ptr() if paged else 0, block_table.stride(0) if paged else 0, slopes,
            out.data_ptr(), H * D, D, lse.data_ptr() if return_lse else 0, H, rw, rw_sb, rw_sh, ws.data_ptr(), size,
            1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), cap, 0 if window is None else min(int(window), 0x7fffffff),
            1 if kv_seq_len.dtype == torch.int64 else 0, B, H, Hkv, D, ctx, k.size(2) if paged else 0, k.size(0) if paged else 0,
            _DT[dt], grid, 0)
        _lib.check(lib.fta_decode_token(p, stream), "fta_decode_token")
    return (out, lse) if return_lse else out


_ws_sizes = {}  # sizes -> bytes of workspace: a function of the sizes and the device alone


def _workspace(lib, index, B, H, Hkv, D, ctx, dt, weights, grid) -> int:
    key = (index, B, H, Hkv, D, ctx if weights else 0, dt, weights, grid)
    size = _ws_sizes.get(key)
    if size is None:
        p = _lib.FtaTokenParams()
        p.B, p.H, p.Hkv, p.D, p.ctx, p.dtype, p.grid_override = B, H, Hkv, D, ctx, _DT[dt], grid
        p.row_weights = 1 if weights else 0
        size = lib.fta_decode_token_workspace_bytes(_lib.byref(p))
        if size < 0:
            raise _lib.FtaError(-size, "fta_decode_token_workspace_bytes")
        if len(_ws_sizes) >= 4096:
            _ws_sizes.clear()
        _ws_sizes[key] = size
    return size


def decode_attention(q, k_cache, v_cache, kv_seq_len, *, max_seq_len_in_batch: Optional[int] = None, sm_scale: Optional[float] = None,
                     kv_group_num: int = 1, softcap: Optional[float] = None, alibi_slopes: Optional[torch.Tensor] = None,
                     window: Optional[int] = None, row_weights: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of one new token per sequence over a dense right-padded cache.

    Args:
        q: [bsz, num_heads, 1, head_dim] fp16/bf16, head_dim 32, 64, 128 or 256.
        k_cache, v_cache: [bsz, num_kv_heads, ctx, head_dim]; rows at or past kv_seq_len[b] are never read.
        kv_seq_len: [bsz] int32/int64, the new token included (its row is the last).
        max_seq_len_in_batch: upper bound of kv_seq_len; never read from the device.
        sm_scale: defaults to 1/sqrt(head_dim).
        kv_group_num: query heads per KV head; head h reads KV head h // kv_group_num.
        softcap: c > 0 replaces a scaled score s by c * tanh(s / c).
        alibi_slopes: [num_heads] fp32; row r of a sequence of L rows gains slope * (r - (L - 1)).
            Distances count cache rows, so this does not go with evict_rows, which closes up gaps.
        window: only the last `window` rows of a sequence are seen.
        row_weights: [bsz, num_kv_heads, ctx] fp32, updated in place: row r of a KV head gains the
            softmax weights that the group's query heads gave it (what evict_rows goes by).
        return_lse: also return the fp32 natural-log LSE [bsz, num_heads, 1].

    An empty sequence gives zeros and an LSE of -inf.  Asynchronous on the current stream of q's
    device, no host synchronisation, capturable in a CUDA graph.  Every call has a workspace of its own.
    """
    return _decode(q, k_cache, v_cache, kv_seq_len, None, max_seq_len_in_batch, sm_scale, kv_group_num, softcap, alibi_slopes, window,
                   row_weights, return_lse)


def decode_attention_paged(q, k_pages, v_pages, block_table, kv_seq_len, *, max_seq_len_in_batch: Optional[int] = None,
                           sm_scale: Optional[float] = None, kv_group_num: int = 1, softcap: Optional[float] = None,
                           alibi_slopes: Optional[torch.Tensor] = None, window: Optional[int] = None,
                           row_weights: Optional[torch.Tensor] = None, return_lse: bool = False):
    """decode_attention over a paged cache.

    k_pages, v_pages: [n_pages, num_kv_heads, page_size, head_dim], page_size a multiple of 64;
    block_table: [bsz, max_pages] int32.  Entries past ceil(kv_seq_len[b] / page_size) are never
    used; an entry in use that lies outside [0, n_pages) takes its page's rows out of the attention.
    """
    return _decode(q, k_pages, v_pages, kv_seq_len, block_table, max_seq_len_in_batch, sm_scale, kv_group_num, softcap, alibi_slopes, window,
                   row_weights, return_lse)


def evict_rows(k_cache, v_cache, kv_seq_len, row_weights, budget: int, recent: int, *, block_table: Optional[torch.Tensor] = None):
    """Bring every sequence longer than `budget` rows back to it, in place, per KV head.

    Kept are the last `recent` rows and, of the others, the budget - recent with the largest
    row_weights (ties: the lower row; NaN counts as largest).  They close up to rows [0, budget) in
    their old order and their weights move with them.

    Args:
        k_cache, v_cache: dense [bsz, num_kv_heads, ctx, head_dim], or pools of pages with
            `block_table`, updated in place; rows at or past the new length keep what they held.
            No page may belong to two sequences: moving one's rows would change the other's.
        kv_seq_len: [bsz] int32/int64 on the device, becomes min(length, budget) in place.
        row_weights: [bsz, num_kv_heads, ctx] fp32 as decode_attention adds them up, updated in place:
            0 from the new length to the old one, so that appended rows start at 0.
        budget, recent: 1 <= budget, 0 <= recent <= budget.

    Returns kept [bsz, num_kv_heads, budget] int32, the old row of every row now in the cache (-1 past
    a shorter sequence's end).  Keys keep the rotary positions they were written with; a caller that
    needs rows' positions keeps them by `kept`.  Asynchronous on the current stream of the caches'
    device, no host synchronisation.
    """
    lib = _lib.load()
    if not k_cache.is_cuda:
        raise RuntimeError("evict_rows runs on CUDA tensors only (no CPU path exists)")
    dt, dev = k_cache.dtype, k_cache.device
    assert dt in _DT and k_cache.dim() == 4, "caches must be fp16 or bf16 [.., num_kv_heads, rows, head_dim]"
    B, Hkv, D = kv_seq_len.size(0) if kv_seq_len.dim() == 1 else -1, k_cache.size(1), k_cache.size(3)
    assert D in (32, 64, 128, 256)
    ctx = _check_caches(k_cache, v_cache, B, Hkv, D, dt, dev, block_table)
    _check_lengths(kv_seq_len, B, dev)
    assert rows_ok(k_cache) and rows_ok(v_cache) and not _overlaps(k_cache) and not _overlaps(v_cache), \
        "caches are updated in place: they must have 16-byte rows and must not be expanded"
    assert B <= 1 or kv_seq_len.stride(0) == 1, "kv_seq_len is updated in place and must be contiguous"
    assert row_weights.dtype == torch.float32 and row_weights.dim() == 3 and row_weights.device == dev and row_weights.size(0) == B \
        and row_weights.size(1) == Hkv and row_weights.size(2) >= ctx and row_weights.stride(2) == 1 and not _overlaps(row_weights), \
        "row_weights must be [bsz, num_kv_heads, ctx] fp32 on the caches' device, unit stride along ctx"
    budget, recent = int(budget), int(recent)
    assert 1 <= budget <= 0x7fffffff and 0 <= recent <= budget, "1 <= budget and 0 <= recent <= budget"
    kept = torch.empty((B, Hkv, budget), dtype=torch.int32, device=dev)
    if B == 0:
        return kept
    ks, vs = k_cache.stride(), v_cache.stride()
    paged = block_table is not None
    p = _lib.pack_evict(
        k_cache.data_ptr(), ks[0], ks[1], ks[2], v_cache.data_ptr(), vs[0], vs[1], vs[2], kv_seq_len.data_ptr(),
        block_table.data_ptr() if paged else 0, block_table.stride(0) if paged else 0,
        row_weights.data_ptr(), row_weights.stride(0), row_weights.stride(1), kept.data_ptr(),
        1 if kv_seq_len.dtype == torch.int64 else 0, B, Hkv, D, ctx, k_cache.size(2) if paged else 0, k_cache.size(0) if paged else 0,
        budget, recent, 0)
    with on_device(dev) as stream:
        _lib.check(lib.fta_evict_rows(p, stream), "fta_evict_rows")
    return kept


def _overlaps(t: torch.Tensor) -> bool:
    """Whether some dimension of an in-place argument is broadcast (stride 0)."""
    return any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride()))
