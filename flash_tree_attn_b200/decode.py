"""The decoding step without a draft tree: attention of one new token per sequence over the cache,
and the eviction of the rows that the attention looked at least.

Shapes, strides, lengths and page tables are those of `flash_decoding_attention` and
`flash_decoding_attention_paged` with q_len = 1; the new token's own key and value are already in
the cache (see `append_tokens`).  All arithmetic happens in libfta.so.

A decoding step makes many small calls, so the checks here read each tensor's attributes once.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib
from ._lib import launch, pack_evict, pack_token, rows_of

_DT = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_LEN = {torch.int32: 0, torch.int64: 1}  # -> is int64
_HEAD_DIMS = (32, 64, 128, 256)
_MOST_ROWS = 0x7fff0000  # of a sequence: row numbers are 32-bit, and loops over them step past the end
_f32 = torch.float32


def check_lengths(kv_seq_len: torch.Tensor, B: int, dev: int) -> int:
    """1 for int64 lengths, 0 for int32 ones."""
    is64 = _LEN.get(kv_seq_len.dtype)
    assert is64 is not None and kv_seq_len.shape == (B,) and kv_seq_len.get_device() == dev, \
        "kv_seq_len must be [bsz] int32 or int64 on the caches' device"
    return is64


def check_caches(k: torch.Tensor, v: torch.Tensor, B: int, Hkv: int, D: int, dtype, dev: int, block_table: Optional[torch.Tensor]):
    """What every entry asks of a dense or paged pair of caches.  Returns (k's pointer and strides, v's,
    rows that a sequence can hold, table's pointer, its row stride, page_size, number of pages)."""
    assert k.dtype is dtype and v.dtype is dtype, "cache dtype must equal the new tokens' dtype"
    assert k.get_device() == dev and v.get_device() == dev, "caches must be on the new tokens' device"
    shape = k.shape
    assert len(shape) == 4 and v.shape == shape and shape[1] == Hkv and shape[3] == D, \
        "caches must be [.., num_kv_heads, rows, head_dim], both alike"
    kr, vr = rows_of(k), rows_of(v)
    assert kr is not None and vr is not None, \
        "caches must have 16-byte rows: unit stride in head_dim, other strides multiples of 8 elements, a 16-byte aligned base"
    if block_table is None:
        assert shape[0] >= B, "dense caches must be [bsz, num_kv_heads, ctx, head_dim]"
        return kr, vr, min(shape[2], _MOST_ROWS), 0, 0, 0, 0
    page = shape[2]
    assert page % 64 == 0 and page > 0, "page_size must be a multiple of 64"
    rows, width = block_table.shape
    assert rows == B, "block_table must be [bsz, max_pages]"
    return kr, vr, min(width * page, _MOST_ROWS), block_table.data_ptr(), block_table.stride(0), page, shape[0]


def table_of(block_table: Optional[torch.Tensor], caches: torch.Tensor) -> Optional[torch.Tensor]:
    """The table as the kernels read it: int32, unit stride along a row, on the caches' device."""
    if block_table is None:
        return None
    assert block_table.dtype in _LEN and block_table.dim() == 2, "block_table must be [bsz, max_pages] int32"
    if block_table.dtype is not torch.int32 or block_table.get_device() != caches.get_device() or block_table.stride(1) != 1:
        block_table = block_table.to(device=caches.device, dtype=torch.int32).contiguous()
    return block_table


def check_in_place(k: torch.Tensor, v: torch.Tensor, kr, vr, kv_seq_len: torch.Tensor, B: int) -> None:
    """kr, vr: the caches' pointers and strides."""
    assert kr[0] != vr[0], "k_cache and v_cache are updated in place and must be two tensors"
    assert (0 not in kr or not _overlaps(k)) and (0 not in vr or not _overlaps(v)), "caches are updated in place and must not be expanded"
    assert B <= 1 or kv_seq_len.stride(0) == 1, "kv_seq_len is updated in place and must be contiguous"


def _overlaps(t: torch.Tensor) -> bool:
    """Whether some dimension is broadcast (stride 0)."""
    return 0 in t.stride() and any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride()))


def check_weights(w: torch.Tensor, B: int, Hkv: int, ctx: int, dev: int):
    """(pointer, strides of the two leading dimensions)"""
    b, h, n = w.shape
    sb, sh, one = w.stride()
    assert w.dtype is _f32 and w.get_device() == dev and b == B and h == Hkv and n >= ctx and (one == 1 or n <= 1) and not _overlaps(w), \
        "row_weights must be [bsz, num_kv_heads, ctx] fp32 on the caches' device, unit stride along ctx"
    return w.data_ptr(), sb, sh


def _decode(q, k, v, kv_seq_len, block_table, max_seq_len_in_batch, sm_scale, kv_group_num, softcap, alibi_slopes, window, row_weights,
            return_lse, grid=0):
    lib = _lib.load()
    if not q.is_cuda:
        raise RuntimeError("decode_attention runs on CUDA tensors only (no CPU path exists)")
    B, H, one, D = q.shape
    dt = q.dtype
    dev = q.get_device()
    code = _DT.get(dt)
    G = int(kv_group_num)
    assert one == 1, "q must be [bsz, num_heads, 1, head_dim]: one new token per sequence"
    assert D in _HEAD_DIMS and code is not None, "q must be fp16 or bf16 with head_dim 32, 64, 128 or 256"
    assert G >= 1 and H % G == 0, "num_heads must be a multiple of kv_group_num"
    Hkv = H // G
    block_table = table_of(block_table, k)
    kr, vr, ctx, table, table_sb, page, n_pages = check_caches(k, v, B, Hkv, D, dt, dev, block_table)
    is64 = check_lengths(kv_seq_len, B, dev)
    if max_seq_len_in_batch is not None:
        ctx = min(ctx, int(max_seq_len_in_batch))
    qr = rows_of(q)
    if qr is None:
        q = q.clone(memory_format=torch.contiguous_format)
        qr = rows_of(q)
    if B > 1 and kv_seq_len.stride(0) != 1:
        kv_seq_len = kv_seq_len.contiguous()
    if softcap is not None:
        softcap = float(softcap)
        assert 0.0 < softcap < math.inf, "softcap must be positive"
    if window is not None:
        window = min(int(window), 0x7fffffff)
        assert window > 0, "window must be positive"
    slopes = 0
    if alibi_slopes is not None:
        assert alibi_slopes.dtype is _f32 and alibi_slopes.shape == (H,) and alibi_slopes.get_device() == dev \
            and alibi_slopes.is_contiguous(), "alibi_slopes must be [num_heads] fp32 on q's device"
        slopes = alibi_slopes.data_ptr()
    weights = row_weights is not None
    rw, rw_sb, rw_sh = check_weights(row_weights, B, Hkv, ctx, dev) if weights else (0, 0, 0)
    out = torch.empty_like(q) if q.is_contiguous() else torch.empty(B, H, 1, D, dtype=dt, device=q.device)
    lse = torch.empty(B, H, 1, dtype=_f32, device=q.device) if return_lse else None
    if B and H:
        size = _workspace(lib, dev, B, H, Hkv, D, ctx, code, weights, window or 0, grid)
        ws = out.new_empty(size) if size else None  # `size` elements of two bytes each
        launch(lib.fta_decode_token, pack_token(
            qr[0], qr[1], qr[2], *kr, *vr, kv_seq_len.data_ptr(), table, table_sb, slopes, out.data_ptr(), H * D, D,
            lse.data_ptr() if return_lse else 0, H, rw, rw_sb, rw_sh, ws.data_ptr() if size else 0, 2 * size,
            1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), softcap or 0.0, window or 0, is64,
            B, H, Hkv, D, ctx, page, n_pages, code, grid, 0), dev, "fta_decode_token")
    return (out, lse) if return_lse else out


_ws_sizes = {}  # sizes -> 16-bit elements of workspace: a function of the sizes and the device alone


def _workspace(lib, *key) -> int:
    size = _ws_sizes.get(key)
    if size is None:
        index, B, H, Hkv, D, ctx, code, weights, window, grid = key
        p = _lib.FtaTokenParams()
        p.B, p.H, p.Hkv, p.D, p.ctx, p.dtype, p.grid_override = B, H, Hkv, D, ctx, code, grid
        p.row_weights, p.window = 1 if weights else 0, window
        with torch.cuda.device(index):
            size = lib.fta_decode_token_workspace_bytes(_lib.byref(p))
        if size < 0:
            raise _lib.FtaError(-size, "fta_decode_token_workspace_bytes")
        size = (size + 1) // 2
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
            softmax weights that the group's query heads gave it (what evict_rows goes by).  The call then
            keeps every score until it ends, 4 bytes x bsz x num_heads x ctx of scratch by the cache's
            capacity, not the lengths: 2 GB for 64 sequences of 131072 rows and 64 heads.
            max_seq_len_in_batch bounds that too.
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
        budget, recent: 1 <= budget <= 2^31 - 2^16, 0 <= recent <= budget.

    Returns kept [bsz, num_kv_heads, budget] int32, the old row of every row now in the cache (-1 past
    a shorter sequence's end).  Keys keep the rotary positions they were written with; a caller that
    needs rows' positions keeps them by `kept`.  Asynchronous on the current stream of the caches'
    device, no host synchronisation.
    """
    lib = _lib.load()
    if not k_cache.is_cuda:
        raise RuntimeError("evict_rows runs on CUDA tensors only (no CPU path exists)")
    dt, dev = k_cache.dtype, k_cache.get_device()
    assert dt in _DT and k_cache.dim() == 4 and kv_seq_len.dim() == 1, \
        "caches must be fp16 or bf16 [.., num_kv_heads, rows, head_dim], kv_seq_len [bsz]"
    B = kv_seq_len.size(0)
    _, Hkv, _, D = k_cache.shape
    assert D in _HEAD_DIMS, "head_dim must be 32, 64, 128 or 256"
    block_table = table_of(block_table, k_cache)
    kr, vr, ctx, table, table_sb, page, n_pages = check_caches(k_cache, v_cache, B, Hkv, D, dt, dev, block_table)
    is64 = check_lengths(kv_seq_len, B, dev)
    check_in_place(k_cache, v_cache, kr, vr, kv_seq_len, B)
    assert row_weights.dim() == 3, "row_weights must be [bsz, num_kv_heads, ctx]"
    rw, rw_sb, rw_sh = check_weights(row_weights, B, Hkv, ctx, dev)
    budget, recent = int(budget), int(recent)
    assert 1 <= budget <= _MOST_ROWS and 0 <= recent <= budget, "1 <= budget <= 2^31 - 2^16 and 0 <= recent <= budget"
    kept = torch.empty(B, Hkv, budget, dtype=torch.int32, device=k_cache.device)
    if B and Hkv:
        launch(lib.fta_evict_rows, pack_evict(*kr, *vr, kv_seq_len.data_ptr(), table, table_sb, rw, rw_sb, rw_sh, kept.data_ptr(),
                                              is64, B, Hkv, D, ctx, page, n_pages, budget, recent, 0), dev, "fta_evict_rows")
    return kept
