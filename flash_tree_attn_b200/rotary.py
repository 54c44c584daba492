"""Rotary positions of queries and keys, and the append of new tokens to the cache.

Frequencies are data: any scheme for long contexts is a list of radians per position, one for each
pair, in 64 bits (`rotary_frequencies` makes the usual ones).  A position is an integer of any size;
angles are taken modulo one turn in whole numbers, so far positions lose nothing.  All arithmetic
happens in libfta.so.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import on_device, rows_ok
from .decode import _DT, _LEN, _check_caches, _check_lengths, _overlaps

_LAYOUT = {"half": _lib.ROTARY_HALF, "interleaved": _lib.ROTARY_INTERLEAVED}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original_len: int = 8192, *,
                       low: float = 1.0, high: float = 4.0, fast: float = 32.0, slow: float = 1.0,
                       device="cuda") -> Tuple[torch.Tensor, float]:
    """inv_freq [rotary_dim / 2] float64 on `device`, and the factor on cosine and sine.

    Pair i turns by base ** (-2 i / rotary_dim) radians a position, changed by `scaling`:
        "none"    nothing
        "linear"  divided by factor (positions are squeezed)
        "base"    the base grows by factor ** (rotary_dim / (rotary_dim - 2)): the longest wavelength by factor
        "bands"   by the turns a pair makes over original_len positions: at most `low`, divided by
                  factor; at least `high`, unchanged; between, a linear blend of the two
        "ramp"    the blend runs linearly over the pair's index between those that make `fast` and
                  `slow` turns, and the factor on cosine and sine is 0.1 ln(factor) + 1
    """
    assert rotary_dim >= 2 and rotary_dim % 2 == 0 and base > 1.0 and factor >= 1.0 and original_len > 0
    assert scaling in ("none", "linear", "base", "bands", "ramp"), "scaling: none, linear, base, bands or ramp"
    n, amplitude = rotary_dim // 2, 1.0
    if scaling == "base":
        assert rotary_dim > 2, "a single pair has no longest wavelength to stretch"
        base = base * factor ** (rotary_dim / (rotary_dim - 2.0))
    plain = [base ** (-2.0 * i / rotary_dim) for i in range(n)]
    keep = [1.0] * n  # the share that stays as it is
    if scaling == "linear":
        keep = [0.0] * n
    elif scaling == "bands":
        assert high > low
        keep = [(original_len * f / (2.0 * math.pi) - low) / (high - low) for f in plain]
    elif scaling == "ramp":
        def index(turns):
            return rotary_dim * math.log(original_len / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

        first, last = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), rotary_dim - 1)
        keep = [1.0 - (i - first) / max(last - first, 0.001) for i in range(n)]
        amplitude = 0.1 * math.log(factor) + 1.0
    keep = [min(1.0, max(0.0, x)) for x in keep]
    return torch.tensor([f * x + f / factor * (1.0 - x) for f, x in zip(plain, keep)], dtype=torch.float64, device=device), amplitude


def _rows(t: torch.Tensor) -> torch.Tensor:
    return t if rows_ok(t) else t.clone(memory_format=torch.contiguous_format)


def _check_frequencies(inv_freq: torch.Tensor, D: int, dev, layout: str) -> int:
    assert layout in _LAYOUT, "layout: half or interleaved"
    n = inv_freq.numel()
    assert inv_freq.dtype == torch.float64 and inv_freq.dim() == 1 and inv_freq.device == dev and inv_freq.is_contiguous(), \
        "inv_freq must be a contiguous float64 vector on q's device"
    assert n > 0 and n % 8 == 0 and 2 * n <= D, "inv_freq must have a multiple of 8 entries, at most head_dim / 2"
    return n


def _check_positions(positions: torch.Tensor, offsets: Optional[torch.Tensor], B: int, Q: int, dev):
    """-> (pointer, stride along bsz, stride along q_len, is int64, offsets' pointer)"""
    assert positions.dtype in _LEN and positions.device == dev and tuple(positions.shape) in ((B,), (B, Q)), \
        "positions must be [bsz] or [bsz, q_len] int32 or int64 on q's device"
    if offsets is not None:
        assert offsets.dtype == torch.int32 and offsets.shape == (Q,) and offsets.device == dev and offsets.is_contiguous(), \
            "offsets must be [q_len] int32 on q's device"
    each = positions.dim() == 2
    if each and positions.stride(1) == 0:  # the same position for every token: stride 0 would mean consecutive ones
        positions = positions.contiguous()
        if positions.stride(1) == 0:
            positions = positions.clone(memory_format=torch.contiguous_format)
    return positions, positions.stride(0), positions.stride(1) if each else 0, 1 if positions.dtype == torch.int64 else 0, \
        0 if offsets is None else offsets.data_ptr()


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 offsets: Optional[torch.Tensor] = None, layout: str = "half", amplitude: float = 1.0, inverse: bool = False):
    """Rotate queries and keys to their positions; returns new tensors (q, k).

    Args:
        q: [bsz, num_heads, q_len, head_dim] fp16/bf16, head_dim 32, 64, 128 or 256.
        k: [bsz, num_kv_heads, q_len, head_dim] of q's dtype, or None.
        positions: [bsz] the first token's position (token i lies offsets[i], or without offsets i,
            further on), or [bsz, q_len] every token's (offsets, if given, are added); int32/int64.
        inv_freq: [n] float64, radians per position of the n pairs; n a multiple of 8.  The first
            2 n elements of a head turn, the others are copied.
        offsets: [q_len] int32, e.g. the depths of a draft tree's nodes (`DraftTree.depth`).
        layout: pairs are elements (i, i + n): "half", or (2 i, 2 i + 1): "interleaved".
        amplitude: factor on cosine and sine.
        inverse: turn back by the same angles (times amplitude).  That is the transpose, so it takes
            the gradients of the outputs to the gradients of the inputs.

    Computed in 32 bits and rounded once.  Asynchronous on the current stream of q's device.
    """
    lib = _lib.load()
    if not q.is_cuda:
        raise RuntimeError("apply_rotary runs on CUDA tensors only (no CPU path exists)")
    B, H, Q, D = q.shape
    dt, dev = q.dtype, q.device
    assert dt in _DT and D in (32, 64, 128, 256), "q must be fp16 or bf16 with head_dim 32, 64, 128 or 256"
    n = _check_frequencies(inv_freq, D, dev, layout)
    q = _rows(q)
    qo = torch.empty((B, H, Q, D), dtype=dt, device=dev)
    Hkv, kp, ks, ko = 0, 0, (0, 0, 0), None
    if k is not None:
        assert k.dtype == dt and k.device == dev and k.dim() == 4 and k.size(0) == B and k.size(2) == Q and k.size(3) == D, \
            "k must be [bsz, num_kv_heads, q_len, head_dim] of q's dtype and on its device"
        k = _rows(k)
        Hkv, kp, ks = k.size(1), k.data_ptr(), k.stride()
        ko = torch.empty((B, Hkv, Q, D), dtype=dt, device=dev)
    positions, psb, psq, is64, off = _check_positions(positions, offsets, B, Q, dev)
    if B == 0 or Q == 0 or H + Hkv == 0:
        return qo, ko
    qs = q.stride()
    p = _lib.pack_rotary(
        q.data_ptr(), qs[0], qs[1], qs[2], kp, ks[0], ks[1], ks[2], 0, 0, 0, 0, qo.data_ptr(), 0 if ko is None else ko.data_ptr(),
        0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, positions.data_ptr(), psb, psq, off, inv_freq.data_ptr(),
        float(amplitude), _LAYOUT[layout], 1 if inverse else 0, n, 0, is64, B, H, Hkv, Q, D, 0, 0, 0, _DT[dt], 0)
    with on_device(dev) as stream:
        _lib.check(lib.fta_apply_rotary(p, stream), "fta_apply_rotary")
    return qo, ko


def append_tokens(k_cache, v_cache, q, k, v, kv_seq_len, *, inv_freq: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                  layout: str = "half", amplitude: float = 1.0, block_table: Optional[torch.Tensor] = None):
    """Rotate new tokens to their positions and append their keys and values to the cache, in place.

    Args:
        k_cache, v_cache: dense [bsz, num_kv_heads, ctx, head_dim], or pools of pages with `block_table`.
        q: [bsz, num_heads, q_len, head_dim] of the new tokens, k, v: [bsz, num_kv_heads, q_len, head_dim].
            q_len is 1 in a decoding step and longer for a chunk of a prompt.
        kv_seq_len: [bsz] int32/int64 on the device, grows by q_len in place (at most to what the cache holds).
        inv_freq, layout, amplitude: as apply_rotary; without inv_freq nothing is rotated.
        positions: [bsz] or [bsz, q_len] as apply_rotary; by default a token's position is its cache row,
            kv_seq_len[b] + i.  Give them where rows have been evicted.

    Token i of sequence b becomes cache row kv_seq_len[b] + i; rows past the cache's end are dropped.
    Returns the rotated q (q itself without inv_freq).  Asynchronous on the current stream, no host
    synchronisation.
    """
    lib = _lib.load()
    if not k_cache.is_cuda:
        raise RuntimeError("append_tokens runs on CUDA tensors only (no CPU path exists)")
    B, Hkv, Q, D = k.shape
    dt, dev = k.dtype, k_cache.device
    assert dt in _DT and D in (32, 64, 128, 256), "k must be fp16 or bf16 with head_dim 32, 64, 128 or 256"
    assert k.device == dev and v.device == dev and v.dtype == dt and v.shape == k.shape, "k and v must be alike, on the caches' device"
    ctx = _check_caches(k_cache, v_cache, B, Hkv, D, dt, dev, block_table)
    _check_lengths(kv_seq_len, B, dev)
    assert rows_ok(k_cache) and rows_ok(v_cache) and not _overlaps(k_cache) and not _overlaps(v_cache), \
        "caches are updated in place: they must have 16-byte rows and must not be expanded"
    assert B <= 1 or kv_seq_len.stride(0) == 1, "kv_seq_len is updated in place and must be contiguous"
    assert q.dim() == 4 and q.size(0) == B and q.size(2) == Q and q.size(3) == D and q.dtype == dt and q.device == dev, \
        "q must be [bsz, num_heads, q_len, head_dim] of k's dtype and on its device"
    n, out, H, qp, qs = 0, q, 0, 0, (0, 0, 0)
    k, v = _rows(k), _rows(v)
    psb = psq = is64 = pos = freq = 0
    if inv_freq is not None:
        n = _check_frequencies(inv_freq, D, dev, layout)
        H = q.size(1)
        q = _rows(q)
        out = torch.empty((B, H, Q, D), dtype=dt, device=dev)
        qp, qs, freq = q.data_ptr(), q.stride(), inv_freq.data_ptr()
        if positions is not None:
            positions, psb, psq, is64, _ = _check_positions(positions, None, B, Q, dev)
            pos = positions.data_ptr()
    if B == 0 or Q == 0 or Hkv == 0:
        return out
    ks, vs, kc, vc = k.stride(), v.stride(), k_cache.stride(), v_cache.stride()
    paged = block_table is not None
    p = _lib.pack_rotary(
        qp, qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], out.data_ptr() if n else 0, 0,
        k_cache.data_ptr(), kc[0], kc[1], kc[2], v_cache.data_ptr(), vc[0], vc[1], vc[2], kv_seq_len.data_ptr(),
        block_table.data_ptr() if paged else 0, block_table.stride(0) if paged else 0, pos, psb, psq, 0, freq,
        float(amplitude), _LAYOUT[layout], 0, n, 1 if kv_seq_len.dtype == torch.int64 else 0, is64, B, H, Hkv, Q, D, ctx,
        k_cache.size(2) if paged else 0, k_cache.size(0) if paged else 0, _DT[dt], 0)
    with on_device(dev) as stream:
        _lib.check(lib.fta_append_tokens(p, stream), "fta_append_tokens")
    return out
