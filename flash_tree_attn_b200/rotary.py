"""Rotary positions of queries and keys, and the append of new tokens to the cache.

Frequencies are data: any scheme for long contexts is a list of radians per position, one for each
pair, in 64 bits (`rotary_frequencies` makes the usual ones).  Positions are integers, and angles are
taken modulo one turn in whole numbers: an angle is off by |position| * (inv_freq / 2 pi * 2^-52 + 2^-65)
of a turn and 2^-26 of a turn for 32-bit cosines, so that positions up to 2^28 lose less than 32 bits
hold.  All arithmetic happens in libfta.so.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import launch, pack_rotary, rows_of
from .decode import _DT, _HEAD_DIMS, _LEN, check_caches, check_in_place, check_lengths, table_of

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


def _rows(t: torch.Tensor):
    """(the tensor or a copy of it with rows that can be copied in 16-byte pieces, its pointer and strides)"""
    r = rows_of(t)
    if r is None:
        t = t.clone(memory_format=torch.contiguous_format)
        r = rows_of(t)
    return t, r


def _check_frequencies(inv_freq: torch.Tensor, D: int, dev: int, layout: str):
    """(number of pairs, layout's code)"""
    code = _LAYOUT.get(layout)
    assert code is not None, "layout: half or interleaved"
    assert inv_freq.dtype is torch.float64 and inv_freq.dim() == 1 and inv_freq.get_device() == dev and inv_freq.is_contiguous(), \
        "inv_freq must be a contiguous float64 vector on q's device"
    n = inv_freq.size(0)
    assert n > 0 and n % 8 == 0 and 2 * n <= D, "inv_freq must have a multiple of 8 entries, at most head_dim / 2"
    return n, code


def _check_positions(positions: torch.Tensor, B: int, Q: int, dev: int):
    """(the tensor or a copy, its pointer, stride along bsz, stride along q_len (0: consecutive positions), is int64)"""
    is64, shape = _LEN.get(positions.dtype), positions.shape
    assert is64 is not None and positions.get_device() == dev and (shape == (B,) or shape == (B, Q)), \
        "positions must be [bsz] or [bsz, q_len] int32 or int64 on q's device"
    if len(shape) == 1:
        return positions, positions.data_ptr(), positions.stride(0), 0, is64
    if positions.stride(1) == 0:  # the same position for every token: as a stride, 0 would mean consecutive ones
        positions = positions.clone(memory_format=torch.contiguous_format)
    return positions, positions.data_ptr(), positions.stride(0), positions.stride(1), is64


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
    dt, dev = q.dtype, q.get_device()
    code = _DT.get(dt)
    assert code is not None and D in _HEAD_DIMS, "q must be fp16 or bf16 with head_dim 32, 64, 128 or 256"
    n, layout = _check_frequencies(inv_freq, D, dev, layout)
    q, qr = _rows(q)
    qo = torch.empty_like(q) if q.is_contiguous() else torch.empty_like(q, memory_format=torch.contiguous_format)
    Hkv, kr, ko, kp = 0, (0, 0, 0, 0), None, 0
    if k is not None:
        assert k.dtype is dt and k.get_device() == dev and k.dim() == 4, "k must be of q's dtype and on its device"
        kb, Hkv, kq, kd = k.shape
        assert kb == B and kq == Q and kd == D, "k must be [bsz, num_kv_heads, q_len, head_dim]"
        k, kr = _rows(k)
        ko = torch.empty_like(k) if k.is_contiguous() else torch.empty_like(k, memory_format=torch.contiguous_format)
        kp = ko.data_ptr()
    positions, pos, psb, psq, is64 = _check_positions(positions, B, Q, dev)
    off = 0
    if offsets is not None:
        assert offsets.dtype is torch.int32 and offsets.shape == (Q,) and offsets.get_device() == dev and offsets.is_contiguous(), \
            "offsets must be [q_len] int32 on q's device"
        off = offsets.data_ptr()
    if B and Q and H + Hkv:
        launch(lib.fta_apply_rotary, pack_rotary(
            *qr, *kr, 0, 0, 0, 0, qo.data_ptr(), kp, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, pos, psb, psq, off, inv_freq.data_ptr(),
            float(amplitude), layout, 1 if inverse else 0, n, 0, is64, B, H, Hkv, Q, D, 0, 0, 0, code, 0), dev, "fta_apply_rotary")
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
    dt, dev = k.dtype, k_cache.get_device()
    code = _DT.get(dt)
    assert code is not None and D in _HEAD_DIMS, "k must be fp16 or bf16 with head_dim 32, 64, 128 or 256"
    assert k.get_device() == dev and v.get_device() == dev and v.dtype is dt and v.shape == k.shape, "k and v must be alike, on the caches' device"
    block_table = table_of(block_table, k_cache)
    kc, vc, ctx, table, table_sb, page, n_pages = check_caches(k_cache, v_cache, B, Hkv, D, dt, dev, block_table)
    len64 = check_lengths(kv_seq_len, B, dev)
    check_in_place(k_cache, v_cache, kc, vc, kv_seq_len, B)
    qb, H, qq, qd = q.shape
    assert qb == B and qq == Q and qd == D and q.dtype is dt and q.get_device() == dev, \
        "q must be [bsz, num_heads, q_len, head_dim] of k's dtype and on its device"
    k, kr = _rows(k)
    v, vr = _rows(v)
    out, qr, qo, n, pos, psb, psq, is64, freq = q, (0, 0, 0, 0), 0, 0, 0, 0, 0, 0, 0
    if inv_freq is not None:
        n, layout = _check_frequencies(inv_freq, D, dev, layout)
        q, qr = _rows(q)
        out = torch.empty_like(q) if q.is_contiguous() else torch.empty_like(q, memory_format=torch.contiguous_format)
        qo, freq = out.data_ptr(), inv_freq.data_ptr()
        if positions is not None:
            positions, pos, psb, psq, is64 = _check_positions(positions, B, Q, dev)
    else:
        layout, H = 0, 0
    if B and Q and Hkv:
        launch(lib.fta_append_tokens, pack_rotary(
            *qr, *kr, *vr, qo, 0, *kc, *vc, kv_seq_len.data_ptr(), table, table_sb, pos, psb, psq, 0, freq,
            float(amplitude), layout, 0, n, len64, is64, B, H, Hkv, Q, D, ctx, page, n_pages, code, 0), dev, "fta_append_tokens")
    return out
