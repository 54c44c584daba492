"""Log probabilities of given tokens under rows of logits: what an acceptance rule goes by.

One pass over the logits gives the log-sum-exp, the entropy, the log probabilities of the given
tokens and the likeliest tokens.  All arithmetic happens in libfta.so, in 32 bits.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import launch, pack_logprob

_DT = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
_LEN = {torch.int32: 0, torch.int64: 1}  # -> is int64
MAX_TOP_K = 64


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]      # [.., n] fp32, of the given tokens
    entropy: torch.Tensor                 # [..] fp32
    lse: torch.Tensor                     # [..] fp32
    top_logprobs: Optional[torch.Tensor]  # [.., top_k] fp32, falling
    top_ids: Optional[torch.Tensor]       # [.., top_k] int64


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0) -> TokenLogprobs:
    """Log probabilities (natural logs) of `tokens` under `logits`.

    Args:
        logits: [.., vocab] fp16, bf16 or fp32, unit stride along the vocabulary; any other strides
            that leave the leading dimensions one row stride apart are used as they are.
        tokens: [.., n] int32/int64, n tokens for every row of logits, or None.
        top_k: number of likeliest tokens wanted, 0 to 64 (and at most vocab).

    A token outside [0, vocab), such as a padding of -1, gets -inf.  Ties among the likeliest go to the
    lower token.  A row of nothing but -inf has lse = -inf, entropy 0 and log probabilities of -inf; a
    NaN logit shows as NaN in all of its row's values, and ranks first.  Asynchronous on the current
    stream of the logits' device, no host synchronisation.
    """
    lib = _lib.load()
    if not logits.is_cuda:
        raise RuntimeError("token_logprobs runs on CUDA tensors only (no CPU path exists)")
    dev, code = logits.get_device(), _DT.get(logits.dtype)
    shape = logits.shape
    assert code is not None and len(shape) >= 1 and shape[-1] > 0, "logits must be [.., vocab] fp16, bf16 or fp32"
    lead, V = shape[:-1], shape[-1]
    top_k = int(top_k)
    assert 0 <= top_k <= MAX_TOP_K and top_k <= V, "top_k must be 0 to 64 and at most the vocabulary"
    if len(shape) != 2:
        logits = logits.reshape(-1, V)
    rows = logits.size(0)
    row_stride, one = logits.stride()
    if one != 1 and V > 1:
        logits = logits.contiguous()
        row_stride = V
    # sizes one by one: a tuple of them costs half as much again to read
    entropy = torch.empty(*lead, dtype=torch.float32, device=logits.device) if lead else logits.new_empty((), dtype=torch.float32)
    lse = torch.empty_like(entropy)
    n = tp = token_stride = t64 = 0
    lp = top_lp = top_ids = None
    if tokens is not None:
        t64 = _LEN.get(tokens.dtype)
        ts = tokens.shape
        assert t64 is not None and tokens.get_device() == dev and len(ts) == len(shape) and ts[:-1] == lead, \
            "tokens must be [.., n] int32 or int64 on the logits' device, with the logits' leading sizes"
        n = ts[-1]
        lp = entropy.new_empty(*ts)
        if len(ts) != 2:
            tokens = tokens.reshape(rows, n)
        token_stride, one = tokens.stride()
        if one != 1 and n > 1:
            tokens = tokens.contiguous()
            token_stride = n
        tp = tokens.data_ptr()
    if top_k:
        top_lp = entropy.new_empty(*lead, top_k)
        top_ids = torch.empty_like(top_lp, dtype=torch.int64)
    if rows:
        launch(lib.fta_token_logprobs, pack_logprob(
            logits.data_ptr(), row_stride, tp, token_stride, lp.data_ptr() if n else 0, entropy.data_ptr(), lse.data_ptr(),
            top_lp.data_ptr() if top_k else 0, top_ids.data_ptr() if top_k else 0, rows, V, n, top_k, code, t64), dev, "fta_token_logprobs")
    return TokenLogprobs(lp, entropy, lse, top_lp, top_ids)
