"""Log probabilities of given tokens under rows of logits: what an acceptance rule goes by.

One pass over the logits gives the log-sum-exp, the entropy, the log probabilities of the given
tokens and the likeliest tokens.  All arithmetic happens in libfta.so, in 32 bits.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import on_device

_DT = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}
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
    dev, dt = logits.device, logits.dtype
    assert dt in _DT, "logits must be fp16, bf16 or fp32"
    assert logits.dim() >= 1 and logits.size(-1) > 0, "logits must be [.., vocab]"
    lead, V = logits.shape[:-1], logits.size(-1)
    top_k = int(top_k)
    assert 0 <= top_k <= min(MAX_TOP_K, V), "top_k must be 0 to 64 and at most the vocabulary"
    if logits.dim() != 2:
        logits = logits.reshape(-1, V)
    rows = logits.size(0)
    if V > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    n, tp, tsr, t64, lp = 0, 0, 0, 0, None
    if tokens is not None:
        assert tokens.dtype in (torch.int32, torch.int64) and tokens.device == dev and tokens.dim() == len(lead) + 1 \
            and tokens.shape[:-1] == lead, "tokens must be [.., n] int32 or int64 on the logits' device, with the logits' leading sizes"
        n = tokens.size(-1)
        if tokens.dim() != 2:
            tokens = tokens.reshape(rows, n)
        if n > 1 and tokens.stride(1) != 1:
            tokens = tokens.contiguous()
        tp, tsr, t64 = tokens.data_ptr(), tokens.stride(0), 1 if tokens.dtype == torch.int64 else 0
        lp = torch.empty((*lead, n), dtype=torch.float32, device=dev)
    entropy, lse = torch.empty((2, *lead), dtype=torch.float32, device=dev).unbind(0)
    top_lp = top_ids = None
    if top_k:
        top_lp = torch.empty((*lead, top_k), dtype=torch.float32, device=dev)
        top_ids = torch.empty((*lead, top_k), dtype=torch.int64, device=dev)
    if rows:
        with on_device(dev) as stream:
            p = [logits.data_ptr(), logits.stride(0), tp, tsr, lp.data_ptr() if n else 0, entropy.data_ptr(), lse.data_ptr(),
                 top_lp.data_ptr() if top_k else 0, top_ids.data_ptr() if top_k else 0, 0, 0, rows, V, n, top_k, _DT[dt], t64]
            size = lib.fta_token_logprobs_workspace_bytes(_lib.pack_logprob(*p))
            if size < 0:
                raise _lib.FtaError(-size, "fta_token_logprobs_workspace_bytes")
            ws = torch.empty(size, dtype=torch.uint8, device=dev)
            p[9], p[10] = ws.data_ptr(), size
            _lib.check(lib.fta_token_logprobs(_lib.pack_logprob(*p), stream), "fta_token_logprobs")
    return TokenLogprobs(lp, entropy, lse, top_lp, top_ids)
