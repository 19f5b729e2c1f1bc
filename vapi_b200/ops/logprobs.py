"""Log probabilities of given tokens, entropy, and the most likely tokens (csrc/logprobs.cu)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import KernelError, _check, _contig, _cuda, _dt, _here, _i32, _lib, _native, _p, _stream

#: alternatives that one call reports at most
LOGPROBS_MAX_TOP = 64


class TokenLogprobs(NamedTuple):
    """Per row of logits, natural logarithms in float32."""

    logprob: torch.Tensor        # [R]: of the given token
    entropy: torch.Tensor        # [R]: of the row's distribution
    top_ids: torch.Tensor        # [R, top] int32: the most likely tokens, most likely first, ties by lower id
    top_logprobs: torch.Tensor   # [R, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0, status: Optional[torch.Tensor] = None,
                   slices: int = 0) -> TokenLogprobs:
    """What the softmax of each row of ``logits`` [R, V] (float32 or bfloat16, rows at any stride) says of ``tokens`` [R] (int32): the
    log probability of the given token, the entropy, and the ``top`` (0..64, at most V) most likely tokens with their log
    probabilities.  The logits are read once.

    A token outside the vocabulary gets NaN and a status.  Logits of -inf are tokens of probability zero, like any other in the
    ranking.  A row with a NaN or +inf, or of nothing but -inf, has NaN for its numbers (which tokens it then ranks is not said; -1 stands
    where there are none).  ``slices``: into how many blocks a row is cut (a power of two up to 8; 0: as many as pay); in another
    cut the sums are added in another order."""
    if logits.is_cuda:
        lib = _lib("logprobs")
        got = _native("logprobs", lib, "vapi_token_logprobs", logits, tokens, top, slices, _p(status))
        if got is not NotImplemented:
            _check(lib, got if type(got) is int else 0, int(logits.shape[0] > 0))
            return TokenLogprobs._make(got)
    if logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise KernelError("logits must be [R, V] with unit inner stride")
    dt = _dt(logits)
    _i32(tokens, "tokens")
    _contig(tokens, "tokens")
    rows, vocab = logits.shape
    if tuple(tokens.shape) != (rows,):
        raise KernelError(f"tokens must be [{rows}], got {tuple(tokens.shape)}")
    if not 0 <= top <= min(LOGPROBS_MAX_TOP, vocab):
        raise KernelError(f"{top} alternatives are outside 0..{min(LOGPROBS_MAX_TOP, vocab)}")
    _cuda(logits, tokens)
    _here(logits, tokens)
    empty = lambda shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=logits.device)
    out = TokenLogprobs(empty(rows), empty(rows), empty((rows, top), torch.int32), empty((rows, top)))
    lib = _lib("logprobs")
    _check(lib, lib.vapi_token_logprobs(_p(logits), dt, rows, vocab, logits.stride(0), _p(tokens), top, out.logprob.data_ptr(),
                                        out.entropy.data_ptr(), out.top_ids.data_ptr(), out.top_logprobs.data_ptr(), slices, _p(status),
                                        _stream()), launches=int(rows > 0))
    return out
