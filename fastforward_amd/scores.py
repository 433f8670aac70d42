"""Scores of given tokens from rows of logits, on gfx950 kernels.

No reference counterpart: the reference scores options by the logit of one letter
(``ops.lm_readout``). An answer that is a text is scored by its tokens' log
probabilities, one row of vocabulary logits per position.

Like the other ops: shape, dtype and device violations raise AssertionError before any
launch, outputs are fresh tensors, inputs are never written, launches go to the current
stream and can be captured (no host sync, no device-dependent grid).
"""
import ctypes
import functools
from typing import NamedTuple, Optional

import torch

from ._lib import call, entry, stream

BF16, F32 = torch.bfloat16, torch.float32
MAX_TOP = 64


class TokenScores(NamedTuple):
    logprobs: torch.Tensor                 # the shape of the tokens, fp32
    entropy: torch.Tensor                  # (T,) fp32
    top_logprobs: Optional[torch.Tensor]   # (T, top) fp32, falling
    top_ids: Optional[torch.Tensor]        # (T, top) int32


@functools.lru_cache(maxsize=1024)
def scores_workspace(t, v, top):
    """Bytes of workspace ff_token_scores needs (0: none)."""
    need = ctypes.c_int64(0)
    call("ff_token_scores_workspace", t, v, top, ctypes.byref(need))
    return need.value


def token_scores(logits, tokens, top=0):
    """Scores of ``tokens`` (T,) or (T, N) int64 under softmax(logits) of rows (T, V), bf16 or
    fp32: ``logprobs`` (the tokens' shape), log p; ``entropy`` (T,), -sum p log p in nats;
    with ``top`` (at most 64) the ``top`` likeliest tokens of each row, ``top_ids`` (lowest
    index first among equals) and their ``top_logprobs``.

    A logit of -inf switches its token off: log p = -inf, nothing in the entropy. A token
    outside [0, V) is none and scores 0 (padding adds nothing to a sum). A row that is
    switched off altogether has log p -inf and entropy 0; a row with a NaN or +inf has NaN
    scores, its ``top_ids`` still in order (NaN first). Sums are fp32 over all but the
    maximum, so that log p of a near-certain token keeps its relative precision."""
    assert logits.dim() == 2 and logits.dtype in (BF16, F32), (logits.shape, logits.dtype)
    t, v = logits.shape
    assert 0 < v < 1 << 31 and t <= 1 << 24, (t, v)
    assert 0 <= top <= min(MAX_TOP, v), (top, v)
    assert tokens.dtype == torch.int64 and tokens.dim() in (1, 2) and tokens.shape[0] == t, (tokens.shape, tokens.dtype)
    n = 1 if tokens.dim() == 1 else tokens.shape[1]
    assert n <= 65536, n
    here = logits.get_device()
    assert here == tokens.get_device() >= 0, f"logits on {logits.device}, tokens on {tokens.device}"
    assert torch._C._cuda_getDevice() == here, f"tensors on GPU {here}, which is not the current one"
    ld, step = logits.stride()
    if step != 1 and v > 1:
        logits, ld = logits.contiguous(), v
    strides = tokens.stride()
    logprobs = torch.empty_like(tokens, dtype=F32, memory_format=torch.contiguous_format)
    entropy = logits.new_empty(t, dtype=F32)
    top_logprobs = logits.new_empty(t, top, dtype=F32) if top else None
    top_ids = logits.new_empty(t, top, dtype=torch.int32) if top else None
    need = scores_workspace(t, v, top)
    ws = logits.new_empty(need, dtype=torch.uint8) if need else None
    entry("ff_token_scores")(logits.data_ptr(), logits.dtype == F32, ld, tokens.data_ptr(), strides[0], strides[-1],
                             logprobs.data_ptr(), entropy.data_ptr(), top_logprobs.data_ptr() if top else 0,
                             top_ids.data_ptr() if top else 0, t, v, n, top, 0 if ws is None else ws.data_ptr(), need,
                             stream())
    return TokenScores(logprobs, entropy, top_logprobs, top_ids)


__all__ = ["token_scores", "TokenScores", "scores_workspace"]
