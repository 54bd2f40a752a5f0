"""Scoring of logits on librlu.so: log probabilities of given tokens, with their rank, the entropy and
the largest alternatives, in one read of the logits.

No counterpart in the reference, which hands the lm_heads' logits to vLLM's sampler; the results are
those of the server's logprobs (token, rank, top alternatives) for the logits of ops.gemm_fp8_block,
ops.gemm_fp8_dense and w4.gemm_w4a16. ops.Fp8TargetHead.logprobs runs head and scoring together.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from ._lib import check, lib, on_device, stream_ptr

_DTYPE_CODE = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}
MAX_TOP = 32
MAX_VOCAB = 500000


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor        # f32 [R]
    rank: torch.Tensor           # int32 [R], 1 = the largest logit
    entropy: torch.Tensor        # f32 [R], nats
    top_logprobs: torch.Tensor   # f32 [R, top_n], falling
    top_ids: torch.Tensor        # int32 [R, top_n]


@functools.lru_cache(maxsize=4096)
def _workspace(dtype: int, rows: int, vocab: int, top_n: int) -> int:
    n = ctypes.c_longlong()
    check(lib().rlu_token_logprobs_workspace(dtype, rows, vocab, top_n, ctypes.byref(n)),
          "rlu_token_logprobs_workspace")
    return n.value


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top_n: int = 0) -> TokenLogprobs:
    """logits [R, V] bf16, f16 or f32 (rows may be apart: logits[:, :n] of a wider buffer), tokens [R]
    int64 or int32 -> TokenLogprobs, all in float32.

    rank counts the logits before the token's in falling order, ties by the lowest id, as the
    alternatives are ordered. A logit of -inf has probability 0; a row of nothing else gives -inf
    and entropy 0, a row with a NaN or +inf gives NaN, rank 0 and ids -1. A negative token asks for
    none (a padded row): logprob 0, rank 0; one past the vocabulary gives NaN, rank 0."""
    if logits.ndim != 2 or logits.dtype not in _DTYPE_CODE or not logits.is_cuda:
        raise ValueError("token_logprobs takes bf16, f16 or f32 logits [R, V] on the GPU")
    rows, vocab = logits.shape
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"token_logprobs: a vocabulary of {vocab} is outside 1..{MAX_VOCAB}")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("token_logprobs: a row's logits must lie next to each other")
    if tokens.shape != (rows,) or tokens.dtype not in (torch.int64, torch.int32) or \
            not tokens.is_contiguous() or tokens.device != logits.device:
        raise ValueError(f"token_logprobs: tokens must be contiguous int64 or int32 [{rows}] "
                         "beside the logits")
    if not 0 <= top_n <= min(MAX_TOP, vocab):
        raise ValueError(f"token_logprobs: top_n={top_n} is outside 0..{min(MAX_TOP, vocab)}")
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError("token_logprobs has no gradient: detach the logits")
    code, dev = _DTYPE_CODE[logits.dtype], logits.device
    out = TokenLogprobs(torch.empty(rows, dtype=torch.float32, device=dev),
                        torch.empty(rows, dtype=torch.int32, device=dev),
                        torch.empty(rows, dtype=torch.float32, device=dev),
                        torch.empty((rows, top_n), dtype=torch.float32, device=dev),
                        torch.empty((rows, top_n), dtype=torch.int32, device=dev))
    if rows == 0:
        return out
    # taken and given back on the current stream, as the outputs are: calls on two streams, or two
    # captured graphs, have their own
    ws = torch.empty(_workspace(code, rows, vocab, top_n), dtype=torch.uint8, device=dev)
    with on_device(dev):
        rc = lib().rlu_token_logprobs(
            logits.data_ptr(), code, logits.stride(0), rows, vocab, tokens.data_ptr(),
            int(tokens.dtype == torch.int64), top_n, *[t.data_ptr() for t in out], ws.data_ptr(),
            stream_ptr())
    check(rc, "rlu_token_logprobs")
    return out
