"""Losses over logits on librlu.so, with the logits' gradient: the clipped policy loss of sampled tokens with a
KL term, and distillation from a teacher's top log probabilities.

No counterpart in the reference, which serves only. What they learn from is what logprobs.token_logprobs gives:
its log probabilities are a rollout's old and reference ones, its alternatives a teacher's list.

  policy_loss, distill_top              for autograd, in eager code
  policy_loss_grad, distill_top_grad    loss and gradient by hand: into a buffer of the caller's, in place of the
                                        logits, in a captured graph
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from ._lib import check, has_tangent, lib, on_device, stream_ptr, written
from .logprobs import _DTYPE_CODE, MAX_VOCAB

MAX_TOP = 32


class PolicyLoss(NamedTuple):
    loss: torch.Tensor           # f32 [R], each row's, times its weight
    logprob: torch.Tensor        # f32 [R], of the row's token; no gradient


@functools.lru_cache(maxsize=4096)
def _workspace(dtype: int, rows: int, vocab: int, top: int) -> int:
    n = ctypes.c_longlong()
    check(lib().rlu_loss_workspace(dtype, rows, vocab, top, ctypes.byref(n)), "rlu_loss_workspace")
    return n.value


def _check_logits(name: str, logits: torch.Tensor) -> None:
    if logits.ndim != 2 or logits.dtype not in _DTYPE_CODE or not logits.is_cuda:
        raise ValueError(f"{name} takes bf16, f16 or f32 logits [R, V] on the GPU")
    vocab = logits.shape[1]
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"{name}: a vocabulary of {vocab} is outside 1..{MAX_VOCAB}")
    if vocab > 1 and logits.stride()[1] != 1:
        raise ValueError(f"{name}: a row's logits must lie next to each other")


def _check_beside(name: str, what: str, t, shape, dtypes, dev) -> None:
    if t.shape != shape or t.dtype not in dtypes or not t.is_contiguous() or t.device != dev:
        raise ValueError(f"{name}: {what} must be contiguous {' or '.join(str(d)[6:] for d in dtypes)} "
                         f"{list(shape)} beside the logits")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} has no gradient of {what}: detach it")


_F32, _I32, _IDS = (torch.float32,), (torch.int32,), (torch.int64, torch.int32)


def _grad_like(logits: torch.Tensor) -> torch.Tensor:
    """A buffer for the gradient whose rows start at the same place within 16 bytes as the logits'."""
    rows, vocab = logits.shape
    size = logits.element_size()
    n = 16 // size
    ld = vocab + ((logits.stride()[0] - vocab) % n if rows > 1 else 0)
    off = logits.data_ptr() // size % n
    if ld == vocab and off == 0:
        return torch.empty(rows, vocab, dtype=logits.dtype, device=logits.device)
    return torch.empty(off + rows * ld, dtype=logits.dtype, device=logits.device).as_strided(
        (rows, vocab), (ld, 1), off)


def _check_out(name: str, out: torch.Tensor, logits: torch.Tensor) -> None:
    rows, vocab = logits.shape
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device or \
            (vocab > 1 and out.stride(1) != 1) or (rows > 1 and out.stride(0) < vocab):
        raise ValueError(f"{name}: out must be {logits.dtype} [{rows}, {vocab}] beside the logits, its rows apart")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name}: out asks for a gradient")
    a, b = logits.data_ptr(), out.data_ptr()
    if a == b and (rows < 2 or logits.stride(0) == out.stride(0)):
        return                                         # in place of the logits
    size = logits.element_size()
    end = lambda t: t.data_ptr() + ((rows - 1) * t.stride(0) + vocab) * size     # noqa: E731
    if rows and a < end(out) and b < end(logits):
        raise ValueError(f"{name}: out overlaps the logits (it may be the logits, or apart from them)")


def _call(logits, grad, top, fn, *args) -> None:
    """Runs fn(logits ..., *args, grad ..., ws, stream)."""
    rows, vocab = logits.shape
    code, dev = _DTYPE_CODE[logits.dtype], logits.device
    if rows == 0:
        return
    # taken and given back on the current stream, as the outputs are: calls on two streams, or two
    # captured graphs, have their own
    ws = torch.empty(_workspace(code, rows, vocab, top), dtype=torch.uint8, device=dev)
    with on_device(dev):
        rc = getattr(lib(), fn)(
            logits.data_ptr(), code, logits.stride()[0], rows, vocab, *args,
            0 if grad is None else grad.data_ptr(),
            0 if grad is None else grad.stride()[0] if rows > 1 else vocab, ws.data_ptr(), stream_ptr())
    check(rc, fn)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


def _policy(logits, tokens, old_logprobs, advantages, ref_logprobs, weight, clip, kl, temperature,
            grad, by=None) -> PolicyLoss | None:
    """by: factors of rows whose gradient is in grad already; the others are written again, and nothing else."""
    args = (tokens.data_ptr(), int(tokens.dtype == torch.int64), old_logprobs.data_ptr(), advantages.data_ptr(),
            _ptr(ref_logprobs), _ptr(weight), clip[0], clip[1], kl, temperature)
    if by is not None:
        return _call(logits, grad, 1, "rlu_policy_grad_by", *args, by.data_ptr(), by.stride(0))
    rows, dev = logits.shape[0], logits.device
    loss = torch.empty(rows, dtype=torch.float32, device=dev)
    logprob = torch.empty(rows, dtype=torch.float32, device=dev)
    _call(logits, grad, 1, "rlu_policy_loss", *args, loss.data_ptr(), logprob.data_ptr())
    return PolicyLoss(loss, logprob)


def _distill(logits, top_ids, top_logprobs, weight, rest, temperature, grad, by=None) -> torch.Tensor | None:
    """by: as for _policy."""
    top = top_ids.shape[1]
    args = (top_ids.data_ptr(), top_logprobs.data_ptr(), top, int(rest), _ptr(weight), temperature)
    if by is not None:
        return _call(logits, grad, top, "rlu_distill_top_grad_by", *args, by.data_ptr(), by.stride(0))
    loss = torch.empty(logits.shape[0], dtype=torch.float32, device=logits.device)
    _call(logits, grad, top, "rlu_distill_top", *args, loss.data_ptr())
    return loss


def _check_temperature(name: str, temperature) -> None:
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"{name}: a temperature of {temperature}")


def _check_policy(name, logits, tokens, old_logprobs, advantages, ref_logprobs, weight, clip, kl,
                  temperature, out=None) -> None:
    _check_logits(name, logits)
    rows, dev = (logits.shape[0],), logits.device
    _check_beside(name, "tokens", tokens, rows, _IDS, dev)
    _check_beside(name, "old_logprobs", old_logprobs, rows, _F32, dev)
    _check_beside(name, "advantages", advantages, rows, _F32, dev)
    if ref_logprobs is not None:
        _check_beside(name, "ref_logprobs", ref_logprobs, rows, _F32, dev)
    if weight is not None:
        _check_beside(name, "weight", weight, rows, _F32, dev)
    if len(clip) != 2 or not 0 <= clip[0] <= 1 or not 0 <= clip[1] < float("inf"):
        raise ValueError(f"{name}: clip={clip}, not (below, above) with 0 <= below <= 1 and above >= 0")
    if not 0 <= kl <= 1e30:
        raise ValueError(f"{name}: kl={kl} is not a factor >= 0")
    if kl and ref_logprobs is None:
        raise ValueError(f"{name}: kl={kl} needs ref_logprobs")
    _check_temperature(name, temperature)
    if has_tangent(logits, old_logprobs, advantages, ref_logprobs, weight, out):
        raise ValueError(f"{name} has no forward-mode derivative")


def _check_distill(name, logits, top_ids, top_logprobs, weight, temperature, out=None) -> None:
    _check_logits(name, logits)
    rows, dev = logits.shape[0], logits.device
    if top_ids.ndim != 2 or top_ids.shape[0] != rows or not 1 <= top_ids.shape[1] <= MAX_TOP:
        raise ValueError(f"{name}: top_ids must be [{rows}, 1..{MAX_TOP}]")
    _check_beside(name, "top_ids", top_ids, top_ids.shape, _I32, dev)
    _check_beside(name, "top_logprobs", top_logprobs, top_ids.shape, _F32, dev)
    if weight is not None:
        _check_beside(name, "weight", weight, (rows,), _F32, dev)
    _check_temperature(name, temperature)
    if has_tangent(logits, top_logprobs, weight, out):
        raise ValueError(f"{name} has no forward-mode derivative")


def _by_hand(name: str, logits: torch.Tensor) -> None:
    if logits.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} returns the gradient itself: detach the logits")


def policy_loss_grad(logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor,
                     advantages: torch.Tensor, ref_logprobs: torch.Tensor | None = None,
                     weight: torch.Tensor | None = None, *, clip: tuple[float, float] = (0.2, 0.2),
                     kl: float = 0.0, temperature: float = 1.0,
                     out: torch.Tensor | None = None) -> tuple[PolicyLoss, torch.Tensor]:
    """policy_loss and the gradient of the rows' sum, [R, V] of the logits' type: into out where given, which
    may be the logits themselves or lie apart from them as a whole (not columns of one buffer side by side)."""
    name = "policy_loss_grad"
    _check_policy(name, logits, tokens, old_logprobs, advantages, ref_logprobs, weight, clip, kl,
                  temperature, out)
    _by_hand(name, logits)
    if out is None:
        out = _grad_like(logits)
    else:
        _check_out(name, out, logits)
        written(out)
    return _policy(logits, tokens, old_logprobs, advantages, ref_logprobs, weight, clip, kl,
                   temperature, out), out


def distill_top_grad(logits: torch.Tensor, top_ids: torch.Tensor, top_logprobs: torch.Tensor,
                     weight: torch.Tensor | None = None, *, rest: bool = True,
                     temperature: float = 1.0,
                     out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """distill_top and the gradient of the rows' sum, [R, V] of the logits' type: into out where given, which
    may be the logits themselves or lie apart from them as a whole (not columns of one buffer side by side)."""
    name = "distill_top_grad"
    _check_distill(name, logits, top_ids, top_logprobs, weight, temperature, out)
    _by_hand(name, logits)
    if out is None:
        out = _grad_like(logits)
    else:
        _check_out(name, out, logits)
        written(out)
    return _distill(logits, top_ids, top_logprobs, weight, rest, temperature, out), out


# ---- for autograd -------------------------------------------------------------------------------
class _Rows(torch.autograd.Function):
    """The rows' losses. Their gradient is made in the forward pass, which has the logits in the cache, and
    handed out once. An incoming factor other than 1 belongs in front of the rounding to 16 bits (float16 has nothing
    below 6e-8 for a loss scale to lift again): such rows are then worked out again from the logits. Float32's are
    multiplied."""

    @staticmethod
    def forward(ctx, logits, op, beside, *how):
        grad = _grad_like(logits)
        out = op(logits, *beside, *how, grad)
        ctx.grad, ctx.op, ctx.how = grad, op, how
        if grad.element_size() == 2:
            ctx.save_for_backward(logits, *beside)
        if isinstance(out, PolicyLoss):
            ctx.mark_non_differentiable(out.logprob)
            return tuple(out)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, by, *_):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a captured graph takes a loss's gradient by hand, without autograd")
        grad, ctx.grad = ctx.grad, None
        if grad is None:
            raise RuntimeError("a loss's gradient is handed out once: compute the loss again for a "
                               "second backward pass")
        none = (None,) * (2 + len(ctx.how))
        if grad.element_size() == 2:
            ctx.op(*ctx.saved_tensors, *ctx.how, grad, by)           # (refuses logits written to since)
        elif grad.numel():
            rows, vocab = grad.shape
            with on_device(grad.device):
                rc = lib().rlu_scale_rows(
                    grad.data_ptr(), _DTYPE_CODE[grad.dtype], grad.stride(0) if rows > 1 else vocab,
                    rows, vocab, by.data_ptr(), by.stride(0), stream_ptr())
            check(rc, "rlu_scale_rows")
        return (grad, *none)


def _differentiable(name: str, logits: torch.Tensor) -> bool:
    if not (logits.requires_grad and torch.is_grad_enabled()):
        return False
    if torch.cuda.is_current_stream_capturing():
        raise ValueError(f"{name}: a captured graph takes {name}_grad, without autograd")
    return True


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logprobs: torch.Tensor,
                advantages: torch.Tensor, ref_logprobs: torch.Tensor | None = None,
                weight: torch.Tensor | None = None, *, clip: tuple[float, float] = (0.2, 0.2),
                kl: float = 0.0, temperature: float = 1.0) -> PolicyLoss:
    """logits [R, V] bf16, f16 or f32 (rows may be apart), the sampled tokens [R] int64 or int32, the log
    probabilities they were sampled with, their advantages, and where kl is not 0 those of a reference policy, f32
    [R] -> each row's loss times its weight, and the token's log probability under softmax(logits / temperature):

      lp = ln p_token, rho = e^(lp - old)
      loss = -min(rho adv, clamp(rho, 1 - clip[0], 1 + clip[1]) adv) + kl (e^(ref - lp) - (ref - lp) - 1)

    A negative token (a padded row) or a weight of 0 gives 0 and no gradient; the logits of such a row may be
    anything. A token past the vocabulary, a NaN or +inf give NaN. A token at -inf has rho = 0, and with a KL term
    an infinite loss. A gradient that comes in as 1 (the factors of a mean in weight, the rows' sum) costs nothing; any other
    one more pass, in which 16-bit rows are worked out again with it, so that a loss scale meets the gradient before its
    rounding: autograd keeps 16-bit logits until then, and refuses a backward pass if they or the other inputs have been
    written to. Backward runs once a loss."""
    _check_policy("policy_loss", logits, tokens, old_logprobs, advantages, ref_logprobs, weight, clip,
                  kl, temperature)
    if not _differentiable("policy_loss", logits):
        return _policy(logits, tokens, old_logprobs, advantages, ref_logprobs, weight, clip, kl,
                       temperature, None)
    return PolicyLoss(*_Rows.apply(logits, _policy, (tokens, old_logprobs, advantages, ref_logprobs, weight), clip, kl,
                                   temperature))


def distill_top(logits: torch.Tensor, top_ids: torch.Tensor, top_logprobs: torch.Tensor,
                weight: torch.Tensor | None = None, *, rest: bool = True,
                temperature: float = 1.0) -> torch.Tensor:
    """A student's logits [R, V] bf16, f16 or f32 (rows may be apart), a teacher's top_ids [R, n] int32 and
    top_logprobs [R, n] f32, n <= 32, as token_logprobs gives them -> the divergence of p = softmax(logits /
    temperature) from the teacher, f32 [R], times the row's weight:

      rest        q_j = e^top_logprobs_j, and the tokens not listed are one outcome of probability 1 - sum q:
                  loss = sum q_j ln(q_j / p_j) + q_rest ln(q_rest / p_rest)
      not rest    q = softmax(top_logprobs / temperature) over the listed (logits will do): sum q_j ln(q_j / p_j)

    A negative id is none, with its value. One past the vocabulary, a NaN or +inf among the logits or the values that
    count, or (rest) a value whose exponential float32 does not hold, give a row of NaN. A weight of 0
    gives 0 and no gradient; the logits of such a row may be anything. An id listed twice has a term for each. Where
    probabilities sum to 1 or more there is no rest (and in the gradient an excess of up to 2^-16 is rounding). Where
    no token is left for the rest, as all are listed or those that are not are at -inf, its term is left out of the
    loss, and the listed tokens' gradient is that loss's, (sum q) p_j - q_j. Weight, backward: as policy_loss."""
    _check_distill("distill_top", logits, top_ids, top_logprobs, weight, temperature)
    if not _differentiable("distill_top", logits):
        return _distill(logits, top_ids, top_logprobs, weight, rest, temperature, None)
    return _Rows.apply(logits, _distill, (top_ids, top_logprobs, weight), rest, temperature)
