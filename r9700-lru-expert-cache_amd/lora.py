"""Low-rank adapters of many requests beside a shared, frozen projection, on librlu.so: for each row the
adapter that its request asks for, out = y + s (x A^T) B^T, and the backward pass that trains them.

No counterpart in the reference. The projection itself is whatever gave y: ops.gemm_fp8_dense, the heads, or
any product of the caller's; rows, adapters and outputs are bf16 or f16. The backward pass is the adapters' alone: what the
frozen projection adds to dx, dy times its weight, is the caller's. ops.gemm_fp8_dense has no gradient and no product with
the transposed weight, so in this package training reaches the adapters of a model's last product, the head.

  plan_rows      a batch's rows by adapter: once, for all the projections that the batch passes
  add_lora       for serving (in place or into another tensor), and for autograd in eager code
  add_lora_grad  the backward pass by hand, also in a captured graph
"""
from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from ._lib import check, has_tangent, lib, on_device, stream_ptr, written

_DTYPE_CODE = {torch.bfloat16: 0, torch.float16: 2}
MAX_RANK = 128
MAX_ADAPTERS = 1024
MAX_FEATURES = 1 << 24


@dataclass(frozen=True)
class LoraStack:
    """n adapters of one projection: hold this on the layer. Adapters of a lower rank are padded with zeros."""
    a: torch.Tensor        # [n, rank, K] bf16 or f16
    b: torch.Tensor        # [n, N, rank], the same type
    scale: torch.Tensor    # f32 [n], usually alpha / rank

    def __post_init__(self):
        a, b, s = self.a, self.b, self.scale
        if a.ndim != 3 or b.ndim != 3 or a.dtype not in _DTYPE_CODE or b.dtype != a.dtype or \
                s.dtype != torch.float32 or b.shape[0] != a.shape[0] or b.shape[2] != a.shape[1] or \
                s.shape != a.shape[:1] or not (a.is_contiguous() and b.is_contiguous() and
                                               s.is_contiguous()):
            raise ValueError("LoraStack: contiguous bf16 or f16 a [n, rank, K] and b [n, N, rank] with "
                             f"float32 scale [n], not {tuple(a.shape)}, {tuple(b.shape)}, {tuple(s.shape)}")
        if not a.is_cuda or b.device != a.device or s.device != a.device:
            raise ValueError("LoraStack: all on one GPU")
        if not (1 <= self.n <= MAX_ADAPTERS and 1 <= self.rank <= MAX_RANK and
                1 <= a.shape[2] <= MAX_FEATURES and 1 <= b.shape[1] <= MAX_FEATURES):
            raise ValueError(f"LoraStack: {tuple(a.shape)}, {tuple(b.shape)}: 1..{MAX_ADAPTERS} adapters of rank "
                             f"1..{MAX_RANK} over 1..{MAX_FEATURES} features")
        if s.requires_grad:
            raise ValueError("LoraStack: the scale has no gradient")

    @property
    def n(self) -> int:
        return self.a.shape[0]

    @property
    def rank(self) -> int:
        return self.a.shape[1]


@dataclass(frozen=True)
class LoraRows:
    """A batch's rows by adapter, as the kernels read them (plan_rows makes it)."""
    order: torch.Tensor    # int32 [rows]: the rows of adapter 0, of adapter 1, ...; without one; ids past the last
    tiles: torch.Tensor    # int32 [cap, 4]
    first: torch.Tensor    # int32 [n + 5]
    rows: int
    n: int                 # adapters that the ids count
    size: int              # rows of a tile


def plan_rows(ids: torch.Tensor, n: int) -> LoraRows:
    """ids [rows] int32 or int64, the adapter of each of a batch's rows in a stack of n: below 0 none; a row whose id
    is n or more becomes NaN. Reads ids on the GPU, without a synchronisation."""
    if ids.ndim != 1 or ids.dtype not in (torch.int32, torch.int64) or not ids.is_cuda or \
            not ids.is_contiguous():
        raise ValueError("plan_rows takes contiguous int32 or int64 ids [rows] on the GPU")
    if not 1 <= n <= MAX_ADAPTERS:
        raise ValueError(f"plan_rows: {n} adapters, not 1..{MAX_ADAPTERS}")
    rows, dev = ids.shape[0], ids.device
    if rows > 1 << 24:
        raise ValueError(f"plan_rows: {rows} rows, at most {1 << 24}")
    # few rows: tiles of 16 (many adapters have fewer); many: an adapter's factors are read once for 64. [2560 -> 10240], R =
    # 16, 8 adapters, tiles of 16 / 64, us forward and backward: 256 rows 9.8 + 19.7 / 11.0 + 16.1, 1023 18.2 + 37.1 / 17.1
    # + 33.9, 2048 30.9 + 50.4 / 25.8 + 44.5; 1023 rows of 64 adapters, [2560 -> 2560] 11.5 + 27.2 / 12.6 + 27.3. The rule goes by
    # the rows alone: below 1024 the forward pass of few rows and batches of many adapters gain, the backward pass of few
    # adapters loses, 8% of a step with 8.
    size = 16 if rows < 1024 else 64
    cap = rows // size + min(rows, n + 2)
    order = torch.empty(rows, dtype=torch.int32, device=dev)
    tiles = torch.empty(cap, 4, dtype=torch.int32, device=dev)
    first = torch.empty(n + 5, dtype=torch.int32, device=dev)
    with on_device(dev):
        rc = lib().rlu_lora_plan(ids.data_ptr(), int(ids.dtype == torch.int64), rows, n, size, cap,
                                 order.data_ptr(), tiles.data_ptr(), first.data_ptr(), stream_ptr())
    check(rc, "rlu_lora_plan")
    return LoraRows(order, tiles, first, rows, n, size)


def _check_rows(name: str, what: str, t: torch.Tensor, rows: int, cols: int, w: LoraStack) -> None:
    if t.shape != (rows, cols) or t.dtype != w.a.dtype or t.device != w.a.device or \
            (t.stride()[1] != 1 and cols > 1):
        raise ValueError(f"{name}: {what} must be {w.a.dtype} [{rows}, {cols}] beside the adapters, a row's elements "
                         "next to each other")


def _check_batch(name: str, w: LoraStack, rows: LoraRows) -> None:
    if rows.n != w.a.shape[0] or rows.order.device != w.a.device:
        raise ValueError(f"{name}: rows planned for {rows.n} adapters on {rows.order.device}, a stack of {w.n} "
                         f"on {w.a.device}")


def _check_hidden(name: str, hidden: torch.Tensor, rows: int, w: LoraStack) -> None:
    if hidden.shape != (rows, w.rank) or hidden.dtype != torch.float32 or \
            not hidden.is_contiguous() or hidden.device != w.a.device or hidden.requires_grad:
        raise ValueError(f"{name}: hidden must be contiguous float32 [{rows}, {w.rank}] beside the adapters")


def _overlap(s: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether the bytes that their rows reach over meet: the one that begins first ends behind the other's beginning."""
    a, b = s.data_ptr(), t.data_ptr()
    if a > b:
        a, b, s, t = b, a, t, s
    rows, cols = s.shape
    return rows > 0 and t.shape[0] > 0 and a + ((rows - 1) * s.stride(0) + cols) * s.element_size() > b


def _ld(t: torch.Tensor) -> int:
    rows, cols = t.shape
    return t.stride()[0] if rows > 1 else cols


def _forward(y, x, w, rows, hidden, out) -> None:
    if rows.rows == 0:
        return
    a, b = w.a, w.b
    n, rank, K = a.shape
    with on_device(x.device):
        rc = lib().rlu_lora_add(
            x.data_ptr(), _ld(x), a.data_ptr(), b.data_ptr(), w.scale.data_ptr(),
            _DTYPE_CODE[x.dtype], rows.order.data_ptr(), rows.tiles.data_ptr(), rows.first.data_ptr(),
            rows.rows, n, rows.size, rows.tiles.shape[0], K, y.shape[1], rank,
            hidden.data_ptr(), y.data_ptr(), _ld(y), out.data_ptr(), _ld(out), stream_ptr())
    check(rc, "rlu_lora_add")


def add_lora(y: torch.Tensor, x: torch.Tensor, w: LoraStack, rows: LoraRows,
             out: torch.Tensor | None = None, hidden: torch.Tensor | None = None) -> torch.Tensor:
    """y [rows, N] + scale (x [rows, K] a^T) b^T with each row's adapter, all of the stack's type; sums and
    x a^T in float32 (of which float16's second product takes 22 bits), rounded once. Rows may be apart (x, y and out of any
    stride). A row without an adapter is y's.
    out: where the result goes, y itself among others; a new tensor without it. What out's rows reach over from the first to
    the last must not meet x's, nor y's unless it is y: not columns of one buffer side by side.
    hidden: float32 [rows, rank] that receives scale x a^T, for add_lora_grad."""
    a, b, M = w.a, w.b, rows.rows
    _check_batch("add_lora", w, rows)
    _check_rows("add_lora", "x", x, M, a.shape[2], w)
    _check_rows("add_lora", "y", y, M, b.shape[1], w)
    if hidden is not None:
        _check_hidden("add_lora", hidden, M, w)
    if has_tangent(y, x, a, b, w.scale, out, hidden):
        raise ValueError("add_lora has no forward-mode derivative")
    grad = (x.requires_grad or y.requires_grad or a.requires_grad or b.requires_grad) and \
        torch.is_grad_enabled()
    if grad and (out is not None or hidden is not None):
        raise ValueError("add_lora: autograd keeps its own hidden and makes its own out; detach the operands for a "
                         "gradient by hand")
    if out is not None:
        _check_rows("add_lora", "out", out, M, b.shape[1], w)
        if M > 1 and out.stride()[0] < out.shape[1]:
            raise ValueError("add_lora: out's rows overlap")
        if out.requires_grad and torch.is_grad_enabled():
            raise ValueError("add_lora: out asks for a gradient")
        same = out.data_ptr() == y.data_ptr() and _ld(out) == _ld(y)
        if (not same and _overlap(out, y)) or _overlap(out, x):
            raise ValueError("add_lora: out overlaps y or x (it may be y, or apart from both)")
    if hidden is not None and M:
        at = hidden.data_ptr()
        for t in (x, y, out):                          # (_overlap, without asking for what is known: a small step's time)
            if t is not None and t.data_ptr() < at + 4 * M * w.rank and \
                    at < t.data_ptr() + 2 * ((M - 1) * t.stride()[0] + t.shape[1]):
                raise ValueError("add_lora: hidden overlaps x, y or out")
    if grad:
        if torch.cuda.is_current_stream_capturing():
            raise ValueError("add_lora: a captured graph takes add_lora_grad, without autograd")
        return _AddLora.apply(y, x, a, b, w, rows)
    if hidden is None:
        hidden = torch.empty(M * a.shape[1], dtype=torch.float32, device=x.device)
    else:
        written(hidden)
    if out is None:
        out = torch.empty(M, b.shape[1], dtype=y.dtype, device=y.device)
    else:
        written(out)
    _forward(y, x, w, rows, hidden, out)
    return out


@functools.lru_cache(maxsize=4096)
def _grad_workspace(dtype: int, rows: int, n: int, size: int, cap: int, K: int, N: int,
                    rank: int) -> int:
    b = ctypes.c_longlong()
    check(lib().rlu_lora_grad_workspace(dtype, rows, n, size, cap, K, N, rank, ctypes.byref(b)),
          "rlu_lora_grad_workspace")
    return b.value


def _backward(dy, x, w, rows, hidden, need):
    a, b, M, dev = w.a, w.b, rows.rows, x.device
    n, rank, K = a.shape
    N = b.shape[1]
    make = torch.empty if M else torch.zeros
    dx = torch.empty(M, K, dtype=x.dtype, device=dev) if need[0] else None
    da = make(n, rank, K, dtype=x.dtype, device=dev) if need[1] else None
    db = make(n, N, rank, dtype=x.dtype, device=dev) if need[2] else None
    if M and (need[0] or need[1] or need[2]):
        code, cap = _DTYPE_CODE[x.dtype], rows.tiles.shape[0]
        # taken and given back on the current stream: calls on two streams, or two captured graphs, have their own
        ws = torch.empty(_grad_workspace(code, M, n, rows.size, cap, K, N, rank), dtype=torch.uint8,
                         device=dev)
        with on_device(dev):
            rc = lib().rlu_lora_grad(
                dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), a.data_ptr(), b.data_ptr(),
                w.scale.data_ptr(), code, rows.order.data_ptr(), rows.tiles.data_ptr(),
                rows.first.data_ptr(), M, n, rows.size, cap, K, N, rank, hidden.data_ptr(),
                0 if dx is None else dx.data_ptr(), K, 0 if da is None else da.data_ptr(),
                0 if db is None else db.data_ptr(), ws.data_ptr(), stream_ptr())
        check(rc, "rlu_lora_grad")
    return dx, da, db


def add_lora_grad(dy: torch.Tensor, x: torch.Tensor, w: LoraStack, rows: LoraRows,
                  hidden: torch.Tensor, need: tuple[bool, bool, bool] = (True, True, True)):
    """From the gradient dy [rows, N] of add_lora's output, its x, rows and the hidden that it filled: the gradients
    (dx [rows, K], da [n, rank, K], db [n, N, rank]) of the stack's type, None where need says no (the pass
    over dy that db comes out of is dx's and da's too). That of y is dy itself. Sums in float32, in an order that the sizes
    and the rows' ids decide."""
    _check_batch("add_lora_grad", w, rows)
    _check_rows("add_lora_grad", "x", x, rows.rows, w.a.shape[2], w)
    _check_rows("add_lora_grad", "dy", dy, rows.rows, w.b.shape[1], w)
    _check_hidden("add_lora_grad", hidden, rows.rows, w)
    if len(need) != 3:
        raise ValueError("add_lora_grad: need says whether dx, da and db are wanted")
    if (dy.requires_grad or x.requires_grad or w.a.requires_grad or w.b.requires_grad) and \
            torch.is_grad_enabled():
        raise ValueError("add_lora_grad returns the gradients itself: detach its operands")
    if has_tangent(dy, x, w.a, w.b, w.scale, hidden):
        raise ValueError("add_lora_grad has no forward-mode derivative")
    return _backward(dy, x, w, rows, hidden, need)


class _AddLora(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, x, a, b, w, rows):
        hidden = torch.empty(rows.rows, a.shape[1], dtype=torch.float32, device=x.device)
        out = torch.empty(rows.rows, y.shape[1], dtype=y.dtype, device=y.device)
        _forward(y, x, w, rows, hidden, out)
        ctx.save_for_backward(x, a, b, hidden, w.scale)
        ctx.w, ctx.rows = w, rows
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("add_lora: a captured graph takes add_lora_grad, without autograd")
        x, _, _, hidden, _ = ctx.saved_tensors         # (refuses a, b or the scale written to since)
        if dy.stride(1) != 1 and dy.shape[1] > 1:
            dy = dy.contiguous()
        need = ctx.needs_input_grad
        return (dy if need[0] else None, *_backward(dy, x, ctx.w, ctx.rows, hidden, need[1:4]), None, None)
