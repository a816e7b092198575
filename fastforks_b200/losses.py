"""Losses of an output layer from hidden states and the layer's weight, without the logits: softmax cross entropy, and distillation from a
teacher's largest logits.

Host side of `b200_head_loss` and `b200_head_grad` (include/b200_training.h). The logits are computed tile by tile where their statistics are
taken, and once more, in pieces of the vocabulary, where their gradients are; nothing of the size of rows times vocabulary is kept from the loss to
its gradients, and of a vocabulary of more than 2048 tokens there is never all of it at a time where rows are many.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .rotary import as_held, refuse_tangent

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
MAX_TOP = 256


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as `[rows, dim]`, rows on 16 bytes; a copy where it does not lie so."""
    t = t.reshape(-1, t.shape[-1])
    if t.stride(1) != 1 or t.stride(0) % 8 or t.stride(0) < t.shape[1] or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _vector(t: torch.Tensor | None) -> torch.Tensor | None:
    """A bias on 16 bytes."""
    return t if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0) else t.clone(memory_format=torch.contiguous_format)


def _check(what: str, x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None, reduction: str) -> None:
    if x.dtype not in (torch.float16, torch.bfloat16) or not x.is_cuda or x.dim() < 1:
        msg = f"{what}: x must be a float16 / bfloat16 CUDA tensor [..., dim], got {tuple(x.shape)} {x.dtype} on {x.device}"
        raise ValueError(msg)
    if w.dtype != x.dtype or w.device != x.device or w.dim() != 2 or w.shape[1] != x.shape[-1] or w.shape[0] < 1:  # noqa: PLR2004
        msg = f"{what}: weight must be {x.dtype} [vocabulary, {x.shape[-1]}] on {x.device}, got {tuple(w.shape)} {w.dtype} on {w.device}"
        raise ValueError(msg)
    if x.shape[-1] % 8 or x.shape[-1] < 8:  # noqa: PLR2004
        msg = f"{what}: dim {x.shape[-1]} must be a multiple of 8"
        raise ValueError(msg)
    if reduction not in _REDUCTIONS:
        msg = f"{what}: reduction {reduction!r} must be one of {tuple(_REDUCTIONS)}"
        raise ValueError(msg)
    if bias is not None and (bias.dtype != x.dtype or bias.device != x.device or bias.shape != w.shape[:1]):
        msg = f"{what}: bias must be {x.dtype} [{w.shape[0]}] on {x.device}, got {tuple(bias.shape)} {bias.dtype} on {bias.device}"
        raise ValueError(msg)
    refuse_tangent(what, "x", x)
    refuse_tangent(what, "weight", w)
    if bias is not None:
        refuse_tangent(what, "bias", bias)


def _args(x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None, top: int, tau: float, reduction: int, *, whole: bool = False) -> _lib.B200HeadArgs:  # noqa: PLR0913
    a = _lib.B200HeadArgs()
    a.struct_size = ctypes.sizeof(a)
    a.whole = whole
    a.dtype, a.rows, a.dim, a.vocab, a.top, a.tau, a.reduction = _DTYPES[x.dtype], x.shape[0], x.shape[1], w.shape[0], top, tau, reduction
    a.x, a.ldx, a.w, a.ldw = x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0)
    if x.shape[0] == 1:
        a.ldx = x.shape[1]
    if w.shape[0] == 1:
        a.ldw = w.shape[1]
    if bias is not None:
        a.bias = bias.data_ptr()
    return a


def _sizes(what: str, a: _lib.B200HeadArgs) -> tuple[int, int, int]:
    state, loss, grad = (ctypes.c_int64(0) for _ in range(3))
    _lib.raise_for_code(_lib.library().b200_head_sizes(ctypes.byref(a), ctypes.byref(state), ctypes.byref(loss), ctypes.byref(grad)), what)
    return state.value, loss.value, grad.value


def _buffer(size: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(size, dtype=torch.uint8, device=like.device)


def _loss(what: str, x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None, targets: torch.Tensor, teacher: torch.Tensor | None, ignore: int, tau: float, reduction: int) -> tuple[torch.Tensor, torch.Tensor]:  # noqa: PLR0913
    """The loss (per row, or one number) and what its gradients need."""
    a = _args(x, w, bias, 0 if teacher is None else targets.shape[1], tau, reduction)
    a.targets, a.target_bytes, a.ignore = targets.data_ptr(), targets.element_size(), ignore
    if teacher is not None:
        a.targets_stride, a.teacher, a.teacher_stride, a.teacher_dtype = targets.stride(0), teacher.data_ptr(), teacher.stride(0), _DTYPES[teacher.dtype]
    loss = torch.empty(x.shape[0] if reduction == 0 else (), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        state_bytes, loss_bytes, _ = _sizes(what, a)
        state, ws = _buffer(state_bytes, x), _buffer(loss_bytes, x)
        a.loss, a.state, a.state_bytes, a.workspace, a.workspace_bytes = loss.data_ptr(), state.data_ptr(), state_bytes, ws.data_ptr(), loss_bytes
        code = _lib.library().b200_head_loss(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(x.device.index))  # noqa: SLF001
    _lib.raise_for_code(code, what)
    _lib.use_fast()
    return loss, state


class _HeadLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, what, x, w, bias, targets, teacher, ignore, tau, reduction, whole):  # noqa: ANN001, ANN205, PLR0913
        loss, state = _loss(what, _rows(x), _rows(w), _vector(bias), targets, teacher, ignore, tau, reduction)
        ctx.save_for_backward(x, w, bias, state)
        ctx.what, ctx.top, ctx.tau, ctx.reduction, ctx.whole = what, 0 if teacher is None else targets.shape[1], tau, reduction, whole
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):  # noqa: ANN001, ANN205
        x, w, bias, state = ctx.saved_tensors
        g = as_held(g)
        rows, weight, vector = _rows(x), _rows(w), _vector(bias)
        a = _args(rows, weight, vector, ctx.top, ctx.tau, ctx.reduction, whole=ctx.whole)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if ctx.needs_input_grad[1] else None
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device) if ctx.needs_input_grad[2] else None
        db = torch.empty(bias.shape, dtype=bias.dtype, device=bias.device) if ctx.needs_input_grad[3] else None
        a.grad, a.grad_stride = g.data_ptr(), g.stride(0) if g.dim() else 0
        a.dx, a.dw, a.dbias = (None if t is None else t.data_ptr() for t in (dx, dw, db))
        with torch.cuda.device(x.device):
            _, _, size = _sizes(f"{ctx.what} gradient", a)
            ws = _buffer(size, x)
            a.state, a.state_bytes, a.workspace, a.workspace_bytes = state.data_ptr(), state.numel(), ws.data_ptr(), size
            code = _lib.library().b200_head_grad(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(x.device.index))  # noqa: SLF001
        _lib.raise_for_code(code, f"{ctx.what} gradient")
        return None, dx, dw, db, None, None, None, None, None, None


def _run(what: str, x: torch.Tensor, w: torch.Tensor, bias: torch.Tensor | None, targets: torch.Tensor, teacher: torch.Tensor | None, ignore: int, tau: float, reduction: str, whole: bool) -> torch.Tensor:  # noqa: FBT001, PLR0913
    shape = x.shape[:-1] if reduction == "none" else ()
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w, bias))
    x, w, bias = (as_held(t) for t in (x, w, bias))
    if x.numel() == 0:
        if grad:
            msg = f"{what}: x {tuple(x.shape)} without a row has no gradient"
            raise ValueError(msg)
        return torch.zeros(shape, dtype=torch.float32, device=x.device)
    if grad:
        loss = _HeadLoss.apply(what, x, w, bias, targets, teacher, ignore, tau, _REDUCTIONS[reduction], bool(whole))
    else:
        loss, _ = _loss(what, _rows(x), _rows(w), _vector(bias), targets, teacher, ignore, tau, _REDUCTIONS[reduction])
    return loss.view(shape)


def linear_cross_entropy(  # noqa: PLR0913
    x: torch.Tensor,
    weight: torch.Tensor,
    targets: torch.Tensor,
    *,
    bias: torch.Tensor | None = None,
    ignore_index: int = -100,
    reduction: str = "mean",
    whole_gradients: bool = False,
) -> torch.Tensor:
    """Softmax cross entropy of the logits `x @ weight^T + bias`, which are never in memory; differentiable (once, backwards) in x, weight and bias.

    `logsumexp(logits) - logits[target]` of each row, products and sums in fp32, the loss in fp32. The gradients of the logits are rounded to
    x's type once, on their way into the two products that give those of x and weight (but see `whole_gradients`). Rows that do not count are left out of all work.

    Args:
        x: Hidden states, CUDA `[..., dim]`, fp16 or bf16, dim a multiple of 8. Rows that do not lie on 16 bytes are copied.
        weight: `[vocabulary, dim]` of x's type.
        targets: int64 or int32 `[...]`, the shape of x without its last dimension. One outside the vocabulary (and not `ignore_index`)
            makes NaN of its row, and `device_status()` reports it.
        bias: `[vocabulary]` of x's type, or None. Its gradient is summed over the rows 64 columns at a time: over few tokens that is most of the time.
        ignore_index: Target of rows that do not count: their loss is 0, they have no gradient, and what x holds there is not looked at.
        reduction: `"mean"` or `"sum"` over the rows that count (0 where none does), or `"none"`: the loss of each row.
        whole_gradients: Multiply what the rounding of the logits' gradients takes, too: the error of the results is then that of their own rounding (else 1.1 to
            1.5 times as much), at half as many operations more and up to twice the scratch. Up to 128 rows or 2^31 products that is so in any case.

    Raises:
        ValueError: Operands outside the contract (checked before the launch), or no row at all where a gradient is wanted.
        KernelUnavailableError: The CUDA library is not built or does not load.
    """
    if _lib.fast is not None:
        done = _lib.fast.head_loss(x, weight, bias, targets, None, ignore_index, 1.0, _REDUCTIONS.get(reduction), whole_gradients)
        if done is not None:
            return done
    what = "linear_cross_entropy"
    _check(what, x, weight, bias, reduction)
    if targets.dtype not in (torch.int64, torch.int32) or targets.shape != x.shape[:-1] or targets.device != x.device:
        msg = f"{what}: targets must be int64 or int32 {tuple(x.shape[:-1])} on {x.device}, got {tuple(targets.shape)} {targets.dtype} on {targets.device}"
        raise ValueError(msg)
    if not -(2**63) <= ignore_index < 2**63:
        msg = f"{what}: ignore_index {ignore_index} is no 64-bit number"
        raise ValueError(msg)
    return _run(what, x, weight, bias, targets.contiguous(), None, ignore_index, 1.0, reduction, whole_gradients)


def linear_distillation(  # noqa: PLR0913
    x: torch.Tensor,
    weight: torch.Tensor,
    teacher_ids: torch.Tensor,
    teacher_logits: torch.Tensor,
    *,
    bias: torch.Tensor | None = None,
    temperature: float = 1.0,
    reduction: str = "mean",
    whole_gradients: bool = False,
) -> torch.Tensor:
    """Divergence of the distribution of the logits `x @ weight^T + bias` from a teacher's largest logits; differentiable (once, backwards) in x,
    weight and bias.

    With p the softmax of the teacher's logits of a row over `temperature`, and q that of all of the row's own logits over `temperature`:
    `temperature ** 2 * sum(p * (log p - log q))` over the teacher's entries, in fp32. Otherwise as `linear_cross_entropy`.

    Args:
        x: Hidden states, CUDA `[..., dim]`, fp16 or bf16, dim a multiple of 8. Rows that do not lie on 16 bytes are copied.
        weight: `[vocabulary, dim]` of x's type.
        teacher_ids: int64 or int32 `[..., entries]`, 1 to 256 entries a row in any order: which tokens the teacher's logits are of. Negative: no
            entry; a row without one does not count. A token that comes twice counts twice. One past the vocabulary makes NaN of its row, and
            `device_status()` reports it.
        teacher_logits: fp16 / bf16 / fp32 of the same shape (log probabilities are logits too). An entry of -inf has no weight; a row whose entries
            all are is NaN.
        bias: `[vocabulary]` of x's type, or None.
        temperature: Positive.
        reduction: `"mean"` or `"sum"` over the rows that count (0 where none does), or `"none"`: the loss of each row, 0 where it does not count.
        whole_gradients: As for `linear_cross_entropy`.

    Raises:
        ValueError: Operands outside the contract (checked before the launch), or no row at all where a gradient is wanted.
        KernelUnavailableError: The CUDA library is not built or does not load.
    """
    if _lib.fast is not None and teacher_logits is not None:
        done = _lib.fast.head_loss(x, weight, bias, teacher_ids, teacher_logits, 0, temperature, _REDUCTIONS.get(reduction), whole_gradients)
        if done is not None:
            return done
    what = "linear_distillation"
    _check(what, x, weight, bias, reduction)
    if teacher_ids.dtype not in (torch.int64, torch.int32) or teacher_ids.dim() != x.dim() or teacher_ids.shape[:-1] != x.shape[:-1] or not 1 <= teacher_ids.shape[-1] <= MAX_TOP or teacher_ids.device != x.device:
        msg = f"{what}: teacher_ids must be int64 or int32 {tuple(x.shape[:-1])} and 1 .. {MAX_TOP} entries on {x.device}, got {tuple(teacher_ids.shape)} {teacher_ids.dtype} on {teacher_ids.device}"
        raise ValueError(msg)
    if teacher_logits.dtype not in _DTYPES or teacher_logits.shape != teacher_ids.shape or teacher_logits.device != x.device:
        msg = f"{what}: teacher_logits must be float {tuple(teacher_ids.shape)} on {x.device}, got {tuple(teacher_logits.shape)} {teacher_logits.dtype} on {teacher_logits.device}"
        raise ValueError(msg)
    if teacher_logits.requires_grad and torch.is_grad_enabled():
        msg = f"{what}: teacher_logits requires a gradient, and is a constant here (detach it)"
        raise ValueError(msg)
    refuse_tangent(what, "teacher_logits", teacher_logits)
    if not 0 < temperature < math.inf:
        msg = f"{what}: temperature {temperature} must be positive and finite"
        raise ValueError(msg)
    k = teacher_ids.shape[-1]
    ids, logits = (t.reshape(-1, k) for t in (teacher_ids, as_held(teacher_logits)))
    ids, logits = (t if t.stride(1) == 1 or k == 1 else t.contiguous() for t in (ids, logits))
    return _run(what, x, weight, bias, ids, logits, 0, float(temperature), reduction, whole_gradients)
