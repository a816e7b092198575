"""Layer norm of rows with its gradients.

Host side of `b200_layer_norm` and `b200_layer_norm_grad` (include/b200_training.h). Encoder forwards (`vit.py`, `sam.py`) run layer norms of
their own inside one native call; this is the operator by itself, for blocks that are trained.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .rotary import as_held, refuse_negation, refuse_tangent, written

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
MAX_DIM = 32768


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as `[rows, dim]` with unit last stride; a copy where its strides do not allow a view."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t.reshape(-1, t.shape[-1])


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _shares(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory that `a` and `b` span meets."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride(), strict=True))) * t.element_size()) for t in (a, b))
    return a0 < b1 and b0 < a1


def _args(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float) -> _lib.B200LayerNormArgs:
    a = _lib.B200LayerNormArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = a.weight_dtype = _DTYPES[x.dtype]
    a.rows, a.dim = x.shape
    a.eps = eps
    a.x, a.x_stride = x.data_ptr(), _row_stride(x)
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            setattr(a, name, t.data_ptr())
            a.weight_dtype = _DTYPES[t.dtype]
    return a


def _forward(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, eps: float, y: torch.Tensor, *, stats: bool) -> torch.Tensor | None:  # noqa: PLR0913
    a = _args(x, weight, bias, eps)
    a.y, a.y_stride = y.data_ptr(), _row_stride(y)
    kept = torch.empty((x.shape[0], 2), dtype=torch.float32, device=x.device) if stats else None
    if kept is not None:
        a.stats = kept.data_ptr()
    with torch.cuda.device(x.device):
        code = _lib.library().b200_layer_norm(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(x.device.index))  # noqa: SLF001
    _lib.raise_for_code(code, "layer_norm")
    _lib.use_fast()
    return kept


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):  # noqa: ANN001, ANN205
        rows = _rows(x)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = _forward(rows, weight, bias, eps, y.view(rows.shape), stats=True)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.eps = eps
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):  # noqa: ANN001, ANN205
        x, weight, bias, stats = ctx.saved_tensors
        rows, g = _rows(x), _rows(as_held(g))
        want_x, want_w, want_b, _ = ctx.needs_input_grad
        a = _args(rows, weight, bias, ctx.eps)
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if want_x else None
        dw = torch.empty_like(weight) if want_w else None
        db = torch.empty_like(bias) if want_b else None
        a.stats, a.dy, a.dy_stride = stats.data_ptr(), g.data_ptr(), _row_stride(g)
        if dx is not None:
            a.dx, a.dx_stride = dx.data_ptr(), a.dim
        for name, t in (("dweight", dw), ("dbias", db)):
            if t is not None:
                setattr(a, name, t.data_ptr())
        lib = _lib.library()
        with torch.cuda.device(x.device):
            if dw is not None or db is not None:
                size = ctypes.c_int64(0)
                _lib.raise_for_code(lib.b200_layer_norm_workspace(ctypes.byref(a), ctypes.byref(size)), "layer_norm workspace")
                ws = torch.empty(size.value, dtype=torch.uint8, device=x.device)
                a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
            code = lib.b200_layer_norm_grad(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(x.device.index))  # noqa: SLF001
        _lib.raise_for_code(code, "layer_norm gradient")
        return dx, dw, db, None


def layer_norm(
    x: torch.Tensor,
    weight: torch.Tensor | None = None,
    bias: torch.Tensor | None = None,
    *,
    eps: float = 1e-5,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """`(x - mean) * rsqrt(var + eps) * weight + bias` over the last dimension of `x`; differentiable in x, weight and bias.

    Computed in fp32 and rounded once; the variance is of the differences from the mean, and the gradients of weight and bias are summed over
    all rows in a fixed order. Differentiable once and backwards.

    Args:
        x: CUDA `[..., dim]`, fp16 / bf16 / fp32, dim up to 32768. Rows on 16 bytes that are a multiple of 16 bytes are fastest; a tensor whose
            rows do not lie equally far apart, or whose last stride is not one, is copied.
        weight: `[dim]` of x's type or float32, or None (ones).
        bias: `[dim]`, of the type of `weight`, or None (zeros).
        eps: Added to the variance.
        out: Gets the result, contiguous; may be `x` itself (without gradients), and shares no memory with the operands otherwise. Autograd
            sees that it was written to.

    Raises:
        ValueError: Operands outside the contract (checked before the launch), or no row at all where a gradient is wanted.
        KernelUnavailableError: The CUDA library is not built or does not load.
    """
    if out is None and _lib.fast is not None:
        done = _lib.fast.layer_norm(x, weight, bias, eps)
        if done is not None:
            return done
    what = "layer_norm"
    x, weight, bias = (as_held(t) for t in (x, weight, bias))
    if x.dtype not in _DTYPES or not x.is_cuda or x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_DIM:
        msg = f"{what}: x must be a float16 / bfloat16 / float32 CUDA tensor [..., 1 .. {MAX_DIM}], got {tuple(x.shape)} {x.dtype} on {x.device}"
        raise ValueError(msg)
    refuse_tangent(what, "x", x)
    affine = [t for t in (weight, bias) if t is not None]
    for t in affine:
        if t.shape != x.shape[-1:] or t.dtype not in (x.dtype, torch.float32) or t.dtype != affine[0].dtype or t.device != x.device or not t.is_contiguous():
            msg = f"{what}: weight and bias must be contiguous [{x.shape[-1]}] of {x.dtype} or float32 (both alike) on {x.device}, got {tuple(t.shape)} {t.dtype} on {t.device}"
            raise ValueError(msg)
        refuse_tangent(what, "weight or bias", t)
    if not eps >= 0 or eps == float("inf"):
        msg = f"{what}: eps {eps} must be finite and not negative"
        raise ValueError(msg)
    grad = torch.is_grad_enabled() and any(t.requires_grad for t in (x, *affine))
    if out is not None and (out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous() or grad or out.requires_grad):
        msg = f"{what}: out must be contiguous {tuple(x.shape)} {x.dtype} on {x.device} and nothing may require a gradient"
        raise ValueError(msg)
    if out is not None:
        refuse_negation(what, "out", out)
    if out is not None and ((_shares(out, x) and not (out.data_ptr() == x.data_ptr() and x.is_contiguous())) or any(_shares(out, t) for t in affine)):
        msg = f"{what}: out shares memory with x, without being x, or with weight or bias"
        raise ValueError(msg)
    if x.numel() >= 2**31 * x.shape[-1]:
        msg = f"{what}: {x.numel() // x.shape[-1]} rows are too many"
        raise ValueError(msg)
    if x.numel() == 0 and not grad:
        return x.clone() if out is None else out
    if x.numel() == 0:
        msg = f"{what}: x {tuple(x.shape)} without a row has no gradient"
        raise ValueError(msg)
    if grad:
        return _LayerNorm.apply(x, weight, bias, float(eps))
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    rows = _rows(x)
    _forward(rows, weight, bias, float(eps), y.view(rows.shape), stats=False)
    if out is not None:
        written(out)
    return y
