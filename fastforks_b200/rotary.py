"""Rotary positions of heads, alone or behind the root-mean-square norm of each head, with their gradients.

Host side of `b200_rotary` (include/b200_decoder.h). `rotary_table` makes the cosines and sines of a context, stretched ones
too; `rotary` turns one tensor of heads, `qk_norm_rotary` norms and turns q and k in one launch. Both are differentiable, once and backwards
(table and positions are constants); tensors that carry a tangent of forward-mode differentiation are refused.
`rope_qk_` remains the in-place call of DINOv3's blocks.
"""

from __future__ import annotations

import ctypes
import math
import threading

import torch

from . import _lib

_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
MAX_HEAD_DIM = 512
_HEADER_BYTES = 256  # the zeroed words in front of the workspace

_WORKSPACES: dict[tuple[int, int], torch.Tensor] = {}
_WORKSPACES_LOCK = threading.Lock()


def rotary_table(  # noqa: PLR0913
    length: int,
    dim: int,
    *,
    base: float = 10000.0,
    scaling: str | None = None,
    factor: float = 1.0,
    original_length: int | None = None,
    beta_fast: float = 32.0,
    beta_slow: float = 1.0,
    device: torch.device | str | None = None,
) -> torch.Tensor:
    """fp32 `[length, 2, dim / 2]` = cos | sin of positions 0 .. length - 1, pair i turning by `position * base ** (-2 i / dim)`.

    Args:
        length: Rows of the table.
        dim: Dimensions of a head that are turned (even).
        base: Base of the frequencies.
        scaling: How a context is stretched `factor` times: None (not), `"linear"` (positions divided by the factor), `"ntk"` (the base
            grows so that the slowest pair is stretched by the factor and the fastest not at all) or `"yarn"` (pairs that turn more than
            `beta_fast` times within `original_length` as they are, those that turn less than `beta_slow` times divided by the factor,
            a ramp between; cosines and sines times `0.1 ln(factor) + 1`).
        factor: See `scaling`; at least 1.
        original_length: Context the model was trained on (`"yarn"`).
        beta_fast: See `scaling`.
        beta_slow: See `scaling`.
        device: Where the table goes.

    Raises:
        ValueError: Arguments outside the contract.
    """
    if length < 1 or dim < 2 or dim % 2 or not base > 0:  # noqa: PLR2004
        msg = f"rotary_table: length {length}, dim {dim} (even) and base {base} must be positive"
        raise ValueError(msg)
    if scaling not in (None, "linear", "ntk", "yarn") or not factor >= 1:
        msg = f"rotary_table: scaling {scaling!r} must be None, 'linear', 'ntk' or 'yarn', with a factor of at least 1 (got {factor})"
        raise ValueError(msg)
    if scaling == "ntk" and dim > 2:  # noqa: PLR2004
        base = base * factor ** (dim / (dim - 2))
    pair = torch.arange(dim // 2, dtype=torch.float64, device=device)
    inv = base ** (-2 * pair / dim)
    size = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if original_length is None or original_length < 1:
            msg = "rotary_table: scaling 'yarn' needs original_length"
            raise ValueError(msg)
        if not base > 1:
            msg = f"rotary_table: scaling 'yarn' needs a base above 1, got {base}"
            raise ValueError(msg)
        # The pair whose number of turns is beta lies at dim / 2 * ln(original_length / (2 pi beta)) / ln(base). The ramp ends on whole pairs; its end may
        # lie behind the last pair, at dim - 1 at most, as in the published method (Peng et al., YaRN, 2023).
        low, high = (dim / 2 * math.log(original_length / (2 * math.pi * beta)) / math.log(base) for beta in (beta_fast, beta_slow))
        low, high = max(math.floor(low), 0), min(math.ceil(high), dim - 1)
        kept = 1 - ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv = inv * kept + inv / factor * (1 - kept)
        size = 0.1 * math.log(factor) + 1
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv
    return (torch.stack((angle.cos(), angle.sin()), 1) * size).float().contiguous()


def _workspace(index: int) -> torch.Tensor:
    """Scratch of the current stream for the sums behind the weights' gradients; a graph that is being captured gets its own."""
    stream = torch._C._cuda_getCurrentRawStream(index)  # noqa: SLF001
    ws = _WORKSPACES.get((index, stream))
    if ws is not None:
        return ws
    size = ctypes.c_int64(0)
    with torch.cuda.device(index):
        _lib.raise_for_code(_lib.library().b200_rotary_workspace(ctypes.byref(size)), "rotary workspace")
        capturing = torch.cuda.is_current_stream_capturing()
        ws = torch.empty(size.value, dtype=torch.uint8, device=torch.device("cuda", index))
        ws[:_HEADER_BYTES].zero_()
    if not capturing:
        with _WORKSPACES_LOCK:
            ws = _WORKSPACES.setdefault((index, stream), ws)
    return ws


def refuse_tangent(what: str, name: str, t: torch.Tensor) -> None:
    """The kernels have no forward derivative: a tensor that carries a tangent would come back without it."""
    if torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
        msg = f"{what}: {name} carries a tangent; forward-mode differentiation is not supported"
        raise ValueError(msg)


def _check_heads(what: str, name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> None:
    if t.dim() != 4 or t.dtype not in _DTYPES or not t.is_cuda:  # noqa: PLR2004
        msg = f"{what}: {name} must be a float16 / bfloat16 / float32 CUDA [batch, tokens, heads, dim] tensor, got {tuple(t.shape)} {t.dtype} on {t.device}"
        raise ValueError(msg)
    if not 1 <= t.shape[3] <= MAX_HEAD_DIM:
        msg = f"{what}: head dim {t.shape[3]} must be 1 .. {MAX_HEAD_DIM}"
        raise ValueError(msg)
    if t.stride(3) != 1 and t.shape[3] > 1:
        msg = f"{what}: {name} must have unit last stride, got strides {t.stride()}"
        raise ValueError(msg)
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[:2] != like.shape[:2] or t.shape[3] != like.shape[3]):
        msg = f"{what}: {name} {tuple(t.shape)} {t.dtype} on {t.device} does not go with {tuple(like.shape)} {like.dtype} on {like.device}"
        raise ValueError(msg)
    refuse_tangent(what, name, t)


def _check_table(what: str, table: torch.Tensor | None, positions: torch.Tensor | None, x: torch.Tensor) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    b, n, _, dim = x.shape
    if table is None:
        return None, None
    if table.dim() != 3 or table.shape[1] != 2 or 2 * table.shape[2] > dim or table.dtype != torch.float32 or table.device != x.device or table.shape[0] < 1:  # noqa: PLR2004
        msg = f"{what}: table must be float32 [rows, 2, <= {dim // 2}] on {x.device}, got {tuple(table.shape)} {table.dtype} on {table.device}"
        raise ValueError(msg)
    if positions is None:
        if table.shape[0] < n:
            msg = f"{what}: a table of {table.shape[0]} rows for {n} tokens"
            raise ValueError(msg)
    elif positions.dtype not in (torch.int32, torch.int64) or positions.device != x.device or tuple(positions.shape) not in ((n,), (b, n)):
        msg = f"{what}: positions must be int32 (or int64) [{n}] or [{b}, {n}] on {x.device}, got {tuple(positions.shape)} {positions.dtype} on {positions.device}"
        raise ValueError(msg)
    else:
        positions = positions if positions.dtype == torch.int32 else positions.clamp(-1, 2**31 - 1).int()  # what 32 bits do not hold is out of range, too
    return table.contiguous(), positions


def _strides(t: torch.Tensor) -> tuple[int, int, int]:
    return t.stride(0), t.stride(1), t.stride(2)


def _launch(  # noqa: PLR0913
    what: str,
    tensors: list[dict[str, torch.Tensor | None]],
    table: torch.Tensor | None,
    positions: torch.Tensor | None,
    *,
    interleaved: bool,
    norm: bool = False,
    eps: float = 0.0,
    backward: bool = False,
) -> None:
    first = tensors[0]["y"]
    a = _lib.B200RotaryArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = a.weight_dtype = _DTYPES[first.dtype]
    a.batch, a.tokens, _, a.head_dim = first.shape
    a.interleaved, a.norm, a.backward, a.tensors, a.eps = interleaved, norm, backward, len(tensors), eps
    if table is not None:
        a.rot, a.cs, a.table_rows = 2 * table.shape[2], table.data_ptr(), table.shape[0]
        if positions is not None:
            a.positions = positions.data_ptr()
            a.pos_stride[:] = (0 if positions.dim() == 1 else positions.stride(0), positions.stride(-1))
    for h, t in zip(a.heads, tensors, strict=False):
        for name in ("x", "y", "g"):
            if t.get(name) is not None:
                setattr(h, name, t[name].data_ptr())
                getattr(h, f"{name}_stride")[:] = _strides(t[name])
        for name in ("w", "dw"):
            if t.get(name) is not None:
                setattr(h, name, t[name].data_ptr())
                a.weight_dtype = _DTYPES[t[name].dtype]
        h.heads = t["y"].shape[2]
    with torch.cuda.device(first.device):
        if any(t.get("dw") is not None for t in tensors):
            ws = _workspace(first.device.index)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        code = _lib.library().b200_rotary(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(first.device.index))  # noqa: SLF001
    _lib.raise_for_code(code, what)
    _lib.use_fast()


def _unit(g: torch.Tensor) -> torch.Tensor:
    return g if g.stride(-1) == 1 or g.shape[-1] == 1 else g.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, table, positions, interleaved):  # noqa: ANN001, ANN205
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        _launch("rotary", [{"x": x, "y": y}], table, positions, interleaved=interleaved)
        ctx.save_for_backward(table, positions)
        ctx.interleaved = interleaved
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):  # noqa: ANN001, ANN205
        table, positions = ctx.saved_tensors
        dx = torch.empty(g.shape, dtype=g.dtype, device=g.device)
        _launch("rotary", [{"g": _unit(g), "y": dx}], table, positions, interleaved=ctx.interleaved, backward=True)
        return dx, None, None, None


def rotary(
    x: torch.Tensor,
    table: torch.Tensor,
    positions: torch.Tensor | None = None,
    *,
    interleaved: bool = False,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The heads `x` `[batch, tokens, heads, dim]` turned by their positions; differentiable in `x`.

    The first `2 * table.shape[2]` dimensions of a head are turned, in pairs `(j, j + half)` or, `interleaved`, `(2 j, 2 j + 1)`; the others
    are copied. Computed in fp32 and rounded once.

    Args:
        x: CUDA tensor, fp16 / bf16 / fp32, unit last stride, any other strides (a view of a packed qkv tensor is fine). Rows on 16 bytes and
            rotated parts in multiples of 16 dimensions are fastest.
        table: `rotary_table`, fp32 `[rows, 2, half]`.
        positions: int32 `[tokens]` or `[batch, tokens]`: the table's row of each token, default 0, 1, 2, ...; negative: not turned (class
            tokens). One past the table is not turned either, and `device_status()` reports it.
        interleaved: Which dimensions are pairs.
        out: Gets the result, may be `x` itself (without gradients).

    Raises:
        ValueError: Operands outside the contract (checked before the launch).
        KernelUnavailableError: The CUDA library is not built or does not load.
    """
    if out is None and _lib.fast is not None:
        done = _lib.fast.rotary(x, table, positions, interleaved)
        if done is not None:
            return done
    _check_heads("rotary", "x", x)
    if table is None:
        msg = "rotary: table is None"
        raise ValueError(msg)
    table, positions = _check_table("rotary", table, positions, x)
    grad = x.requires_grad and torch.is_grad_enabled()
    if out is not None:
        _check_heads("rotary", "out", out, x)
        if grad or out.requires_grad or out.shape != x.shape:
            msg = f"rotary: out must be {tuple(x.shape)} and neither it nor x may require a gradient"
            raise ValueError(msg)
    if x.numel() == 0:
        return x.clone() if out is None else out
    if grad:
        return _Rotary.apply(x, table, positions, interleaved)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    _launch("rotary", [{"x": x, "y": y}], table, positions, interleaved=interleaved)
    return y


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, table, positions, eps, interleaved):  # noqa: ANN001, ANN205, PLR0913
        yq, yk = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
        _launch("qk_norm_rotary", [{"x": q, "y": yq, "w": wq}, {"x": k, "y": yk, "w": wk}], table, positions, interleaved=interleaved, norm=True, eps=eps)
        ctx.save_for_backward(q, k, wq, wk, table, positions)
        ctx.eps, ctx.interleaved = eps, interleaved
        return yq, yk

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):  # noqa: ANN001, ANN205
        q, k, wq, wk, table, positions = ctx.saved_tensors
        tensors = []
        for i, (x, g, w) in enumerate(((q, gq, wq), (k, gk, wk))):
            dw = torch.empty_like(w) if w is not None and ctx.needs_input_grad[2 + i] else None
            tensors.append({"x": x, "g": _unit(g), "w": w, "y": torch.empty(x.shape, dtype=x.dtype, device=x.device), "dw": dw})
        _launch("qk_norm_rotary", tensors, table, positions, interleaved=ctx.interleaved, norm=True, eps=ctx.eps, backward=True)
        return tensors[0]["y"], tensors[1]["y"], tensors[0]["dw"], tensors[1]["dw"], None, None, None, None


def qk_norm_rotary(  # noqa: PLR0913
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    table: torch.Tensor | None,
    positions: torch.Tensor | None = None,
    *,
    eps: float = 1e-6,
    interleaved: bool = False,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """q and k with each head divided by its root mean square, times a weight, and turned by its position, in one launch.

    `x * rsqrt(mean(x ** 2) + eps) * weight`, then `rotary`, in fp32 and rounded once; differentiable in q, k and both weights (their
    gradients are summed over all heads and tokens in a fixed order).

    Args:
        q: CUDA `[batch, tokens, heads, dim]`, fp16 / bf16 / fp32, unit last stride.
        k: The same with its own count of heads.
        q_weight: `[dim]` of q's type or float32, or None (ones).
        k_weight: The same for k; of the type of `q_weight`.
        table: As for `rotary`, or None: nothing is turned.
        positions: As for `rotary`.
        eps: Added to the mean square.
        interleaved: As for `rotary`.
        out: Get the results, may be q and k themselves (without gradients).

    Raises:
        ValueError: Operands outside the contract (checked before the launch).
        KernelUnavailableError: The CUDA library is not built or does not load.
    """
    if out is None and _lib.fast is not None:
        done = _lib.fast.qk_norm_rotary(q, k, q_weight, k_weight, table, positions, eps, interleaved)
        if done is not None:
            return done
    what = "qk_norm_rotary"
    _check_heads(what, "q", q)
    _check_heads(what, "k", k, q)
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.shape != (q.shape[3],) or w.dtype not in (q.dtype, torch.float32) or w.dtype != weights[0].dtype or w.device != q.device or not w.is_contiguous():
            msg = f"{what}: weights must be contiguous [{q.shape[3]}] of {q.dtype} or float32 (both alike) on {q.device}, got {tuple(w.shape)} {w.dtype} on {w.device}"
            raise ValueError(msg)
        refuse_tangent(what, "a weight", w)
    if not eps >= 0:
        msg = f"{what}: eps {eps} must not be negative"
        raise ValueError(msg)
    if positions is not None and table is None:
        msg = f"{what}: positions without a table"
        raise ValueError(msg)
    table, positions = _check_table(what, table, positions, q)
    grad = torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, *weights))
    if out is not None:
        for name, t, x in (("out[0]", out[0], q), ("out[1]", out[1], k)):
            _check_heads(what, name, t, x)
            if grad or t.requires_grad or t.shape != x.shape:
                msg = f"{what}: {name} must be {tuple(x.shape)} and nothing may require a gradient"
                raise ValueError(msg)
    if q.numel() == 0 or k.numel() == 0:
        msg = f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)} must not be empty"
        raise ValueError(msg)
    if grad:
        return _QkNormRotary.apply(q, k, q_weight, k_weight, table, positions, float(eps), interleaved)
    yq, yk = out if out is not None else (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k))
    _launch(what, [{"x": q, "y": yq, "w": q_weight}, {"x": k, "y": yk, "w": k_weight}], table, positions, interleaved=interleaved, norm=True, eps=float(eps))
    return yq, yk
