"""A token decoder's operators from their definitions, in float64 (torch, on whatever device the operands are).

TEST INFRASTRUCTURE: only `tests/` may import this file; the product never does.
"""

from __future__ import annotations

import math

import torch

BLOCK = 16


def rotate(x: torch.Tensor, table: torch.Tensor | None, positions: torch.Tensor | None, *, interleaved: bool, back: bool = False) -> torch.Tensor:
    """x `[B, N, H, D]` as float64, its first dimensions turned pair by pair; negative positions and those past the table are not."""
    x = x.double().clone()
    b, n, _, _ = x.shape
    if table is None:
        return x
    half = table.shape[2]
    at = torch.arange(n, device=x.device).expand(b, n) if positions is None else positions.long().expand(b, n)
    still = (at < 0) | (at >= table.shape[0])
    row = table.double()[at.clamp(0, table.shape[0] - 1)]
    cos = torch.where(still[..., None], 1.0, row[:, :, 0])[:, :, None]
    sin = torch.where(still[..., None], 0.0, row[:, :, 1])[:, :, None] * (-1 if back else 1)
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    p, q = x[..., first].clone(), x[..., second].clone()
    x[..., first], x[..., second] = p * cos - q * sin, q * cos + p * sin
    return x


def norm_rotate(x: torch.Tensor, w: torch.Tensor | None, table: torch.Tensor | None, positions: torch.Tensor | None, *, eps: float, interleaved: bool) -> torch.Tensor:
    h = x.double() / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps)
    return rotate(h if w is None else h * w.double(), table, positions, interleaved=interleaved)


def norm_rotate_backward(x: torch.Tensor, g: torch.Tensor, w: torch.Tensor | None, table: torch.Tensor | None, positions: torch.Tensor | None, *, eps: float, interleaved: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """(gradient of x, gradient of w) by the formula."""
    t = rotate(g, table, positions, interleaved=interleaved, back=True)
    r = 1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + eps)
    hat = x.double() * r
    tw = t if w is None else t * w.double()
    return r * (tw - hat * (tw * hat).mean(-1, keepdim=True)), (t * hat).sum((0, 1, 2))


# ---- the 4-bit cache, byte by byte ----


def byte_places(dim: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Byte of each code of K and of V in a block, `[16, dim]`, and of each token's four parameters `[16, 4]`."""
    t, d = torch.arange(BLOCK)[:, None], torch.arange(dim)
    row = 8 * dim + t // 2 * (dim + 16)
    return t * (dim // 2) + d // 2, row + 4 * (d // 4) + 2 * (t % 2) + d % 4 // 2, row + dim + 8 * (t % 2) + 2 * torch.arange(4)


def decode(cache: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(K values, V values, parameters) of every slot of a cache: float64 `[pages, heads, page, dim]` twice and `[.., page, 4]`."""
    dim = cache.shape[3] // BLOCK - 8
    at_k, at_v, at_p = (x.to(cache.device) for x in byte_places(dim))
    high = torch.arange(dim, device=cache.device) % 2 == 1
    low_byte, high_byte = cache[..., at_p].int(), cache[..., at_p + 1].int()
    pairs = ((low_byte << 16) | (high_byte << 24)).view(torch.float32).double()
    got = []
    for at, pair in ((at_k, 0), (at_v, 2)):
        byte = cache[..., at]
        code = torch.where(high, byte >> 4, byte & 15).double()
        got.append((pairs[..., pair, None] * code + pairs[..., pair + 1, None]).flatten(2, 3))
    return got[0], got[1], pairs.flatten(2, 3)


def quantise(x: torch.Tensor) -> torch.Tensor:
    """Values that a group along the last axis is held as: codes by fp32 arithmetic, as the definition has it, values in float64."""
    x = x.float()
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = high - low
    step, least = (span * torch.tensor(1 / 15, dtype=torch.float32, device=x.device)).bfloat16().float(), low.bfloat16().float()
    step = torch.where(step < 2.0**-126, 0.0, step)
    code = torch.where(step > 0, ((x - least) * (1 / step)).round().clamp(0, 15), 0.0)
    held = least.double() + step.double() * code.double()
    return torch.where(span.isfinite() & step.isfinite() & least.isfinite(), held, math.nan)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """One sequence: q `[n, Hq, D]`, the last n of k, v `[H, T, D]`'s tokens. Returns the output and the softmax weights `[n, Hq, T]`."""
    n, hq, _ = q.shape
    h, t, _ = k.shape
    logits = torch.einsum("nhgd,htd->nhgt", q.double().unflatten(1, (h, hq // h)), k) * scale
    last = t - n + torch.arange(n, device=q.device)
    logits = logits.masked_fill(torch.arange(t, device=q.device) > last[:, None, None, None], -math.inf)
    p = torch.where((last < 0)[:, None, None, None], 0.0, torch.softmax(logits, -1)).nan_to_num(0.0) if t else logits
    return torch.einsum("nhgt,htd->nhgd", p, v).flatten(1, 2), p.flatten(1, 2)
