"""Layer norm, and an output layer's cross entropy and distillation, from their definitions in float64 (torch, on whatever device the operands
are). Gradients by the formulas. The `*_size` results are sums of magnitudes, which errors are proportional to.

TEST INFRASTRUCTURE: only `tests/` may import this file; the product never does.
"""

from __future__ import annotations

import dataclasses

import torch


@dataclasses.dataclass
class Norm:
    y: torch.Tensor
    hat: torch.Tensor
    rstd: torch.Tensor
    dx: torch.Tensor | None = None
    dw: torch.Tensor | None = None
    db: torch.Tensor | None = None


def layer_norm(x: torch.Tensor, w: torch.Tensor | None, b: torch.Tensor | None, eps: float, dy: torch.Tensor | None = None) -> Norm:
    """Of rows `[T, D]`."""
    x = x.double()
    w64 = torch.ones_like(x[0]) if w is None else w.double()
    b64 = torch.zeros_like(x[0]) if b is None else b.double()
    rstd = 1 / torch.sqrt(x.var(1, unbiased=False, keepdim=True) + eps)
    hat = (x - x.mean(1, keepdim=True)) * rstd
    r = Norm(hat * w64 + b64, hat, rstd)
    if dy is not None:
        t = dy.double() * w64
        r.dx = rstd * (t - t.mean(1, keepdim=True) - hat * (t * hat).mean(1, keepdim=True))
        r.dw, r.db = (dy.double() * hat).sum(0), dy.double().sum(0)
    return r


@dataclasses.dataclass
class Head:
    rows: torch.Tensor  # loss of each row, 0 where it does not count
    loss: torch.Tensor  # reduced
    counts: torch.Tensor
    q: torch.Tensor  # softmax of the logits / tau
    dl: torch.Tensor | None = None  # gradient of the logits
    dx: torch.Tensor | None = None
    dw: torch.Tensor | None = None
    db: torch.Tensor | None = None


def head(x: torch.Tensor, w: torch.Tensor, p: torch.Tensor, entropy: torch.Tensor, counts: torch.Tensor, tau: float, reduction: str, g: torch.Tensor | None, bias: torch.Tensor | None) -> Head:  # noqa: PLR0913
    """p `[T, V]` over the vocabulary; entropy = sum p log p; g: gradient of the result (a number, or one for each row)."""
    x = torch.where(counts[:, None], x.double(), 0.0)
    z = (x @ w.double().T + (0.0 if bias is None else bias.double())) / tau
    logq = z - torch.logsumexp(z, 1, keepdim=True)
    rows = torch.where(counts, tau**2 * (entropy - (p * torch.where(p > 0, logq, 0.0)).sum(1)), 0.0)
    n = counts.sum().clamp(min=1)
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / n}[reduction]
    r = Head(rows, loss, counts, logq.exp())
    if g is not None:
        each = g.double().expand(rows.shape) / (n if reduction == "mean" else 1)
        r.dl = torch.where(counts[:, None], (each * tau)[:, None] * (r.q - p), 0.0)
        r.dx, r.dw, r.db = r.dl @ w.double(), r.dl.T @ x, r.dl.sum(0)
    return r


def cross_entropy(x: torch.Tensor, w: torch.Tensor, targets: torch.Tensor, ignore: int, reduction: str, g: torch.Tensor | None = None, bias: torch.Tensor | None = None) -> Head:  # noqa: PLR0913
    counts = targets != ignore
    p = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    p[counts, targets[counts].long()] = 1.0
    return head(x, w, p, torch.zeros_like(p[:, 0]), counts, 1.0, reduction, g, bias)


def distillation(x: torch.Tensor, w: torch.Tensor, ids: torch.Tensor, teacher: torch.Tensor, tau: float, reduction: str, g: torch.Tensor | None = None, bias: torch.Tensor | None = None) -> Head:  # noqa: PLR0913
    there = ids >= 0
    counts = there.any(1)
    z = (teacher.double() / tau).masked_fill(~there, -torch.inf)
    logp = z - torch.where(counts, torch.logsumexp(z, 1), 0.0)[:, None]
    each = logp.exp()
    entropy = torch.where(each > 0, each * logp, 0.0).sum(1)
    p = torch.zeros(x.shape[0], w.shape[0], dtype=torch.float64, device=x.device)
    p.scatter_add_(1, ids.clamp(min=0).long(), each)
    return head(x, w, p, entropy, counts, tau, reduction, g, bias)
