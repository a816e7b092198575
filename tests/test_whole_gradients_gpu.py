"""`whole_gradients` of the losses on a B200: gradients without what the rounding of the logits' gradients to 16 bits takes.

Tolerances are those of tests/test_losses_gpu.py but for the logits' gradient, of which two roundings after one another leave U^2 instead of U (the second is of
what the first took, at most U of a value); fp16 flushes below 2^-40 of the largest row's as there. The errors' 2-norms: the results' own rounding, and a fiftieth
of it for all that fp32 leaves (U is 2^13 or 2^16 times u, and sums of thousands of terms are off by some hundred u).
"""

from __future__ import annotations

import pytest
import torch

import fastforks_b200 as ff
from fastforks_b200 import _lib
from oracle import training_oracle as oracle
from test_losses_gpu import DTYPES, F32, TINY, integers, layer, logit_error, near, normal

pytestmark = pytest.mark.gpu

# rows, vocabulary, dim, entries: past 2^31 products; in several pieces of the vocabulary; in parts of the rows; of few rows and of few products, where they are whole anyhow
SIZES = [(300, 30000, 264, 0), (300, 30000, 264, 9), (1025, 16001, 512, 0), (2049, 70001, 64, 5), (40000, 300, 256, 0), (100, 500, 64, 0), (300, 1000, 136, 5)]


@pytest.fixture(autouse=True)
def _kernels_ran_to_the_end():  # noqa: ANN202
    yield
    assert ff.device_status() == 0


def problem(rows: int, vocab: int, dim: int, entries: int, dtype: torch.dtype, reduction: str):  # noqa: ANN201, PLR0913
    """A call of x, weight, bias and keywords; these; a gradient of its result; the result in 64 bits; the temperature."""
    x, w, y = layer(rows, vocab, dim, dtype)
    y[::11] = -100
    bias = normal(vocab, dtype=dtype, seed=3)
    g = normal(rows, seed=5) if reduction == "none" else torch.tensor(-1.7, device="cuda")
    if entries:
        ids, teacher = integers(0, vocab, (rows, entries), 7), normal(rows, entries, seed=8)
        ids[::11] = -1
        call = lambda a, b, c, **kw: ff.linear_distillation(a, b, ids, teacher, bias=c, temperature=2.0, reduction=reduction, **kw)  # noqa: E731
        return call, (x, w, bias), g, oracle.distillation(x, w, ids, teacher, 2.0, reduction, g, bias), 2.0
    call = lambda a, b, c, **kw: ff.linear_cross_entropy(a, b, y, bias=c, reduction=reduction, **kw)  # noqa: E731
    return call, (x, w, bias), g, oracle.cross_entropy(x, w, y, -100, reduction, g, bias), 1.0


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_the_error_is_that_of_the_results_rounding(size: tuple[int, int, int, int], dtype: str, reduction: str) -> None:
    t = DTYPES[dtype]
    call, operands, g, r, tau = problem(*size, t, reduction)
    leaves = [o.detach().requires_grad_(True) for o in operands]
    loss = call(*leaves, whole_gradients=True)
    grads = dict(zip(("dx", "dw", "db"), torch.autograd.grad(loss, leaves, g, retain_graph=True), strict=True))
    x, w, bias = operands
    half, n = torch.finfo(t).eps / 2, int(r.counts.sum().clamp(min=1))
    d = logit_error(x, w, r.counts, bias.double()) / tau
    each = torch.where(r.counts, g.double().abs().expand(r.rows.shape) * tau / (n if reduction == "mean" else 1), 0.0)[:, None]
    flushed = each.max() * 2.0**-39 if t == torch.float16 else 0.0
    e_dl = half**2 * r.dl.abs() + (1 + half) * each * r.q * (2 * d + 40 * F32)[:, None] + flushed * r.counts[:, None]
    xz = torch.where(r.counts[:, None], x.double(), 0.0)
    ones = torch.ones(1, size[0], dtype=torch.float64, device="cuda")
    for name, left, right, error in (("dx", r.dl, w.double(), e_dl), ("dw", r.dl.T, xz, e_dl.T), ("db", r.dl.T, ones.T, e_dl.T)):
        ref = getattr(r, name)
        terms = left.shape[1] * (2 if name != "db" else 1)  # G, and what its rounding took
        e = (error @ right.abs() + 2 * F32 * (terms / 16 + 64) * (left.abs() @ right.abs())).view(ref.shape)
        near(grads[name], ref, half * (ref.abs() + e) + e + TINY[t], name)
        own = float((ref.to(t).double() - ref).norm())
        assert float((grads[name].double() - ref).norm()) <= 1.02 * own + float(e.norm()), name
    again = torch.autograd.grad(loss, leaves, g)
    assert all(torch.equal(a, b) for a, b in zip(again, grads.values(), strict=True))
    with torch.no_grad():
        assert torch.equal(call(*operands), loss)  # the loss does not depend on it


@pytest.mark.parametrize("entries", [0, 5])
def test_both_ways_of_a_call_and_each_gradient_alone(entries: int, monkeypatch: pytest.MonkeyPatch) -> None:
    call, operands, g, _, _ = problem(400, 9000, 640, entries, torch.bfloat16, "mean")

    def gradients(wanted: tuple[int, ...], **kw: bool) -> list[torch.Tensor]:
        leaves = [o.detach().requires_grad_(i in wanted) for i, o in enumerate(operands)]
        return list(torch.autograd.grad(call(*leaves, **kw), [leaves[i] for i in wanted], g))

    ff.layer_norm(torch.zeros(1, 8, device="cuda"))
    assert _lib.fast is not None
    whole, rounded = gradients((0, 1, 2), whole_gradients=True), gradients((0, 1, 2))
    assert not any(torch.equal(a, b) for a, b in zip(whole[:2], rounded, strict=False))
    monkeypatch.setattr(_lib, "fast", None)
    monkeypatch.setattr(_lib, "use_fast", lambda: None)
    for want, kw in ((whole, {"whole_gradients": True}), (rounded, {"whole_gradients": False})):
        assert all(torch.equal(a, b) for a, b in zip(gradients((0, 1, 2), **kw), want, strict=True))
        assert torch.equal(gradients((2,), **kw)[0], want[2])
        for wanted in ((0,), (1,), (0, 2), (1, 2)):  # other parts of k may be added up in another order: fp32's difference, and a rounding that goes the other way
            for i, got in zip(wanted, gradients(wanted, **kw), strict=True):
                assert float((got.double() - want[i].double()).norm()) < 2.0**-9 * float(want[i].double().norm())


def test_small_calls_are_whole_anyhow() -> None:
    for rows, vocab, dim in ((128, 20000, 1024), (1000, 1000, 2048)):
        call, operands, g, _, _ = problem(rows, vocab, dim, 0, torch.bfloat16, "mean")
        leaves = [o.detach().requires_grad_(True) for o in operands]
        pairs = zip(torch.autograd.grad(call(*leaves), leaves, g), torch.autograd.grad(call(*leaves, whole_gradients=True), leaves, g), strict=True)
        assert all(torch.equal(a, b) for a, b in pairs)


def test_in_a_graph() -> None:
    call, operands, g, _, _ = problem(500, 9000, 512, 0, torch.float16, "none")

    def step() -> list[torch.Tensor]:
        leaves = [o.detach().requires_grad_(True) for o in operands]
        return list(torch.autograd.grad(call(*leaves, whole_gradients=True), leaves, g))

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for t in out:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want, strict=True))
