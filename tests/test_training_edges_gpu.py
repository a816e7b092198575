"""Edges of `layer_norm`, `linear_cross_entropy` and `linear_distillation` on a B200, on the full way and on the way of repeated calls.
Tolerances are those of tests/test_layer_norm_gpu.py and tests/test_losses_gpu.py."""

from __future__ import annotations

from typing import TYPE_CHECKING

import pytest
import torch

import fastforks_b200 as ff
from fastforks_b200 import _lib
from oracle import training_oracle as oracle
from test_losses_gpu import check, integers, layer, normal

if TYPE_CHECKING:
    from collections.abc import Callable

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _kernels_ran_to_the_end():  # noqa: ANN202
    yield
    assert ff.device_status() == 0


@pytest.fixture(params=["full", "repeated"])
def way(request: pytest.FixtureRequest, monkeypatch: pytest.MonkeyPatch) -> str:
    """Both ways of a call: the Python side's, and the host extension's once it is loaded."""
    if request.param == "full":
        monkeypatch.setattr(_lib, "fast", None)
        monkeypatch.setattr(_lib, "use_fast", lambda: None)
    else:
        ff.layer_norm(torch.zeros(1, 8, device="cuda"))
        assert _lib.fast is not None
    return request.param


def negated(t: torch.Tensor) -> torch.Tensor:
    """`t` as a tensor that holds -t and a bit that says so, as the imaginary part of a conjugate does."""
    view = torch._neg_view(-t)  # noqa: SLF001
    assert view.is_neg()
    assert torch.equal(view, t)
    return view


def operators() -> dict[str, tuple[Callable[..., torch.Tensor], tuple[torch.Tensor, ...]]]:
    """Name -> call, its differentiable operands."""
    x, w, y = layer(40, 300, 64, torch.bfloat16)
    ids, teacher = integers(0, 300, (40, 5), 3), normal(40, 5)
    bias = normal(300, dtype=torch.bfloat16, seed=4)
    heads, table = normal(2, 7, 3, 64, dtype=torch.float16, seed=5), ff.rotary_table(7, 64, device="cuda")
    weight = 1 + 0.2 * normal(64, seed=6)
    return {
        "ce none": (lambda a, b, c: ff.linear_cross_entropy(a, b, y, bias=c, reduction="none"), (x, w, bias)),
        "ce mean": (lambda a, b, c: ff.linear_cross_entropy(a, b, y, bias=c), (x, w, bias)),
        "kd none": (lambda a, b: ff.linear_distillation(a, b, ids, teacher, reduction="none"), (x, w)),
        "layer norm": (lambda a, b, c: ff.layer_norm(a, b, c), (x, w[0], w[1])),
        "layer norm of odd rows": (lambda a: ff.layer_norm(a), (normal(9, 33),)),
        "rotary": (lambda a: ff.rotary(a, table), (heads,)),
        "norm and rotary": (lambda a, b: torch.cat(ff.qk_norm_rotary(a, a * 2, b, b, table), 2), (heads, weight)),
    }


OPERATORS = ("ce none", "ce mean", "kd none", "layer norm", "layer norm of odd rows", "rotary", "norm and rotary")


@pytest.mark.usefixtures("way")
@pytest.mark.parametrize("name", OPERATORS)
def test_gradients_that_come_in_with_a_lazy_negation(name: str) -> None:
    call, operands = operators()[name]
    leaves = [t.detach().clone().requires_grad_(True) for t in operands]
    result = call(*leaves)
    g = normal(result.numel(), dtype=result.dtype, seed=9).view(result.shape)
    want = torch.autograd.grad(result, leaves, g, retain_graph=True)
    got = torch.autograd.grad(result, leaves, negated(g), retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))
    if result.dtype == torch.float32:  # as it comes about: the imaginary part of a conjugate, every second number in memory
        strided = torch.complex(g, -g).conj().imag
        assert strided.is_neg()
        got = torch.autograd.grad(result, leaves, strided)
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


@pytest.mark.usefixtures("way")
@pytest.mark.parametrize("name", OPERATORS)
def test_operands_with_a_lazy_negation(name: str) -> None:
    call, operands = operators()[name]
    leaves = [t.detach().clone().requires_grad_(True) for t in operands]
    want = call(*leaves)
    g = normal(want.numel(), dtype=want.dtype, seed=9).view(want.shape)
    grads = torch.autograd.grad(want, leaves, g)
    for i in range(len(leaves)):
        result = call(*(negated(t) if j == i else t for j, t in enumerate(leaves)))
        assert torch.equal(result, want)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(result, leaves, g), grads, strict=True))
        with torch.no_grad():
            assert torch.equal(call(*(negated(t) if j == i else t for j, t in enumerate(leaves))), want)


@pytest.mark.usefixtures("way")
def test_a_teacher_a_table_and_an_out_with_a_lazy_negation() -> None:
    x, w, _ = layer(40, 300, 64, torch.float16)
    ids, teacher = integers(0, 300, (40, 5), 3), normal(40, 5)
    assert torch.equal(ff.linear_distillation(x, w, ids, negated(teacher)), ff.linear_distillation(x, w, ids, teacher))
    heads, table = x.view(2, 10, 2, 64).clone(), ff.rotary_table(10, 64, device="cuda")
    assert torch.equal(ff.rotary(heads, negated(table)), ff.rotary(heads, table))
    before = x.clone()
    for refused in (
        lambda: ff.layer_norm(x, out=negated(x.clone())),
        lambda: ff.layer_norm(x, out=torch._neg_view(x)),  # noqa: SLF001
        lambda: ff.rotary(heads, table, out=negated(heads.clone())),
        lambda: ff.qk_norm_rotary(heads, heads, None, None, table, out=(heads, negated(heads.clone()))),
    ):
        with pytest.raises(ValueError, match="negat"):
            refused()
    assert torch.equal(x, before)


@pytest.mark.usefixtures("way")
@pytest.mark.parametrize("saved_by", ["cross entropy", "distillation", "layer norm"])
def test_a_saved_tensor_that_a_norm_writes_to_is_noticed(saved_by: str) -> None:
    x, w, y = layer(40, 300, 64, torch.float16)
    weight = w.detach().requires_grad_(True) if saved_by != "layer norm" else torch.ones(64, device="cuda", dtype=torch.float16, requires_grad=True)
    call = {
        "cross entropy": lambda t: ff.linear_cross_entropy(t, weight, y),
        "distillation": lambda t: ff.linear_distillation(t, weight, y[:, None], torch.zeros(40, 1, device="cuda")),
        "layer norm": lambda t: ff.layer_norm(t, weight).sum(),
    }[saved_by]
    for out in (lambda t: t, lambda t: t[3:5]):  # itself, and a part of it
        held = x.clone()
        loss = call(held)
        ff.layer_norm(out(held), out=out(held))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, weight)
    held = x.clone()
    loss = call(held)
    ff.layer_norm(held, out=torch.empty_like(held))  # another tensor: nothing is noticed, as nothing happened
    torch.autograd.grad(loss, weight)


@pytest.mark.usefixtures("way")
def test_tensors_of_inference_mode_are_written_to() -> None:
    x = normal(5, 64)
    with torch.inference_mode():
        kept = torch.empty_like(x)
        inside = ff.layer_norm(x, out=torch.empty_like(x))
    assert ff.layer_norm(x, out=kept) is kept  # they have no version
    assert torch.equal(kept, ff.layer_norm(x))
    assert torch.equal(inside, kept)


@pytest.mark.usefixtures("way")
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("rows", "vocab"), [(40, 300), (300, 1000), (3000, 10)])
def test_no_row_counts_under_a_gradient_that_is_not_finite(rows: int, vocab: int, dtype: torch.dtype) -> None:
    """A sum divided by the number of rows that count: with none of them its gradient is infinite, and nothing is added to nothing."""
    x, w, y = layer(rows, vocab, 64, dtype)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, normal(vocab, dtype=dtype, seed=4))]
    for g in (float("inf"), float("nan")):
        loss = ff.linear_cross_entropy(leaves[0], leaves[1], torch.full_like(y, -100), bias=leaves[2], reduction="sum")
        for grad in torch.autograd.grad(loss, leaves, torch.tensor(g, device="cuda")):
            assert not grad.any()


@pytest.mark.parametrize("size", [1e-40, 1e-30, 1e-3, 1e25, 1e37])
def test_row_gradients_of_any_size_in_bfloat16(size: float) -> None:
    """bfloat16 has fp32's range: nothing is flushed or infinite. Below 2^-126 gradients themselves have fewer digits than fp32's 24 (1e-40: some 16), and the
    results are subnormal numbers, steps of 2^-133 apart: half of one is in the bounds."""
    x, w, y = layer(100, 400, 64, torch.bfloat16)
    x, w, b = x.requires_grad_(True), w.requires_grad_(True), normal(400, dtype=torch.bfloat16, seed=3).requires_grad_(True)
    g = normal(100, seed=5).clamp(-4, 4) * size
    g[::7] = 0
    loss = ff.linear_cross_entropy(x, w, y, bias=b, reduction="none")
    dx, dw, db = torch.autograd.grad(loss, (x, w, b), g)
    r = oracle.cross_entropy(x.detach(), w.detach(), y, -100, "none", g, b.detach())
    assert not dx[::7].any()
    check(r, x, w, 1.0, loss, {"dx": dx, "dw": dw, "db": db}, g, "none", b)


def test_row_gradients_past_the_range_of_float16() -> None:
    """Infinities of the right sign, rows without a gradient 0, nothing NaN. (65520 lies half a step past the largest number; a sixteenth to either side
    is left to the roundings before it.)"""
    x, w, y = layer(100, 400, 64, torch.float16)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    g = normal(100, seed=5) * 1e25
    g[::7] = 0
    dx, dw = torch.autograd.grad(ff.linear_cross_entropy(x, w, y, reduction="none"), (x, w), g)
    r = oracle.cross_entropy(x.detach(), w.detach(), y, -100, "none", g)
    for got, ref in ((dx, r.dx), (dw, r.dw)):
        assert not got.isnan().any()
        sure = ref.abs() > 65520 * 17 / 16
        # of what is computed from numbers of size 1e25 the last 2^-11 (and 2^-24 of a sum's size) is not known: all that matters is that it is far above 65520
        sure &= ref.abs() > ref.abs().amax() * 2.0**-8
        assert torch.equal(got[sure].double(), ref[sure].sign() * float("inf"))
    assert not dx[::7].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("kind", ["cross entropy", "distillation"])
@pytest.mark.parametrize(("rows", "vocab", "dim"), [(300, 30000, 264), (2049, 8191, 136), (100, 500, 64)])
def test_row_gradients_that_lie_decades_apart(rows: int, vocab: int, dim: int, kind: str, dtype: torch.dtype) -> None:
    """A power of two is taken out of all rows together, so a row's gradients of logits have what fp16's subnormal numbers leave of them: the bounds' 2^-39 of
    the largest row's. The first two sizes are past 128 rows and 2^31 products, where what is rounded off is not multiplied."""
    x, w, y = layer(rows, vocab, dim, dtype)
    y[::11] = -100
    x, w, b = x.requires_grad_(True), w.requires_grad_(True), normal(vocab, dtype=dtype, seed=3).requires_grad_(True)
    g = torch.exp(-14 * torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(6), device="cuda")) * normal(rows, seed=5).sign()  # 1 to 1e-6
    if kind == "cross entropy":
        loss = ff.linear_cross_entropy(x, w, y, bias=b, reduction="none")
        r = oracle.cross_entropy(x.detach(), w.detach(), y, -100, "none", g, b.detach())
        tau = 1.0
    else:
        ids, teacher, tau = integers(0, vocab, (rows, 9), 7), normal(rows, 9, seed=8), 2.0
        ids[::11] = -1
        loss = ff.linear_distillation(x, w, ids, teacher, bias=b, temperature=tau, reduction="none")
        r = oracle.distillation(x.detach(), w.detach(), ids, teacher, tau, "none", g, b.detach())
    dx, dw, db = torch.autograd.grad(loss, (x, w, b), g)
    check(r, x, w, tau, loss, {"dx": dx, "dw": dw, "db": db}, g, "none", b)
    # and each row by itself: of its own size, but for what is flushed
    near = (dx.detach().double() - r.dx).norm(dim=1)
    flushed = float(g.abs().max()) * tau * 2.0**-39 if dtype == torch.float16 else 0.0
    counted = r.counts
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 * dim**0.5
    size = 2 * torch.finfo(dtype).eps / 2 * (r.dl.abs() @ w.detach().double().abs()).norm(dim=1)
    assert bool((near[counted] <= (size + flushed * float(w.detach().double().abs().sum(0).norm()) + tiny)[counted]).all())
