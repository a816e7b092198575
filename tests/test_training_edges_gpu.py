"""Edges of `layer_norm`, `linear_cross_entropy` and `linear_distillation` on a B200, on the full way and on the way of repeated calls.
Tolerances are those of tests/test_layer_norm_gpu.py and tests/test_losses_gpu.py."""

from __future__ import annotations

from typing import TYPE_CHECKING

import pytest
import torch

import fastforks_b200 as ff
from fastforks_b200 import _lib
from test_losses_gpu import integers, layer, normal

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
