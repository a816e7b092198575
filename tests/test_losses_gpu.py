"""`linear_cross_entropy` and `linear_distillation` on a B200 against their definitions in 64 bits, forward and gradients.

Tolerances. u = 2^-24, U half a step of the operands' type. A logit is a chain of dim / 16 products of sixteen terms, each of which may lose a unit of
fp32 (2 u) of what has been summed up, at most the sum of magnitudes M: D = 2 u (dim / 16 + 16) M, and with it softmax is off by 2 D relative to itself
(its own logit, and the sum's) and by 40 u (exponential, sums of exponentials, logarithm), the loss of a row by 2 D / tau and 40 u of |z| + |loss|, times tau^2.
The logits' gradient is rounded to 16 bits on its way into the products: U of |q - p|; fp16 holds it times 2^15, down to 2^-40 of the largest row's. dx and dw are
sums of it over V and T, in chains like a logit's, rounded once more.
"""

from __future__ import annotations

import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import fastforks_b200 as ff
from oracle import training_oracle as oracle

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-133}
F32 = 2.0**-24
TARGET = 1 << 23


@pytest.fixture(autouse=True)
def _kernels_ran_to_the_end(request: pytest.FixtureRequest):  # noqa: ANN202
    yield
    assert ff.device_status() == (TARGET if "reports" in request.node.name else 0)


def normal(*shape: int, dtype: torch.dtype = torch.float32, seed: int = 0, scale: float = 1.0) -> torch.Tensor:
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def integers(low: int, high: int, shape: tuple[int, ...], seed: int = 0) -> torch.Tensor:
    return torch.randint(low, high, shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def layer(rows: int, vocab: int, dim: int, dtype: torch.dtype, seed: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Hidden states that lean to their targets, the layer's weight, the targets."""
    w = normal(vocab, dim, dtype=dtype, seed=seed, scale=1.5 / dim**0.5)
    y = integers(0, vocab, (rows,), seed + 1)
    lean = 4 * torch.rand(rows, 1, generator=torch.Generator(device="cuda").manual_seed(seed + 2), device="cuda")
    return (normal(rows, dim, seed=seed + 3) + lean * w[y].float()).to(dtype), w, y


def logit_error(x: torch.Tensor, w: torch.Tensor, counts: torch.Tensor, bias: torch.Tensor | float) -> torch.Tensor:
    """Of each row, the largest."""
    x = torch.where(counts[:, None], x.double(), 0.0)
    return 2 * F32 * (x.shape[1] / 16 + 16) * (x.abs() @ w.double().abs().T + abs(bias)).amax(1)


def near(got: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    assert got.shape == ref.shape, what
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), f"{what}: worst {float((off / bound).max()):.2f} bounds"


def check(r: oracle.Head, x: torch.Tensor, w: torch.Tensor, tau: float, loss: torch.Tensor, grads: dict, g: torch.Tensor | None, reduction: str, bias: torch.Tensor | None = None) -> None:  # noqa: PLR0913
    x, w, b64 = x.detach(), w.detach(), 0.0 if bias is None else bias.detach().double()
    d = logit_error(x, w, r.counts, b64) / tau
    z = ((torch.where(r.counts[:, None], x.double(), 0.0) @ w.double().T + b64) / tau).abs().amax(1)
    e_rows = torch.where(r.counts, tau**2 * (2 * d + 40 * F32 * (z + 3)) + 40 * F32 * r.rows.abs(), 0.0)
    n = int(r.counts.sum().clamp(min=1))
    e_loss = {"none": e_rows, "sum": e_rows.sum(), "mean": e_rows.sum() / n}[reduction]
    near(loss.detach(), r.loss, e_loss, "loss")
    if g is None:
        return
    half = torch.finfo(x.dtype).eps / 2
    each = (g.double().abs().expand(r.rows.shape) * tau / (n if reduction == "mean" else 1))[:, None]
    each = torch.where(r.counts[:, None], each, 0.0)
    flushed = each.max() * 2.0**-39 if x.dtype == torch.float16 else 0.0
    e_dl = half * r.dl.abs() + (1 + half) * each * r.q * (2 * d + 40 * F32)[:, None] + flushed * r.counts[:, None]
    xz = torch.where(r.counts[:, None], x.double(), 0.0)
    for name, left, right, error in (("dx", r.dl, w.double(), e_dl), ("dw", r.dl.T, xz, e_dl.T)):
        if name in grads:
            ref = getattr(r, name)
            size = left.abs() @ right.abs()
            e = error @ right.abs() + 2 * F32 * (left.shape[1] / 16 + 64) * size
            near(grads[name].detach(), ref, half * (ref.abs() + e) + e + TINY[x.dtype], name)
    if "db" in grads:
        e = e_dl.sum(0) + 2 * F32 * (x.shape[0] / 32 + 64) * r.dl.abs().sum(0)
        near(grads["db"].detach(), r.db, half * (r.db.abs() + e) + e + TINY[x.dtype], "db")


SHAPES = [
    # rows, vocabulary, dim
    (1, 1, 8), (1, 10, 64), (2, 300, 40), (63, 129, 64), (64, 64, 128), (65, 1000, 136), (255, 257, 264), (256, 256, 256), (257, 2049, 520), (300, 5003, 768), (520, 777, 1032), (130, 20011, 72),
    (17, 4000, 4104), (100, 700, 2056), (250, 300, 2056), (300, 600, 2056), (16, 5000, 1096),
]  # fmt: skip


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_cross_entropy(shape: tuple[int, int, int], dtype: str, reduction: str) -> None:
    rows, vocab, dim = shape
    x, w, y = layer(rows, vocab, dim, DTYPES[dtype])
    y[integers(0, 100, (rows,), 9) < 20] = -100  # noqa: PLR2004
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = ff.linear_cross_entropy(x, w, y, reduction=reduction)
    g = normal(rows, seed=5) if reduction == "none" else torch.tensor(-1.7, device="cuda")
    dx, dw = torch.autograd.grad(loss, (x, w), g)
    check(oracle.cross_entropy(x.detach(), w.detach(), y, -100, reduction, g), x, w, 1.0, loss, {"dx": dx, "dw": dw}, g, reduction)
    with torch.no_grad():
        assert torch.equal(ff.linear_cross_entropy(x, w, y.int(), reduction=reduction), loss)


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("shape", "top", "tau"), [((1, 10, 64), 1, 1.0), ((65, 1000, 136), 7, 2.0), ((257, 300, 520), 256, 0.7), ((300, 5003, 768), 64, 4.0), ((130, 20011, 72), 33, 1.0)])
def test_distillation(shape: tuple[int, int, int], top: int, tau: float, dtype: str, reduction: str) -> None:
    rows, vocab, dim = shape
    x, w, y = layer(rows, vocab, dim, DTYPES[dtype])
    ids = integers(0, vocab, (rows, top), 6)  # the same token twice among them
    ids[:, 0] = y
    ids[integers(0, 100, (rows, top), 7) < 20] = -1  # noqa: PLR2004
    ids[integers(0, 100, (rows,), 8) < 10] = -5  # noqa: PLR2004
    teacher = normal(rows, top, seed=4, scale=3.0)
    teacher[integers(0, 100, (rows, top), 10) < 5] = -1e4  # noqa: PLR2004
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = ff.linear_distillation(x, w, ids, teacher, temperature=tau, reduction=reduction)
    g = normal(rows, seed=5) if reduction == "none" else torch.tensor(0.3, device="cuda")
    dx, dw = torch.autograd.grad(loss, (x, w), g)
    r = oracle.distillation(x.detach(), w.detach(), ids, teacher, tau, reduction, g)
    check(r, x, w, tau, loss, {"dx": dx, "dw": dw}, g, reduction)
    with torch.no_grad():
        order = torch.rand(rows, top, device="cuda").argsort(1)  # entries in another order: the same sums but for their order
        other = ff.linear_distillation(x, w, ids.gather(1, order).int(), teacher.gather(1, order), temperature=tau, reduction=reduction)
        check(r, x, w, tau, other, {}, None, reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("shape", "top"), [((1, 10, 64), 0), ((40, 300, 72), 5), ((64, 1000, 2056), 0), ((130, 20011, 72), 3), ((300, 1000, 768), 0), ((257, 777, 1096), 20), ((2048, 70001, 64), 0)])
def test_a_bias(shape: tuple[int, int, int], top: int, dtype: str) -> None:
    rows, vocab, dim = shape
    x, w, y = layer(rows, vocab, dim, DTYPES[dtype])
    bias = normal(vocab, dtype=DTYPES[dtype], seed=11)
    y[::5] = -100
    leaves = [t.detach().requires_grad_(True) for t in (x, w, bias)]
    if top:
        ids, teacher = integers(0, vocab, (rows, top), 6), normal(rows, top, seed=4)
        ids[::5] = -1
        call = lambda a, b, c: ff.linear_distillation(a, b, ids, teacher, bias=c, temperature=2.0)  # noqa: E731
    else:
        call = lambda a, b, c: ff.linear_cross_entropy(a, b, y, bias=c)  # noqa: E731
    g = torch.tensor(1.5, device="cuda")
    tau = 2.0 if top else 1.0
    r = oracle.distillation(x, w, ids, teacher, 2.0, "mean", g, bias) if top else oracle.cross_entropy(x, w, y, -100, "mean", g, bias)
    loss = call(*leaves)
    grads = dict(zip(("dx", "dw", "db"), torch.autograd.grad(loss, leaves, g), strict=True))
    check(r, x, w, tau, loss, grads, g, "mean", bias)
    odd = torch.cat((bias[:1], bias))[1:].requires_grad_(True)  # two bytes off: copied; and its gradient alone
    loss = call(x, w, odd)
    check(r, x, w, tau, loss, {"db": torch.autograd.grad(loss, odd, g)[0]}, g, "mean", bias)
    same = call(*leaves)
    again = torch.autograd.grad(same, leaves[2], g)[0]
    assert torch.equal(again, grads["db"])
    with torch.no_grad():
        assert torch.equal(call(*leaves), loss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [0.0, 0.5, 0.99, 1.0])
@pytest.mark.parametrize("shape", [(2500, 40, 72), (8191, 10, 32), (4097, 300, 264), (9000, 100, 1032), (700, 2, 8)])
def test_small_vocabularies(shape: tuple[int, int, int], masked: float, dtype: str) -> None:  # dw in parts, of which there are fewer where few rows count
    rows, vocab, dim = shape
    x, w, y = layer(rows, vocab, dim, DTYPES[dtype])
    y[torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda") < masked] = -100
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    for reduction, g in (("mean", torch.tensor(2.5, device="cuda")), ("none", normal(rows, seed=5))):
        loss = ff.linear_cross_entropy(x, w, y, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (x, w), g, retain_graph=True)
        check(oracle.cross_entropy(x.detach(), w.detach(), y, -100, reduction, g), x, w, 1.0, loss, {"dx": dx, "dw": dw}, g, reduction)
        again = torch.autograd.grad(loss, (x, w), g)
        assert torch.equal(again[0], dx)
        assert torch.equal(again[1], dw)
        alone = ff.linear_cross_entropy(x.detach(), w, y, reduction=reduction)
        (dw,) = torch.autograd.grad(alone, w, g)
        check(oracle.cross_entropy(x.detach(), w.detach(), y, -100, reduction, g), x, w, 1.0, alone, {"dw": dw}, g, reduction)


@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("masked", [0.0, 0.3, 0.999, 1.0])
@pytest.mark.parametrize("shape", [(16385, 19, 64), (40001, 700, 32), (20000, 10001, 16)])
def test_many_rows(shape: tuple[int, int, int], masked: float, reduction: str) -> None:
    rows, vocab, dim = shape
    x, w, y = layer(rows, vocab, dim, torch.bfloat16)
    y[torch.rand(rows, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda") < masked] = -100
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    g = normal(rows, seed=5) if reduction == "none" else torch.tensor(2.5, device="cuda")
    loss = ff.linear_cross_entropy(x, w, y, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (x, w), g)
    check(oracle.cross_entropy(x.detach(), w.detach(), y, -100, reduction, g), x, w, 1.0, loss, {"dx": dx, "dw": dw}, g, reduction)
    ids = torch.where(y < 0, -1, y)[:, None]
    one = ff.linear_distillation(x, w, ids, torch.zeros(rows, 1, device="cuda"), reduction=reduction)
    assert torch.equal(one, loss)
    two, teacher = torch.cat((ids, -torch.ones_like(ids)), 1), torch.zeros(rows, 2, device="cuda")
    other = ff.linear_distillation(x, w, two, teacher, reduction=reduction)
    check(oracle.distillation(x.detach(), w.detach(), two, teacher, 1.0, reduction), x, w, 1.0, other, {}, None, reduction)


def test_one_entry_is_cross_entropy() -> None:
    x, w, y = layer(200, 900, 128, torch.bfloat16)
    a = ff.linear_distillation(x, w, y[:, None], normal(200, 1, seed=3), reduction="none")
    assert torch.equal(a, ff.linear_cross_entropy(x, w, y, reduction="none"))


@pytest.mark.parametrize("teacher_type", [torch.float16, torch.bfloat16, torch.float32])
def test_teachers_of_every_type_and_stride(teacher_type: torch.dtype) -> None:
    x, w, _ = layer(70, 500, 64, torch.float16)
    ids, teacher = integers(0, 500, (70, 40), 1), normal(70, 40, dtype=teacher_type, seed=2)
    want = ff.linear_distillation(x, w, ids[:, :20].contiguous(), teacher[:, :20].contiguous(), reduction="none")
    assert torch.equal(ff.linear_distillation(x, w, ids[:, :20], teacher[:, :20], reduction="none"), want)
    assert torch.equal(ff.linear_distillation(x, w, ids.t().contiguous().t()[:, :20], teacher.t().contiguous().t()[:, :20], reduction="none"), want)
    r = oracle.distillation(x, w, ids[:, :20], teacher[:, :20], 1.0, "none")
    check(r, x, w, 1.0, want, {}, None, "none")


@pytest.mark.parametrize("rows", [3, 300])
def test_small_losses_keep_their_digits(rows: int) -> None:
    """Logits of a single product are exact. The target's is the largest, of about 100, the others lie 4 to 20 below: losses of 1e-3 to 0.2. What is left is
    fp32's error of a sum of about 1 (8 u: each half tile's, their sum's, the logarithm's), 2^-21 of the other terms (exponential and sums), and log2(e)'s
    rounding, u of the distances that the terms have."""
    x = torch.zeros(rows, 64, dtype=torch.bfloat16, device="cuda")
    x[:, 0] = 8.0
    w = torch.zeros(1000, 64, dtype=torch.bfloat16, device="cuda")
    w[:, 0] = 10.0 + 1.5 * torch.rand(1000, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    y = torch.zeros(rows, dtype=torch.int64, device="cuda")
    w[0, 0] = 12.5
    r = oracle.cross_entropy(x, w, y, -100, "none")
    assert 1e-3 < float(r.rows.min()) < 0.2  # noqa: PLR2004
    z = x.double() @ w.double().T
    others = r.q[:, 1:].sum(1)
    bound = 8 * F32 + 2.0**-21 * others + F32 * (r.q * (z - z[:, :1]).abs()).sum(1) + F32 * r.rows
    near(ff.linear_cross_entropy(x, w, y, reduction="none"), r.rows, bound, "loss")


def test_large_weights_of_the_vocabulary_in_several_pieces() -> None:
    """More columns than a piece holds, and a last piece that is nearly empty: dx is the sum of all pieces."""
    rows, vocab, dim = 4096, 32768 + 8 + 32768, 64
    x, w, y = layer(rows, vocab, dim, torch.bfloat16)
    y[::3] = -100
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = ff.linear_cross_entropy(x, w, y)
    dx, dw = torch.autograd.grad(loss, (x, w))
    g = torch.ones((), device="cuda")
    check(oracle.cross_entropy(x.detach(), w.detach(), y, -100, "mean", g), x, w, 1.0, loss, {"dx": dx, "dw": dw}, g, "mean")


@pytest.mark.parametrize("frozen", ["x", "w"])
def test_a_frozen_operand(frozen: str) -> None:
    x, w, y = layer(300, 3000, 256, torch.float16)
    y[:40] = -100
    leaf = (w if frozen == "x" else x).requires_grad_(True)
    loss = ff.linear_cross_entropy(x, w, y, reduction="sum")
    (got,) = torch.autograd.grad(loss, leaf)
    g = torch.ones((), device="cuda")
    check(oracle.cross_entropy(x.detach(), w.detach(), y, -100, "sum", g), x, w, 1.0, loss, {"dw" if frozen == "x" else "dx": got}, g, "sum")


def test_what_rows_that_do_not_count_hold_is_not_looked_at() -> None:
    x, w, y = layer(300, 700, 128, torch.bfloat16)
    out = integers(0, 100, (300,), 3) < 30  # noqa: PLR2004
    y[out] = -100
    results = []
    for filling in (0.0, float("nan"), float("inf")):
        leaf, weight = x.masked_fill(out[:, None], filling).requires_grad_(True), w.detach().requires_grad_(True)
        loss = ff.linear_cross_entropy(leaf, weight, y)
        dx, dw = torch.autograd.grad(loss, (leaf, weight))
        assert not dx[out].any()
        results.append((loss, dx, dw))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(other, results[0], strict=True))
    g = torch.ones((), device="cuda")
    loss, dx, dw = results[0]
    check(oracle.cross_entropy(x, w.detach(), y, -100, "mean", g), x, w, 1.0, loss, {"dx": dx, "dw": dw}, g, "mean")


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_no_row_counts(reduction: str) -> None:
    x, w, _ = layer(100, 300, 64, torch.float16)
    x, w = x.fill_(float("nan")).requires_grad_(True), w.requires_grad_(True)
    for loss in (
        ff.linear_cross_entropy(x, w, torch.full((100,), 7, device="cuda"), ignore_index=7, reduction=reduction),
        ff.linear_distillation(x, w, torch.full((100, 3), -1, device="cuda"), torch.zeros(100, 3, device="cuda"), reduction=reduction),
    ):
        assert not loss.any()
        dx, dw = torch.autograd.grad(loss, (x, w), torch.ones_like(loss))
        assert not dx.any()
        assert not dw.any()
    assert ff.linear_cross_entropy(x[:0].detach(), w.detach(), torch.empty(0, dtype=torch.int64, device="cuda"), reduction=reduction).sum() == 0


@pytest.mark.parametrize("kind", ["cross entropy", "distillation"])
def test_a_token_past_the_vocabulary_reports_and_makes_nan_of_its_row(kind: str) -> None:
    x, w, y = layer(100, 300, 64, torch.bfloat16)
    x = x.requires_grad_(True)
    if kind == "cross entropy":
        bad = y.clone()
        bad[17], bad[50], bad[99] = 300, 2**40, -3
        good = torch.tensor([i not in (17, 50, 99) for i in range(100)], device="cuda")
        losses = [ff.linear_cross_entropy(x, w, t, reduction="none") for t in (y, bad)]
    else:
        ids, teacher = integers(0, 300, (100, 5), 2), normal(100, 5)
        bad = ids.clone()
        bad[17, 2], bad[50, 0], bad[99, 4] = 300, 2**40, 2**31 - 1
        good = torch.tensor([i not in (17, 50, 99) for i in range(100)], device="cuda")
        losses = [ff.linear_distillation(x, w, t, teacher, reduction="none") for t in (ids, bad)]
    grads = [torch.autograd.grad(loss, x, torch.ones_like(loss))[0] for loss in losses]
    assert torch.equal(losses[0][good], losses[1][good])
    assert bool(losses[1][~good].isnan().all())
    assert torch.equal(grads[0][good], grads[1][good])
    assert bool(grads[1][~good].isnan().all())


def test_teachers_with_infinities() -> None:
    x, w, _ = layer(8, 300, 64, torch.bfloat16)
    ids, teacher = integers(0, 300, (8, 6), 2), normal(8, 6)
    inf = float("inf")
    teacher[0, 1:], teacher[1], teacher[2, 3], teacher[3, 3] = -inf, -inf, inf, float("nan")
    teacher[4, 2], ids[4, 2] = float("nan"), -1  # not an entry
    ids[5], ids[6, 1:] = -1, -1
    loss = ff.linear_distillation(x, w, ids, teacher, reduction="none")
    assert loss.isnan().tolist() == [False, True, True, True, False, False, False, False]
    assert float(loss[5]) == 0.0
    assert torch.equal(loss[[0, 6]], ff.linear_cross_entropy(x, w, ids[:, 0].clamp(min=0), reduction="none")[[0, 6]])


def test_any_shape_stride_and_alignment() -> None:
    x, w, y = layer(60, 500, 96, torch.float16)
    want = ff.linear_cross_entropy(x, w, y, reduction="none")
    wide = torch.zeros(60, 3, 112, dtype=torch.float16, device="cuda")
    wide[:, 1, 8:104] = x
    odd = torch.zeros(60 * 96 + 1, dtype=torch.float16, device="cuda")[1:].view(60, 96).copy_(x)
    weights = torch.zeros(500, 104, dtype=torch.float16, device="cuda")
    weights[:, :96] = w
    for leaf in (wide[:, 1, 8:104], odd, x.t().contiguous().t(), x.view(3, 20, 96), x.view(3, 20, 96).transpose(0, 1)):
        for weight in (w, weights[:, :96]):
            t = y.view(3, 20) if leaf.dim() == 3 else y  # noqa: PLR2004
            t = t.t() if leaf.shape[0] == 20 else t  # noqa: PLR2004
            a, b = leaf.detach().requires_grad_(True), weight.detach().requires_grad_(True)
            loss = ff.linear_cross_entropy(a, b, t, reduction="none")
            assert torch.equal(loss.t().reshape(-1) if leaf.shape[0] == 20 else loss.reshape(-1), want)  # noqa: PLR2004
            g = torch.ones(1, device="cuda").expand(loss.shape)  # of stride zero
            dx, dw = torch.autograd.grad(loss, (a, b), g)
            r = oracle.cross_entropy(x, w, y, -100, "none", torch.ones(60, device="cuda"))
            dx = (dx.transpose(0, 1) if leaf.shape[0] == 20 else dx).reshape(60, 96)  # noqa: PLR2004
            check(r, x, w, 1.0, want, {"dx": dx, "dw": dw}, torch.ones(60, device="cuda"), "none")


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e25])
def test_row_gradients_of_any_size(size: float) -> None:
    x, w, y = layer(100, 400, 64, torch.float16)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    g = normal(100, seed=5) * size
    g[::7] = 0
    dx, dw = torch.autograd.grad(ff.linear_cross_entropy(x, w, y, reduction="none"), (x, w), g)
    r = oracle.cross_entropy(x.detach(), w.detach(), y, -100, "none", g)
    if size < 1:
        check(r, x, w, 1.0, r.loss.float(), {"dx": dx, "dw": dw}, g, "none")
    else:  # past fp16's range: infinite, not wrong
        assert bool((dx.isinf() | (r.dx.abs() < 65520)).all())  # noqa: PLR2004
    dx, _ = torch.autograd.grad(ff.linear_cross_entropy(x, w, y, reduction="none"), (x, w), torch.zeros(100, device="cuda"))
    assert not dx.any()


def test_gradients_agree_with_differences() -> None:
    x, w, y = layer(40, 200, 64, torch.bfloat16)
    ids, teacher = integers(0, 200, (40, 5), 3), normal(40, 5)
    calls = (lambda a, b: ff.linear_cross_entropy(a, b, y), lambda a, b: ff.linear_distillation(a, b, ids, teacher, temperature=2.0))
    for call in calls:
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        grads = torch.autograd.grad(call(a, b), (a, b))
        for i, grad in enumerate(grads):
            # steps that bfloat16 holds exactly: to the neighbour of each value, up and down by the same
            leaf = (x, w)[i]
            exponent = torch.frexp(leaf.float())[1]
            step = torch.ldexp(torch.ones_like(leaf, dtype=torch.float32), exponent - 5) * torch.sign(normal(*leaf.shape, seed=30 + i))
            step = torch.where(grad.float() * step > 0, step, -step)  # all uphill
            up, down = (leaf.float() + s * step for s in (1, -1))
            up, down = up.bfloat16(), down.bfloat16()
            ends = [float(call(*((t, w) if i == 0 else (x, t)))) for t in (up, down)]
            along = (up.double() - down.double()) / 2
            want = float((grad.double() * along).sum())
            # third order: steps are a sixteenth of the values; the gradient's own rounding of 2^-8 of each term
            assert abs((ends[0] - ends[1]) / 2 - want) < 0.05 * abs(want), (i, ends, want)


def test_the_gradients_may_be_asked_for_twice_and_from_another_thread() -> None:
    x, w, y = layer(500, 2000, 128, torch.bfloat16)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    loss = ff.linear_cross_entropy(x, w, y)
    first = torch.autograd.grad(loss, (x, w), retain_graph=True)
    got: list = []
    thread = threading.Thread(target=lambda: got.extend(torch.autograd.grad(loss, (x, w), retain_graph=True)))
    thread.start()
    thread.join()
    assert all(torch.equal(a, b) for a, b in zip(got, first, strict=True))
    with pytest.raises(RuntimeError):
        dx = torch.autograd.grad(loss, x, create_graph=True)[0]
        torch.autograd.grad(dx.float().sum(), x)


def test_gradients_are_the_first_thing_that_autograds_thread_does() -> None:
    """Autograd runs them in a thread of its own, which has no context until it makes a CUDA call: a process whose first gradients these are."""
    code = """
import torch, fastforks_b200 as ff
x, w = (torch.randn(n, 64, device="cuda").half().requires_grad_(True) for n in (300, 500))
loss = ff.linear_cross_entropy(x, w, torch.zeros(300, dtype=torch.int64, device="cuda"))
assert all(g.isfinite().all() for g in torch.autograd.grad(loss, (x, w)))
assert ff.device_status() == 0
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parent.parent, capture_output=True, text=True, timeout=300, check=False)
    assert done.returncode == 0, done.stderr


def test_a_single_row_without_a_batch() -> None:
    x, w, y = layer(1, 50, 64, torch.bfloat16)
    for reduction in ("none", "sum", "mean"):
        for way in range(2):
            leaf = x[0].detach().requires_grad_(True)
            if way:  # two bytes off: copied
                leaf = torch.cat((x[0, :1], x[0]))[1:].detach().requires_grad_(True)
            loss = ff.linear_cross_entropy(leaf, w, y[0], reduction=reduction)
            assert loss.shape == ()
            (dx,) = torch.autograd.grad(loss, leaf)
            g = torch.ones(1, device="cuda")
            r = oracle.cross_entropy(x, w, y, -100, "none", g)
            check(r, x, w, 1.0, loss.reshape(1), {"dx": dx.reshape(1, 64)}, g, "none")


def test_rows_whose_offsets_pass_32_bits() -> None:
    if torch.cuda.mem_get_info()[0] < 6 * 2**30:
        pytest.skip("no room")
    x, w, y = layer(70, 300, 64, torch.float16)
    stride = 2**25 + 8
    far = torch.zeros(70 * stride, dtype=torch.float16, device="cuda").as_strided((70, 64), (stride, 1))
    far.copy_(x)
    y[::4] = -100
    assert torch.equal(ff.linear_cross_entropy(far, w, y, reduction="none"), ff.linear_cross_entropy(x, w, y, reduction="none"))


def test_a_stream_and_two_graphs_at_once() -> None:
    hidden, weight, y = layer(600, 3000, 256, torch.bfloat16)
    ids, teacher = integers(0, 3000, (600, 20), 3), normal(600, 20)

    def step() -> tuple[torch.Tensor, ...]:
        x, w = (t.detach().requires_grad_(True) for t in (hidden, weight))  # of the stream that the step runs on
        a, b = ff.linear_cross_entropy(x, w, y), ff.linear_distillation(x, w, ids, teacher, temperature=2.0)
        return (a, b, *torch.autograd.grad(a, (x, w)), *torch.autograd.grad(b, (x, w)))

    want = [t.detach().clone() for t in step()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, c) for a, c in zip(got, want, strict=True))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out, torch.cuda.Stream()))
    y[::2] = -100  # the graphs follow what the tensors hold
    want = [t.detach().clone() for t in step()]
    torch.cuda.synchronize()
    for _ in range(4):
        for graph, _, s in graphs:
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, _ in graphs:
        assert all(torch.equal(a.detach(), c) for a, c in zip(out, want, strict=True))


def test_a_training_step_of_norm_and_both_losses() -> None:
    """As they are used: rows normed, both losses of one output layer, gradients of everything at once, against 64 bits with the roundings between
    them: the normed rows and their gradients, each loss's gradients and their sum, all to bfloat16."""
    rows, dim, vocab = 300, 256, 1500
    h, dy_seed = normal(rows, dim, dtype=torch.bfloat16, scale=2.0), 3
    nw, nb = (normal(dim, seed=i, scale=0.2).add(i == 1).bfloat16() for i in (1, 2))
    w = normal(vocab, dim, dtype=torch.bfloat16, seed=dy_seed, scale=1.5 / 16)
    y, ids, teacher = integers(0, vocab, (rows,), 4), integers(0, vocab, (rows, 10), 5), normal(rows, 10, seed=6)
    y[:30] = -100
    leaves = [t.detach().requires_grad_(True) for t in (h, nw, nb, w)]
    x = ff.layer_norm(*leaves[:3])
    loss = ff.linear_cross_entropy(x, leaves[3], y) + 0.5 * ff.linear_distillation(x, leaves[3], ids, teacher, temperature=2.0)
    got = torch.autograd.grad(loss, leaves)
    exact = [t.double().requires_grad_(True) for t in (h, nw, nb, w)]
    x64 = torch.nn.functional.layer_norm(exact[0], (dim,), exact[1], exact[2], 1e-5)
    x64 = x64 + (x.detach().double() - x64).detach()  # the rounded rows
    logits = x64 @ exact[3].T
    ce = torch.nn.functional.cross_entropy(logits, y)
    p, logq = torch.softmax(teacher.double() / 2, 1), torch.log_softmax(logits / 2, 1)
    kd = 4 * (p * (p.log() - logq.gather(1, ids))).sum(1).mean()
    want = torch.autograd.grad(ce + 0.5 * kd, exact)
    assert abs(float(loss.detach()) - float((ce + 0.5 * kd).detach())) < 1e-4  # noqa: PLR2004
    for name, a, b in zip(("h", "norm weight", "norm bias", "weight"), got, want, strict=True):
        # a rounding to bfloat16 is off by 2^-8 / sqrt(3) of a value at most, in the mean; up to five of them follow one another, none helps another
        assert float((a.double() - b).norm() / b.norm()) < 5**0.5 * 2.0**-8 / 3**0.5, name
