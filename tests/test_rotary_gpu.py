"""`rotary` and `qk_norm_rotary` on a B200 against their definitions in 64 bits, forward and gradients.

Tolerances: results are rounded once from fp32, so an element may be off by half a unit in the last place of its type (U, relative to
it) plus the fp32 error of what went into it. A rotation has three roundings of terms |a| + |b|; the norm's factor adds those of a
sum of squares (a chain of 16 products in a lane, 5 shuffles) and of rsqrt (2 units): 32 * 2^-24 covers both. The sum over tokens behind
a weight's gradient runs through chains of at most 64 + 4 * 75 additions at these sizes: 400 * 2^-24 of the sum of magnitudes.
"""

from __future__ import annotations

import pytest
import torch

import fastforks_b200 as ff
from oracle import decoder_oracle as do

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-133, torch.float32: 2.0**-149}
F32 = 2.0**-24


@pytest.fixture(autouse=True)
def _kernels_ran_to_the_end(request: pytest.FixtureRequest):  # noqa: ANN202
    yield
    assert ff.device_status() == (0 if "reports" not in request.node.name else 1 << 20)


def normal(*shape: int, dtype: torch.dtype, seed: int = 0, scale: float = 1.0) -> torch.Tensor:
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def pair_size(x: torch.Tensor, half: int, *, interleaved: bool) -> torch.Tensor:
    """|a| + |b| at both places of each pair, |x| elsewhere."""
    m = x.double().abs()
    if half == 0:
        return m
    head = m[..., : 2 * half].unflatten(-1, (half, 2) if interleaved else (2, half))
    s = head.sum(-1 if interleaved else -2, keepdim=True).expand_as(head).flatten(-2)
    return torch.cat((s, m[..., 2 * half :]), -1)


def close(got: torch.Tensor, ref: torch.Tensor, size: torch.Tensor | float, units: float, what: str = "") -> None:
    bound = U[got.dtype] * ref.abs() + units * F32 * size + TINY[got.dtype]
    bad = (got.double() - ref).abs() > bound
    assert got.shape == ref.shape
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double() - ref).abs() / bound).max()):.2f} bounds"


SHAPES = [
    # batch, tokens, heads, dim, rot
    (1, 1, 1, 64, 64), (3, 1, 32, 128, 128), (2, 37, 5, 128, 64), (1, 257, 3, 256, 256), (2, 9, 4, 96, 96), (2, 9, 4, 80, 32),
    (1, 33, 2, 72, 72), (2, 17, 3, 64, 22), (1, 5, 2, 40, 6), (1, 3, 7, 2, 2), (1, 4, 1, 9, 8), (1, 3, 2, 512, 512), (1, 3, 2, 300, 128),
]  # fmt: skip


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary(shape: tuple[int, ...], dtype: str, interleaved: bool) -> None:
    b, n, h, d, rot = shape
    x = normal(b, n, h, d, dtype=DTYPES[dtype], seed=n).requires_grad_(True)
    table = ff.rotary_table(300, rot, device="cuda")
    positions = torch.randint(-1, 300, (b, n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).int()
    y = ff.rotary(x, table, positions, interleaved=interleaved)
    close(y, do.rotate(x.detach(), table, positions, interleaved=interleaved), pair_size(x.detach(), rot // 2, interleaved=interleaved), 3)
    g = normal(b, n, h, d, dtype=DTYPES[dtype], seed=7)
    (dx,) = torch.autograd.grad(y, x, g)
    close(dx, do.rotate(g, table, positions, interleaved=interleaved, back=True), pair_size(g, rot // 2, interleaved=interleaved), 3)
    with torch.no_grad():
        assert torch.equal(ff.rotary(x, table, positions, interleaved=interleaved), y)
        kept = x.detach().clone()
        same = ff.rotary(kept, table, positions, interleaved=interleaved, out=kept)
        assert same is kept
        assert torch.equal(kept, y)


def test_rotary_takes_row_i_by_default_and_positions_of_either_shape() -> None:
    x, table = normal(2, 7, 3, 64, dtype=torch.bfloat16), ff.rotary_table(7, 64, device="cuda")
    y = ff.rotary(x, table)
    at = torch.arange(7, device="cuda")
    assert torch.equal(y, ff.rotary(x, table, at))
    assert torch.equal(y, ff.rotary(x, table, at.int().expand(2, 7)))
    assert torch.equal(y, ff.rotary(x, table, at.int()[None].repeat(2, 2)[:, ::1][:, :7]))
    close(y, do.rotate(x, table, None, interleaved=False), pair_size(x, 32, interleaved=False), 3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_strides(dtype: str) -> None:
    """Views: of a packed tensor, heads in front of tokens, one element past an aligned address, a gradient that is broadcast."""
    t = DTYPES[dtype]
    table = ff.rotary_table(11, 64, device="cuda")
    packed = normal(2, 11, 3, 4, 64, dtype=t)
    heads_first = normal(2, 4, 11, 64, dtype=t).transpose(1, 2)
    shifted = normal(2 * 11 * 4 * 64 + 1, dtype=t)[1:].view(2, 11, 4, 64)
    narrow = normal(2, 11, 4, 67, dtype=t)[..., 1:65]
    for x in (packed[:, :, 1], heads_first, shifted, narrow, packed[:, ::2, 2].repeat(1, 2, 1, 1)[:, :11], packed[:1, :1, 0].expand(2, 11, 4, 64)):
        for interleaved in (False, True):
            close(ff.rotary(x, table, interleaved=interleaved), do.rotate(x, table, None, interleaved=interleaved), pair_size(x, 32, interleaved=interleaved), 3)
    x = heads_first.detach().requires_grad_(True)
    ff.rotary(x, table).sum().backward()
    g = torch.ones_like(x)
    close(x.grad, do.rotate(g, table, None, interleaved=False, back=True), pair_size(g, 32, interleaved=False), 3)


def test_rotary_reports_a_position_past_the_table() -> None:
    x, table = normal(1, 4, 2, 64, dtype=torch.float16), ff.rotary_table(3, 64, device="cuda")
    at = torch.tensor([0, 2, 3, 2**31 - 1], device="cuda", dtype=torch.int32)
    y = ff.rotary(x, table, at)
    assert torch.equal(y[:, 2:], x[:, 2:])
    close(y, do.rotate(x, table, at, interleaved=False), pair_size(x, 32, interleaved=False), 3)


def test_rotary_of_nothing() -> None:
    table = ff.rotary_table(4, 64, device="cuda")
    assert ff.rotary(torch.empty(0, 4, 2, 64, device="cuda"), table).shape == (0, 4, 2, 64)
    assert ff.rotary(torch.empty(2, 0, 2, 64, device="cuda"), table).shape == (2, 0, 2, 64)


NORM_SHAPES = [
    # batch, tokens, q heads, kv heads, dim, rot
    (1, 1, 1, 1, 64, 64), (4, 1, 32, 8, 128, 128), (2, 37, 6, 6, 64, 64), (2, 61, 5, 1, 128, 64), (1, 19, 4, 2, 96, 40), (1, 23, 3, 2, 72, 72),
    (1, 3, 2, 1, 10, 0), (1, 5, 1, 1, 512, 256), (3, 300, 8, 2, 128, 128),
]  # fmt: skip


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weights", ["alike", "fp32", "none"])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_norm_rotary(shape: tuple[int, ...], weights: str, dtype: str, interleaved: bool) -> None:
    b, n, hq, hk, d, rot = shape
    t, eps = DTYPES[dtype], 1e-5
    q, k = normal(b, n, hq, d, dtype=t, seed=1).requires_grad_(True), normal(b, n, hk, d, dtype=t, seed=2, scale=3).requires_grad_(True)
    w = [None, None] if weights == "none" else [(1 + 0.3 * normal(d, dtype=torch.float32, seed=s)).to(t if weights == "alike" else torch.float32).requires_grad_(True) for s in (3, 4)]
    table = ff.rotary_table(n + 3, rot, device="cuda") if rot else None
    positions = torch.arange(n, device="cuda").int() - 1 if rot else None
    got = ff.qk_norm_rotary(q, k, w[0], w[1], table, positions, eps=eps, interleaved=interleaved)
    gs = normal(b, n, hq, d, dtype=t, seed=5), normal(b, n, hk, d, dtype=t, seed=6)
    grads = torch.autograd.grad(got, (q, k, *(x for x in w if x is not None)), gs)
    again = torch.autograd.grad(ff.qk_norm_rotary(q, k, w[0], w[1], table, positions, eps=eps, interleaved=interleaved), (q, k, *(x for x in w if x is not None)), gs)
    assert all(torch.equal(x, y) for x, y in zip(grads, again, strict=True))  # sums are taken in a fixed order
    with torch.no_grad():
        plain = ff.qk_norm_rotary(q, k, w[0], w[1], table, positions, eps=eps, interleaved=interleaved)
    for i, (x, y, g) in enumerate(zip((q, k), got, gs, strict=True)):
        assert torch.equal(plain[i], y)
        xd, wd = x.detach(), None if w[i] is None else w[i].detach()
        h = do.norm_rotate(xd, wd, None, None, eps=eps, interleaved=interleaved)
        close(y, do.norm_rotate(xd, wd, table, positions, eps=eps, interleaved=interleaved), pair_size(h, rot // 2, interleaved=interleaved), 32, "y")
        dx, dw = do.norm_rotate_backward(xd, g, wd, table, positions, eps=eps, interleaved=interleaved)
        r = 1 / torch.sqrt(xd.double().square().mean(-1, keepdim=True) + eps)
        hat, tw = xd.double() * r, pair_size(g, rot // 2, interleaved=interleaved) * (1 if wd is None else wd.double().abs())
        close(grads[i], dx, r * (tw + hat.abs() * (tw * hat.abs()).mean(-1, keepdim=True)), 96, "dx")
        if wd is not None:
            size = (pair_size(g, rot // 2, interleaved=interleaved) * hat.abs()).sum((0, 1, 2))
            close(grads[2 + i], dw, size, 400, "dw")


def test_norm_rotary_gradient_against_differences() -> None:
    """Central differences of the 64-bit definition along random directions: the error of a step of 1e-4 is of order 1e-8."""
    b, n, hq, hk, d, eps = 2, 5, 3, 1, 64, 1e-6
    table = ff.rotary_table(n, 32, device="cuda")
    args = [normal(b, n, hq, d, dtype=torch.float32, seed=1), normal(b, n, hk, d, dtype=torch.float32, seed=2), 1 + 0.2 * normal(d, dtype=torch.float32, seed=3), 1 + 0.2 * normal(d, dtype=torch.float32, seed=4)]
    gs = normal(b, n, hq, d, dtype=torch.float32, seed=5).double(), normal(b, n, hk, d, dtype=torch.float32, seed=6).double()

    def loss(q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor) -> float:
        return float(sum((do.norm_rotate(x, w, table, None, eps=eps, interleaved=True) * g).sum() for x, w, g in ((q, wq, gs[0]), (k, wk, gs[1]))))

    leaves = [x.clone().requires_grad_(True) for x in args]
    out = ff.qk_norm_rotary(*leaves, table, eps=eps, interleaved=True)
    grads = torch.autograd.grad(out, leaves, [g.float() for g in gs])
    for i in range(4):
        way = normal(*args[i].shape, dtype=torch.float32, seed=10 + i).double()
        h = 1e-4
        up, down = ([a.double() + (s * h * way if j == i else 0) for j, a in enumerate(args)] for s in (1, -1))
        slope = (loss(*up) - loss(*down)) / (2 * h)
        along = float((grads[i].double() * way).sum())
        size = float((grads[i].double() * way).abs().sum())
        assert abs(slope - along) <= 1e-6 * size + 1e-6


def test_norm_rotary_of_extreme_heads() -> None:
    """A head of zeros gives zeros (and finite gradients), a large one stays in range, one with an infinity spoils itself alone."""
    table = ff.rotary_table(4, 64, device="cuda")
    q = normal(1, 4, 2, 64, dtype=torch.bfloat16)
    q[0, 0] = 0
    q[0, 1, 0] = 1e18
    q[0, 2, 1, 5] = torch.inf
    q.requires_grad_(True)
    y, _ = ff.qk_norm_rotary(q, q, None, None, table, eps=1e-6)
    assert torch.equal(y[0, 0], torch.zeros_like(y[0, 0]))
    assert y[0, 1].isfinite().all()
    assert not y[0, 2, 1].isfinite().all()
    rest = torch.ones(4, 2, dtype=torch.bool, device="cuda")
    rest[2, 1] = False
    assert y[0][rest].isfinite().all()
    (dq,) = torch.autograd.grad(y, q, torch.ones_like(y))
    assert dq[0][rest].isfinite().all()


def test_norm_rotary_on_another_stream_and_in_a_graph() -> None:
    table = ff.rotary_table(64, 128, device="cuda")
    data = normal(2, 64, 8, 128, dtype=torch.bfloat16, seed=1), normal(2, 64, 2, 128, dtype=torch.bfloat16, seed=2), *torch.ones(2, 128, device="cuda", dtype=torch.bfloat16)
    gs = normal(2, 64, 8, 128, dtype=torch.bfloat16, seed=3), normal(2, 64, 2, 128, dtype=torch.bfloat16, seed=4)

    def step() -> tuple[torch.Tensor, ...]:
        leaves = [t.detach().requires_grad_(True) for t in data]  # of the stream that the step runs on
        out = ff.qk_norm_rotary(*leaves, table)
        return (*out, *torch.autograd.grad(out, leaves, gs))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got, strict=True))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        for t in held:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, held, strict=True))


def test_a_second_derivative_is_refused() -> None:
    table = ff.rotary_table(4, 64, device="cuda")
    x = normal(1, 4, 2, 64, dtype=torch.float32).requires_grad_(True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    for _ in range(2):  # the full way, and the way of repeated calls
        for y in (ff.rotary(x, table), ff.qk_norm_rotary(x, x, w, w, table)[0]):
            (dx,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
            with pytest.raises(RuntimeError, match="once_differentiable"):
                dx.sum().backward()


def test_gradients_of_what_needs_them() -> None:
    """Parts of the inputs alone, an output that is not used, an output that is used twice, and outputs changed in place."""
    table = ff.rotary_table(6, 64, device="cuda")
    q, k, wq, wk = normal(2, 6, 4, 64, dtype=torch.bfloat16, seed=1), normal(2, 6, 2, 64, dtype=torch.bfloat16, seed=2), *torch.ones(2, 64, device="cuda", dtype=torch.bfloat16)
    g = normal(2, 6, 4, 64, dtype=torch.bfloat16, seed=3)
    full = [t.detach().requires_grad_(True) for t in (q, k, wq, wk)]
    want = torch.autograd.grad(ff.qk_norm_rotary(*full, table)[0], full, g, allow_unused=True)
    assert not want[1].any()
    assert not want[3].any()
    for needs in ((0,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(i in needs) for i, t in enumerate((q, k, wq, wk))]
        out = ff.qk_norm_rotary(*leaves, table)[0]
        assert out.requires_grad
        got = torch.autograd.grad(out, [leaves[i] for i in needs], g)
        assert all(torch.equal(a, want[i]) for a, i in zip(got, needs, strict=True))
    x = q.detach().requires_grad_(True)
    y = ff.rotary(x, table)
    (dx,) = torch.autograd.grad(y, x, g, retain_graph=True)
    (twice,) = torch.autograd.grad((y, y), x, (g, g))
    assert torch.equal(twice, 2 * dx)
    z = ff.rotary(x, table)
    z.mul_(2)
    (scaled,) = torch.autograd.grad(z, x, g)
    assert torch.equal(scaled, 2 * dx)
    with torch.no_grad():
        assert not ff.rotary(x, table).requires_grad


def test_refusals_on_the_device() -> None:
    x, table = normal(1, 4, 2, 64, dtype=torch.float16), ff.rotary_table(4, 64, device="cuda")
    w = torch.ones(64, device="cuda", dtype=torch.float16)
    for call, word in [
        (lambda: ff.rotary(x.double(), table), "float16"),
        (lambda: ff.rotary(x[0], table), "batch, tokens"),
        (lambda: ff.rotary(x.transpose(2, 3), table), "last stride"),
        (lambda: ff.rotary(x, table.half()), "table"),
        (lambda: ff.rotary(x[..., :32], table), "table"),
        (lambda: ff.rotary(x, table[:3]), "rows"),
        (lambda: ff.rotary(x, None), "None"),
        (lambda: ff.rotary(x, table, torch.arange(5, device="cuda")), "positions"),
        (lambda: ff.rotary(x, table, torch.arange(4.0, device="cuda")), "positions"),
        (lambda: ff.rotary(x, table, torch.arange(4)), "positions"),
        (lambda: ff.rotary(x, table, out=x[:, :3]), "out"),
        (lambda: ff.rotary(x.clone().requires_grad_(True), table, out=x), "gradient"),
        (lambda: ff.qk_norm_rotary(x, x.float(), w, w, table), "does not go with"),
        (lambda: ff.qk_norm_rotary(x, x, w[:32], w, table), "weights"),
        (lambda: ff.qk_norm_rotary(x, x, w, w.float(), table), "weights"),
        (lambda: ff.qk_norm_rotary(x, x, w, w, table, eps=-1), "eps"),
        (lambda: ff.qk_norm_rotary(x, x, w, w, None, torch.arange(4, device="cuda")), "without a table"),
        (lambda: ff.qk_norm_rotary(x[:, :0], x[:, :0], w, w, table), "empty"),
    ]:
        with pytest.raises(ValueError, match=word):
            call()
