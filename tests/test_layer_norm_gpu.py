"""`layer_norm` on a B200 against its definition in 64 bits, forward and gradients.

Tolerances. u = 2^-24, U half a step of the result's type. A sum over a row is a chain of at most 32 values in a thread and ten steps of a
tree: 42 u of the sum of magnitudes. With A the mean of |x|: the mean is off by 42 u A, a difference from it by that and u of itself; the variance's
error from the mean is of second order, its own sum 42 u + 3 u; r = 1 / sqrt(..) half of that and 2 u: 25 u. So h is off by E = 42 u A r + 30 u |h|.
The sums over rows run through at most `rows` additions in a thread and 64 more.
"""

from __future__ import annotations

import pytest
import torch

import fastforks_b200 as ff
from oracle import training_oracle as oracle

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-133, torch.float32: 2.0**-149}
F32 = 2.0**-24
EPS = 1e-5


@pytest.fixture(autouse=True)
def _kernels_ran_to_the_end():  # noqa: ANN202
    yield
    assert ff.device_status() == 0


def normal(*shape: int, dtype: torch.dtype, seed: int = 0, scale: float = 1.0) -> torch.Tensor:
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def within(got: torch.Tensor, ref: torch.Tensor, error: torch.Tensor, what: str) -> None:
    assert got.shape == ref.shape, what
    bound = torch.finfo(got.dtype).eps / 2 * (ref.abs() + error) + error + TINY[got.dtype]
    off = (got.double() - ref).abs()
    assert bool((off <= bound).all()), f"{what}: worst {float((off / bound).max()):.2f} bounds"


def check(x: torch.Tensor, w: torch.Tensor | None, b: torch.Tensor | None, y: torch.Tensor, dy: torch.Tensor | None = None, grads: dict | None = None, eps: float = EPS) -> None:
    x, y = (t.detach().reshape(-1, t.shape[-1]) for t in (x, y))
    w, b = (None if t is None else t.detach() for t in (w, b))
    dy = None if dy is None else dy.reshape(x.shape)
    r = oracle.layer_norm(x, w, b, eps, dy)
    aw = 1.0 if w is None else w.double().abs()
    size = x.double().abs().mean(1, keepdim=True)
    e_hat = F32 * (42 * size * r.rstd + 30 * r.hat.abs())
    within(y, r.y, e_hat * aw + 3 * F32 * (r.y.abs() + (r.hat * aw).abs()), "y")
    if grads is None:
        return
    t = dy.double() * (1.0 if w is None else w.double())
    mean_t, mean_th = t.abs().mean(1, keepdim=True), (t * r.hat).abs().mean(1, keepdim=True)
    e_mean_th = 45 * F32 * mean_th + (t.abs() * e_hat).mean(1, keepdim=True)
    e_dx = r.rstd * (4 * F32 * t.abs() + 45 * F32 * mean_t + r.hat.abs() * e_mean_th + e_hat * mean_th + 4 * F32 * (mean_t + r.hat.abs() * mean_th)) + 30 * F32 * r.dx.abs()
    chain = (x.shape[0] + 64) * F32
    if "dx" in grads:
        within(grads["dx"].reshape(x.shape), r.dx, e_dx, "dx")
    if "dw" in grads:
        within(grads["dw"], r.dw, chain * (dy.double() * r.hat).abs().sum(0) + (dy.double().abs() * e_hat).sum(0), "dw")
    if "db" in grads:
        within(grads["db"], r.db, chain * dy.double().abs().sum(0), "db")


SHAPES = [
    (1, 1), (3, 1), (1, 64), (5, 7), (2, 8), (7, 768), (197, 768), (33, 100), (300, 1024), (3, 1025), (129, 384), (40, 513), (64, 2048), (9, 2056), (10, 4096), (6, 4104),
    (5, 8192), (3, 9000), (3, 10001), (2, 16384), (2, 16385), (2, 32768), (1201, 192), (2500, 520),
]  # fmt: skip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape: tuple[int, int], dtype: str) -> None:
    rows, dim = shape
    t = DTYPES[dtype]
    x = (normal(rows, dim, dtype=t, seed=dim) * 2 + normal(dim, dtype=t, seed=1)).requires_grad_(True)
    w, b = (normal(dim, dtype=t, seed=i).add(i == 2).requires_grad_(True) for i in (2, 3))  # noqa: PLR2004
    dy = normal(rows, dim, dtype=t, seed=4)
    y = ff.layer_norm(x, w, b, eps=EPS)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (dx.dtype, dw.dtype, db.dtype) == (t, t, t)
    check(x, w, b, y, dy, {"dx": dx, "dw": dw, "db": db})
    with torch.no_grad():
        assert torch.equal(ff.layer_norm(x, w, b, eps=EPS), y)
        same = x.detach().clone()
        assert ff.layer_norm(same, w, b, eps=EPS, out=same) is same
        assert torch.equal(same, y)


@pytest.mark.parametrize(("rows", "dim"), [(9601, 504), (2401, 776), (4801, 1024), (2401, 2040), (1201, 2056), (1201, 4096), (4801, 2600), (4801, 4096), (1185, 1001), (593, 1901), (601, 2047), (300, 4095), (300, 5001), (20, 8191)])
def test_many_rows(rows: int, dim: int) -> None:  # odd: the last has no other to go with, where rows go two at a time
    x, w, b = normal(rows, dim, dtype=torch.bfloat16, seed=dim), normal(dim, dtype=torch.bfloat16, seed=1), normal(dim, dtype=torch.bfloat16, seed=2)
    y = torch.full((rows + 3, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    ff.layer_norm(x, w, b, eps=EPS, out=y[:rows])
    assert bool((y[rows:] == 7.0).all())  # noqa: PLR2004
    check(x, w, b, y[:rows])
    same = x.clone()
    assert torch.equal(ff.layer_norm(same, w, b, eps=EPS, out=same), y[:rows])


@pytest.mark.parametrize("wanted", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1), (1, 0, 1), (1, 1, 0)])
@pytest.mark.parametrize("dim", [72, 768, 1500])
def test_only_the_gradients_that_are_asked_for(dim: int, wanted: tuple[int, int, int]) -> None:
    leaves = [normal(50, dim, dtype=torch.bfloat16), normal(dim, dtype=torch.bfloat16, seed=1), normal(dim, dtype=torch.bfloat16, seed=2)]
    for t, on in zip(leaves, wanted, strict=True):
        t.requires_grad_(bool(on))
    dy = normal(50, dim, dtype=torch.bfloat16, seed=3)
    y = ff.layer_norm(*leaves, eps=EPS)
    got = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], dy)
    names = [n for n, on in zip(("dx", "dw", "db"), wanted, strict=True) if on]
    check(*leaves, y, dy, dict(zip(names, got, strict=True)))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_weights_in_32_bits_and_without_them(dtype: str) -> None:
    x, dy = normal(37, 640, dtype=DTYPES[dtype]).requires_grad_(True), normal(37, 640, dtype=DTYPES[dtype], seed=1)
    w, b = (normal(640, dtype=torch.float32, seed=i).requires_grad_(True) for i in (2, 3))
    for weight, bias in ((w, b), (w, None), (None, b), (None, None)):
        y = ff.layer_norm(x, weight, bias, eps=EPS)
        leaves = {"dx": x} | ({"dw": weight} if weight is not None else {}) | ({"db": bias} if bias is not None else {})
        got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy), strict=True))
        assert all(t.dtype == torch.float32 for n, t in got.items() if n != "dx")
        check(x, weight, bias, y, dy, got)


def test_strides_and_alignments() -> None:
    base = normal(6, 5, 3, 776, dtype=torch.float16)
    w, b = normal(768, dtype=torch.float16, seed=1), normal(768, dtype=torch.float16, seed=2)
    odd_w = torch.cat((w[:1], w))[1:]  # two bytes off
    for x in (base[..., :768], base[..., 1:769], base[:, :, 1, :768], base[:, :, 1, 3:771], base.permute(2, 1, 0, 3)[..., :768], base[:1, :1, :1, 5:773], base[..., :768].transpose(1, 3)):
        for weight in (w, odd_w) if x.shape[-1] == 768 else (None,):  # noqa: PLR2004
            leaf = x.detach().requires_grad_(True)
            y = ff.layer_norm(leaf, weight, b if weight is not None else None, eps=EPS)
            g = normal(*y.shape[::-1], dtype=torch.float16, seed=5).permute(*range(y.dim())[::-1])  # strides of its own
            (dx,) = torch.autograd.grad(y, leaf, g)
            check(x, weight, b if weight is not None else None, y, g, {"dx": dx})
    row = normal(768, dtype=torch.float16, seed=9).expand(40, 768)  # the same row forty times
    assert torch.equal(ff.layer_norm(row, w, b), ff.layer_norm(row[:1], w, b).expand(40, 768))


def test_rows_without_spread_and_rows_far_from_zero() -> None:
    x = torch.full((4, 1000), 3.0, device="cuda")
    b = normal(1000, dtype=torch.float32)
    y = ff.layer_norm(x, None, b, eps=EPS)
    assert torch.equal(y, b.expand(4, 1000))  # 3 is exact, so are the sums: differences of zero
    x = normal(16, 1000, dtype=torch.float32) + 1000.0
    check(x, None, b, ff.layer_norm(x, None, b, eps=EPS))


def test_nan_and_infinity_stay_in_their_rows() -> None:
    x = normal(9, 520, dtype=torch.bfloat16)
    clean = ff.layer_norm(x)
    x[2, 5], x[6, 0] = float("nan"), float("inf")
    y = ff.layer_norm(x)
    bad = torch.tensor([2, 6], device="cuda")
    assert bool(y[bad].isnan().all())
    keep = [i for i in range(9) if i not in (2, 6)]
    assert torch.equal(y[keep], clean[keep])


def test_no_rows() -> None:
    assert ff.layer_norm(torch.empty(0, 64, device="cuda")).shape == (0, 64)


def test_gradients_agree_with_differences() -> None:
    x, w, b = (normal(*s, dtype=torch.float32, seed=i).requires_grad_(True) for i, s in enumerate(((5, 96), (96,), (96,))))
    dy = normal(5, 96, dtype=torch.float32, seed=7)
    got = torch.autograd.grad(ff.layer_norm(x, w, b), (x, w, b), dy)
    for i, (leaf, grad) in enumerate(zip((x, w, b), got, strict=True)):
        along = normal(*leaf.shape, dtype=torch.float32, seed=20 + i)
        h = 1e-2
        ends = []
        for sign in (1, -1):
            moved = [t.detach() for t in (x, w, b)]
            moved[i] = moved[i] + sign * h * along
            ends.append(float((ff.layer_norm(*moved).double() * dy).sum()))
        # the difference's own error: h^2 / 6 of a third derivative (some ten times the function's size), and 480 roundings of values of about 1
        want = float((grad.double() * along).sum())
        assert abs((ends[0] - ends[1]) / (2 * h) - want) < 10 * h**2 / 6 * float(dy.abs().sum()) + 480 * 4 * F32 / h


def test_another_stream_a_graph_and_twice_the_same_bits() -> None:
    data = [normal(700, 1024, dtype=torch.bfloat16), *(normal(1024, dtype=torch.bfloat16, seed=i) for i in (2, 3))]
    dy = normal(700, 1024, dtype=torch.bfloat16, seed=1)

    def step() -> tuple[torch.Tensor, ...]:
        leaves = [t.detach().requires_grad_(True) for t in data]  # of the stream that the step runs on
        y = ff.layer_norm(*leaves)
        return (y, *torch.autograd.grad(y, leaves, dy))

    want = [t.clone() for t in step()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, c) for a, c in zip(got, want, strict=True))
    graphs = []
    for _ in range(2):  # two graphs at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for (graph, out), s in zip(graphs, streams, strict=True):
            with torch.cuda.stream(s):
                for t in out:
                    t.detach().zero_()
                graph.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a.detach(), c.detach()) for a, c in zip(out, want, strict=True))


def test_more_rows_than_fit_32_bits_of_offset() -> None:
    """Row strides whose products pass 2^31 elements."""
    rows, stride = 70, 2**25 + 8
    if torch.cuda.mem_get_info()[0] < 6 * 2**30:
        pytest.skip("no room")
    base = torch.zeros(rows * stride, dtype=torch.float16, device="cuda")
    x = base.as_strided((rows, 64), (stride, 1))
    x.copy_(normal(rows, 64, dtype=torch.float16))
    assert torch.equal(ff.layer_norm(x), ff.layer_norm(x.contiguous()))


def test_out_that_shares_memory_is_refused() -> None:
    base = normal(20 * 64, dtype=torch.bfloat16)
    x, w, b = base[: 10 * 64].view(10, 64), normal(64, dtype=torch.bfloat16, seed=1), normal(64, dtype=torch.bfloat16, seed=2)
    want = ff.layer_norm(x, w, b)
    before = base.clone()
    for out in (base[64 : 11 * 64], base[1 : 10 * 64 + 1], base[9 * 64 + 63 : 19 * 64 + 63]):
        with pytest.raises(ValueError, match="shares memory"):
            ff.layer_norm(x, w, b, out=out.view(10, 64))
    wide = base.view(10, 128)[:, :64]  # out would lie over its rows
    with pytest.raises(ValueError, match="shares memory"):
        ff.layer_norm(wide, w, b, out=x)
    with pytest.raises(ValueError, match="shares memory"):
        ff.layer_norm(x, base[19 * 64 :], b, out=base[10 * 64 :].view(10, 64))
    assert torch.equal(base, before)
    assert torch.equal(ff.layer_norm(x, w, b, out=base[10 * 64 :].view(10, 64)), want)  # side by side
    assert torch.equal(ff.layer_norm(x, w, b, out=x), want)


@pytest.mark.parametrize(("rows", "dim"), [(4001, 101), (1301, 1001), (2401, 1024), (700, 2600)])
def test_a_chain_in_place_without_waiting(rows: int, dim: int) -> None:
    x, w = normal(rows, dim, dtype=torch.bfloat16), 1 + 0.2 * normal(dim, dtype=torch.bfloat16, seed=1)
    apart = x
    for _ in range(30):
        apart = ff.layer_norm(apart, w)
        torch.cuda.synchronize()
    for _ in range(30):
        ff.layer_norm(x, w, out=x)
    assert torch.equal(x, apart)
