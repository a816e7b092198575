"""Edges of `rotary` and `qk_norm_rotary` on a B200 against their definitions in 64 bits. Tolerances are those of tests/test_rotary_gpu.py."""

from __future__ import annotations

import pytest
import torch

import fastforks_b200 as ff
from oracle import decoder_oracle as do
from test_rotary_gpu import DTYPES, normal, pair_size
from test_rotary_gpu import close as close_where_finite

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _kernels_ran_to_the_end(request: pytest.FixtureRequest):  # noqa: ANN202
    yield
    assert ff.device_status() == (0 if "reports" not in request.node.name else 1 << 20)


def close(got: torch.Tensor, ref: torch.Tensor, *rest: object) -> None:
    """NaN is not close to anything, which a comparison for "too far" does not see."""
    assert got.isfinite().all(), f"{int((~got.isfinite()).sum())} of {got.numel()} not finite"
    close_where_finite(got, ref, *rest)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(3, 5), (6, 6), (7, 1)])
@pytest.mark.parametrize(("dim", "rot"), [(64, 64), (64, 22), (72, 72), (10, 4), (300, 128)])
def test_gradients_without_eps(dim: int, rot: int, heads: tuple[int, int], dtype: str) -> None:
    """With eps = 0 a head of zeros has no norm, but there is none here: places of a CTA that have no head or token count for nothing."""
    b, n, t = 2, 37, DTYPES[dtype]
    x = [normal(b, n, h, dim, dtype=t, seed=s).requires_grad_(True) for s, h in enumerate(heads)]
    w = [(1 + 0.3 * normal(dim, dtype=torch.float32, seed=s)).to(t).requires_grad_(True) for s in (3, 4)]
    g = [normal(b, n, h, dim, dtype=t, seed=5 + s) for s, h in enumerate(heads)]
    table = ff.rotary_table(n, rot, device="cuda")
    grads = torch.autograd.grad(ff.qk_norm_rotary(*x, *w, table, eps=0.0), (*x, *w), g)
    for i in range(2):
        xd, wd = x[i].detach(), w[i].detach()
        dx, dw = do.norm_rotate_backward(xd, g[i], wd, table, None, eps=0.0, interleaved=False)
        r = 1 / torch.sqrt(xd.double().square().mean(-1, keepdim=True))
        hat, turned = xd.double() * r, pair_size(g[i], rot // 2, interleaved=False)
        tw = turned * wd.double().abs()
        close(grads[i], dx, r * (tw + hat.abs() * (tw * hat.abs()).mean(-1, keepdim=True)), 96, "dx")
        close(grads[2 + i], dw, (turned * hat.abs()).sum((0, 1, 2)), 400, "dw")


def test_forward_mode_is_refused() -> None:
    """The kernels have no forward derivative: a tensor that carries a tangent is refused rather than answered without it, also where no
    gradient is recorded, on the full way and on the way of repeated calls. Without a tangent the same calls go on."""
    from torch.autograd import forward_ad

    table = ff.rotary_table(4, 64, device="cuda")
    x, w = normal(1, 4, 2, 64, dtype=torch.float32), torch.ones(64, device="cuda")
    h = x.half()
    cache, pages = ff.kv4_cache(1, 2, 64, page=16), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    lengths = torch.full((1,), 4, dtype=torch.int32, device="cuda")

    def calls(x: torch.Tensor, w: torch.Tensor, h: torch.Tensor) -> list:
        out = torch.empty_like(h)
        return [
            (lambda: ff.rotary(x, table), x),
            (lambda: ff.rotary(x, table, out=torch.empty_like(x)), x),
            (lambda: ff.qk_norm_rotary(x, x.detach(), None, None, table), x),
            (lambda: ff.qk_norm_rotary(w.new_ones(1, 4, 2, 64), w.new_ones(1, 4, 2, 64), w, w, table), w),
            (lambda: ff.kv4_append_(cache, h, h, pages, lengths, table=table), h),
            (lambda: ff.kv4_append_(cache, h.detach(), h.detach(), pages, lengths, table=table, q=h), h),
            (lambda: ff.kv4_attention(h, cache, pages, lengths), h),
            (lambda: ff.kv4_attention(h, cache, pages, lengths, out=out), h),
        ]

    for call, _ in calls(x, w, h):
        call()
    for grad in (False, True):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w, h)]
            for i, (call, _) in enumerate(calls(*dual)):
                with pytest.raises(ValueError, match="forward-mode"):
                    call()
                    pytest.fail(f"call {i} went through")
            for call, _ in calls(x, w, h):
                call()


@pytest.mark.parametrize("norm", [False, True])
def test_a_call_reports_positions_of_64_bits(norm: bool) -> None:
    """int64 positions mean what they say: one past 32 bits is past the table, one far below zero is negative, and neither is turned."""
    x, table = normal(1, 5, 2, 64, dtype=torch.float32), ff.rotary_table(8, 64, device="cuda")
    at = torch.tensor([3, 2**32 + 3, -(2**32) + 3, 2**31, -(2**63)], device="cuda")
    want = torch.tensor([3, -1, -1, -1, -1], device="cuda", dtype=torch.int32)
    if norm:
        w = torch.ones(64, device="cuda")
        got, ref = (ff.qk_norm_rotary(x, x, w, w, table, p)[0] for p in (at, want))
    else:
        got, ref = (ff.rotary(x, table, p) for p in (at, want))
    assert torch.equal(got, ref)
