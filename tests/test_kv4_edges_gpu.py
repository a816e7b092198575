"""Edges of attention over the 4-bit cache, of few rows of a kv head and of many (49 and more go to kernels of their own), against 64 bits.

Tolerance, element by element: the output's own rounding (U |o|); a weight is rounded to fp16, 2^-11 of it and never less than 2^-25 of a
range that ends at 2^7, times values up to |v| (shared over the keys seen); a logit is off by 2^-18 of the sum of its magnitudes (fp32
sums, an fp16 q of 11 bits that is exact but for values 2^-20 below a row's largest) and an exponential by 2^-21. Where q is bfloat16 and rows are
many, K and V are rounded to fp16 themselves: least + 8 step once and the value once more, 2^-11 of either, and, below 2^-14 of the
range, 2^-25 of it, where V's range ends at the largest value of the sequence (2^-38 of that) and K's at the largest of a step. An error d of a logit
moves the output by at most d times (|v| + |o|), weighed, to first order; 1.25 d stands for the rest as long as d < 0.2.
"""

from __future__ import annotations

import math

import pytest
import torch

import fastforks_b200 as ff
from oracle import decoder_oracle as do
from test_kv4_gpu import DTYPES, STATUS_PAGE, U, check_attention, fill, held_tokens, normal, pages_of

pytestmark = pytest.mark.gpu
# queries and q heads on one kv head: rows for the kernel of few rows, for one tile of 128, for two, and for more
ROWS = {"few": (3, 4), "tile": (20, 4), "two tiles": (50, 4), "more tiles": (75, 4)}


@pytest.fixture(autouse=True)
def _kernels_ran_to_the_end():  # noqa: ANN202
    yield
    assert ff.device_status() == 0


def check(got: torch.Tensor, q: torch.Tensor, cache: torch.Tensor, pages: torch.Tensor, lengths: torch.Tensor, scale: float) -> None:
    hk = cache.shape[1]
    group = q.shape[2] // hk
    rounded = q.dtype == torch.bfloat16 and q.shape[1] * group > 48  # noqa: PLR2004
    for b, length in enumerate(lengths.tolist()):
        if length == 0:
            assert not got[b].any()
            continue
        k, v, pairs = held_tokens(cache, pages, b, length)
        o, p = do.attention(q[b], k, v, scale)
        ks, kl, vs, vl = (x.repeat_interleave(group, 0) for x in pairs.unbind(-1))  # [hq, length]
        ka, va = (x.abs().repeat_interleave(group, 0) for x in (k, v))  # [hq, length, dim]
        qa = q[b].double().abs()  # [n, hq, dim]
        logit = scale * qa.sum(-1)[..., None] * (15 * ks + kl.abs()) * 2.0**-18 + 2.0**-21
        off_v = torch.zeros_like(va)
        if rounded:
            rest = (kl + 8 * ks).abs()
            top = ka.amax(-1).amax(-1)[:, None, None]
            logit = logit + scale * torch.einsum("nhd,htd->nht", qa, 2.0**-11 * (ka + rest[..., None]) + 2.0**-37 * top)
            off_v = 2.0**-11 * (va + (vl + 8 * vs).abs()[..., None]) + 2.0**-37 * va.amax(-1).amax(-1)[:, None, None]
        assert float(torch.where(p > 0, logit, 0.0).max()) < 0.2, "the bound does not hold for such operands"
        moved = torch.einsum("nht,htd->nhd", p * (1.25 * logit + 2.0**-11), va) + (p * 1.25 * logit).sum(-1)[..., None] * o.abs()
        floor = 2.0**-32 * va.amax(1) * length
        bound = U[q.dtype] * o.abs() + moved + torch.einsum("nht,htd->nhd", p, off_v) + floor + 2.0**-25
        bad = ~((got[b].double() - o).abs() <= bound)
        assert not bad.any(), f"sequence {b}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got[b].double() - o).abs() / bound).max()):.2f} bounds"
        assert not got[b, : max(0, q.shape[1] - length)].any()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("zero", ["q and keys", "q", "keys"])
def test_zero_queries_and_keys(zero: str, rows: str, dtype: str, dim: int) -> None:
    """A logit of zero weighs as one, however it came about: the mean of the values that a query sees."""
    n, group = ROWS[rows]
    t, lens = DTYPES[dtype], [n, 300, 130]
    pages, total = pages_of(3, 5)
    cache = ff.kv4_cache(total, 2, dim, page=64)
    k, v = (normal(3, 300, 2, dim, dtype=t, seed=s) for s in (1, 2))
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    ff.kv4_append_(cache, torch.zeros_like(k) if zero != "q" else k, v, pages, lengths)
    q = normal(3, n, 2 * group, dim, dtype=t, seed=3)
    q = q if zero == "keys" else torch.zeros_like(q)
    check(ff.kv4_attention(q, cache, pages, lengths), q, cache, pages, lengths, dim**-0.5)


def check_finite(got: torch.Tensor, q: torch.Tensor, cache: torch.Tensor, pages: torch.Tensor, lengths: torch.Tensor, scale: float) -> None:
    """The tolerance of tests/test_kv4_gpu.py (a weight times V's step is what is rounded), which NaN would pass."""
    assert got.isfinite().all(), f"{int((~got.isfinite()).sum())} of {got.numel()} not finite"
    check_attention(got, q, cache, pages, lengths, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("size", [1e-30, 1e-20, 1e-4, 1.0, 3e3, 1e20, 1e36, 1e37])
def test_sizes_of_q(size: float, rows: str, dtype: str) -> None:
    """Queries of any size their type has, with a scale that brings the logits back."""
    if dtype == "fp16" and not 1e-4 <= size <= 3e3:  # noqa: PLR2004
        pytest.skip("out of fp16's range")
    n, group = ROWS[rows]
    cache, pages, lengths = fill(2, 2, 64, 16, [n + 60, 7])
    q = (normal(2, n, 2 * group, 64, dtype=torch.float32, seed=3) * size).to(DTYPES[dtype])
    scale = 0.125 / size
    check_finite(ff.kv4_attention(q, cache, pages, lengths, scale), q, cache, pages, lengths, scale)


@pytest.mark.parametrize("rows", ROWS)
def test_a_small_scale_on_zero_queries(rows: str) -> None:
    n, group = ROWS[rows]
    cache, pages, lengths = fill(2, 2, 128, 32, [n + 60, 7])
    q = torch.zeros(2, n, 2 * group, 128, dtype=torch.bfloat16, device="cuda")
    check_finite(ff.kv4_attention(q, cache, pages, lengths, 1e-30), q, cache, pages, lengths, 1e-30)
