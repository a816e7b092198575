"""Edges of attention over the 4-bit cache, of few rows of a kv head and of many (49 and more go to kernels of their own), against 64 bits.

Tolerance of `check_finite`: that of tests/test_kv4_gpu.py. Tolerance of `check`, for weights that are all alike (powers of two, whose product with
V's step is exact in fp16): the output's own rounding (U |o|); 2^-11 of a weight and never less than 2^-25 of a
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


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("flip", [False, True])
def test_values_of_many_sizes(flip: bool, rows: str) -> None:
    """V of tokens from 2^-12 to 2^12, small first and large first."""
    n, group = ROWS[rows]
    d, tokens = 128, 400
    pages, total = pages_of(1, 7)
    cache = ff.kv4_cache(total, 1, d, page=64)
    size = torch.exp2(torch.linspace(-12, 12, tokens, device="cuda"))
    size = size.flip(0) if flip else size
    k, v = normal(1, tokens, 1, d, dtype=torch.float32, seed=1).bfloat16(), (normal(1, tokens, 1, d, dtype=torch.float32, seed=2) * size[:, None, None]).bfloat16()
    lengths = torch.tensor([tokens], dtype=torch.int32, device="cuda")
    ff.kv4_append_(cache, k, v, pages, lengths)
    q = normal(1, n, group, d, dtype=torch.float32, seed=3).bfloat16()
    check_finite(ff.kv4_attention(q, cache, pages, lengths), q, cache, pages, lengths, d**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("which", ["k", "v"])
def test_nan_and_infinite_tokens(which: str, rows: str, dtype: str) -> None:
    """A token that is held as NaN shows in the queries that see it, all of their output, and changes no bit of the others."""
    d, t = 64, DTYPES[dtype]
    n, group = ROWS[rows]
    tokens = n + 137
    for at in (tokens - 2, tokens - n + 1, 130):  # of the last queries, of all but one, of all
        cache, pages, lengths = fill(1, 2, d, 16, [tokens], seed=5)
        q = normal(1, n, 2 * group, d, dtype=t, seed=3)
        k, v = ff.kv4_read(cache, pages, lengths, tokens, torch.float16)
        ff.kv4_append_(cache, k, v, pages, lengths)
        want = ff.kv4_attention(q, cache, pages, lengths)
        (k if which == "k" else v)[0, at, 1, 9] = math.inf if at % 2 else math.nan
        ff.kv4_append_(cache, k, v, pages, lengths)
        got = ff.kv4_attention(q, cache, pages, lengths)
        sees = torch.zeros(n, 2 * group, dtype=torch.bool, device="cuda")
        sees[max(0, n - tokens + at) :, group:] = True
        assert want.isfinite().all()
        assert got[0][sees].isnan().all()
        # the others' weights and values are what they were; but for powers of two of a step's range, so is their arithmetic
        assert torch.allclose(got[0][~sees].double(), want[0][~sees].double(), rtol=4 * U[t], atol=2.0**-11)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", ROWS)
def test_strides_and_out(rows: str, dtype: str) -> None:
    n, group = ROWS[rows]
    t = DTYPES[dtype]
    cache, pages, lengths = fill(3, 2, 128, 32, [n + 100, 1, 57])
    packed = normal(3, n, 2 * group + 4, 128, dtype=t, seed=3)
    q = packed[:, :, 2 : 2 * group + 2]
    want = ff.kv4_attention(q.contiguous(), cache, pages, lengths)
    check_finite(want, q, cache, pages, lengths, 128**-0.5)
    assert torch.equal(ff.kv4_attention(q, cache, pages, lengths), want)
    assert torch.equal(ff.kv4_attention(q.transpose(1, 2).contiguous().transpose(1, 2), cache, pages, lengths), want)
    wide = torch.zeros(3, n, 2 * group, 160, dtype=t, device="cuda")
    out = wide[..., 16:144]
    assert ff.kv4_attention(q, cache, pages, lengths, out=out) is out
    assert torch.equal(out, want)
    assert not wide[..., :16].any()
    assert not wide[..., 144:].any()
    one = q[:, :, :1].expand_as(q)  # all heads read the same
    assert torch.equal(ff.kv4_attention(one, cache, pages, lengths), ff.kv4_attention(one.contiguous(), cache, pages, lengths))


@pytest.mark.parametrize("rows", ROWS)
def test_a_graph_follows_the_lengths_and_streams_do_not_meet(rows: str) -> None:
    n, group = ROWS[rows]
    b, hk, d, most = 4, 2, 128, 700
    cache, pages, lengths = fill(b, hk, d, 64, [most] * b)
    q = normal(b, n, hk * group, d, dtype=torch.bfloat16, seed=3)
    sets = [[700, 1, 77, 300], [3, 0, 500, 16], [700, 700, 700, 700]]
    want = [ff.kv4_attention(q, cache, pages, torch.tensor(s, dtype=torch.int32, device="cuda")) for s in sets]
    for s, ref in zip(sets, want, strict=True):
        check_finite(ref, q, cache, pages, torch.tensor(s), d**-0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ff.kv4_attention(q, cache, pages, lengths)
    for s, ref in zip(sets * 2, want * 2, strict=True):
        lengths.copy_(torch.tensor(s, dtype=torch.int32))
        graph.replay()
        assert torch.equal(got, ref)
    lengths.fill_(most)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ff.kv4_attention(q, cache, pages, lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[2]) for o in outs)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize(("queries", "lens"), [(70, [3, 0, 70, 69]), (300, [300, 1, 299, 128]), (513, [513, 257, 0, 600])])
def test_whole_prompts_and_padding(queries: int, lens: list[int], dtype: str) -> None:
    """Prompts whose queries are the whole sequence, padded on the left to the longest: rows that see nothing are zeros, whole tiles of them too."""
    cache, pages, lengths = fill(4, 2, 128, 16, lens)
    q = normal(4, queries, 8, 128, dtype=DTYPES[dtype], seed=3)
    check_finite(ff.kv4_attention(q, cache, pages, lengths), q, cache, pages, lengths, 128**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("bad", [-1, "past", 2**31 - 1])
def test_a_page_outside_the_cache_shows_in_the_queries_that_see_it(bad: int | str, rows: str, page: int, dtype: str) -> None:
    """Nothing stands in for such a page, least of all another sequence's tokens: queries that see a place of it get NaN, the others what they
    get without it, and the status says so."""
    d, t = 64, DTYPES[dtype]
    n, group = ROWS[rows]
    tokens = n + 150
    cache, pages, lengths = fill(2, 2, d, page, [tokens, tokens], seed=5)
    q = normal(2, n, 2 * group, d, dtype=t, seed=3)
    want = ff.kv4_attention(q, cache, pages, lengths)
    assert want.isfinite().all()
    for column in (0, 1, (tokens - n // 2) // page, (tokens - 1) // page):
        broken = pages.clone()
        broken[1, column] = cache.shape[0] if bad == "past" else bad
        got = ff.kv4_attention(q, cache, broken, lengths)
        assert ff.device_status() == STATUS_PAGE
        assert torch.equal(got[0], want[0])
        sees = tokens - n + torch.arange(n, device="cuda") >= column * page
        assert got[1][sees].isnan().all()
        assert torch.allclose(got[1][~sees].double(), want[1][~sees].double(), rtol=4 * U[t], atol=2.0**-11)


@pytest.mark.parametrize("rows", ["few", "tile"])
@pytest.mark.parametrize("blocks", [1_875_000, 1_875_001])
def test_blocks_behind_32_bits_of_a_page(blocks: int, rows: str) -> None:
    """One page that holds a whole sequence of thirty million tokens: its last blocks lie more than 2^31 bytes behind its first. All but the
    last tokens are zeros, which weigh exp(0) each beside logits of some 70 at most."""
    d, new = 64, 40
    n, group = ROWS[rows][0], ROWS[rows][1]
    tokens = 16 * blocks
    cache = ff.kv4_cache(1, 1, d, page=tokens)
    pages, lengths = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([tokens], dtype=torch.int32, device="cuda")
    k, v = (4 * normal(1, new, 1, d, dtype=torch.bfloat16, seed=1)), normal(1, new, 1, d, dtype=torch.bfloat16, seed=2)
    ff.kv4_append_(cache, k, v, pages, lengths)
    q = 4 * normal(1, n, group, d, dtype=torch.bfloat16, seed=3)
    got = ff.kv4_attention(q, cache, pages, lengths)
    small = ff.kv4_cache(4, 1, d, page=16)  # the last blocks alone: as many whole ones, with what they hold at the same places
    small[:] = cache[:, :, -4:].transpose(0, 2)
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    held_k, held_v, pairs = held_tokens(small, table, 0, 64)
    logits = torch.einsum("nhd,td->nht", q[0].double(), held_k[0]) * d**-0.5
    at, last = tokens - 64 + torch.arange(64, device="cuda"), tokens - n + torch.arange(n, device="cuda")
    logits = logits.masked_fill(at > last[:, None, None], -math.inf)
    most = logits.amax(-1, keepdim=True).clamp(min=0.0)
    weights = torch.exp(logits - most)
    p = weights / (weights.sum(-1, keepdim=True) + (tokens - 64) * torch.exp(-most))
    o = p @ held_v[0]
    ks, kl, vs, _ = pairs[0].unbind(-1)
    logit = d**-0.5 * q[0].double().abs().sum(-1)[..., None] * (15 * ks + kl.abs()) * 2.0**-18 + 2.0**-21
    if rows == "tile":  # bfloat16 keys go to the tensor cores in fp16
        logit = logit + d**-0.5 * torch.einsum("nhd,td->nht", q[0].double().abs(), 2.0**-11 * (held_k[0].abs() + (kl + 8 * ks).abs()[:, None]) + 2.0**-37 * held_k.abs().max())
    assert float(torch.where(p > 0, logit, 0.0).max()) < 0.5  # noqa: PLR2004
    size = held_v[0].abs() + 15 * vs[:, None]
    bound = U[q.dtype] * o.abs() + torch.einsum("nht,td->nhd", p * (2 * logit + 2.0**-10), size) + (2 * p * logit).sum(-1)[..., None] * o.abs() + 2.0**-20
    assert ((got[0].double() - o).abs() <= bound).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_zeros_of_more_than_32_bits_of_rows(dim: int) -> None:
    """A sequence without tokens in a call whose output has 2^34 values of 16 bits and a few more: all of them are zeros. The queries are one row."""
    heads, queries = 8, 2**34 // (8 * dim) + 3
    cache = ff.kv4_cache(1, heads, dim, page=16)
    pages, lengths = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    q = normal(1, 1, 1, dim, dtype=torch.bfloat16, seed=3).expand(1, queries, heads, dim)
    out = torch.full((1, queries, heads, dim), 1.0, dtype=torch.bfloat16, device="cuda")
    ff.kv4_attention(q, cache, pages, lengths, out=out)
    for part in out.flatten().split(2**30):
        assert not part.any()
    assert ff.device_status() == 0
