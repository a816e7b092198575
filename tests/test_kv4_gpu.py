"""The paged 4-bit cache and its attention on a B200 against their definitions.

Writing is elementwise fp32 arithmetic with a fixed order of roundings, so what the cache holds has to be equal to the definition's, and
bytes that belong to no new token have to stay.

Tolerance of attention, element by element against 64 bits on the values that the cache holds: the output's own rounding (U |o|); the
softmax weight times V's step is rounded to fp16 (2^-11 of it, and never less than 2^-25 of the range's 2^7, shared over the keys) and
multiplies codes up to 15; a weight is off by the error of its logit: fp32 sums of dim products of q and codes with an fp16 q of 11
bits or more (exact for 16-bit inputs but for values 2^-20 below a row's largest), 2^-18 of the sum of the magnitudes, and of its
exponential (2^-21).
"""

from __future__ import annotations

import math

import pytest
import torch

import fastforks_b200 as ff
from oracle import decoder_oracle as do

pytestmark = pytest.mark.gpu
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
STATUS_POSITION, STATUS_PAGE = 1 << 20, 1 << 21


@pytest.fixture(autouse=True)
def _kernels_ran_to_the_end():  # noqa: ANN202
    yield
    assert ff.device_status() == 0


def gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(*shape: int, dtype: torch.dtype, seed: int = 0) -> torch.Tensor:
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(dtype)


def pages_of(batch: int, columns: int, seed: int = 0) -> tuple[torch.Tensor, int]:
    """A page table of pages in any order, and how many there are (one is nobody's)."""
    n = batch * columns + 1
    return torch.randperm(n, generator=gen(seed), device="cuda")[: batch * columns].view(batch, columns).int(), n


def held_tokens(cache: torch.Tensor, table: torch.Tensor, b: int, length: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """K, V `[heads, length, dim]` and parameters of a sequence."""
    pages = table[b].long()
    return tuple(x[pages].transpose(0, 1).flatten(1, 2)[:, :length] for x in do.decode(cache))


APPENDS = [
    # batch, tokens, q heads, kv heads, dim, rot, page, lengths
    (1, 1, 1, 1, 64, 64, 16, [1]),
    (3, 1, 8, 2, 128, 128, 64, [1, 64, 65]),
    (4, 5, 6, 3, 64, 32, 32, [5, 0, 3, 77]),
    (2, 37, 4, 4, 128, 22, 16, [37, 90]),
    (2, 16, 5, 1, 128, 0, 16, [16, 31]),
    (1, 200, 2, 2, 64, 64, 128, [333]),
]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", APPENDS)
def test_append(case: tuple, dtype: str, interleaved: bool) -> None:
    b, n, hq, hk, d, rot, page, lens = case
    t = DTYPES[dtype]
    pages, total = pages_of(b, -(-max(lens) // page) + 1)
    cache = torch.randint(0, 256, (total, hk, page // 16, 16 * (d + 8)), generator=gen(3), device="cuda", dtype=torch.uint8)
    before = cache.clone()
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q, k, v = normal(b, n, hq + 2 * hk, d, dtype=t, seed=4).split((hq, hk, hk), 2)
    table = ff.rotary_table(max(lens), rot, device="cuda") if rot else None
    out = ff.kv4_append_(cache, k, v, pages, lengths, table=table, interleaved=interleaved, q=q)
    at = lengths[:, None] - n + torch.arange(n, device="cuda")
    assert torch.equal(out, ff.rotary(q, table, at.int(), interleaved=interleaved) if rot else q)
    # k turned in fp32, not rounded to 16 bits before its codes are taken
    turned = ff.rotary(k.float(), table, at.int(), interleaved=interleaved) if rot else k.float()
    want_k, want_v = do.quantise(turned).double(), do.quantise(v).double()
    touched = torch.zeros_like(cache, dtype=torch.bool)
    at_k, at_v, at_p = (x.cuda() for x in do.byte_places(d))
    for s in range(b):
        got_k, got_v, _ = held_tokens(cache, pages, s, max(lens[s], 1))
        for i in range(max(0, n - lens[s]), n):
            p = lens[s] - n + i
            assert torch.equal(got_k[:, p], want_k[s, i]), (s, i)
            assert torch.equal(got_v[:, p], want_v[s, i]), (s, i)
            block = touched[int(pages[s, p // page]), :, p % page // 16]
            for place in (at_k[p % 16], at_v[p % 16], at_p[p % 16], at_p[p % 16] + 1):
                block[:, place] = True
    assert torch.equal(cache[~touched], before[~touched])
    # values are read back as they are held, zeros in front of a sequence's start
    for as_type in (torch.float16, torch.bfloat16):
        read_k, read_v = ff.kv4_read(cache, pages, lengths, n, as_type)
        there = (at >= 0)[:, :, None, None]
        assert torch.equal(read_k, torch.where(there, want_k.float(), 0.0).to(as_type))
        assert torch.equal(read_v, torch.where(there, want_v.float(), 0.0).to(as_type))
    again = before.clone()
    assert ff.kv4_append_(again, k, v, pages, lengths, table=table, interleaved=interleaved) is None
    assert torch.equal(again, cache)


def test_append_one_by_one_is_append_at_once() -> None:
    b, n, h, d = 2, 45, 2, 128
    pages, total = pages_of(b, 2)
    caches = [ff.kv4_cache(total, h, d, page=32) for _ in range(2)]
    k, v = normal(b, n, h, d, dtype=torch.float16, seed=1), normal(b, n, h, d, dtype=torch.float16, seed=2)
    table = ff.rotary_table(64, d, device="cuda")
    ff.kv4_append_(caches[0], k, v, pages, torch.full((b,), n, dtype=torch.int32, device="cuda"), table=table)
    for i in range(n):
        ff.kv4_append_(caches[1], k[:, i : i + 1], v[:, i : i + 1], pages, torch.full((b,), i + 1, dtype=torch.int32, device="cuda"), table=table)
    assert torch.equal(*caches)


def test_append_of_extreme_groups() -> None:
    """Constant, tiny, huge and non-finite groups; each spoils nothing but itself."""
    d = 64
    rows = torch.stack([
        torch.zeros(d), torch.full((d,), 3.25), torch.linspace(-1, 1, d) * 2.0**-130, torch.linspace(-1, 1, d) * 2.0**-120,
        torch.linspace(-1, 1, d) * 2.0**120, torch.linspace(-1, 1, d) * 3e38, torch.linspace(0, 15, d), torch.linspace(-1e-3, 1e4, d),
    ])  # fmt: skip
    odd = torch.linspace(-1, 1, d).repeat(3, 1)
    odd[0, 7], odd[1, 63], odd[2, 0] = math.nan, math.inf, -math.inf
    k = torch.cat((rows, odd)).bfloat16().cuda()[None, :, None]
    n = k.shape[1]
    pages, total = pages_of(1, 1)
    cache = ff.kv4_cache(total, 1, d, page=16)
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    ff.kv4_append_(cache, k, k.flip(1), pages, lengths)
    got_k, got_v, _ = held_tokens(cache, pages, 0, n)
    want = do.quantise(k[0, :, 0]).double()
    for got, ref in ((got_k[0], want), (got_v[0], want.flip(0))):
        assert torch.equal(got.isnan(), ref.isnan())
        assert torch.equal(got.nan_to_num(0.0), ref.nan_to_num(0.0))
    assert want[:5].isfinite().all()
    assert want[8:].isnan().all()


@pytest.mark.parametrize(("what", "status"), [("page", STATUS_PAGE), ("negative page", STATUS_PAGE), ("length", STATUS_PAGE | STATUS_POSITION), ("position", STATUS_POSITION)])
def test_append_leaves_out_what_lies_outside(what: str, status: int) -> None:
    d, page = 64, 16
    pages, total = pages_of(2, 2)
    cache = torch.randint(0, 256, (total, 1, 1, 16 * (d + 8)), generator=gen(3), device="cuda", dtype=torch.uint8)
    before = cache.clone()
    lengths = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    k = normal(2, 1, 1, d, dtype=torch.float16)
    table = ff.rotary_table(32, d, device="cuda")
    good = cache.clone()
    ff.kv4_append_(good, k, k, pages, lengths, table=table)
    if what == "page":
        pages[1, 1] = total
    elif what == "negative page":
        pages[1, 1] = -5
    elif what == "length":
        lengths[1] = 2 * page + 1
    else:
        table = table[:19]
    ff.kv4_append_(cache, k, k, pages, lengths, table=table)
    assert ff.device_status() == status
    if what == "position":
        ff.kv4_append_(before, k, k, pages, lengths)
        assert torch.equal(cache, before)
    else:
        mine = int(pages[0, 1])
        assert torch.equal(cache[mine], good[mine])
        others = torch.arange(total, device="cuda") != mine
        assert torch.equal(cache[others], before[others])


def fill(b: int, hk: int, d: int, page: int, lens: list[int], seed: int = 0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """A cache of such sequences, written by the framework; slots behind a sequence's end hold NaN and infinite parameters."""
    pages, total = pages_of(b, max(1, -(-max(lens) // page)), seed)
    cache = torch.full((total, hk, page // 16, 16 * (d + 8)), 255, dtype=torch.uint8, device="cuda")  # bfloat16 0xffff: NaN
    cache[:, :, ::2, -8:] = 0x7F  # NaN of the other sign
    n = max(lens)
    if n:
        large = 1 + 3 * (torch.rand(1, 1, hk, d, generator=gen(seed + 1), device="cuda") < 0.05)
        k = (torch.randn(b, n, hk, d, generator=gen(seed + 2), device="cuda") * large).half()
        v = (torch.randn(b, n, hk, d, generator=gen(seed + 3), device="cuda") * torch.exp(torch.randn(b, n, hk, 1, generator=gen(seed + 4), device="cuda"))).half()
        ff.kv4_append_(cache, k, v, pages, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    return cache, pages, torch.tensor(lens, dtype=torch.int32, device="cuda")


def check_attention(got: torch.Tensor, q: torch.Tensor, cache: torch.Tensor, pages: torch.Tensor, lengths: torch.Tensor, scale: float) -> None:
    n, hq = q.shape[1], q.shape[2]
    hk = cache.shape[1]
    for b, length in enumerate(lengths.tolist()):
        k, v, pairs = held_tokens(cache, pages, b, length)
        if length == 0:
            assert torch.equal(got[b], torch.zeros_like(got[b]))
            continue
        o, p = do.attention(q[b], k, v, scale)
        qabs = q[b].double().abs().sum(-1)  # [n, hq]
        ks, kl, vs, _ = (x.repeat_interleave(hq // hk, 0) for x in pairs.unbind(-1))  # [hq, length]
        logit = scale * qabs[..., None] * (15 * ks + kl.abs()) * 2.0**-18 + 2.0**-21
        per_key = p * (2.0**-11 + logit) * (15 * vs + 0 * vs)
        floor = 2.0**-32 * 15 * vs.amax(-1) * length
        spread = (p * logit).sum(-1)[..., None] * o.abs()
        bound = U[q.dtype] * o.abs() + per_key.sum(-1)[..., None] + floor[:, None] + spread + 2.0**-25
        bad = (got[b].double() - o).abs() > bound
        assert not bad.any(), f"sequence {b}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got[b].double() - o).abs() / bound).max()):.2f} bounds"
        early = n - length
        if early > 0:
            assert torch.equal(got[b, :early], torch.zeros_like(got[b, :early]))


ATTENTIONS = [
    # batch, queries, q heads, kv heads, dim, page, lengths
    (1, 1, 1, 1, 64, 16, [1]),
    (1, 1, 8, 1, 128, 16, [17]),
    (3, 1, 32, 8, 128, 64, [0, 1, 1000]),
    (5, 1, 16, 1, 128, 32, [16, 15, 33, 0, 2]),
    (2, 1, 17, 1, 64, 16, [129, 300]),
    (2, 1, 40, 1, 128, 16, [129, 300]),
    (1, 1, 100, 1, 64, 128, [500]),
    (4, 5, 12, 12, 64, 16, [5, 3, 0, 777]),
    (2, 7, 6, 2, 128, 32, [7, 450]),
    (2, 9, 10, 2, 128, 64, [4, 2100]),
    (1, 65, 4, 1, 128, 16, [65]),
    (2, 100, 8, 2, 64, 64, [100, 1033]),
    (1, 333, 5, 1, 128, 128, [1500]),
    (40, 1, 4, 2, 128, 16, list(range(0, 400, 10))),
    (1, 1, 2, 2, 128, 64, [30000]),
    (1, 4, 64, 1, 128, 16, [9001]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", ATTENTIONS)
def test_attention(case: tuple, dtype: str) -> None:
    b, n, hq, hk, d, page, lens = case
    cache, pages, lengths = fill(b, hk, d, page, lens)
    q = (1.5 * normal(b, n, hq, d, dtype=torch.float32, seed=9)).to(DTYPES[dtype])
    got = ff.kv4_attention(q, cache, pages, lengths)
    check_attention(got, q, cache, pages, lengths, d**-0.5)
    assert torch.equal(got, ff.kv4_attention(q, cache, pages, lengths))  # parts are joined in a fixed order


@pytest.mark.parametrize("size", [1e-30, 1e-4, 1.0, 3e4, 1e20])
def test_attention_of_any_size_of_q(size: float) -> None:
    cache, pages, lengths = fill(2, 2, 64, 16, [40, 7])
    q = (normal(2, 1, 4, 64, dtype=torch.float32, seed=3) * size).bfloat16()
    scale = 0.125 / max(size, 1e-30)
    check_attention(ff.kv4_attention(q, cache, pages, lengths, scale), q, cache, pages, lengths, scale)


def test_attention_over_steps_of_many_sizes() -> None:
    """V of tokens from 2^-40 to 2^20, small first and large first: the shared power of two is raised on the way, and a large step at a
    token that has no weight does not drown the others."""
    d, n = 128, 320
    for flip in (False, True):
        pages, total = pages_of(1, n // 64)
        cache = ff.kv4_cache(total, 1, d, page=64)
        size = torch.exp2(torch.linspace(-40, 20, n, device="cuda"))
        size = size.flip(0) if flip else size
        k, v = normal(1, n, 1, d, dtype=torch.float32, seed=1).bfloat16(), (normal(1, n, 1, d, dtype=torch.float32, seed=2) * size[:, None, None]).bfloat16()
        lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
        ff.kv4_append_(cache, k, v, pages, lengths)
        q = normal(1, 3, 4, d, dtype=torch.float32, seed=3).bfloat16()
        check_attention(ff.kv4_attention(q, cache, pages, lengths), q, cache, pages, lengths, d**-0.5)
    # one token of 2^13 times the others' size whose logit is far below
    v = normal(1, 64, 1, d, dtype=torch.float32, seed=2)
    v[:, 3] *= 2.0**13
    q = normal(1, 1, 1, d, dtype=torch.float32, seed=3).bfloat16()
    k = normal(1, 64, 1, d, dtype=torch.float32, seed=1).bfloat16()
    k[:, 3] = -4 * q[:, 0]
    lengths = torch.tensor([64], dtype=torch.int32, device="cuda")
    ff.kv4_append_(cache, k, v.bfloat16(), pages, lengths)
    got = ff.kv4_attention(q, cache, pages, lengths)
    ks, vs, _ = held_tokens(cache, pages, 0, 64)
    o, p = do.attention(q[0], ks, vs, d**-0.5)
    assert float(p[..., 3].max()) < 1e-12
    assert float((got[0].double() - o).norm() / o.norm()) < 2.0**-7


def test_attention_of_nan_and_infinite_values() -> None:
    """A token that is held as NaN shows in the queries that see it and in no other, be it in K or in V."""
    d, n, queries = 64, 70, 12
    for which in ("k", "v"):
        cache, pages, lengths = fill(1, 2, d, 16, [n], seed=5)
        k, v = ff.kv4_read(cache, pages, lengths, n, torch.float16)
        bad = k if which == "k" else v
        bad[0, n - 4, 1, 9] = math.inf
        ff.kv4_append_(cache, k, v, pages, lengths)
        q = normal(1, queries, 4, d, dtype=torch.float16, seed=3)
        got = ff.kv4_attention(q, cache, pages, lengths)
        sees = torch.zeros(queries, 4, dtype=torch.bool, device="cuda")
        sees[queries - 4 :, 2:] = True
        assert torch.equal(got[0].isnan().all(-1), sees)
        assert got[0][~sees].isfinite().all()


def test_attention_strides_and_out() -> None:
    cache, pages, lengths = fill(3, 2, 128, 32, [100, 1, 57])
    packed = normal(3, 4, 8, 128, dtype=torch.bfloat16, seed=3)
    q = packed[:, :, 2:6]
    want = ff.kv4_attention(q.contiguous(), cache, pages, lengths)
    assert torch.equal(ff.kv4_attention(q, cache, pages, lengths), want)
    assert torch.equal(ff.kv4_attention(q.transpose(1, 2).contiguous().transpose(1, 2), cache, pages, lengths), want)
    wide = torch.zeros(3, 4, 4, 160, dtype=torch.bfloat16, device="cuda")
    out = wide[..., 16:144]
    assert ff.kv4_attention(q, cache, pages, lengths, out=out) is out
    assert torch.equal(out, want)
    assert not wide[..., :16].any()
    assert not wide[..., 144:].any()
    table = torch.full((3, 9), -7, dtype=torch.int32, device="cuda")  # columns behind a sequence's pages are not looked at
    table[:, : pages.shape[1]] = pages
    assert torch.equal(ff.kv4_attention(q, cache, table, lengths), want)


def test_attention_past_32_bits() -> None:
    """Pages behind the first four gigabytes of a cache."""
    d, page, hk = 128, 128, 8
    per = hk * page * (d + 8)
    total = (2**32 + 2**28) // per
    cache = torch.zeros(total, hk, page // 16, 16 * (d + 8), dtype=torch.uint8, device="cuda")
    pages = torch.tensor([[total - 1, 0, total - 2]], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([300], dtype=torch.int32, device="cuda")
    k, v = normal(1, 300, hk, d, dtype=torch.bfloat16, seed=1), normal(1, 300, hk, d, dtype=torch.bfloat16, seed=2)
    ff.kv4_append_(cache, k, v, pages, lengths)
    small = torch.stack((cache[total - 1], cache[0], cache[total - 2]))
    q = normal(1, 2, 32, d, dtype=torch.bfloat16, seed=3)
    got = ff.kv4_attention(q, cache, pages, lengths)
    small_pages = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    assert torch.equal(got, ff.kv4_attention(q, small, small_pages, lengths))
    check_attention(got, q, small, small_pages, lengths, d**-0.5)
    want, read = ff.kv4_read(small, small_pages, lengths, 300), ff.kv4_read(cache, pages, lengths, 300)
    assert all(torch.equal(x, y) for x, y in zip(want, read, strict=True))


@pytest.mark.parametrize("what", ["page", "length"])
def test_attention_reports_what_lies_outside(what: str) -> None:
    cache, pages, lengths = fill(2, 1, 64, 16, [40, 33])
    q = normal(2, 1, 2, 64, dtype=torch.float16, seed=3)
    want = ff.kv4_attention(q, cache, pages, lengths)
    if what == "page":
        pages[1, 0] = cache.shape[0]
    else:
        lengths[1] = 49
    got = ff.kv4_attention(q, cache, pages, lengths)
    assert ff.device_status() == STATUS_PAGE
    assert torch.equal(got[0], want[0])
    ff.kv4_attention(q, cache, pages, lengths)
    assert ff.device_status() == STATUS_PAGE


def test_a_graph_follows_the_lengths_and_streams_do_not_meet() -> None:
    b, hk, d, most = 4, 2, 128, 500
    cache, pages, lengths = fill(b, hk, d, 64, [most] * b)
    q = normal(b, 1, 8, d, dtype=torch.bfloat16, seed=3)
    sets = [[500, 1, 77, 300], [3, 0, 500, 16], [500, 500, 500, 500]]
    want = [ff.kv4_attention(q, cache, pages, torch.tensor(s, dtype=torch.int32, device="cuda")) for s in sets]
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


def test_steps_of_a_decoder_agree_with_the_whole_prompt() -> None:
    """Token by token, in pieces and at once: the same cache, and outputs within the tolerance of one another's."""
    b, n, hq, hk, d = 2, 75, 8, 2, 128
    pages, total = pages_of(b, 5)
    table = ff.rotary_table(80, d, device="cuda")
    q, k, v = (normal(b, n, h, d, dtype=torch.bfloat16, seed=s) for s, h in ((1, hq), (2, hk), (3, hk)))
    outs = []
    for pieces in ([n], [40, 34, 1], [1] * n):
        cache = ff.kv4_cache(total, hk, d, page=16)
        at, got = 0, []
        for m in pieces:
            lengths = torch.full((b,), at + m, dtype=torch.int32, device="cuda")
            part = slice(at, at + m)
            turned = ff.kv4_append_(cache, k[:, part], v[:, part], pages, lengths, table=table, q=q[:, part])
            o = ff.kv4_attention(turned, cache, pages, lengths)
            check_attention(o, turned, cache, pages, lengths, d**-0.5)
            got.append(o)
            at += m
        outs.append((cache, torch.cat(got, 1)))
    for cache, _ in outs[1:]:
        assert torch.equal(cache, outs[0][0])


def test_refusals_on_the_device() -> None:
    cache, pages, lengths = fill(2, 2, 64, 16, [20, 5])
    q = normal(2, 1, 4, 64, dtype=torch.float16)
    k = q[:, :, :2].contiguous()
    shifted = normal(2 * 4 * 64 + 1, dtype=torch.float16)[1:].view(2, 1, 4, 64)
    table = ff.rotary_table(32, 64, device="cuda")
    for call, word in [
        (lambda: ff.kv4_attention(q, cache.int(), pages, lengths), "cache"),
        (lambda: ff.kv4_attention(q, cache[:, :, :, :-16], pages, lengths), "contiguous"),
        (lambda: ff.kv4_attention(q, cache[:, :, :, :-16].contiguous(), pages, lengths), "head dim"),
        (lambda: ff.kv4_attention(q, cache, pages.long(), lengths), "page_table"),
        (lambda: ff.kv4_attention(q, cache, pages[:1], lengths), "page_table"),
        (lambda: ff.kv4_attention(q, cache, pages, lengths.long()), "lengths"),
        (lambda: ff.kv4_attention(q, cache, pages, lengths.cpu()), "lengths"),
        (lambda: ff.kv4_attention(q.float(), cache, pages, lengths), "float16"),
        (lambda: ff.kv4_attention(q[..., :32], cache, pages, lengths), "float16"),
        (lambda: ff.kv4_attention(q[:, :, :3], cache, pages, lengths), "multiple"),
        (lambda: ff.kv4_attention(shifted, cache, pages, lengths), "aligned"),
        (lambda: ff.kv4_attention(q, cache, pages, lengths, 0.0), "scale"),
        (lambda: ff.kv4_attention(q, cache, pages, lengths, math.inf), "scale"),
        (lambda: ff.kv4_attention(q, cache, pages, lengths, out=q.bfloat16()), "out"),
        (lambda: ff.kv4_attention(q.clone().requires_grad_(True), cache, pages, lengths), "grad"),
        (lambda: ff.kv4_append_(cache, q, q, pages, lengths), "heads"),
        (lambda: ff.kv4_append_(cache, k, k.bfloat16(), pages, lengths), "does not go"),
        (lambda: ff.kv4_append_(cache, k, k, pages, lengths, table=table.double()), "table"),
        (lambda: ff.kv4_append_(cache, k, k, pages, lengths, out=q), "without q"),
        (lambda: ff.kv4_append_(cache, k, k, pages, lengths, q=q.bfloat16()), "does not go"),
        (lambda: ff.kv4_read(cache, pages, lengths, 3, torch.float32), "float16"),
        (lambda: ff.kv4_read(cache, pages, lengths, -1), "negative"),
    ]:
        with pytest.raises(ValueError, match=word):
            call()
    assert ff.kv4_attention(q[:, :0], cache, pages, lengths).shape == (2, 0, 4, 64)
    assert ff.kv4_read(cache, pages, lengths, 0)[0].shape == (2, 0, 2, 64)
