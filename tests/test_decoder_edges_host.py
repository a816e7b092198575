"""Edges of a token decoder's layers that need no GPU: what device code does by its text, compiled for the host or read."""

from __future__ import annotations

import math
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import fastforks_b200 as ff
from fastforks_b200 import _lib


def header(name: str) -> str:
    return next(p for p in _lib.HEADERS if p.name == name).read_text()


SPLIT_ROWS = r"""
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <map>
#define __device__
#define __forceinline__ inline
static float row_memory[1024], *row = row_memory;
static std::map<int, int> writer;  // float of the row -> the lane that stored it
static int lane_now, bad, stored;
static void __syncwarp() {}
static float __ldg(const float* p) { return *p; }
static float __fmul_rn(float a, float b) { return a * b; }
static float __fadd_rn(float a, float b) { return a + b; }
template <typename T> void store8(T* to, const float*) {
  for (int i = 0; i < 8; ++i) {
    const int at = static_cast<int>(to - row) + i;
    if (!writer.emplace(at, lane_now).second || at >= 1024) ++bad;
    ++stored;
  }
}
%(forms)s
%(places)s
template <int FORM> struct Turns;
%(turns)s
struct { int rot, dim; } p;
int main() {
  for (p.dim = 8; p.dim <= 512; p.dim += 8) {
    p.rot = p.dim >= 6 ? p.dim - 2 : p.dim;
    int lanes = 1;
    while (16 * lanes < p.dim) lanes *= 2;
    writer.clear();
    bad = stored = 0;
    for (int j = 0; j < lanes; ++j) {
      constexpr int FORM = kRowSplit;
      lane_now = j;
%(kernel)s
      (void)place_b;
      float f[16] = {};
      Turns<FORM> turns;
      turns.load(nullptr, a, b, p.rot, 1.f);
      turns.template apply<false>(f, row, p.dim, false);
    }
    printf("%%d %%d %%d\n", p.dim, bad, stored);
  }
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_each_place_of_a_split_row_is_stored_by_one_lane(tmp_path: Path) -> None:
    """Halves whose partners are looked up in shared memory: a row's lanes store its values there without a barrier between one another, so
    no float may have two writers. A row of 72, 80 or 96 has lanes that hold none of it. The kernel's own lines, run lane by lane."""
    text = header("rotary_sm100.cuh")

    def part(begin: str, end: str, start: int = 0) -> str:
        at = text.index(begin, start)
        return text[at : text.index(end, at) + len(end)]

    kernel = text.index("rotary_stream_kernel(const RotaryParams p)")
    source = SPLIT_ROWS % {
        "forms": part("enum RowForm", ";"),
        "places": part("template <int FORM>\n__device__ __forceinline__ void lane_places", "\n}\n"),
        "turns": part("template <>\nstruct Turns<kRowSplit>", "\n};\n"),
        "kernel": part("int a, b;", "constexpr bool kWhole", kernel).replace("constexpr bool kWhole", ""),
    }
    src, exe = tmp_path / "rows.cpp", tmp_path / "rows"
    src.write_text(source)
    subprocess.run(["g++", "-std=c++17", "-Wno-unused", "-o", str(exe), str(src)], check=True)
    lines = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")[:-1]
    got = {int(dim): (int(bad), int(stored)) for dim, bad, stored in (line.split() for line in lines)}
    assert sorted(got) == list(range(8, 513, 8))
    assert {dim: n for dim, (n, _) in got.items() if n} == {}
    assert all(stored == dim for dim, (_, stored) in got.items())  # and every float is stored


def test_copies_in_flight_are_waited_for_on_every_path() -> None:
    """The loader of the attention over many rows has asked for everything long before the others are through: a wait that runs out in
    another warp then ends the CTA with copies on their way into its shared memory, unless the loader waits for the last of either
    buffer whatever it has seen, with a limit and on a word that nobody raises. (Read, not run: no wait runs out on a healthy GPU.) The phases that
    are waited for are counted here for any number of steps."""
    source = header("kv4_tiles_sm100.cuh")
    body = next(b for b in source.split("__global__")[1:] if "kv4_tiles_kernel(" in b)
    loader = body[body.index("// ---- loads ----") : body.index("// ---- products ----")]
    wait = "for (uint32_t i = steps < 2 ? 0 : steps - 2; i < steps; ++i) mbar_wait(bars + kBarRawFull + (i & 1), (i >> 1) & 1, abort_flag + 2);"
    at = loader.index(wait)
    begin = loader.index("if (lane == 0) {")
    depth = loader[begin:at].count("{") - loader[begin:at].count("}")
    assert depth == 1, "the wait is under a condition"
    assert at > loader.rindex("bulk_load(")
    assert not re.search(r"\breturn\b", loader[begin:at])
    for steps in range(9):
        waited = [(i & 1, (i >> 1) & 1) for i in range(max(0, steps - 2), steps)]
        last = {i & 1: (i >> 1) & 1 for i in range(steps)}  # of each buffer, the phase of its last copy
        assert dict(waited) == last and len(waited) == len(last)


@pytest.mark.parametrize(("dim", "base", "original", "factor"), [(128, 1e4, 131072, 4.0), (64, 1e4, 65536, 8.0), (128, 1e4, 2048, 4.0), (64, 500.0, 4096, 2.0), (2, 1e4, 1000, 2.0)])
def test_yarn_divides_each_pair_by_its_number_of_turns(dim: int, base: float, original: int, factor: float) -> None:
    """A pair's share of the plain frequency goes from one, at beta_fast turns within the original length, to none, at beta_slow, evenly over the
    logarithm of the turns (the pairs in between are evenly spaced there): also where the slowest pair still turns more often than beta_slow.
    The ends of the ramp lie on whole pairs, the nearest ones outside of it, which moves a pair's share by two pairs' worth at most."""
    fast, slow = 32.0, 1.0
    table = ff.rotary_table(2, dim, base=base, scaling="yarn", factor=factor, original_length=original)
    plain = base ** (-2 * torch.arange(dim // 2).double() / dim)
    ratio = torch.atan2(table[1, 1].double(), table[1, 0].double()) / plain
    kept = (ratio - 1 / factor) / (1 - 1 / factor)
    turns = original * plain / (2 * math.pi)
    want = (turns.log() - math.log(slow)) / (math.log(fast) - math.log(slow))
    pairs = dim / 2 * math.log(fast / slow) / math.log(base)  # of the ramp
    assert ((kept - want.clamp(0, 1)).abs() <= 2 / pairs + 1e-4).all()
    assert (kept[turns < slow] <= 1e-4 + 2 / pairs).all()
    last = float(want[-1])
    if last > 2 / pairs:
        assert float(kept[-1]) > 0.0
    assert (kept.diff() <= 1e-5).all()


@pytest.mark.parametrize("base", [1.0, 0.5])
def test_yarn_needs_pairs_that_get_slower(base: float) -> None:
    with pytest.raises(ValueError, match="rotary_table"):
        ff.rotary_table(8, 64, base=base, scaling="yarn", factor=2.0, original_length=4)


def test_operands_without_dimensions_are_refused_as_any_others() -> None:
    nothing, none = torch.zeros(()), torch.zeros((), dtype=torch.int32)
    cache = ff.kv4_cache(2, 2, 64, page=16, device="cpu")
    pages, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (
        lambda: ff.rotary(nothing, ff.rotary_table(4, 64)),
        lambda: ff.qk_norm_rotary(nothing, nothing, None, None, None),
        lambda: ff.kv4_append_(cache, nothing.half(), nothing.half(), pages, lengths),
        lambda: ff.kv4_read(cache, pages, none, 1),
        lambda: ff.kv4_attention(nothing.half(), cache, pages, lengths),
        lambda: ff.kv4_attention(torch.zeros(1, 1, 2, 64).half(), nothing, pages, lengths),
        lambda: ff.kv4_attention(torch.zeros(1, 1, 2, 64).half(), cache, none, none),
    ):
        with pytest.raises(ValueError, match=r"rotary|kv4_"):
            call()
