"""A token decoder's layers without a GPU: the C structs, what the calls refuse before any launch, and the tables of positions."""

from __future__ import annotations

import ctypes
import math
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import fastforks_b200 as ff
from fastforks_b200 import _lib
from oracle import decoder_oracle as do

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "b200_decoder.h"


@pytest.fixture(scope="module")
def lib() -> ctypes.CDLL:
    if _lib.needs_build():
        _lib.build()
    _lib.library.cache_clear()
    return _lib.library()


def test_header_declares_the_expected_entry_points(lib: ctypes.CDLL) -> None:
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    assert sorted(re.findall(r"^int (b200_\w+)\s*\(", text, flags=re.M)) == sorted(_lib.DECODER_EXPORTS)
    for name in _lib.DECODER_EXPORTS:
        assert hasattr(lib, name)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_ctypes_structs_match_the_c_structs(tmp_path: Path) -> None:
    structs = (_lib.B200Heads, _lib.B200RotaryArgs, _lib.B200Kv4Args, _lib.B200Kv4AttnArgs)
    want = {f"{s.__name__}.{f}": getattr(s, f).offset for s in structs for f, *_ in s._fields_}  # noqa: SLF001
    want |= {s.__name__: ctypes.sizeof(s) for s in structs}
    lines = "\n".join(f'  printf("{name} %zu\\n", {"offsetof(" + name.replace(".", ", ") + ")" if "." in name else "sizeof(" + name + ")"});' for name in want)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{\n{lines}\n  return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert {name: int(offset) for name, offset in (line.split() for line in out)} == want


def rotary_args(**kw: object) -> _lib.B200RotaryArgs:
    a = _lib.B200RotaryArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = a.weight_dtype = _lib.BF16
    a.batch, a.tokens, a.head_dim, a.rot, a.tensors, a.cs, a.table_rows, a.eps = 2, 5, 64, 64, 1, 0x10000, 5, 1e-6
    a.heads[0].x = a.heads[0].y = 0x10000
    a.heads[0].heads = 3
    for name, v in kw.items():
        if name.startswith("h_"):
            setattr(a.heads[0], name[2:], v)
        else:
            setattr(a, name, v)
    return a


@pytest.mark.parametrize(
    ("kw", "code", "word"),
    [
        ({"struct_size": 8}, _lib.BAD_CONFIG, "struct_size"),
        ({"dtype": 7}, _lib.BAD_CONFIG, "dtype"),
        ({"norm": 1, "weight_dtype": _lib.F16}, _lib.BAD_CONFIG, "weight_dtype"),
        ({"batch": 0}, _lib.BAD_CONFIG, "batch"),
        ({"tensors": 3}, _lib.BAD_CONFIG, "tensors"),
        ({"head_dim": 513}, _lib.UNSUPPORTED, "head_dim"),
        ({"rot": 7}, _lib.UNSUPPORTED, "rot"),
        ({"rot": 66}, _lib.UNSUPPORTED, "rot"),
        ({"cs": 0}, _lib.BAD_CONFIG, "table"),
        ({"cs": 0x10004}, _lib.UNSUPPORTED, "aligned"),
        ({"norm": 1, "eps": -1.0}, _lib.BAD_CONFIG, "eps"),
        ({"h_heads": 0}, _lib.BAD_CONFIG, "heads"),
        ({"h_y": 0}, _lib.BAD_CONFIG, "NULL"),
        ({"h_x": 0}, _lib.BAD_CONFIG, "NULL"),
        ({"backward": 1}, _lib.BAD_CONFIG, "NULL"),
        ({"h_x": 0x10001}, _lib.UNSUPPORTED, "aligned"),
        ({"tokens": 2**31 - 1}, _lib.UNSUPPORTED, "at most"),
    ],
)
def test_rotary_rejects(lib: ctypes.CDLL, kw: dict, code: int, word: str) -> None:
    assert lib.b200_rotary(ctypes.byref(rotary_args(**kw)), None) == code
    assert word in _lib.last_error()


def kv4_args(kind: type, **kw: object) -> ctypes.Structure:
    a = kind()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = _lib.BF16
    a.batch, a.q_heads, a.kv_heads, a.head_dim, a.page, a.pages, a.table_pages, a.table_stride = 2, 8, 2, 128, 64, 10, 4, 4
    a.cache = a.page_table = a.lengths = a.q = 0x10000
    strides = (5 * 8 * 128, 8 * 128, 128)
    if kind is _lib.B200Kv4Args:
        a.tokens, a.rot, a.cs, a.table_rows = 5, 128, 0x10000, 256
        for name in ("q", "k", "v", "q_out", "k_out", "v_out"):
            setattr(a, name, 0x10000)
            getattr(a, f"{name}_stride")[:] = strides
    else:
        a.queries, a.scale, a.o, a.workspace, a.counters = 5, 0.1, 0x10000, 0x10000, 0x10000
        a.q_stride[:] = a.o_stride[:] = strides
    for name, v in kw.items():
        if isinstance(v, tuple):
            getattr(a, name)[:] = v
        else:
            setattr(a, name, v)
    return a


COMMON = [
    ({"struct_size": 8}, _lib.BAD_CONFIG, "struct_size"),
    ({"dtype": _lib.F32}, _lib.BAD_CONFIG, "dtype"),
    ({"head_dim": 96}, _lib.UNSUPPORTED, "head_dim"),
    ({"batch": 0}, _lib.BAD_CONFIG, "batch"),
    ({"page": 24}, _lib.UNSUPPORTED, "page"),
    ({"page": 0}, _lib.UNSUPPORTED, "page"),
    ({"pages": 0}, _lib.BAD_CONFIG, "pages"),
    ({"table_pages": 2**26}, _lib.BAD_CONFIG, "page table"),
    ({"cache": 0}, _lib.BAD_CONFIG, "NULL"),
    ({"lengths": 0}, _lib.BAD_CONFIG, "NULL"),
    ({"cache": 0x10008}, _lib.UNSUPPORTED, "aligned"),
]


@pytest.mark.parametrize(
    ("kw", "code", "word"),
    [
        *COMMON,
        ({"rot": 130}, _lib.UNSUPPORTED, "rot"),
        ({"table_rows": 0}, _lib.BAD_CONFIG, "table"),
        ({"k": 0}, _lib.BAD_CONFIG, "NULL"),
        ({"v": 0x10002}, _lib.UNSUPPORTED, "aligned"),
        ({"k_stride": (5 * 8 * 128, 8 * 128, 132)}, _lib.UNSUPPORTED, "multiples of 8"),
        ({"q_out": 0}, _lib.BAD_CONFIG, "NULL"),
        ({"q_heads": 0}, _lib.BAD_CONFIG, "q heads"),
    ],
)
def test_append_rejects(lib: ctypes.CDLL, kw: dict, code: int, word: str) -> None:
    assert lib.b200_kv4_append(ctypes.byref(kv4_args(_lib.B200Kv4Args, **kw)), None) == code
    assert word in _lib.last_error()


@pytest.mark.parametrize(("kw", "code", "word"), [*COMMON, ({"k_out": 0}, _lib.BAD_CONFIG, "NULL"), ({"v_out_stride": (4, 8, 8)}, _lib.UNSUPPORTED, "multiples of 8")])
def test_read_rejects(lib: ctypes.CDLL, kw: dict, code: int, word: str) -> None:
    assert lib.b200_kv4_read(ctypes.byref(kv4_args(_lib.B200Kv4Args, **kw)), None) == code
    assert word in _lib.last_error()


@pytest.mark.parametrize(
    ("kw", "code", "word"),
    [
        *COMMON,
        ({"q_heads": 9}, _lib.BAD_CONFIG, "multiple"),
        ({"scale": 0.0}, _lib.UNSUPPORTED, "scale"),
        ({"scale": math.nan}, _lib.UNSUPPORTED, "scale"),
        ({"q": 0}, _lib.BAD_CONFIG, "NULL"),
        ({"o": 0x10008}, _lib.UNSUPPORTED, "aligned"),
    ],
)
def test_attention_rejects(lib: ctypes.CDLL, kw: dict, code: int, word: str) -> None:
    assert lib.b200_kv4_attention(ctypes.byref(kv4_args(_lib.B200Kv4AttnArgs, **kw)), None) == code
    assert word in _lib.last_error()


def test_null_args(lib: ctypes.CDLL) -> None:
    for name in _lib.DECODER_EXPORTS:
        arguments = (None, None) if len(getattr(lib, name).argtypes) == 2 else (None,)  # noqa: PLR2004
        assert getattr(lib, name)(*arguments) == _lib.BAD_CONFIG


def test_cpu_tensors_are_refused() -> None:
    x, table = torch.zeros(1, 2, 2, 64), ff.rotary_table(4, 64)
    cache = ff.kv4_cache(2, 2, 64, page=16, device="cpu")
    pages, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (
        lambda: ff.rotary(x, table),
        lambda: ff.qk_norm_rotary(x, x, None, None, table),
        lambda: ff.kv4_append_(cache, x.half(), x.half(), pages, lengths),
        lambda: ff.kv4_read(cache, pages, lengths, 1),
        lambda: ff.kv4_attention(x.half(), cache, pages, lengths),
    ):
        with pytest.raises(ValueError, match="CUDA"):
            call()


@pytest.mark.parametrize("kw", [{"head_dim": 96}, {"page": 8}, {"page": 40}, {"pages": 0}, {"kv_heads": 0}])
def test_cache_refuses(kw: dict) -> None:
    with pytest.raises(ValueError, match="kv4_cache"):
        ff.kv4_cache(**({"pages": 4, "kv_heads": 2, "head_dim": 64, "page": 16, "device": "cpu"} | kw))


def test_cache_shape() -> None:
    cache = ff.kv4_cache(5, 3, 128, page=48, device="cpu")
    assert cache.shape == (5, 3, 3, 16 * 136)
    assert cache.dtype == torch.uint8
    places = torch.cat([x.flatten() for x in do.byte_places(128)])
    assert places.max() < 16 * 136


@pytest.mark.parametrize("kw", [{"length": 0}, {"dim": 7}, {"dim": 0}, {"base": 0.0}, {"scaling": "other"}, {"scaling": "linear", "factor": 0.5}, {"scaling": "yarn", "factor": 2.0}])
def test_table_refuses(kw: dict) -> None:
    with pytest.raises(ValueError, match="rotary_table"):
        ff.rotary_table(**({"length": 8, "dim": 64} | kw))


def test_table_is_cosines_and_sines() -> None:
    t = ff.rotary_table(100, 64, base=500.0)
    angle = torch.arange(100).double()[:, None] * 500.0 ** (-torch.arange(32).double() / 32)
    assert t.shape == (100, 2, 32)
    assert torch.equal(t[:, 0], angle.cos().float())
    assert torch.equal(t[:, 1], angle.sin().float())


def test_scaled_tables() -> None:
    """Linear: position 4 p of a table stretched fourfold is position p. NTK: the fastest pair is untouched, the slowest stretched by the
    factor. YaRN: pairs of many turns are untouched, of few turns stretched, none goes beyond, and everything is larger by a constant."""
    plain = ff.rotary_table(64, 128)
    linear = ff.rotary_table(256, 128, scaling="linear", factor=4.0)
    assert torch.allclose(linear[::4], plain, atol=1e-6)
    angle = lambda t: torch.atan2(t[1, 1].double(), t[1, 0].double())  # noqa: E731  of one position
    ntk = angle(ff.rotary_table(2, 128, scaling="ntk", factor=4.0))
    assert torch.allclose(ntk[0], angle(plain)[0])
    assert torch.allclose(ntk[-1], angle(plain)[-1] / 4, rtol=1e-5)
    yarn = ff.rotary_table(2, 128, scaling="yarn", factor=4.0, original_length=2048)
    size = 0.1 * math.log(4) + 1
    assert torch.allclose(yarn.double().square().sum(1), torch.full((2, 64), size**2, dtype=torch.float64), rtol=1e-6)
    ratio = angle(yarn) / angle(plain)
    turns = 2048 * angle(plain) / (2 * math.pi)
    assert torch.allclose(ratio[turns > 40], torch.ones(()).double(), rtol=1e-5)
    assert torch.allclose(ratio[turns < 0.7], torch.full((), 0.25).double(), rtol=1e-5)
    assert (ratio.diff() <= 1e-6).all()
    assert torch.equal(ff.rotary_table(9, 64, scaling="yarn", factor=1.0, original_length=64), ff.rotary_table(9, 64))


def test_oracle_of_the_cache_round_trips() -> None:
    """The oracle's own places: each byte of a block is one place's, and a group comes back within half a step."""
    for dim in (64, 128):
        at_k, at_v, at_p = do.byte_places(dim)
        every = torch.cat((at_k[:, ::2].flatten(), at_v[:, ::2].flatten(), at_p.flatten(), at_p.flatten() + 1))
        assert torch.equal(every.sort().values, torch.arange(16 * (dim + 8)))
    x = torch.randn(50, 128)
    step = (x.amax(-1) - x.amin(-1)) / 15
    assert ((do.quantise(x) - x.double()).abs().amax(-1) <= step * (0.5 + 15 * 2.0**-9) + x.amin(-1).abs() * 2.0**-8).all()


def test_tiles_of_many_rows_hold_and_free_tensor_memory_in_order() -> None:
    """The attention over many rows allocates before it lets the next kernel start, and frees behind a wait for all of its products that
    hangs on no flag: another warp's wait may run out after this warp has looked at one. (Read, not run.)"""
    source = next(p for p in _lib.HEADERS if p.name == "kv4_tiles_sm100.cuh").read_text()
    body = next(b for b in source.split("__global__")[1:] if "kv4_tiles_kernel(" in b)
    assert body.index("tmem_alloc(") < body.index("grid_launch_dependents();")
    drained = re.search(r"if \(!ok\) give_up\(\);\s*(//[^\n]*\s*)*if \(elect_one\(\)\) umma_commit\(&drain\);\s*__syncwarp\(\);\s*mbar_wait\(&drain, 0, abort_flag \+ 2\);", body)
    assert drained, "products are not waited for, or only under a condition"
    assert drained.end() < body.index("tmem_dealloc(")
    assert not re.search(r"abort_flag\[2\] = [^0a]|abort_flag \+ 2, 1", body)  # the word that this wait looks at stays zero
