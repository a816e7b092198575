"""Layer norm and the losses of an output layer without a GPU: the C structs, what the calls refuse before any launch, and the kernels that hold
tensor memory by name."""

from __future__ import annotations

import ctypes
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

import fastforks_b200 as ff
from fastforks_b200 import _lib

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "b200_training.h"


@pytest.fixture(scope="module")
def lib() -> ctypes.CDLL:
    if _lib.needs_build():
        _lib.build()
    _lib.library.cache_clear()
    return _lib.library()


def test_header_declares_the_expected_entry_points(lib: ctypes.CDLL) -> None:
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    assert sorted(re.findall(r"^int (b200_\w+)\s*\(", text, flags=re.M)) == sorted(_lib.TRAINING_EXPORTS)
    for name in _lib.TRAINING_EXPORTS:
        assert hasattr(lib, name)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_ctypes_structs_match_the_c_structs(tmp_path: Path) -> None:
    structs = (_lib.B200LayerNormArgs, _lib.B200HeadArgs)
    want = {f"{s.__name__}.{f}": getattr(s, f).offset for s in structs for f, *_ in s._fields_}  # noqa: SLF001
    want |= {s.__name__: ctypes.sizeof(s) for s in structs}
    lines = "\n".join(f'  printf("{name} %zu\\n", {"offsetof(" + name.replace(".", ", ") + ")" if "." in name else "sizeof(" + name + ")"});' for name in want)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{HEADER}"\nint main(void) {{\n{lines}\n  return 0;\n}}\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-o", str(exe), str(src)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert {name: int(offset) for name, offset in (line.split() for line in out)} == want


def norm_args(**kw: object) -> _lib.B200LayerNormArgs:
    a = _lib.B200LayerNormArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype = a.weight_dtype = _lib.BF16
    a.rows, a.dim, a.eps = 5, 64, 1e-5
    a.x = a.y = a.dy = a.dx = a.stats = 0x10000
    a.x_stride = a.y_stride = a.dy_stride = a.dx_stride = 64
    for name, v in kw.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize(
    ("kw", "code", "word"),
    [
        ({"struct_size": 8}, _lib.BAD_CONFIG, "struct_size"),
        ({"dtype": 5}, _lib.BAD_CONFIG, "dtype"),
        ({"weight_dtype": _lib.F16}, _lib.BAD_CONFIG, "weight_dtype"),
        ({"dim": 0}, _lib.UNSUPPORTED, "dim"),
        ({"dim": 32769}, _lib.UNSUPPORTED, "dim"),
        ({"rows": 0}, _lib.UNSUPPORTED, "rows"),
        ({"rows": 2**31}, _lib.UNSUPPORTED, "rows"),
        ({"eps": -1.0}, _lib.BAD_CONFIG, "eps"),
        ({"eps": float("nan")}, _lib.BAD_CONFIG, "eps"),
        ({"x": 0}, _lib.BAD_CONFIG, "x is NULL"),
        ({"x": 0x10001}, _lib.UNSUPPORTED, "aligned"),
        ({"x_stride": -64}, _lib.UNSUPPORTED, "stride"),
        ({"weight": 0x10001}, _lib.UNSUPPORTED, "weight"),
    ],
)
def test_layer_norm_rejects_before_launch(lib: ctypes.CDLL, kw: dict, code: int, word: str) -> None:
    for call in (lib.b200_layer_norm, lib.b200_layer_norm_grad):
        assert call(ctypes.byref(norm_args(**kw)), None) == code
        assert word in lib.b200_attn_last_error().decode()


def test_layer_norm_rejects_what_belongs_to_one_direction(lib: ctypes.CDLL) -> None:
    assert lib.b200_layer_norm(ctypes.byref(norm_args(y_stride=63)), None) == _lib.UNSUPPORTED
    assert lib.b200_layer_norm(ctypes.byref(norm_args(bias=0x10001)), None) == _lib.UNSUPPORTED
    assert lib.b200_layer_norm_grad(ctypes.byref(norm_args(dx_stride=0)), None) == _lib.UNSUPPORTED
    assert lib.b200_layer_norm_grad(ctypes.byref(norm_args(stats=0)), None) == _lib.BAD_CONFIG
    assert lib.b200_layer_norm_grad(ctypes.byref(norm_args(dweight=0x10001)), None) == _lib.UNSUPPORTED
    for call in (lib.b200_layer_norm, lib.b200_layer_norm_grad):
        assert call(None, None) == _lib.BAD_CONFIG


def head_args(**kw: object) -> _lib.B200HeadArgs:
    a = _lib.B200HeadArgs()
    a.struct_size = ctypes.sizeof(a)
    a.dtype, a.rows, a.dim, a.vocab, a.top, a.reduction, a.target_bytes, a.tau, a.teacher_dtype = _lib.F16, 100, 64, 500, 0, 2, 8, 1.0, _lib.F32
    a.x = a.w = a.targets = a.teacher = a.loss = a.state = a.workspace = a.grad = a.dx = a.dw = a.bias = a.dbias = 0x10000
    a.ldx = a.ldw = 64
    a.state_bytes = a.workspace_bytes = 1 << 40
    for name, v in kw.items():
        setattr(a, name, v)
    return a


@pytest.mark.parametrize(
    ("kw", "code", "word"),
    [
        ({"struct_size": 8}, _lib.BAD_CONFIG, "struct_size"),
        ({"dtype": _lib.F32}, _lib.BAD_CONFIG, "dtype"),
        ({"rows": 0}, _lib.UNSUPPORTED, "rows"),
        ({"rows": 2**24 + 1}, _lib.UNSUPPORTED, "rows"),
        ({"dim": 60}, _lib.UNSUPPORTED, "dim"),
        ({"dim": 0}, _lib.UNSUPPORTED, "dim"),
        ({"dim": 2**17 + 8}, _lib.UNSUPPORTED, "dim"),
        ({"vocab": 0}, _lib.UNSUPPORTED, "vocab"),
        ({"vocab": 2**26 + 1}, _lib.UNSUPPORTED, "vocab"),
        ({"rows": 2**24, "vocab": 2**26}, _lib.UNSUPPORTED, "too large"),
        ({"top": -1}, _lib.UNSUPPORTED, "top"),
        ({"top": 257}, _lib.UNSUPPORTED, "top"),
        ({"reduction": 3}, _lib.BAD_CONFIG, "reduction"),
        ({"top": 4, "tau": 0.0}, _lib.UNSUPPORTED, "tau"),
        ({"top": 4, "tau": float("nan")}, _lib.UNSUPPORTED, "tau"),
        ({"top": 4, "tau": 1e30}, _lib.UNSUPPORTED, "tau"),
        ({"x": 0}, _lib.BAD_CONFIG, "x is NULL"),
        ({"w": 0x10008}, _lib.UNSUPPORTED, "w is not"),
        ({"ldx": 56}, _lib.UNSUPPORTED, "x: row stride"),
        ({"ldw": 68}, _lib.UNSUPPORTED, "w: row stride"),
        ({"ldx": 2**38}, _lib.UNSUPPORTED, "x: row stride"),
        ({"bias": 0x10008}, _lib.UNSUPPORTED, "bias"),
        ({"state": 0x10010}, _lib.BAD_CONFIG, "state"),
        ({"state_bytes": 100}, _lib.BAD_CONFIG, "state"),
        ({"workspace": 0}, _lib.BAD_CONFIG, "workspace"),
    ],
)
def test_the_losses_reject_before_launch(lib: ctypes.CDLL, kw: dict, code: int, word: str) -> None:
    for call in (lib.b200_head_loss, lib.b200_head_grad):
        assert call(ctypes.byref(head_args(**kw)), None) == code
        assert word in lib.b200_attn_last_error().decode()


@pytest.mark.parametrize(
    ("kw", "word"),
    [({"targets": 0}, "targets"), ({"targets": 0x10004}, "targets"), ({"target_bytes": 2}, "targets"), ({"loss": 0}, "loss"), ({"loss": 0x10002}, "loss"),
     ({"top": 3, "teacher": 0}, "teacher"), ({"top": 3, "teacher_dtype": 7}, "teacher_dtype"), ({"top": 3, "teacher": 0x10002}, "teacher"), ({"top": 3, "teacher_stride": -1}, "strides")],
)  # fmt: skip
def test_the_forward_call_looks_at_its_own(lib: ctypes.CDLL, kw: dict, word: str) -> None:
    assert lib.b200_head_loss(ctypes.byref(head_args(**kw)), None) in (_lib.BAD_CONFIG, _lib.UNSUPPORTED)
    assert word in lib.b200_attn_last_error().decode()


def test_the_gradient_call_looks_at_its_own(lib: ctypes.CDLL) -> None:
    for kw in ({"grad": 0}, {"grad": 0x10002}, {"grad_stride": -1}, {"dx": 0x10008}, {"dw": 0x10008}, {"dbias": 0x10008}):
        assert lib.b200_head_grad(ctypes.byref(head_args(**kw)), None) in (_lib.BAD_CONFIG, _lib.UNSUPPORTED)
    assert lib.b200_head_grad(ctypes.byref(head_args(dx=0, dw=0, dbias=0)), None) == _lib.OK  # nothing asked for
    for call in (lib.b200_head_loss, lib.b200_head_grad):
        assert call(None, None) == _lib.BAD_CONFIG


def test_layer_norm_refuses_on_the_host() -> None:
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        ff.layer_norm(x)


def test_losses_refuse_on_the_host() -> None:
    x, w = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(5, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ff.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="CUDA"):
        ff.linear_distillation(x, w, torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))


@pytest.mark.gpu
def test_layer_norm_refuses() -> None:
    x, w = torch.zeros(4, 8, device="cuda", dtype=torch.float16), torch.zeros(8, device="cuda", dtype=torch.float16)
    bad = [
        lambda: ff.layer_norm(x.double()),
        lambda: ff.layer_norm(x[0, 0]),
        lambda: ff.layer_norm(x[:, :0]),
        lambda: ff.layer_norm(torch.zeros(1, 32776, device="cuda")),
        lambda: ff.layer_norm(x, w[:4]),
        lambda: ff.layer_norm(x, w.bfloat16()),
        lambda: ff.layer_norm(x, w, w.float()),
        lambda: ff.layer_norm(x, w.cpu()),
        lambda: ff.layer_norm(x, torch.zeros(16, device="cuda", dtype=torch.float16)[::2]),
        lambda: ff.layer_norm(x, w, eps=-1.0),
        lambda: ff.layer_norm(x, w, eps=float("nan")),
        lambda: ff.layer_norm(x, out=torch.empty(4, 9, device="cuda", dtype=torch.float16)),
        lambda: ff.layer_norm(x, out=torch.empty(8, 4, device="cuda", dtype=torch.float16).t()),
        lambda: ff.layer_norm(x, out=x.float()),
        lambda: ff.layer_norm(x.clone().requires_grad_(True), out=torch.empty_like(x)),
        lambda: ff.layer_norm(x[:0].requires_grad_(True)),
    ]
    for call in bad:
        with pytest.raises(ValueError, match="layer_norm"):
            call()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="tangent"):
        ff.layer_norm(torch.autograd.forward_ad.make_dual(x, x))


@pytest.mark.gpu
def test_losses_refuse() -> None:
    x, w, y = (torch.zeros(4, 8, device="cuda", dtype=torch.float16), torch.zeros(5, 8, device="cuda", dtype=torch.float16), torch.zeros(4, device="cuda", dtype=torch.int64))
    ids, teacher = torch.zeros(4, 3, device="cuda", dtype=torch.int64), torch.zeros(4, 3, device="cuda")
    bad = [
        lambda: ff.linear_cross_entropy(x.float(), w.float(), y),
        lambda: ff.linear_cross_entropy(x, w.bfloat16(), y),
        lambda: ff.linear_cross_entropy(x, w[:, :4], y),
        lambda: ff.linear_cross_entropy(x, w[:0], y),
        lambda: ff.linear_cross_entropy(x, w[0], y),
        lambda: ff.linear_cross_entropy(x, w.cpu(), y),
        lambda: ff.linear_cross_entropy(x[:, :4], w[:, :4], y),
        lambda: ff.linear_cross_entropy(x, w, y, bias=w[:, 0].float()),
        lambda: ff.linear_cross_entropy(x, w, y, bias=x[:, 0]),
        lambda: ff.linear_cross_entropy(x, w, y, bias=w[:, 0].cpu()),
        lambda: ff.linear_distillation(x, w, ids, teacher, bias=w[:, :1]),
        lambda: ff.linear_cross_entropy(x, w, y[:3]),
        lambda: ff.linear_cross_entropy(x, w, y.float()),
        lambda: ff.linear_cross_entropy(x, w, y.cpu()),
        lambda: ff.linear_cross_entropy(x, w, y, reduction="median"),
        lambda: ff.linear_cross_entropy(x, w, y, ignore_index=2**63),
        lambda: ff.linear_cross_entropy(x[:0].requires_grad_(True), w, y[:0]),
        lambda: ff.linear_distillation(x, w, ids[:3], teacher[:3]),
        lambda: ff.linear_distillation(x, w, ids, teacher[:, :2]),
        lambda: ff.linear_distillation(x, w, ids.float(), teacher),
        lambda: ff.linear_distillation(x, w, ids, teacher.double()),
        lambda: ff.linear_distillation(x, w, ids, teacher.cpu()),
        lambda: ff.linear_distillation(x, w, ids[:, :0], teacher[:, :0]),
        lambda: ff.linear_distillation(x, w, ids[:, :1].expand(4, 257), teacher[:, :1].expand(4, 257)),
        lambda: ff.linear_distillation(x, w, ids, teacher, temperature=0.0),
        lambda: ff.linear_distillation(x, w, ids, teacher, temperature=float("nan")),
        lambda: ff.linear_distillation(x, w, ids, teacher, temperature=1e30),
        lambda: ff.linear_distillation(x, w, ids, teacher.clone().requires_grad_(True)),
    ]
    for call in bad:
        with pytest.raises(ValueError, match="linear_"):
            call()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(ValueError, match="tangent"):
        ff.linear_cross_entropy(torch.autograd.forward_ad.make_dual(x, x), w, y)


HEAD = (ROOT / "fastforks_b200" / "csrc" / "head_sm100.cuh").read_text()


@pytest.mark.parametrize(("name", "end", "pair"), [("head_products", "// The map of tiles", "_pair"), ("head_few", "// ---- sums: dx and dw", "")])
def test_the_pipelines_of_the_losses_hold_their_tensor_memory(name: str, end: str, pair: str) -> None:
    """What the kernels of products run on: tensor memory is held before the next kernel may start, products end before it is freed. (Read, not run:
    nothing makes a wait run out on a healthy GPU.)"""
    body = HEAD[HEAD.index(f"void {name}(") : HEAD.index(end)]
    assert body.count(f"tmem_alloc{pair}(") == body.count(f"tmem_dealloc{pair}(") == 1
    assert body.index(f"tmem_alloc{pair}(") < body.index("grid_launch_dependents();")
    drained, freed = body.index(f"umma_commit{pair}(&sm.drain)"), body.index(f"tmem_dealloc{pair}(")
    assert drained < body.index("mbar_wait(&sm.drain", drained) < freed
    landed = body.index("for (int j = (g > ")  # copies in flight when a loader gives up
    assert landed < body.index("mbar_wait(&sm.full[j %", landed) < freed


def test_a_pair_of_ctas_waits_for_the_last_signals_of_the_other() -> None:
    body = HEAD[HEAD.index("void head_products(") : HEAD.index("// The map of tiles")]
    assert body.index("mbar_wait(&sm.acc_empty[lane]") < body.index("tmem_dealloc_pair(")


def test_the_kernels_of_products_by_name() -> None:
    kernels = re.findall(r"__global__ [^{]*?(head_\w+_kernel)\(", HEAD)
    on = {k: re.findall(r"head_products\(|head_few<", HEAD[HEAD.index(f"{k}(const") : HEAD.index("\n}", HEAD.index(f"{k}(const"))]) for k in kernels}
    assert {k: v[0] for k, v in on.items() if v} == {
        "head_stats_kernel": "head_products(", "head_few_kernel": "head_few<", "head_grads_kernel": "head_products(", "head_sums_kernel": "head_products(",
    }  # fmt: skip


def test_rows_on_their_way_land_before_a_layer_norm_that_gives_up_ends() -> None:
    text = (ROOT / "fastforks_b200" / "csrc" / "layer_norm_sm100.cuh").read_text()
    body = text[text.index("norm_ring_grad_kernel(const") :]
    assert body.index("ring.drain(&sm.abort);") < body.index("joined = ")
    assert "mbar_wait(&full[i]" in text[text.index("void drain(") : text.index("__device__ __forceinline__ LnRing ln_ring(")]
