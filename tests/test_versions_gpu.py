"""What the operators write to in place is noticed by autograd: the version of a tensor moves on with every call that writes to it, on the full way and on
the way of repeated calls, so that a gradient that needs what was there raises instead of taking what is."""

from __future__ import annotations

import pytest
import torch

import fastforks_b200 as ff
from fastforks_b200 import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["full", "repeated"])
def way(request: pytest.FixtureRequest, monkeypatch: pytest.MonkeyPatch) -> str:
    if request.param == "full":
        monkeypatch.setattr(_lib, "fast", None)
        monkeypatch.setattr(_lib, "use_fast", lambda: None)
    else:
        ff.layer_norm(torch.zeros(1, 8, device="cuda"))
        assert _lib.fast is not None
    return request.param


def normal(*shape: int, dtype: torch.dtype = torch.float16, seed: int = 0) -> torch.Tensor:
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def calls() -> dict:
    """Name -> a call, and the tensors that it writes to."""
    x, w = normal(32, 64), normal(64, 64, seed=1)
    heads, other, table = normal(2, 16, 4, 64, seed=2), normal(2, 16, 2, 64, seed=3), ff.rotary_table(16, 64, device="cuda")
    k, v, out = (normal(2, 16, 2, 64, seed=s) for s in (4, 5, 6))
    cache, pages = ff.kv4_cache(2, 2, 64, page=16), torch.arange(2, dtype=torch.int32, device="cuda")[:, None]
    lengths = torch.full((2,), 16, dtype=torch.int32, device="cuda")
    qkv, cs = normal(2, 17, 3, 4, 64, seed=7), ff.rope_table(4, 4, device="cuda")
    empty, result = torch.empty_like(heads), torch.empty_like(x)
    return {
        "gemm": (lambda: ff.gemm(x, w, out=result), [result]),
        "gemm, residual in place": (lambda: ff.gemm(x, w, res=x, out=x), [x]),
        "attention": (lambda: ff.attention(heads, heads, heads, layout="bnhd", out=empty), [empty]),
        "rope": (lambda: ff.rope_qk_(qkv, cs), [qkv]),
        "rotary": (lambda: ff.rotary(heads, table, out=heads), [heads]),
        "norm and rotary": (lambda: ff.qk_norm_rotary(heads, other, None, None, table, out=(heads, other)), [heads, other]),
        "append": (lambda: ff.kv4_append_(cache, k, v, pages, lengths), [cache]),
        "append with queries": (lambda: ff.kv4_append_(cache, k, v, pages, lengths, table=table, q=heads, out=heads), [cache, heads]),
        "cache attention": (lambda: ff.kv4_attention(heads, cache, pages, lengths, out=empty), [empty]),
        "layer norm": (lambda: ff.layer_norm(x, out=result), [result]),
    }


@pytest.mark.usefixtures("way")
@pytest.mark.parametrize("name", ["gemm", "gemm, residual in place", "attention", "rope", "rotary", "norm and rotary", "append", "append with queries", "cache attention", "layer norm"])
def test_the_version_moves_on(name: str) -> None:
    call, written = calls()[name]
    for _ in range(3):
        before = [t._version for t in written]  # noqa: SLF001
        call()
        assert all(t._version > n for t, n in zip(written, before, strict=True))  # noqa: SLF001
    assert ff.device_status() == 0


@pytest.mark.usefixtures("way")
def test_a_gradient_that_needs_what_was_there_raises() -> None:
    x, w = normal(32, 64), normal(64, 64, seed=1)
    leaf = w.detach().requires_grad_(True)
    loss = ff.linear_cross_entropy(x, leaf, torch.zeros(32, dtype=torch.int64, device="cuda"))
    ff.gemm(x, w, out=x[:, :])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, leaf)


@pytest.mark.usefixtures("way")
def test_tensors_of_inference_mode_are_written_to() -> None:
    with torch.inference_mode():
        tensors = calls()
    for call, _ in tensors.values():
        call()
    assert ff.device_status() == 0
