"""Operands of the forward operators that torch keeps with a sign to be turned later (the imaginary part of a conjugate) count with their values, on the full way
and on the way of repeated calls; what is written to is refused with one. (The differentiable operators: tests/test_training_edges_gpu.py.)"""

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


def negated(t: torch.Tensor) -> torch.Tensor:
    view = torch._neg_view(-t)  # noqa: SLF001
    assert view.is_neg()
    return view


def calls() -> dict:
    """Name -> a call, its operands."""
    x, w, b, s = normal(32, 64), normal(64, 64, seed=1), normal(64, seed=2), normal(64, dtype=torch.float32, seed=3)
    q, k, v = (normal(2, 16, 4, 64, seed=i) for i in (4, 5, 6))
    bias, rel = normal(2, 4, 16, 16, seed=7), (normal(2, 4, 16, 4, seed=8), normal(2, 4, 16, 4, seed=9))
    kv_k, kv_v, table = normal(2, 16, 2, 64, seed=10), normal(2, 16, 2, 64, seed=11), ff.rotary_table(16, 64, device="cuda")
    pages, lengths = torch.arange(2, dtype=torch.int32, device="cuda")[:, None], torch.full((2,), 16, dtype=torch.int32, device="cuda")
    qkv, cs = normal(2, 17, 3, 4, 64, seed=12), ff.rope_table(4, 4, device="cuda")
    filled = ff.kv4_cache(2, 2, 64, page=16)
    ff.kv4_append_(filled, kv_k, kv_v, pages, lengths)

    def append(a: torch.Tensor, b: torch.Tensor, c: torch.Tensor, t: torch.Tensor) -> tuple[torch.Tensor, ...]:
        cache = ff.kv4_cache(2, 2, 64, page=16)
        turned = ff.kv4_append_(cache, a, b, pages, lengths, table=t, q=c)
        return turned, *ff.kv4_read(cache, pages, lengths, 16, torch.float16)

    return {
        "gemm": (lambda x, w, b, s, r: ff.gemm(x, w, b, scale=s, res=r), (x, w, b, s, x[:, :])),
        "attention": (lambda q, k, v: ff.attention(q, k, v, layout="bnhd"), (q, k, v)),
        "attention with a bias": (lambda q, k, v, m: ff.attention(q, k, v, layout="bnhd", bias=m), (q, k, v, bias)),
        "attention with relative positions": (lambda q, k, v, h, w: ff.attention(q, k, v, layout="bnhd", rel=(h, w)), (q, k, v, *rel)),
        "rope": (lambda t: ff.rope_qk_(qkv.clone(), t), (cs,)),
        "append": (append, (kv_k, kv_v, q, table)),
        "cache attention": (lambda t: ff.kv4_attention(t, filled, pages, lengths), (q,)),
        "relative terms": (lambda q, h, w: ff.sam_rel_terms(q, h, w, 4), (q, normal(7, 64, seed=13), normal(7, 64, seed=14))),
    }


@pytest.mark.usefixtures("way")
@pytest.mark.parametrize("name", ["gemm", "attention", "attention with a bias", "attention with relative positions", "rope", "append", "cache attention", "relative terms"])
def test_operands_count_with_their_values(name: str) -> None:
    call, operands = calls()[name]
    want = call(*operands)
    for i in range(len(operands)):
        got = call(*(negated(t) if j == i else t for j, t in enumerate(operands)))
        for a, b in zip(*((t,) if isinstance(t, torch.Tensor) else t for t in (got, want)), strict=True):
            assert torch.equal(a, b), i
    assert ff.device_status() == 0


@pytest.mark.usefixtures("way")
def test_what_is_written_to_is_refused() -> None:
    x, w = normal(32, 64), normal(64, 64, seed=1)
    heads, kv, table = normal(2, 16, 4, 64), normal(2, 16, 2, 64), ff.rotary_table(16, 64, device="cuda")
    cache, pages, lengths = ff.kv4_cache(2, 2, 64, page=16), torch.arange(2, dtype=torch.int32, device="cuda")[:, None], torch.full((2,), 16, dtype=torch.int32, device="cuda")
    qkv, cs = normal(2, 17, 3, 4, 64, seed=12), ff.rope_table(4, 4, device="cuda")
    for call in (
        lambda: ff.gemm(x, w, out=negated(x)),
        lambda: ff.attention(heads, heads, heads, layout="bnhd", out=negated(heads)),
        lambda: ff.rope_qk_(negated(qkv), cs),
        lambda: ff.kv4_append_(cache, kv, kv, pages, lengths, table=table, q=heads, out=negated(heads)),
        lambda: ff.kv4_attention(heads, cache, pages, lengths, out=negated(heads)),
    ):
        with pytest.raises(ValueError, match="negat"):
            call()
