"""The example of a token decoder runs, its ways of decoding agree and its gradient step does what a gradient says.

Two ways of decoding write the same cache and differ by the rounding of attention's weights and of layers in bfloat16: a few units of
2^-8 in each of two layers' four products, 0.03 of the result's norm at most."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest

import fastforks_b200 as ff

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


@pytest.mark.parametrize(("batch", "prompt", "steps"), [(1, 5, 3), (4, 100, 16)])
def test_decoding(batch: int, prompt: int, steps: int) -> None:
    import token_decoder

    assert token_decoder.decode(token_decoder.Config(), batch, prompt, steps) < 0.03  # noqa: PLR2004
    assert ff.device_status() == 0


def test_learning() -> None:
    import token_decoder

    before, after = token_decoder.learn(token_decoder.Config())
    assert 0.5e-3 < before - after < 1.5e-3
    assert ff.device_status() == 0
