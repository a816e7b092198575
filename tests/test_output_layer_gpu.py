"""The example's step on the last norm and the output layer runs, and its gradients are those of 64 bits.

Roundings to bfloat16 follow one another: the normed rows, each loss's gradients for them, their sum, and the results; a rounding is off by 2^-8 / sqrt(3)
of a value at most, in the mean, and none helps another."""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

import fastforks_b200 as ff

pytestmark = pytest.mark.gpu
sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))


@pytest.mark.parametrize(("batch", "tokens", "vocabulary"), [(1, 9, 77), (3, 100, 1000)])
def test_the_gradients_of_the_output_layer(batch: int, tokens: int, vocabulary: int) -> None:
    import token_decoder

    r = token_decoder.output_layer(token_decoder.Config(), batch, tokens, vocabulary)
    assert ff.device_status() == 0
    leaves = [r[name].detach().double().requires_grad_(True) for name in ("norm", "shift", "head")]
    x = torch.nn.functional.layer_norm(r["states"].double(), r["states"].shape[-1:], leaves[0], leaves[1], 1e-5)
    logits = (x @ leaves[2].T).flatten(0, 1)
    ce = torch.nn.functional.cross_entropy(logits, r["targets"].flatten())
    ids = r["teacher_ids"].flatten(0, 1)
    counts = ids[:, 0] >= 0
    p, logq = torch.softmax(r["teacher_logits"].flatten(0, 1)[counts].double() / 2, 1), torch.log_softmax(logits[counts] / 2, 1)
    loss = ce + 0.5 * 4 * (p * (p.log() - logq.gather(1, ids[counts]))).sum(1).mean()
    # the normed rows' rounding moves a logit by 2^-8 / sqrt(3) of its size (about 1 here) at most, a row's loss by a few times that
    assert abs(float(r["loss"]) - float(loss.detach())) < 4 * 2.0**-8
    for name, want in zip(("norm", "shift", "head"), torch.autograd.grad(loss, leaves), strict=True):
        got = r[f"d{name}"].double()
        assert float((got - want).norm() / want.norm()) < 6**0.5 * 2.0**-8 / 3**0.5, name
