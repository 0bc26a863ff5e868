"""Beam selection over logits so large that their log-sum-exp is their maximum even in 64 bits: the differences still count."""

import math

import pytest
import torch

from test_beams_gpu import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("level", [torch.finfo(torch.float32).min, torch.finfo(torch.float32).max, -1e30, 2.0 ** 60])
@pytest.mark.parametrize("groups, beams, vocab", [(2, 3, 50), (1, 4, 50257), (3, 8, 4099)])
def test_rows_of_one_large_value(flint, level, groups, beams, vocab):
    """A row of nothing but the lowest number (every token masked) has equal tokens, of log-probability -log(vocab)."""
    step = Step(groups, beams, vocab)
    step.logits[:, :vocab] = level
    out = step.call(flint)
    step.check(out)
    assert abs(out[0][0].item() - (step.scores[:beams].max().item() - math.log(vocab))) < 1e-4


def test_neighbours_of_a_large_value(flint):
    """Beside 2^30 and the FP32 number below it, 2^6 less, the rest is minus 2^70."""
    step = Step(2, 4, 1000)
    step.logits[:, :1000] = -2.0 ** 70
    step.logits[:, 500] = 2.0 ** 30
    step.logits[:, 20] = 2.0 ** 30
    step.logits[:, 40] = 2.0 ** 30 - 2.0 ** 6
    out = step.call(flint)
    step.check(out)
    assert abs(out[0][0].item() - (step.scores[:4].max().item() - math.log(2))) < 1e-5
