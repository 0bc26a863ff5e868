"""Beams whose totals divided by a power of their length are equal: by beam, and by nothing else."""

import pytest
import torch

from test_beams_gpu import DEV, Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [1, 2, 3])
@pytest.mark.parametrize("lengths", [[1, 49], [49, 1], [3, 98, 1, 49, 5, 7, 41, 47], [60, 59, 58, 57, 56, 55, 54, 53, 52, 51, 50, 49, 48, 47],
                                     list(range(1, 33))], ids=len)
def test_equal_quotients(flint, power, lengths):
    """Finished beams of the scores -3 length^power, which are FP32 numbers: their ranks are -3, exactly. (The quotient of two FP64
    numbers is exact where there is an exact one.) A reciprocal in the quotient's place is off for 49, among others."""
    beams = len(lengths)
    step = Step(2, beams, 40, end=5, power=float(power), history=100)
    step.finished.fill_(1)
    step.lengths[:] = torch.tensor(lengths * 2)
    step.scores[:] = -3.0 * step.lengths.double() ** power
    step.scores[beams:] *= torch.linspace(1.5, 0.5, beams)[torch.randperm(beams, generator=torch.Generator().manual_seed(power))]
    out = step.call(flint)
    assert out[1][:beams].tolist() == list(range(beams))
    step.check(out)


@pytest.mark.parametrize("fp32", [False, True])
def test_equal_quotients_among_continuations(flint, fp32):
    """Beams of the same logits that go on, one of them finished already: a total of a length's multiple against one of another's."""
    step = Step(1, 3, 8, 8, fp32, end=7, power=1.0, history=100)
    step.logits[:] = 0.0                    # every token's log-probability is -log 8
    step.logits[:, 1:] = float("-inf")      # and here 0
    step.finished[:] = torch.tensor([0, 1, 0], dtype=torch.int32)
    step.lengths[:] = torch.tensor([48, 7, 97], dtype=torch.int32)
    step.scores[:] = torch.tensor([-98.0, -14.0, -196.0])
    out = step.call(flint)
    assert out[1].tolist() == [0, 1, 2] and out[4].tolist() == [49, 7, 98]
    assert out[0].tolist() == [-98.0, -14.0, -196.0]
