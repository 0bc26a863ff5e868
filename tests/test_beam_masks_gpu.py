"""Beam selection where many logits are equal: tokens that may not come at a finite number, few left that may."""

import pytest
import torch

from test_beams_gpu import DEV, Step

pytestmark = pytest.mark.gpu


def masked(step, allowed, fill, seed=0):
    """Of each row `allowed` tokens keep their logits."""
    keep = torch.rand(step.rows, step.vocab, generator=torch.Generator().manual_seed(seed)).argsort(1)[:, :allowed]
    low = torch.full_like(step.logits, fill)
    low.scatter_(1, keep, step.logits.gather(1, keep))
    low[:, step.vocab:] = float("inf")
    step.logits = low
    return step


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("fill", ["lowest", -1e4])
@pytest.mark.parametrize("allowed", [0, 1, 5, 40, 300])
@pytest.mark.parametrize("groups, beams, vocab", [(2, 6, 9001), (3, 31, 4099), (1, 4, 50257), (1, 32, 65536)])
def test_masks_of_a_finite_number(flint, fp32, fill, allowed, groups, beams, vocab):
    step = Step(groups, beams, vocab, None, fp32, seed=allowed)
    masked(step, allowed, torch.finfo(step.logits.dtype).min if fill == "lowest" else fill)
    step.check(step.call(flint))
    assert not flint.kernel_fault()


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("levels", [1, 2, 3, 17])
@pytest.mark.parametrize("groups, beams, vocab", [(2, 7, 20011), (4, 32, 3000), (1, 13, 65529)])
def test_few_different_values(flint, fp32, levels, groups, beams, vocab):
    """Every level has many tokens; the highest few, some rows fewer than beams."""
    step = Step(groups, beams, vocab, None, fp32)
    g = torch.Generator().manual_seed(levels)
    at = (torch.rand(step.rows, step.cols, generator=g) ** 0.25 * levels).long()
    step.logits[:, :vocab] = (at.to(step.logits.dtype) * -1.5 + 3)[:, :vocab]
    for row in range(0, step.rows, 3):      # zeros of both signs are equal
        step.logits[row, :vocab][step.logits[row, :vocab] == 3] = 0.0
        step.logits[row, 1:vocab:7] = -0.0
    step.check(step.call(flint))


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("places", ["ascending", "descending", "last"])
def test_values_that_rise_behind_equal_ones(flint, fp32, places):
    """The bound is one that many have; behind them come more values above it than there is room for at a time."""
    step = Step(2, 32, 30000, None, fp32)
    step.logits[:, :30000] = -5.0
    rise = torch.linspace(-4, 4, 700)
    if places == "ascending":
        step.logits[:, 20000:20700] = rise
    elif places == "descending":
        step.logits[:, 10000:10700] = rise.flip(0)
    else:
        step.logits[:, 29300:30000] = 2.0
        step.logits[:, 29990:30000] = 3.0
    step.check(step.call(flint))


def best_time(call):
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(5):
            call()
    times = []
    for _ in range(6):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        times.append(begin.elapsed_time(end))
    return min(times)


def test_masked_rows_take_no_pass_per_beam(flint):
    """31 beams of 1,240 rows of 32,001 FP32 logits: one more pass over the rows, from L2, and not 31 (50 times as long)."""
    step = Step(40, 31, 32001, 32008)
    out, given = step.buffers(), step.inputs()
    workspace = torch.empty(flint.beam_select_workspace(40, 31), dtype=torch.uint8, device=DEV)
    ordinary = best_time(lambda: step.call(flint, out, given, workspace))
    given[0] = masked(step, 3, torch.finfo(torch.float32).min).logits.to(DEV)
    assert best_time(lambda: step.call(flint, out, given, workspace)) < 6 * ordinary
