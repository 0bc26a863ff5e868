"""Beam selection against 64 bits on the host: every candidate of a group, sorted."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
INF = float("inf")


class Step:
    def __init__(self, groups, beams, vocab, cols=None, fp32=True, seed=0, end=-1, power=0.0, history=None):
        self.groups, self.beams, self.vocab, self.fp32, self.end, self.power = groups, beams, vocab, fp32, end, power
        self.cols = cols or (vocab + 7) // 8 * 8
        self.rows = rows = groups * beams
        g = torch.Generator().manual_seed(seed)
        self.logits = torch.randn(rows, self.cols, generator=g).mul(3).to(torch.float32 if fp32 else torch.half)
        self.logits[:, vocab:] = INF          # columns that do not count
        self.scores = -torch.rand(rows, generator=g) * 5
        self.finished = self.lengths = self.histories = None
        if end >= 0:
            self.finished = (torch.rand(rows, generator=g) < 0.3).to(torch.int32)
        if history or power:
            self.lengths = torch.randint(0, history or 50, (rows,), generator=g, dtype=torch.int32)
        if history:
            self.histories = torch.randint(0, 60000, (rows, history), generator=g, dtype=torch.int32)

    def buffers(self):
        whole = lambda *shape: torch.full(shape, -7, dtype=torch.int32, device=DEV)
        return [torch.full((self.rows,), 7.0, device=DEV), whole(self.rows),
                whole(self.rows).to(torch.uint16), whole(self.rows) if self.finished is not None else None,
                whole(self.rows) if self.lengths is not None else None,
                torch.full(self.histories.shape, 9, dtype=torch.int32, device=DEV).to(torch.uint16)
                if self.histories is not None else None]

    def inputs(self):
        moved = lambda t: None if t is None else t.to(DEV)
        histories = None if self.histories is None else self.histories.to(torch.uint16).to(DEV)
        return [moved(self.logits), moved(self.scores), moved(self.finished), moved(self.lengths), histories]

    def call(self, flint, out=None, given=None, workspace=None, stream=None):
        out, given = out or self.buffers(), given or self.inputs()
        if workspace is None:
            workspace = torch.full((flint.beam_select_workspace(self.groups, self.beams),), 255, dtype=torch.uint8, device=DEV)
        flint.beam_select(*out, *given, self.fp32, self.groups, self.beams, self.vocab, self.cols,
                          self.histories.shape[1] if self.histories is not None else 0, self.end, self.power, workspace,
                          stream=stream)
        return out

    def want(self):
        """Per row: (total, parent, token), and ranks that are too close to tell."""
        rows = []
        x = self.logits[:, :self.vocab].double()
        log_p = torch.log_softmax(x, 1)
        bad = x.isnan().any(1) | (x == INF).any(1)
        for g in range(self.groups):
            found = []
            for b in range(self.beams):
                row = g * self.beams + b
                score = self.scores[row].double().item()
                if not math.isfinite(score):
                    continue
                length = self.lengths[row].item() if self.lengths is not None else 0
                if self.finished is not None and self.finished[row]:
                    found.append((score / max(length, 1) ** self.power, score, b, max(self.end, 0)))
                elif not bad[row]:
                    totals = score + log_p[row]
                    for c in torch.topk(totals, min(self.beams, self.vocab)).indices.tolist():
                        found.append((totals[c].item() / (length + 1) ** self.power, totals[c].item(), b, c))
                    # (topk leaves open which of equal ones it takes: all of them.)
                    least = torch.topk(totals, min(self.beams, self.vocab)).values[-1]
                    for c in (totals == least).nonzero()[:, 0].tolist()[:self.beams]:
                        found.append((totals[c].item() / (length + 1) ** self.power, totals[c].item(), b, c))
            found = sorted({f for f in found if f[0] > -INF}, key=lambda f: (-f[0], f[2], f[3]))
            for place in range(self.beams):
                if place < len(found):
                    rows.append((*found[place][1:], found[place][0]))
                else:
                    row = g * self.beams + place
                    over = self.finished is not None and bool(self.finished[row])
                    rows.append((-INF, place, max(self.end, 0) if over else 0, -INF))
        return rows

    def check(self, out):
        scores, parents, tokens, finished, lengths, histories = [None if t is None else t.cpu() for t in out]
        tokens = tokens.to(torch.int32)
        histories = None if histories is None else histories.to(torch.int32)
        for row, (total, parent, token, _) in enumerate(self.want()):
            parent += row // self.beams * self.beams
            assert (parents[row].item(), tokens[row].item()) == (parent, token), row
            # One rounding to FP32, of a total whose lse is off by some of FP32's roundings of its size.
            assert scores[row].item() == total or abs(scores[row].item() - total) <= 2.0 ** -22 * (abs(total) + 20), row
            over = self.finished is not None and bool(self.finished[parent])
            if finished is not None:
                assert finished[row].item() == int(over or token == self.end)
            if lengths is not None:
                length = self.lengths[parent].item()
                full = histories is not None and length == self.histories.shape[1]
                assert lengths[row].item() == (length if over or full else length + 1)
            if histories is not None:
                line = [9] * self.histories.shape[1]
                line[:length] = self.histories[parent][:length].tolist()
                if not over and not full:
                    line[length] = token
                assert histories[row].tolist() == line, row


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("groups, beams, vocab, cols", [
    (1, 1, 1, 8), (1, 1, 50257, 50304), (3, 4, 3, 8), (2, 8, 500, 504), (5, 5, 1000, 1000), (1, 32, 32, 32),
    (2, 32, 65536, 65536), (7, 31, 4099, 4112), (1, 4, 50257, 50304), (300, 2, 777, 800), (40, 8, 20011, 20016),
    (150, 6, 9001, 9008)])
def test_sizes(flint, fp32, groups, beams, vocab, cols):
    step = Step(groups, beams, vocab, cols, fp32, seed=vocab)
    if not fp32:
        # (Ties between beams are as good as none, ties within a beam common.)
        step.scores += torch.arange(step.rows) * 1e-3
    step.check(step.call(flint))
    assert not flint.kernel_fault()


@pytest.mark.parametrize("fp32, vocab", [(False, 36000), (True, 20000)])
def test_many_rows_in_one_part_each(flint, fp32, vocab):
    """20,000 rows: a warp has a whole one, whose maxima are noted for two chunks together. Some groups are checked."""
    groups, beams = 10000, 2
    g = torch.Generator(device=DEV).manual_seed(5)
    logits = torch.empty(groups * beams, vocab, dtype=torch.float32 if fp32 else torch.half, device=DEV)
    for part in logits.split(1000):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV) * 3)
    scores = torch.rand(groups * beams, generator=g, device=DEV) * -5
    whole = Step(1, 2, 8)
    whole.groups, whole.rows, whole.vocab, whole.cols, whole.fp32 = groups, groups * beams, vocab, vocab, fp32
    out = whole.call(flint, given=[logits, scores, None, None, None])
    for at in [0, 1, 4999, 9998, 9999, *range(37, 10000, 997)]:
        rows = slice(at * beams, (at + 1) * beams)
        one = Step(1, beams, vocab, vocab, fp32)
        one.logits, one.scores = logits[rows].cpu(), scores[rows].cpu()
        one.check([out[0][rows], out[1][rows] - at * beams, out[2][rows], None, None, None])


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("power", [0.0, 0.6, 1.0, 2.5])
@pytest.mark.parametrize("groups, beams, vocab", [(9, 4, 3000), (3, 20, 12007)])
def test_finished_beams_lengths_and_histories(flint, fp32, power, groups, beams, vocab):
    for seed in range(3):
        step = Step(groups, beams, vocab, None, fp32, seed, end=vocab // 3, power=power, history=61)
        step.logits[::3, vocab // 3] = 9.0        # the end is likely
        step.check(step.call(flint))
    assert not flint.kernel_fault()


def test_all_finished(flint):
    step = Step(2, 5, 100, end=7, history=20)
    step.finished.fill_(1)
    step.logits.fill_(float("nan"))     # (of rows that are not read)
    step.check(step.call(flint))


def test_finished_without_an_end(flint):
    step = Step(6, 4, 400, end=7, history=20)
    step.end = -1
    step.check(step.call(flint))


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("vocab", [40, 3001, 50257])
def test_equal_logits(flint, fp32, vocab):
    """The lowest tokens of the lowest beams, whether few or all are equal."""
    step = Step(3, 6, vocab, None, fp32)
    step.logits[:, :vocab] = 1.5
    step.scores[:] = torch.arange(step.rows) % 6 * -0.25
    step.scores[1] = step.scores[0]
    out = step.call(flint)
    assert out[1].view(3, 6)[2].tolist() == [12] * 6 and out[2].to(torch.int32)[12:].tolist() == list(range(6))
    assert out[1].view(3, 6)[0].tolist() == [0] * 6
    step.check(out)
    step.logits[:, :vocab:3] = 2.0
    step.check(step.call(flint))


@pytest.mark.parametrize("fp32", [False, True])
def test_first_step(flint, fp32):
    """Beams that are not in use give no continuations."""
    step = Step(4, 5, 2000, None, fp32)
    step.scores.view(4, 5)[:, 1:] = -INF
    step.check(step.call(flint))


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("allowed", [0, 1, 3])
def test_tokens_that_cannot_come(flint, fp32, allowed):
    """Fewer continuations than beams: the places left keep their beams at minus infinity."""
    step = Step(5, 4, 3000, None, fp32, end=2, history=9)
    step.finished[:] = 0
    step.finished[1] = 1
    step.lengths.clamp_(max=8)
    keep = torch.rand(step.rows, 3000).argsort(1)[:, :allowed]
    masked = torch.full_like(step.logits, -INF)
    masked.scatter_(1, keep, step.logits.gather(1, keep))
    masked[4:8] = -INF
    masked[4, 17] = 1.0
    step.logits = masked
    step.check(step.call(flint))
    step.scores[:] = -INF
    step.check(step.call(flint))


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), INF])
@pytest.mark.parametrize("vocab", [300, 40000])
def test_rows_that_are_not_numbers(flint, fp32, bad, vocab):
    step = Step(4, 3, vocab, None, fp32)
    step.logits[1, vocab - 1] = bad
    step.logits[3:6, 5] = bad
    step.scores[7], step.scores[8] = float("nan"), INF
    step.check(step.call(flint))


@pytest.mark.parametrize("fp32", [False, True])
def test_logits_far_from_zero(flint, fp32):
    step = Step(3, 4, 5000, None, fp32)
    step.logits[:4, :5000] -= 60000.0
    step.logits[4:8, :5000] += 30000.0
    step.logits[8, :5000] = -65504.0
    step.scores += torch.arange(12) * 0.01
    step.logits[::2, 100:2000] = -INF
    # An lse of 60,000 is off by FP32's roundings of that size.
    out = [t if t is None else t.cpu() for t in step.call(flint)]
    for row, (total, parent, token, _) in enumerate(step.want()):
        assert (out[1][row].item() % 4, out[2].to(torch.int32)[row].item()) == (parent, token)
        assert abs(out[0][row].item() - total) <= 2.0 ** -22 * (abs(total) + 20)


@pytest.mark.parametrize("power", [3.0, 16.0])
def test_long_lengths_and_large_powers(flint, power):
    step = Step(3, 4, 300, end=5, power=power)
    step.lengths[:] = torch.tensor([0, 1, 2, 3, 1000, 999, 1001, 1 << 20, (1 << 31) - 2, (1 << 31) - 3, 1, 0])
    step.finished[:] = 0
    step.finished[[0, 7]] = 1
    flint.kernel_fault()
    out = step.call(flint)
    assert not flint.kernel_fault()
    for row, (total, parent, token, _) in enumerate(step.want()):
        assert (out[1][row].item() % 4, out[2].to(torch.int32)[row].item()) == (parent, token), row
    assert out[4].to(torch.int64).min().item() >= 0
    step.lengths[8] = (1 << 31) - 1
    step.call(flint)
    assert flint.kernel_fault()


def test_full_histories_are_reported(flint):
    step = Step(2, 3, 100, end=5, history=6)
    step.lengths[:] = torch.tensor([6, 2, 5, 6, 6, 0])
    step.finished[:] = 0
    step.finished[4] = 1
    flint.kernel_fault()
    step.check(step.call(flint))
    assert flint.kernel_fault()
    step.lengths[0] = 7
    step.call(flint)
    assert flint.kernel_fault()
    step.lengths[0] = -1
    step.call(flint)
    assert flint.kernel_fault()


@pytest.mark.parametrize("groups, beams, vocab, fp32", [(1, 4, 50257, True), (50, 8, 30000, False)])
def test_results_repeat_and_replay(flint, groups, beams, vocab, fp32):
    step = Step(groups, beams, vocab, None, fp32, end=3, power=0.6, history=40)
    out, given = step.buffers(), step.inputs()
    workspace = torch.empty(flint.beam_select_workspace(groups, beams), dtype=torch.uint8, device=DEV)
    want = [t.clone() for t in step.call(flint, out, given, workspace)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step.call(flint, out, given, workspace)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        for t in out[:2]:
            t.zero_()
        workspace.fill_(255)
        graph.replay()
        for got, old in zip(out, want):
            assert torch.equal(got, old)


def test_two_streams_at_once(flint):
    steps = [Step(20, 6, 15000, None, bool(s), seed=s) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, givens = [s.buffers() for s in steps], [s.inputs() for s in steps]
    spaces = [torch.empty(flint.beam_select_workspace(20, 6), dtype=torch.uint8, device=DEV) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for step, stream, out, given, space in zip(steps, streams, outs, givens, spaces):
            step.call(flint, out, given, space, stream=stream)
    torch.cuda.synchronize()
    for step, out in zip(steps, outs):
        step.check(out)
