"""The packed forward kernel over pages of 8 bits as it hands over probabilities in two parts, model-checked like
test_paged8_protocol.py, whose producer and converting warps it takes over.

What FP16 leaves of a step's probabilities lies in the place of its scores, so that the next step's scores have to wait for the
product with V. The model lets products of either kind overtake each other (only a commit waits for what was issued before it) and shows a
block's scales to no warp that has not waited for them.
"""

import random
import re

import pytest

import test_warp_waits
from test_paged8_protocol import CASES, PIECES, SCALES, SLOTS, WARPS, Eight, Violation, need


class TwoParts(Eight):
    def __init__(self, pieces, seed, variant="kernel", few=False):
        super().__init__(pieces, seed, variant)
        self.few = few                     # several copies of a tile's rows: scores are read once, and zeros fill up P
        self.rng = random.Random(seed)
        self.has_read = set()              # (step, quadrant, half)

    def mma(self):
        tiles = iter(range(2 * len(self.steps)))
        issued, claimed = [0], [None]

        def tile(kind, n):
            k = next(tiles)
            s = k % SLOTS
            yield from self.wait(("slot_full", s), k // SLOTS)
            need(self.slot[s] == (kind, n), f"slot {s} holds {self.slot[s]}, not {kind} {n}")
            self.slot_readers[s] += 1
            return s

        def claim(n):
            claimed[0] = None
            r, j = self.steps[n] if n < len(self.steps) else (len(self.pieces), 0)
            if j == 0:
                yield from self.wait(("piece_full", r % PIECES), r // PIECES)
                need(self.ring[r % PIECES] == r, "another piece's description")
            if n == len(self.steps):
                return
            if j == 0:
                yield from self.wait(("q_full", r & 1), r >> 1)
                need(self.q[r & 1] == r, "another piece's queries")
            claimed[0] = yield from tile("k", n)

        def scores():
            if claimed[0] is None:
                return
            n = issued[0]
            r, j = self.steps[n]
            if n > 0 and self.variant != "no_values_done":
                yield from self.wait("pv_done", n - 1)
            self.q_readers[r & 1] += 1
            self.pipe += [("scores", n, claimed[0], r & 1), ("commit", "s_full"), ("commit", ("slot_empty", claimed[0]))]
            if j + 1 == self.pieces[r]:
                self.pipe.append(("commit", ("q_empty", r & 1)))
            issued[0] += 1

        yield from claim(0)
        yield from scores()
        n = 0
        while n < issued[0]:
            yield from claim(n + 1)
            s = yield from tile("v", n)
            if self.variant != "no_p_ready":
                yield from self.wait("p_ready", n)
            self.pipe += [("values", n, s), ("commit", "pv_done"), ("commit", ("slot_empty", s))]
            yield from scores()
            n += 1
            yield

    def softmax(self, quadrant, half):
        n, met = 0, 0
        seen = [0] * SCALES                # phases of each entry's barrier that this warp has waited for

        def meet():
            nonlocal met
            self.bar["pair", quadrant].arrive()
            if self.variant != "no_meeting":
                yield from self.wait(("pair", quadrant), met)
            met += 1

        def scales():
            need(seen[n % SCALES] == n // SCALES + 1, "scales that this warp has not waited for")
            need(self.scales[n % SCALES] == n, f"scales of step {self.scales[n % SCALES]}, not {n}")

        for r in range(len(self.pieces) + 1):
            yield from self.wait(("piece_full", r % PIECES), r // PIECES)
            need(self.ring[r % PIECES] == r, f"description of piece {self.ring[r % PIECES]}, not {r}")
            if r == len(self.pieces):
                return
            for j in range(self.pieces[r]):
                yield from self.wait("s_full", n)
                phase = n // SCALES - (1 if self.variant == "scales_a_phase_early" else 0)
                if phase >= 0 and self.variant != "no_scales_full":
                    yield from self.wait(("scales_full", n % SCALES), phase)
                    seen[n % SCALES] = phase + 1
                need(self.scores_of == n, f"scores of step {self.scores_of}, not {n}")
                scales()
                yield
                if self.few:
                    self.has_read.add((n, quadrant, half))
                self.maxima[n & 1, quadrant, half] = n
                yield from meet()
                need(self.maxima.get((n & 1, quadrant, 1 - half)) == n, "the other half's maximum of another step")
                if n > 0 and self.variant != "no_pv_done":
                    yield from self.wait("pv_done", n - 1)
                yield
                need(self.scores_of == n, "scores overwritten before their second reading")
                scales()
                self.has_read.add((n, quadrant, half))
                need(n == 0 or n - 1 in self.values_done, f"P of step {n} over step {n - 1}'s")
                if self.few:
                    need((n, quadrant, 1 - half) in self.has_read, "scores overwritten before the other half has read them")
                yield
                self.scale_reads[n] = self.scale_reads.get(n, 0) + 1
                self.wrote_p[n] = self.wrote_p.get(n, 0) + 1
                self.bar["p_ready"].arrive()
                n += 1
                yield
            yield from self.wait("pv_done", n - 1)
            need(n - 1 in self.values_done and n not in self.values_done, "O read too early or too late")
            yield
            self.o_read[r] = self.o_read.get(r, 0) + 1
            yield from meet()

    def step_pipe(self):
        """One product, or the commits at the head of the line."""
        if self.pipe[0][0] == "commit":
            self.bar[self.pipe.pop(0)[1]].arrive()
            return
        kind = self.rng.choice(sorted({op[0] for op in self.pipe} - {"commit"}))
        op = self.pipe.pop(next(i for i, op in enumerate(self.pipe) if op[0] == kind))
        if kind == "scores":
            _, n, s, b = op
            need(n == 0 or n - 1 in self.values_done, f"scores of step {n} over the probabilities before")
            self.scores_of = n
            self.q_readers[b] -= 1
        else:
            _, n, s = op
            need(self.wrote_p.get(n, 0) == WARPS, f"P of step {n} used before it is whole")
            need(self.scores_of == n, "the second part of P overwritten")
            r, j = self.steps[n]
            need(j > 0 or r == 0 or self.o_read.get(r - 1, 0) == WARPS, "O overwritten before it is read")
            self.values_done.add(n)
        self.slot_readers[s] -= 1

    def run(self):
        roles = [self.producer(), self.converter(0), self.converter(1), self.mma(),
                 *(self.softmax(q, h) for q in range(4) for h in range(2))]
        idle = 0
        while roles or self.tma or self.pipe:
            choice = self.rng.random()
            before = (len(self.tma), len(self.pipe), [b.completed for b in self.bar.values()])
            if self.tma and choice < 0.2:
                name, land = self.tma.pop(self.rng.randrange(len(self.tma)))
                land()
                self.bar[name].arrive()
            elif self.pipe and choice < 0.4:
                self.step_pipe()
            elif roles:
                role = self.rng.choice(roles)
                try:
                    next(role)
                except StopIteration:
                    roles.remove(role)
            after = (len(self.tma), len(self.pipe), [b.completed for b in self.bar.values()])
            idle = 0 if before != after else idle + 1
            need(idle < 20000, "deadlock")
        need(len(self.values_done) == len(self.steps), "steps left out")


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("pieces", CASES, ids=str)
def test_every_schedule_finds_its_data(pieces, few):
    for seed in range(40):
        TwoParts(pieces, seed, few=few).run()


@pytest.mark.parametrize("variant", ["no_raw_empty", "no_slot_empty", "no_scales_full", "scales_a_phase_early", "no_values_done",
                                     "no_p_ready", "no_meeting"])
def test_planted_mistakes_are_found(variant):
    found = 0
    for seed in range(120):
        try:
            TwoParts([9, 2, 4], seed, variant, few=True).run()
        except Violation:
            found += 1
    assert found > 0


def test_the_kernel_has_the_models_order():
    """Keys claimed, the product with V issued behind the probabilities, then the next scores behind that product."""
    text = (test_warp_waits.CSRC / "packed_forward.cu").read_text()
    issue = text[text.index("auto issue_scores = "):text.index("} else if (kEight && warp < kFirstSoftmax)")]
    steps = re.findall(r"kEight \? bar\.pv_done\(\) : bar\.s_free\(\)|mma_commit\(bar\.s_full\(\)\)|\bclaim\(\);|\bissue_scores\(\);"
                       r"|if \(!?kEight\)|bar\.p_ready\(\)|mma_f16_ts_at<1>\(tmem_o, tmem_[ps]|mma_commit\(bar\.pv_done\(\)\)", issue)
    assert steps == ["kEight ? bar.pv_done() : bar.s_free()", "mma_commit(bar.s_full())", "claim();", "issue_scores();",
                     "claim();", "if (!kEight)", "issue_scores();", "bar.p_ready()", "mma_f16_ts_at<1>(tmem_o, tmem_p",
                     "if (kEight)", "mma_f16_ts_at<1>(tmem_o, tmem_s", "mma_commit(bar.pv_done())", "if (kEight)",
                     "issue_scores();"]
