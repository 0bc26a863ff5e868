"""The packed forward kernel's synchronisation, model-checked on the CPU, and its waits in the source.

`fb_packed_forward_tiles` (flint_b200/csrc/packed_forward.cu) hands key tiles, scores, probabilities and descriptions
of its pieces from warp to warp through mbarriers whose waits carry a phase parity only. As for the kernel
for equal lengths (test_attention_protocol.py) this file restates the protocol as cooperating generators, runs
it under random schedules with loads that complete in any order, and requires at every access that the data are those
it needs and at every wait that the phase meant has completed. Planted mistakes must be found.
"""

import random
import re

import pytest

import test_attention_protocol as attention
import test_warp_waits
from test_attention_protocol import Barrier, Violation, need

SLOTS, PIECES, WARPS = 4, 8, 8


class Model:
    def __init__(self, pieces, seed, variant="kernel"):
        self.pieces = pieces               # steps (key tiles) of each piece
        self.variant = variant
        self.rng = random.Random(seed)
        names = ["s_full", "pv_done", *((n, b) for n in ("q_full", "q_empty") for b in range(2)),
                 *(("slot_full", s) for s in range(SLOTS)), *(("slot_empty", s) for s in range(SLOTS)),
                 *(("piece_full", i) for i in range(PIECES))]
        self.bar = {n: Barrier(str(n), 1) for n in names}
        self.bar.update({n: Barrier(n, WARPS) for n in ("s_free", "p_ready")})
        self.bar.update({("pair", q): Barrier(f"pair{q}", 2) for q in range(4)})
        self.steps = [(r, j) for r, count in enumerate(pieces) for j in range(count)]
        self.ring, self.slot_readers = [None] * PIECES, [0] * SLOTS
        self.slot = [None] * SLOTS
        self.q, self.q_readers = [None, None], [0, 0]
        self.tma, self.pipe = [], []
        self.scores_of = None              # the step whose scores the buffer holds
        self.read_scores, self.wrote_p = {}, {}
        self.scores_done, self.values_done = set(), set()
        self.o_read = {}                   # piece -> warps that have read O
        self.maxima = {}                   # (step parity, quadrant, half) -> step

    def wait(self, name, phase):
        bar = self.bar[name]
        while not bar.passed(phase & 1):
            yield
        need(bar.completed > phase, f"aliased wait on {bar.name}: meant phase {phase}, {bar.completed} completed")

    def producer(self):
        at, place = [0], {}

        def load(kind, n):
            s, use = at[0] % SLOTS, at[0] // SLOTS
            if use > 0:
                yield from self.wait(("slot_empty", s), use - 1)
            need(self.slot_readers[s] == 0, f"slot {s} reloaded while read")
            self.slot[s] = None
            self.tma.append((("slot_full", s), lambda: self.slot.__setitem__(s, (kind, n))))
            at[0] += 1

        waiting = []
        for n, (r, j) in enumerate(self.steps):
            if j == 0:
                if r >= 2:
                    yield from self.wait(("q_empty", r & 1), (r >> 1) - 1)
                need(self.q_readers[r & 1] == 0, "queries reloaded while read")
                self.ring[r % PIECES] = r
                self.bar["piece_full", r % PIECES].arrive()
                self.q[r & 1] = None
                self.tma.append((("q_full", r & 1), lambda r=r: self.q.__setitem__(r & 1, r)))
                yield
            yield from load("k", n)
            waiting.append(n)
            if len(waiting) == 2:
                yield from load("v", waiting.pop(0))
            yield
        self.ring[len(self.pieces) % PIECES] = len(self.pieces)
        self.bar["piece_full", len(self.pieces) % PIECES].arrive()
        for n in waiting:
            yield from load("v", n)

    def mma(self):
        at, issued = [0], [0]

        def tile(kind, n):
            s, use = at[0] % SLOTS, at[0] // SLOTS
            yield from self.wait(("slot_full", s), use)
            need(self.slot[s] == (kind, n), f"slot {s} holds {self.slot[s]}, not {kind} {n}")
            self.slot_readers[s] += 1
            at[0] += 1
            return s

        def scores():
            n = issued[0]
            r, j = self.steps[n] if n < len(self.steps) else (len(self.pieces), 0)
            if j == 0:
                yield from self.wait(("piece_full", r % PIECES), r // PIECES)
                need(self.ring[r % PIECES] == r, "another piece's description")
            if n == len(self.steps):
                return
            if j == 0:
                yield from self.wait(("q_full", r & 1), r >> 1)
                need(self.q[r & 1] == r, "another piece's queries")
            s = yield from tile("k", n)
            if n > 0 and self.variant != "no_s_free":
                yield from self.wait("s_free", n - 1)
            self.q_readers[r & 1] += 1
            self.pipe.append(("scores", n, s, r & 1))
            self.pipe.append(("commit", "s_full"))
            self.pipe.append(("commit", ("slot_empty", s)))
            if j + 1 == self.pieces[r]:
                self.pipe.append(("commit", ("q_empty", r & 1)))
            issued[0] += 1

        yield from scores()
        n = 0
        while n < issued[0]:
            yield from scores()
            s = yield from tile("v", n)
            yield from self.wait("p_ready", n)
            self.pipe.append(("values", n, s))
            self.pipe.append(("commit", "pv_done"))
            self.pipe.append(("commit", ("slot_empty", s)))
            n += 1
            yield

    def softmax(self, quadrant, half):
        n, met = 0, 0

        def meet():
            nonlocal met
            self.bar["pair", quadrant].arrive()
            yield from self.wait(("pair", quadrant), met)
            met += 1

        for r in range(len(self.pieces) + 1):
            yield from self.wait(("piece_full", r % PIECES), r // PIECES)
            need(self.ring[r % PIECES] == r, f"description of piece {self.ring[r % PIECES]}, not {r}")
            if r == len(self.pieces):
                return
            for j in range(self.pieces[r]):
                yield from self.wait("s_full", n)
                need(self.scores_of == n, f"scores of step {self.scores_of}, not {n}")
                yield
                self.maxima[n & 1, quadrant, half] = n
                yield from meet()
                need(self.maxima[n & 1, quadrant, 1 - half] == n, "the other half's maximum of another step")
                if n > 0 and self.variant != "no_pv_done":
                    yield from self.wait("pv_done", n - 1)
                yield
                need(self.scores_of == n, "scores overwritten before their second reading")
                self.read_scores[n] = self.read_scores.get(n, 0) + 1
                self.bar["s_free"].arrive()
                yield
                need(n == 0 or n - 1 in self.values_done, f"P of step {n} over step {n - 1}'s")
                self.wrote_p[n] = self.wrote_p.get(n, 0) + 1
                self.bar["p_ready"].arrive()
                n += 1
                yield
            yield from self.wait("pv_done", n - 1)
            need(n - 1 in self.values_done and n not in self.values_done, "O read too early or too late")
            yield
            self.o_read[r] = self.o_read.get(r, 0) + 1
            yield from meet()

    def run(self):
        roles = [self.producer(), self.mma(), *(self.softmax(q, h) for q in range(4) for h in range(2))]
        idle = 0
        while roles or self.tma or self.pipe:
            choice = self.rng.random()
            before = (len(self.tma), len(self.pipe), [b.completed for b in self.bar.values()])
            if self.tma and choice < 0.2:
                name, land = self.tma.pop(self.rng.randrange(len(self.tma)))
                land()
                self.bar[name].arrive()
            elif self.pipe and choice < 0.45:
                op = self.pipe.pop(0)
                if op[0] == "commit":
                    self.bar[op[1]].arrive()
                elif op[0] == "scores":
                    _, n, s, b = op
                    need(self.read_scores.get(n - 1, WARPS) == WARPS, f"scores of step {n} over unread ones")
                    self.scores_of = n
                    self.scores_done.add(n)
                    self.slot_readers[s] -= 1
                    self.q_readers[b] -= 1
                else:
                    _, n, s = op
                    need(self.wrote_p.get(n, 0) == WARPS, f"P of step {n} used before it is whole")
                    r, j = self.steps[n]
                    need(j > 0 or r == 0 or self.o_read.get(r - 1, 0) == WARPS, "O overwritten before it is read")
                    self.values_done.add(n)
                    self.slot_readers[s] -= 1
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


CASES = [[1], [3], [1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1, 1], [2, 5, 1, 1, 4], [1, 7, 1], [6, 1, 1, 1, 1, 1, 1, 1, 1, 2]]


@pytest.mark.parametrize("pieces", CASES, ids=str)
def test_every_schedule_finds_its_data(pieces):
    for seed in range(60):
        Model(pieces, seed).run()


@pytest.mark.parametrize("variant", ["no_s_free", "no_pv_done"])
def test_planted_mistakes_are_found(variant):
    found = 0
    for seed in range(60):
        try:
            Model([3, 2, 4], seed, variant).run()
        except Violation:
            found += 1
    assert found > 0


def test_the_model_has_the_kernels_sizes():
    text = (test_warp_waits.CSRC / "packed_forward.cu").read_text()
    for name, value in (("kSlots", SLOTS), ("kPieces", PIECES), ("kSoftmaxWarps", WARPS)):
        assert int(re.search(rf"constexpr int {name} = (\d+);", text).group(1)) == value
    assert attention.Barrier is Barrier


@pytest.mark.parametrize("source, least", [("packed_forward.cu", 12), ("packed_backward.cu", 10)])
def test_lanes_of_a_warp_do_not_decide_for_themselves(source, least):
    """As test_warp_waits.py has it for the other kernels: a warp's waits have one outcome, or the lanes go along and
    agree afterwards, or one lane waits alone."""
    text = (test_warp_waits.CSRC / source).read_text()
    assert len(list(test_warp_waits.waits(text, "sm100::mbar_wait_warp"))) >= least
    for statement, headers in test_warp_waits.waits(text, "sm100::mbar_wait"):
        alone = any(re.search(r"\blane == 0\b", header) for header in headers)
        agreed = re.search(r"\b(there|ok) = .*(&& (there|ok))?$", statement) and "if (" not in statement
        assert alone or agreed, statement


class Copies:
    """The end of a piece in the few-rows forms: eight warps put their rows' copies together through shared memory, with
    a barrier of eight that they meet at nine times. Nothing else is taken to hold them together between pieces."""

    def __init__(self, subsets, pieces, seed, missing=None):
        self.apart, self.subsets, self.pieces, self.missing = 4 // subsets, subsets, pieces, missing
        self.rng = random.Random(seed)
        self.bar = Barrier("meeting", WARPS)
        self.merge, self.staging = [None] * WARPS, [None] * WARPS

    def warp(self, half, quadrant):
        met = 0

        def meet(which):
            nonlocal met
            if which == self.missing:
                return
            self.bar.arrive()
            while not self.bar.passed(met & 1):
                yield
            need(self.bar.completed > met, "aliased wait")
            met += 1

        others = [quadrant % self.apart + s * self.apart for s in range(self.subsets)]
        for r in range(self.pieces):
            self.merge[half * 4 + quadrant] = r
            yield
            yield from meet("maxima and sums")
            for other in others:
                need(self.merge[other] == r and self.merge[4 + other] == r, "maxima and sums of another piece")
                yield
            for part in range(4):
                self.staging[half * 4 + quadrant] = (r, part)
                yield
                yield from meet("columns written")
                for other in others:
                    need(self.staging[half * 4 + other] == (r, part), "columns of another copy or round")
                    yield
                yield from meet("columns read")

    def run(self):
        roles = [self.warp(h, q) for h in range(2) for q in range(4)]
        steps = 0
        while roles:
            role = self.rng.choice(roles)
            try:
                next(role)
            except StopIteration:
                roles.remove(role)
            steps += 1
            need(steps < 200000, "deadlock")


@pytest.mark.parametrize("subsets", [2, 4])
def test_copies_of_few_rows_are_put_together(subsets):
    for seed in range(40):
        Copies(subsets, 4, seed).run()
    for missing in ("maxima and sums", "columns written", "columns read"):
        found = 0
        for seed in range(40):
            try:
                Copies(subsets, 4, seed, missing).run()
            except Violation:
                found += 1
        assert found > 0, missing


def test_the_copies_meet_where_the_model_does():
    text = (test_warp_waits.CSRC / "packed_forward.cu").read_text()
    merge = text[text.index("merge_max[quadrant][lane] = m;"):text.index("// This thread's columns of O:")]
    steps = re.findall(r"meeting\.meet\(\)|top = max3_nan\(top, merge_max|merge_sum\[other\]|r < 4|st\.shared\.v2|ld\.shared\.v2", merge)
    assert steps == ["meeting.meet()", "top = max3_nan(top, merge_max", "merge_sum[other]", "r < 4", "st.shared.v2",
                     "meeting.meet()", "ld.shared.v2", "meeting.meet()"]
