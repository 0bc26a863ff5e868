"""The packed forward kernel over pages of 8 bits: what its two converting warps add to the hand-overs of
test_packed_protocol.py, model-checked in the same way.

Raw tiles land in a ring of their own with the scales of their keys; the converting warps turn each into a slot of the FP16 ring, half a
tile each, and the scales into what the softmax warps read."""

import importlib.util
import re
from pathlib import Path

import pytest

import test_packed_protocol
import test_warp_waits

RAW, SCALES = 2, 8


def packed_with(slots):
    """test_packed_protocol.py once more, with another number of slots."""
    spec = importlib.util.spec_from_file_location("packed_protocol_8", Path(test_packed_protocol.__file__))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.SLOTS = slots
    return module


packed = packed_with(3)
Barrier, Violation, need, SLOTS, PIECES, WARPS = (getattr(packed, n) for n in (
    "Barrier", "Violation", "need", "SLOTS", "PIECES", "WARPS"))


class Eight(packed.Model):
    def __init__(self, pieces, seed, variant="kernel"):
        super().__init__(pieces, seed, variant)
        self.bar.update({("slot_full", s): Barrier(f"slot_full{s}", 2) for s in range(SLOTS)})
        self.bar.update({("raw_full", r): Barrier(f"raw_full{r}", 2) for r in range(RAW)})      # bytes, scales
        self.bar.update({("raw_empty", r): Barrier(f"raw_empty{r}", 2) for r in range(RAW)})
        self.bar.update({("scales_full", i): Barrier(f"scales_full{i}", 1) for i in range(SCALES)})
        steps = len(self.steps)
        self.order = [("k", 0)]
        for n in range(1, steps):
            self.order += [("k", n), ("v", n - 1)]
        self.order.append(("v", steps - 1))
        self.raw, self.raw_readers = [None] * RAW, [0] * RAW
        self.raw_scales, self.scales = [None] * SCALES, [None] * SCALES
        self.scales_of = [None] * RAW
        self.scale_reads = {}
        self.halves = [[None, None] for _ in range(SLOTS)]

    def producer(self):
        at = [0]

        def load(kind, n):
            r, use = at[0] % RAW, at[0] // RAW
            if use > 0 and self.variant != "no_raw_empty":
                yield from self.wait(("raw_empty", r), use - 1)
            need(self.raw_readers[r] == 0, f"raw slot {r} reloaded while read")
            self.raw[r] = None
            if kind == "k":
                need(n < SCALES or self.scale_reads.get(n - SCALES, 0) == WARPS, "scales that are still read")
                self.raw_scales[n % SCALES] = None
            self.scales_of[r] = n % SCALES if kind == "k" else -1
            yield
            self.tma.append((("raw_full", r), lambda: self.raw.__setitem__(r, (kind, n))))
            self.tma.append((("raw_full", r), lambda: self.raw_scales.__setitem__(n % SCALES, n) if kind == "k" else None))
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

    def converter(self, half):
        k = known = piece = 0
        while True:
            if k == 2 * known:
                yield from self.wait(("piece_full", piece % PIECES), piece // PIECES)
                need(self.ring[piece % PIECES] == piece, "another piece's description")
                if piece == len(self.pieces):
                    return
                known += self.pieces[piece]
                piece += 1
            r, s = k % RAW, k % SLOTS
            yield from self.wait(("raw_full", r), k // RAW)
            if k >= SLOTS and self.variant != "no_slot_empty":
                yield from self.wait(("slot_empty", s), k // SLOTS - 1)
            kind, n = self.order[k]
            need(self.raw[r] == (kind, n), f"raw slot {r} holds {self.raw[r]}, not {kind} {n}")
            need(self.slot_readers[s] == 0, f"slot {s} overwritten while read")
            need(self.scales_of[r] == (n % SCALES if kind == "k" else -1), "another tile's scales")
            self.raw_readers[r] += 1
            if half == 0 and kind == "k":
                need(self.raw_scales[n % SCALES] == n, "scales that have not come")
                need(n < SCALES or self.scale_reads.get(n - SCALES, 0) == WARPS, "scales overwritten before they are read")
                self.scales[n % SCALES] = n
            yield
            self.halves[s][half] = (kind, n)
            self.slot[s] = (kind, n) if self.halves[s][0] == self.halves[s][1] else None
            self.raw_readers[r] -= 1
            yield
            self.bar["slot_full", s].arrive()
            self.bar["raw_empty", r].arrive()
            if half == 0 and kind == "k":
                self.bar["scales_full", n % SCALES].arrive()
            k += 1
            yield

    def softmax(self, quadrant, half):
        # (The steps of the base model with the scales beside them.)
        inner = super().softmax(quadrant, half)
        n, checked = 0, set()
        for _ in inner:
            # The base yields behind its wait for scores and again behind the maxima's exchange and P's.
            if self.maxima.get((n & 1, quadrant, half)) == n and n not in checked:
                if self.variant != "no_scales_full":
                    yield from self.wait(("scales_full", n % SCALES), n // SCALES)
                need(self.scales[n % SCALES] == n, f"scales of step {self.scales[n % SCALES]}, not {n}")
                checked.add(n)
            if n in checked and self.mine.get((quadrant, half), 0) > n:
                need(self.scales[n % SCALES] == n, "scales overwritten before their second reading")
                self.scale_reads[n] = self.scale_reads.get(n, 0) + 1
                n += 1
            yield

    def run(self):
        self.mine = {}
        bar = self.bar["p_ready"]
        # Which step's probabilities each softmax warp has written: its arrivals, told apart by who runs.
        roles = {}
        original = bar.arrive

        def arrive():
            self.mine[roles["now"]] = self.mine.get(roles["now"], 0) + 1
            original()

        bar.arrive = arrive
        base = super()
        softmax = self.softmax

        def marked(quadrant, half):
            role = softmax(quadrant, half)
            while True:
                roles["now"] = (quadrant, half)
                try:
                    next(role)
                except StopIteration:
                    return
                yield

        self.softmax = marked
        producer = self.producer
        extra = [self.converter(0), self.converter(1)]

        def with_converters():
            """The producer's place in the schedule, shared at random with the converting warps."""
            those = [producer(), *extra]
            while those:
                role = self.rng.choice(those)
                try:
                    next(role)
                except StopIteration:
                    those.remove(role)
                yield

        self.producer = with_converters
        base.run()


CASES = [[1], [3], [1] * 13, [2, 5, 1, 1, 4], [1, 7, 1], [6, 1, 1, 1, 1, 1, 1, 1, 1, 2], [20], [9, 9]]


@pytest.mark.parametrize("pieces", CASES, ids=str)
def test_every_schedule_finds_its_data(pieces):
    for seed in range(40):
        Eight(pieces, seed).run()


@pytest.mark.parametrize("variant", ["no_raw_empty", "no_slot_empty", "no_scales_full", "no_s_free", "no_pv_done"])
def test_planted_mistakes_are_found(variant):
    found = 0
    for seed in range(120):
        try:
            Eight([3, 2, 4], seed, variant).run()
        except Violation:
            found += 1
    if variant == "no_scales_full":
        # (Scores follow their K tile, whose scales come first: the wait says what the order of the hand-overs has already.)
        assert found == 0
    else:
        assert found > 0


def test_the_model_has_the_kernels_sizes():
    text = (test_warp_waits.CSRC / "packed_forward.cu").read_text()
    for name, value in (("kSlots8", SLOTS), ("kRawSlots", RAW), ("kScaleSteps", SCALES), ("kPieces", PIECES)):
        assert int(re.search(rf"constexpr int {name} = (\d+);", text).group(1)) == value
    for barrier, count in (("slot_full(s)", "kEight ? 2 : 1"), ("raw_full(r)", "1 + 32"), ("raw_empty(r)", "2"),
                           ("scales_full(i)", "1")):
        assert f"sm100::mbar_init(bar.{barrier}, {count});" in text
