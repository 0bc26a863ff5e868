"""The packed backward kernel's synchronisation, model-checked on the CPU.

`fb_packed_backward` (flint_b200/csrc/packed_backward.cu) takes items one by one from a list, hands their numbers on
through a ring, copies an item's two resident tiles into tensor memory while the item before is finished, and runs two score
buffers and a ring of streamed tiles through all items. Its two kinds of items share this protocol. As in
test_packed_protocol.py the roles are generators under random schedules, and every access is checked.
"""

import random
import re

import pytest

import test_warp_waits
from test_attention_protocol import Barrier, Violation, need

STAGES, ITEMS, WARPS = 4, 8, 16


class Model:
    def __init__(self, items, seed, missing=None):
        self.items = items                 # sub-steps of each item that this CTA takes
        self.missing = missing             # a wait that is left out
        self.rng = random.Random(seed)
        names = ["resident", "done", *(("scores_full", b) for b in range(2)), *(("stage_full", s) for s in range(STAGES)),
                 *(("stage_empty", s) for s in range(STAGES)), *(("item_full", i) for i in range(ITEMS))]
        self.bar = {n: Barrier(str(n), 1) for n in names}
        self.bar.update({n: Barrier(str(n), WARPS) for n in ("a_ready", ("operands_ready", 0), ("operands_ready", 1))})
        self.ring = [None] * ITEMS
        self.resident = None               # the item whose tiles are in shared memory
        self.installed = {}                # item -> warps that have copied their part into tensor memory
        self.operand = None                # the item whose tiles tensor memory holds
        self.stage = [None] * STAGES
        self.tma, self.pipe = [], []
        self.scores = [None, None]         # the sub-step in each buffer
        self.scored, self.wrote, self.added = set(), {}, set()
        self.sums_of, self.sums_read = None, {}

    def wait(self, name, phase):
        if (name if isinstance(name, str) else name[0]) == self.missing:
            return
        bar = self.bar[name]
        while not bar.passed(phase & 1):
            yield
        need(bar.completed > phase, f"aliased wait on {bar.name}: meant phase {phase}, {bar.completed} completed")

    def take(self, r):
        self.ring[r % ITEMS] = r
        self.bar["item_full", r % ITEMS].arrive()

    def item(self, r):
        """Whether there is an item in this round."""
        yield from self.wait(("item_full", r % ITEMS), r // ITEMS)
        need(self.ring[r % ITEMS] == r, f"item {self.ring[r % ITEMS]}, not {r}")
        return r < len(self.items)

    def producer(self):
        count = 0
        for r, steps in enumerate(self.items):
            self.take(r)
            yield
            if r > 0:
                yield from self.wait("a_ready", r - 1)
                need(self.installed.get(r - 1, 0) == WARPS, "resident tiles reloaded before they were copied")
            self.resident = None
            self.tma.append(("resident", lambda r=r: setattr(self, "resident", r)))
            for _ in range(steps):
                s, use = count % STAGES, count // STAGES
                if use > 0:
                    yield from self.wait(("stage_empty", s), use - 1)
                need(use == 0 or count - STAGES in self.added, f"stage {s} reloaded while read")
                self.stage[s] = None
                self.tma.append((("stage_full", s), lambda s=s, count=count: self.stage.__setitem__(s, count)))
                count += 1
                yield
        self.take(len(self.items))

    def mma(self):
        before, r = 0, 0
        while (yield from self.item(r)):
            yield from self.wait("a_ready", r)
            steps = self.items[r]

            def issue(step):
                count = before + step
                yield from self.wait(("stage_full", count % STAGES), count // STAGES)
                need(self.stage[count % STAGES] == count, "another sub-step's tile")
                self.pipe += [("scores", count, r), ("commit", ("scores_full", count & 1))]

            yield from issue(0)
            for step in range(steps):
                if step + 1 < steps:
                    yield from issue(step + 1)
                count = before + step
                yield from self.wait(("operands_ready", count & 1), count >> 1)
                self.pipe += [("sums", count, r, step == 0), ("commit", ("stage_empty", count % STAGES))]
                if step + 1 == steps:
                    self.pipe.append(("commit", "done"))
                yield
            before += steps
            r += 1

    def compute(self):
        before = 0

        def install(r):
            yield from self.wait("resident", r)
            need(self.resident == r, f"tiles of item {self.resident}, not {r}")
            need(all(c in self.scored for c in range(before)), "operands overwritten while products read them")
            self.operand = r
            self.installed[r] = self.installed.get(r, 0) + 1
            self.bar["a_ready"].arrive()
            yield

        r = 0
        there = yield from self.item(0)
        if there:
            yield from install(0)
        while there:
            for step in range(self.items[r]):
                count = before + step
                yield from self.wait(("scores_full", count & 1), count >> 1)
                need(self.scores[count & 1] == count, f"scores of sub-step {self.scores[count & 1]}, not {count}")
                yield
                yield from self.wait(("stage_full", count % STAGES), count // STAGES)     # (the rows' statistics)
                need(self.stage[count % STAGES] == count, "statistics of another sub-step")
                yield
                need(self.scores[count & 1] == count, "scores overwritten while read")
                self.wrote[count] = self.wrote.get(count, 0) + 1
                self.bar["operands_ready", count & 1].arrive()
                yield
            before += self.items[r]
            there = yield from self.item(r + 1)
            if there:
                yield from install(r + 1)
            yield from self.wait("done", r)
            need(self.sums_of == r and all(c in self.added for c in range(before)), "sums read too early or too late")
            yield
            need(self.sums_of == r, "sums overwritten while read")
            self.sums_read[r] = self.sums_read.get(r, 0) + 1
            r += 1

    def step_pipe(self):
        op = self.pipe.pop(0)
        if op[0] == "commit":
            self.bar[op[1]].arrive()
        elif op[0] == "scores":
            _, count, r = op
            need(self.operand == r and self.installed.get(r, 0) == WARPS, "products of operands that are not whole")
            need(self.stage[count % STAGES] == count, "another sub-step's tile")
            need(count < 2 or count - 2 in self.added, "scores over operands that were not used yet")
            self.scores[count & 1] = count
            self.scored.add(count)
        else:
            _, count, r, first = op
            need(self.wrote.get(count, 0) == WARPS, "probabilities used before they are whole")
            need(self.stage[count % STAGES] == count, "another sub-step's tile")
            need(not first or r == 0 or self.sums_read.get(r - 1, 0) == WARPS, "sums overwritten before they are read")
            self.sums_of = r
            self.added.add(count)

    def run(self):
        roles = [self.producer(), self.mma(), *(self.compute() for _ in range(WARPS))]
        idle = 0
        while roles or self.tma or self.pipe:
            choice = self.rng.random()
            before = (len(self.tma), len(self.pipe), [b.completed for b in self.bar.values()])
            if self.tma and choice < 0.1:
                name, land = self.tma.pop(self.rng.randrange(len(self.tma)))
                land()
                self.bar[name].arrive()
            elif self.pipe and choice < 0.25:
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
        need(len(self.added) == sum(self.items) and len(self.sums_read) == len(self.items), "work left out")


CASES = [[], [1], [5], [1] * 11, [2, 1, 7, 1, 1, 3], [9, 4], [1, 1, 6, 1, 2, 1, 1, 1, 5, 1]]


@pytest.mark.parametrize("items", CASES, ids=str)
def test_every_schedule_finds_its_data(items):
    for seed in range(25):
        Model(items, seed).run()


@pytest.mark.parametrize("missing", ["item_full", "a_ready", "resident", "stage_full", "stage_empty", "scores_full",
                                     "operands_ready", "done"])
def test_every_wait_is_needed(missing):
    found = 0
    for seed in range(25):
        try:
            Model([3, 1, 6, 2, 1, 1, 1, 1, 1, 1, 2], seed, missing).run()
        except Violation:
            found += 1
    assert found > 0


def test_the_model_has_the_kernels_sizes():
    text = (test_warp_waits.CSRC / "packed_backward.cu").read_text()
    for name, value in (("kStages", STAGES), ("kItems", ITEMS), ("kComputeWarps", WARPS)):
        assert int(re.search(rf"constexpr int {name} = (\d+);", text).group(1)) == value
    # Both kinds of items, the same waits and commits; only the keys' kind reads statistics from the stages.
    halves = text[text.index("void key_items("):text.index("void query_items(")], text[text.index("void query_items("):]
    halves = halves[0], halves[1][:halves[1].index("__global__")]
    waits = [re.findall(r"mbar_wait(?:_warp)?\(bar\.(\w+)\(", half) for half in halves]
    assert [name for name in waits[0] if name != "stage_full"] == [name for name in waits[1] if name != "stage_full"]
    assert (waits[0].count("stage_full"), waits[1].count("stage_full")) == (2, 1)
    assert [re.findall(r"mma_commit\(bar\.(\w+)\(", half) for half in halves] == [["scores_full", "stage_empty", "done"]] * 2
