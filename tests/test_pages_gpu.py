"""A paged cache's tables: fork, reserve, truncate, compact and the copies that they ask for, against lists on the host."""

import random

import pytest
import torch

from flint_b200 import PageArrays, PagePool

pytestmark = pytest.mark.gpu
DEV = "cuda"


def integers(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def empty(*shape):
    return torch.full(shape, -7, dtype=torch.int32, device=DEV)


class Pool:
    """Lists of pages per sequence and the references to them, with the library's arrays beside them."""

    def __init__(self, sequences, pages, size, stride, seed=0):
        self.sequences, self.pages, self.size, self.stride = sequences, pages, size, stride
        self.shape = PagePool(sequences, stride, pages, size)
        self.rows, self.lengths = [[] for _ in range(sequences)], [0] * sequences
        self.references = [0] * pages
        self.rng = random.Random(seed)

    def fill(self, longest):
        """Every sequence a length, shuffled pages of its own as far as they go, and some shared with its neighbour."""
        free = list(range(self.pages))
        self.rng.shuffle(free)
        for s in range(self.sequences):
            length = self.rng.randrange(longest + 1)
            need = -(-length // self.size)
            row = []
            if s and self.rng.random() < 0.5:
                row = self.rows[s - 1][:self.rng.randrange(len(self.rows[s - 1]) + 1)][:need]
            while len(row) < need and free:
                row.append(free.pop())
            self.rows[s] = row
            self.lengths[s] = min(length, len(row) * self.size)
            self.rows[s] = row[:-(-self.lengths[s] // self.size)]
            for page in self.rows[s]:
                self.references[page] += 1

    def arrays(self):
        """Anything behind a sequence's pages."""
        table = [row + [self.rng.choice([-1, 0, 1 << 30])] * 0 + [self.rng.choice([-1, 0, 1 << 30])
                                                                  for _ in range(self.stride - len(row))] for row in self.rows]
        return (integers(table).view(self.sequences, self.stride), integers(self.lengths), integers(self.references))

    def check(self, table, lengths, references, tail=True):
        assert lengths.tolist() == self.lengths
        for got, row in zip(table.tolist(), self.rows):
            assert got[:len(row)] == row
            if tail:
                assert got[len(row):] == [-1] * (self.stride - len(row))
        assert references.tolist() == self.references

    def fork(self, parents):
        rows = [list(self.rows[p]) if p >= 0 else [] for p in parents]
        lengths = [self.lengths[p] if p >= 0 else 0 for p in parents]
        for row in self.rows:
            for page in row:
                self.references[page] -= 1
        for row in rows:
            for page in row:
                self.references[page] += 1
        self.rows, self.lengths = rows, lengths

    def reserve(self, added):
        """(moves, missing)."""
        writers = {}
        for s, n in enumerate(added):
            if n and self.lengths[s] % self.size:
                writers.setdefault(self.rows[s][-1], []).append(s)
        copying = {s for page, those in writers.items()
                   for s in (those if self.references[page] > len(those) else those[1:])}
        free = [page for page, count in enumerate(self.references) if count == 0]
        need = len(copying) + sum(-(-(have + n) // self.size) - -(-have // self.size) for have, n in zip(self.lengths, added))
        if need > len(free):
            return [], need - len(free)
        free, moves = iter(free), []
        for s, n in enumerate(added):
            if s in copying:
                page = next(free)
                moves.append([self.rows[s][-1], page])
                self.references[self.rows[s][-1]] -= 1
                self.references[page] = 1
                self.rows[s][-1] = page
            self.lengths[s] += n
            while len(self.rows[s]) * self.size < self.lengths[s]:
                page = next(free)
                self.references[page] = 1
                self.rows[s].append(page)
        return moves, 0

    def truncate(self, keep):
        for s, n in enumerate(keep):
            self.lengths[s] = min(self.lengths[s], n)
            while len(self.rows[s]) > -(-self.lengths[s] // self.size):
                self.references[self.rows[s].pop()] -= 1

    def compact(self):
        """(moves, pages in use)."""
        count = sum(n > 0 for n in self.references)
        sources = [p for p in range(count, self.pages) if self.references[p] > 0]
        holes = [p for p in range(count) if self.references[p] == 0]
        number = dict(zip(sources, holes))
        self.rows = [[number.get(page, page) for page in row] for row in self.rows]
        references = [0] * self.pages
        for page, n in enumerate(self.references):
            if n > 0:
                references[number.get(page, page)] = n
        self.references = references
        return [list(pair) for pair in number.items()], count


def check_moves(got, moves):
    got = got.tolist()
    assert got[:len(moves)] == moves
    assert all(row == [-1, -1] for row in got[len(moves):])


SHAPES = [(1, 4, 16, 3, 40), (7, 40, 16, 9, 100), (64, 2000, 32, 70, 2000), (300, 1500, 64, 6, 200), (2500, 9000, 16, 4, 50),
          (3, 70000, 16, 5, 60), (1, 1, 1024, 1, 1024)]


@pytest.mark.parametrize("sequences, pages, size, stride, longest", SHAPES)
def test_fork(flint, sequences, pages, size, stride, longest):
    for seed in range(3):
        pool = Pool(sequences, pages, size, stride, seed)
        pool.fill(longest)
        table, lengths, references = pool.arrays()
        before = [t.clone() for t in (table, lengths, references)]
        parents = [pool.rng.choice([-1, s, pool.rng.randrange(sequences), 0]) for s in range(sequences)]
        out = empty(sequences, stride), empty(sequences), empty(pages)
        flint.pages_fork(*out, table, lengths, references, integers(parents), pool.shape)
        pool.fork(parents)
        pool.check(*out)
        for old, now in zip(before, (table, lengths, references)):
            assert torch.equal(old, now)
    assert not flint.kernel_fault()


@pytest.mark.parametrize("sequences, pages, size, stride, longest", SHAPES)
@pytest.mark.parametrize("most", [1, 40])
def test_reserve(flint, sequences, pages, size, stride, longest, most):
    missed = 0
    for seed in range(4):
        pool = Pool(sequences, pages, size, stride, seed)
        pool.fill(longest // 2)
        # Copies of sequences, so that partly filled pages are shared, by all or by some who grow.
        pool.fork([pool.rng.randrange(s + 1) if pool.rng.random() < 0.6 else s for s in range(sequences)])
        added = [pool.rng.choice([0, 1, pool.rng.randrange(most + 1)]) for _ in range(sequences)]
        added = [min(n, stride * size - have) for n, have in zip(added, pool.lengths)]
        arrays = pool.arrays()
        before = [t.clone() for t in arrays]
        moves, counts = empty(sequences, 2), empty(2)
        workspace = torch.full((flint.pages_workspace(pool.shape),), 255, dtype=torch.uint8, device=DEV)
        flint.pages_reserve(*arrays, moves, counts, integers(added), pool.shape, workspace)
        want, missing = pool.reserve(added)
        assert counts.tolist() == [len(want), missing]
        check_moves(moves, want)
        pool.check(*arrays, tail=False)
        if missing:
            missed += 1
            for old, now in zip(before, arrays):
                assert torch.equal(old, now)
    assert not flint.kernel_fault()


def test_reserve_says_how_many_pages_are_missing(flint):
    pool = Pool(3, 5, 16, 40)
    pool.rows, pool.lengths, pool.references = [[4], [4], [1]], [5, 5, 16], [0, 1, 0, 0, 2]
    arrays = pool.arrays()
    workspace = torch.empty(flint.pages_workspace(pool.shape), dtype=torch.uint8, device=DEV)
    for added, missing in (([1, 1, 32], 0), ([0, 0, 1], 1), ([300, 1, 0], 19), ([0, 0, 0], 0)):
        moves, counts = empty(3, 2), empty(2)
        flint.pages_reserve(*arrays, moves, counts, integers(added), pool.shape, workspace)
        want, lacking = pool.reserve(added)
        assert counts.tolist() == [len(want), lacking] and lacking == missing
        check_moves(moves, want)
        pool.check(*arrays, tail=False)


def test_more_pages_than_32_bits_count_are_missing(flint):
    sequences, stride = 600, 1 << 22
    pool = PagePool(sequences, stride, 4, 16)
    table = torch.full((sequences, stride), -1, dtype=torch.int32, device=DEV)
    lengths, references = torch.zeros(sequences, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)
    moves, counts = empty(sequences, 2), empty(2)
    workspace = torch.empty(flint.pages_workspace(pool), dtype=torch.uint8, device=DEV)
    flint.pages_reserve(table, lengths, references, moves, counts, torch.full_like(lengths, 1 << 26), pool, workspace)
    assert counts.tolist() == [0, (1 << 31) - 1]
    assert (lengths == 0).all() and (references == 0).all() and (moves == -1).all()


@pytest.mark.parametrize("sequences, pages, size, stride, longest", SHAPES)
def test_truncate(flint, sequences, pages, size, stride, longest):
    pool = Pool(sequences, pages, size, stride, 5)
    pool.fill(longest)
    arrays = pool.arrays()
    keep = [pool.rng.choice([0, 1 << 30, pool.rng.randrange(longest + 1), max(0, n - 1)]) for n in pool.lengths]
    flint.pages_truncate(*arrays, integers(keep), pool.shape)
    pool.truncate(keep)
    pool.check(*arrays, tail=False)
    assert not flint.kernel_fault()


@pytest.mark.parametrize("sequences, pages, size, stride, longest", SHAPES)
def test_compact(flint, sequences, pages, size, stride, longest):
    for seed in range(3):
        pool = Pool(sequences, pages, size, stride, seed)
        pool.fill(longest)
        table, lengths, references = pool.arrays()
        out = empty(sequences, stride), empty(pages)
        moves, counts = empty(max(pages // 2, 1), 2), empty(2)
        workspace = torch.full((flint.pages_workspace(pool.shape),), 255, dtype=torch.uint8, device=DEV)
        flint.pages_compact(*out, moves, counts, table, lengths, references, pool.shape, workspace)
        want, count = pool.compact()
        assert counts.tolist() == [len(want), count]
        if pages > 1:
            check_moves(moves, want)
        pool.check(out[0], lengths, out[1])
    assert not flint.kernel_fault()


@pytest.mark.parametrize("pages", [1, 5, 40000])
def test_no_sequences(flint, pages):
    """References stand as they are, and counts say that nothing is to be copied."""
    pool = PagePool(0, 3, pages, 16)
    references = torch.randint(0, 3, (pages,), dtype=torch.int32, device=DEV)
    after, counts = empty(pages), empty(2)
    workspace = torch.empty(flint.pages_workspace(pool), dtype=torch.uint8, device=DEV)
    flint.pages_fork(None, None, after, None, None, references, None, pool)
    assert torch.equal(after, references)
    flint.pages_reserve(None, None, after, None, counts, None, pool, workspace)
    assert counts.tolist() == [0, 0] and torch.equal(after, references)
    moves = empty(max(1, pages // 2), 2)
    flint.pages_compact(None, after, moves if pages > 1 else None, counts, None, None, references, pool, workspace)
    used = references > 0
    assert counts[1].item() == used.sum().item() and torch.equal((after > 0).int().cumprod(0).sum(), used.sum())
    assert torch.equal(after.sort().values, references.sort().values)


@pytest.mark.parametrize("widths", [[64], [4, 8192, 12, 8196, 24580], [1 << 20, 16]])
@pytest.mark.parametrize("count", [0, 1, 5])
def test_copy(flint, widths, count):
    """Pages of any multiple of 4 bytes; moves behind the count, and -1 among them, are nothing."""
    pages = 12
    g = torch.Generator(device=DEV).manual_seed(1)
    tensors = [torch.randint(0, 256, (pages, w), generator=g, device=DEV, dtype=torch.uint8) for w in widths]
    moves = [[0, 3], [0, 5], [-1, -1], [7, 1], [2, 11], [6, 4], [8, 9]]
    want = [t.clone() for t in tensors]
    for a, b in moves[:count]:
        if a >= 0:
            for t in want:
                t[b] = t[a]
    flint.pages_copy(PageArrays(tensors), integers(moves), integers([count, 0]), len(moves))
    for got, old in zip(tensors, want):
        assert torch.equal(got, old)
    assert not flint.kernel_fault()


def test_copy_in_most_arrays(flint):
    tensors = [torch.full((4, 20 + 4 * i), i, dtype=torch.uint8, device=DEV) for i in range(128)]
    for i, t in enumerate(tensors):
        t[1] = 255 - i
    flint.pages_copy(PageArrays(tensors), integers([[1, 2]]), integers([1, 0]), 1)
    for i, t in enumerate(tensors):
        assert (t[2] == 255 - i).all() and (t[3] == i).all() and (t[0] == i).all()


def test_copy_beyond_32_bits(flint):
    pages, width = 5, 1 << 28
    t = torch.empty(pages * 4, width, dtype=torch.uint8, device=DEV)
    t[19] = 7
    t[2] = 1
    flint.pages_copy(PageArrays([t]), integers([[19, 18], [2, 0]]), integers([2, 0]), 2)
    assert (t[18] == 7).all() and (t[0] == 1).all()


def test_numbers_out_of_range_are_reported(flint):
    pool = Pool(3, 6, 16, 2)
    pool.rows, pool.lengths, pool.references = [[0, 1], [2], [3]], [20, 16, 3], [1, 1, 1, 1, 0, 0]
    table, lengths, references = pool.arrays()
    out = empty(3, 2), empty(3), empty(6)
    workspace = torch.empty(flint.pages_workspace(pool.shape), dtype=torch.uint8, device=DEV)
    flint.kernel_fault()
    flint.pages_fork(*out, table, lengths, references, integers([3, -2, 1]), pool.shape)
    assert flint.kernel_fault()
    pool.fork([-1, -1, 1])
    pool.check(*out)
    bad = table.clone()
    bad[0, 1] = 6
    flint.pages_fork(*out, bad, lengths, references, integers([0, 1, 2]), pool.shape)
    assert flint.kernel_fault()
    for numbers in ([-1, 16, 3], [33, 16, 3]):
        flint.pages_fork(*out, table, integers(numbers), references, integers([0, 1, 2]), pool.shape)
        assert flint.kernel_fault()
    copy = [t.clone() for t in (table, lengths, references)]
    flint.pages_truncate(*copy, integers([-1, 16, 3]), pool.shape)
    assert flint.kernel_fault() and copy[1].tolist() == [0, 16, 3]
    copy = [t.clone() for t in (table, lengths, references)]
    flint.pages_reserve(*copy, empty(3, 2), empty(2), integers([100, -4, 0]), pool.shape, workspace)
    assert flint.kernel_fault() and copy[1].tolist() == [32, 16, 3]
    t = torch.arange(24, dtype=torch.int32, device=DEV).view(6, 4)
    want = t.clone()
    flint.pages_copy(PageArrays([t]), integers([[0, 6], [-1, 2], [9, 1]]), integers([3, 0]), 3)
    assert flint.kernel_fault() and torch.equal(t, want)
    flint.pages_copy(PageArrays([t]), integers([[0, 1]]), integers([1 << 30, 0]), 1)     # (no more than most_moves)
    want[1] = want[0]
    assert torch.equal(t, want)


def test_a_life_of_a_pool(flint):
    """Many steps of every kind, twice captured and replayed, with the pages' contents followed."""
    pool = Pool(24, 400, 16, 20, 9)
    pool.fill(60)
    arrays = list(pool.arrays())
    cache = torch.randint(0, 1 << 30, (400, 6), dtype=torch.int32, device=DEV)
    held = cache.tolist()
    workspace = torch.empty(flint.pages_workspace(pool.shape), dtype=torch.uint8, device=DEV)
    moves, counts = empty(200, 2), empty(2)
    parents, numbers = empty(24), empty(24)
    spare = [torch.empty_like(t) for t in arrays]
    copies = PageArrays([cache])

    def step():
        flint.pages_fork(*spare, *arrays, parents, pool.shape)
        flint.pages_reserve(*spare, moves, counts, numbers, pool.shape, workspace)
        flint.pages_copy(copies, moves, counts, 24)
        for old, now in zip(arrays, spare):
            old.copy_(now)

    def host(want):
        for a, b in want:
            held[b] = held[a]

    graph = None
    for i in range(30):
        parents.copy_(integers([pool.rng.choice([s, s, pool.rng.randrange(24), -1 if i % 5 == 4 else s]) for s in range(24)]))
        numbers.copy_(integers([pool.rng.choice([0, 1, 1, 3]) for _ in range(24)]))
        numbers.copy_(torch.minimum(numbers, 320 - arrays[1][parents.clamp(min=0).long()]))
        if graph is None and i == 3:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=side):
                    step()
            torch.cuda.current_stream().wait_stream(side)
        if graph is None:
            step()
        else:
            graph.replay()
        pool.fork(parents.tolist())
        want, missing = pool.reserve(numbers.tolist())
        assert counts.tolist() == [len(want), missing]
        host(want)
        pool.check(*arrays, tail=False)
        if i % 4 == 1:
            keep = [max(0, n - pool.rng.choice([0, 1, 7, 40])) for n in pool.lengths]
            flint.pages_truncate(*arrays, integers(keep), pool.shape)
            pool.truncate(keep)
            pool.check(*arrays, tail=False)
        if i % 7 == 5:
            flint.pages_compact(spare[0], spare[2], moves, counts, *arrays, pool.shape, workspace)
            flint.pages_copy(copies, moves, counts, 200)
            want, count = pool.compact()
            assert counts.tolist() == [len(want), count]
            host(want)
            arrays[0].copy_(spare[0])
            arrays[2].copy_(spare[2])
            pool.check(*arrays)
        for row in pool.rows:
            for page in row:
                assert cache[page].tolist() == held[page]
    assert not flint.kernel_fault()
