"""A paged cache: new tokens' keys and values stored into pages, and their attention over them,
against 64 bits."""

import pytest
import torch

import ragged
from flint_b200 import PackedShape, PagedShape

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 0.125


class Cache:
    """Sequences of total[s] positions, the last new[s] of them this call's. Slots that no sequence
    uses are NaN, and so are table entries' pages behind a sequence's end (they do not exist)."""

    def __init__(self, new, total, heads, kv_heads, page_size, seed=0, spare=3, longest=None):
        self.new, self.total, self.heads, self.kv_heads, self.size = new, total, heads, kv_heads, page_size
        self.rows = sum(new) + 2
        g = torch.Generator(device=DEV).manual_seed(seed + sum(total) + 7 * heads + page_size)
        self.width = (heads + 2 * kv_heads) * 64
        self.qkv = torch.randn(self.rows, self.width, generator=g, device=DEV).half()
        first = [0]
        for n in new:
            first.append(first[-1] + n)
        self.first = first
        self.qkv[first[-1]:] = float("nan")
        integers = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        self.starts, self.lengths = integers(first), integers(total)
        counts = [-(-t // page_size) for t in total]
        pages = sum(counts) + spare
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        self.table = torch.full((len(new), max([*counts, 1]) + 2), 1 << 30, dtype=torch.int32, device=DEV)
        self.k_pages, self.v_pages = (torch.full((pages, kv_heads, page_size, 64), float("nan"), dtype=torch.half,
                                                 device=DEV) for _ in range(2))
        self.k, self.v = [], []       # every position's keys and values [total, kv_heads, 64]
        at = 0
        for s, (n, t) in enumerate(zip(new, total)):
            self.table[s, :counts[s]] = order[at:at + counts[s]]
            at += counts[s]
            fresh = self.qkv[first[s]:first[s + 1], heads * 64:].view(n, 2, kv_heads, 64)
            for which, (cache, kept) in enumerate(((self.k_pages, self.k), (self.v_pages, self.v))):
                every = torch.randn(t, kv_heads, 64, generator=g, device=DEV).half()
                old = max(t - n, 0)
                self.put(cache, s, 0, every[:old])
                every[old:] = fresh[n - (t - old):, which]
                kept.append(every)
        self.shape = PagedShape(len(new), self.rows, heads, kv_heads, 64, self.width, self.width, heads * 64, pages,
                                page_size, self.table.shape[1], longest or max(max(new), 1))

    def put(self, cache, s, first, values):
        positions = torch.arange(first, first + values.shape[0], device=DEV)
        cache[self.table[s].long()[positions // self.size], :, positions % self.size] = values

    def store(self, flint, stream=None):
        k, v = self.qkv[:, self.heads * 64:], self.qkv[:, (self.heads + self.kv_heads) * 64:]
        flint.paged_store(self.k_pages, self.v_pages, k, v, self.starts, self.lengths, self.table, self.shape,
                          stream=stream)

    def attend(self, flint, stream=None):
        o = torch.full((self.rows, self.heads * 64), 7.0, dtype=torch.half, device=DEV)
        lse = torch.full((self.heads, self.rows), 7.0, device=DEV)
        workspace = torch.full((flint.paged_attention_workspace(self.shape),), 255, dtype=torch.uint8, device=DEV)
        flint.paged_attention(o, lse, self.qkv, self.k_pages, self.v_pages, self.starts, self.lengths, self.table,
                              self.shape, SCALE, workspace, stream=stream)
        return o, lse

    def check(self, o, lse):
        group = self.heads // self.kv_heads
        for s, (n, t) in enumerate(zip(self.new, self.total)):
            rows = slice(self.first[s], self.first[s + 1])
            for h in range(self.heads):
                g = h // group
                want = ragged.Head(self.qkv[rows, 64 * h:64 * h + 64], self.k[s][:, g], self.v[s][:, g], t - n, SCALE)
                assert ragged.within(o[rows, 64 * h:64 * h + 64], want.o, want.o_bound) <= 1
                assert ragged.within(lse[h, rows], want.lse, ragged.LSE_BOUND) <= 1
        assert (o[self.first[-1]:] == 7).all() and (lse[:, self.first[-1]:] == 7).all()


@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("new, total", [([5], [5]), ([1, 1, 1], [1, 130, 700]), ([3, 0, 40, 1], [17, 9, 300, 129])])
def test_store(flint, page_size, new, total):
    cache = Cache(new, total, 6, 2, page_size)
    before = [t.clone() for t in (cache.k_pages, cache.v_pages)]
    cache.store(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    for kept, pages, old in ((cache.k, cache.k_pages, before[0]), (cache.v, cache.v_pages, before[1])):
        for s, every in enumerate(kept):
            cache.put(old, s, 0, every)
        assert torch.equal(pages.view(torch.int16), old.view(torch.int16))


NEW = [([1], [1]), ([1], [1000]), ([1, 1, 1, 1], [2, 128, 129, 2000]), ([1, 0, 1], [500, 64, 3]),
       ([7], [7]), ([5, 16, 2], [900, 16, 2]), ([130], [130]), ([64, 1, 300], [64, 777, 1300]), ([2], [9000])]


@pytest.mark.parametrize("new, total", NEW, ids=lambda n: "-".join(map(str, n)))
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (12, 12), (8, 2), (8, 1), (5, 1), (48, 2)])
@pytest.mark.parametrize("page_size", [16, 64, 256])
def test_attention(flint, new, total, heads, kv_heads, page_size):
    cache = Cache(new, total, heads, kv_heads, page_size)
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)


@pytest.mark.parametrize("longest", [1, 2, 17, 1000])
def test_longest_bounds_nothing(flint, longest):
    """Whatever `longest` says, every token is worked on."""
    cache = Cache([1, 90, 5], [400, 90, 260], 8, 2, 32, longest=longest)
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)


@pytest.mark.parametrize("heads, kv_heads, page_size", [(4, 4, 128), (16, 2, 16)])
def test_many_sequences(flint, heads, kv_heads, page_size):
    g = torch.Generator().manual_seed(heads)
    total = torch.randint(1, 700, (200,), generator=g).tolist()
    cache = Cache([1] * 200, total, heads, kv_heads, page_size)
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)


@pytest.mark.parametrize("heads, kv_heads, new, total", [(4, 1, [1], [40000]), (8, 1, [1, 3], [20001, 300]),
                                                         (16, 2, [9, 1], [33000, 17000]), (2, 2, [70], [25000])])
def test_long_caches(flint, heads, kv_heads, new, total):
    """Tiles in many parts, which are joined on their own."""
    cache = Cache(new, total, heads, kv_heads, 128)
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)


@pytest.mark.parametrize("heads, kv_heads", [(12, 12), (8, 1)])
@pytest.mark.parametrize("count", [5, 40, 130])
def test_many_chunks(flint, count, heads, kv_heads):
    """Chunks of prompts behind what is there, some with tokens that have no position."""
    g = torch.Generator().manual_seed(count)
    new = torch.randint(0, 200, (count,), generator=g).tolist()
    total = [max(n + int(d), 0) for n, d in zip(new, torch.randint(-20, 600, (count,), generator=g))]
    cache = Cache(new, total, heads, kv_heads, 64)
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)


@pytest.mark.parametrize("longest", [1, 64])
def test_tokens_without_a_position(flint, longest):
    """A length below the number of new tokens: the first ones have no position, nothing to see."""
    cache = Cache([4, 3, 2, 64], [2, 0, 300, 40], 4, 2, 16, longest=longest)
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)
    assert (o[:2] == 0).all() and (o[4:7] == 0).all() and (lse[:, :2] == float("-inf")).all()


@pytest.mark.parametrize("longest", [1, 64])
def test_two_sequences_on_the_same_pages(flint, longest):
    """A prefix that two sequences share, read from the same pages."""
    cache = Cache([1, 1], [200, 200], 8, 2, 16, longest=longest)
    cache.store(flint)
    cache.table[1, :12] = cache.table[0, :12]     # 192 positions
    for kept in (cache.k, cache.v):
        kept[1][:192] = kept[0][:192]
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)


@pytest.mark.parametrize("longest", [1, 64])
@pytest.mark.parametrize("page", [-1, 1 << 30])
def test_page_numbers_out_of_range_are_reported(flint, longest, page):
    cache = Cache([1, 2], [100, 300], 4, 2, 16, longest=longest)
    cache.store(flint)
    cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.table[1, 3] = page
    cache.attend(flint)
    torch.cuda.synchronize()
    assert flint.kernel_fault()
    cache.table[1, 18] = page       # where the new tokens go
    cache.store(flint)
    torch.cuda.synchronize()
    assert flint.kernel_fault()
    cache.lengths[0] = 1 << 30
    cache.attend(flint)
    torch.cuda.synchronize()
    assert flint.kernel_fault()
    cache.lengths[0] = -3
    cache.attend(flint)
    torch.cuda.synchronize()
    assert flint.kernel_fault()


@pytest.mark.parametrize("heads, kv_heads, new, total", [(12, 12, [1] * 5, [100, 3000, 64, 700, 1]),
                                                         (8, 2, [70, 1, 300], [700, 900, 300])])
def test_results_repeat_and_replay(flint, heads, kv_heads, new, total):
    cache = Cache(new, total, heads, kv_heads, 32)
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    workspace = torch.empty(flint.paged_attention_workspace(cache.shape), dtype=torch.uint8, device=DEV)
    again, again_lse = torch.full_like(o, 7.0), torch.full_like(lse, 7.0)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        cache.store(flint)
        flint.paged_attention(again, again_lse, cache.qkv, cache.k_pages, cache.v_pages, cache.starts, cache.lengths,
                              cache.table, cache.shape, SCALE, workspace)
    for _ in range(3):
        again.fill_(7), again_lse.fill_(7), workspace.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert not flint.kernel_fault()
        assert torch.equal(o, again) and torch.equal(lse, again_lse)


@pytest.mark.parametrize("heads, kv_heads, new, total", [(128, 1, [1, 2], [300, 40]), (64, 1, [1], [129]),
                                                         (33, 1, [1, 1], [500, 1]), (1024, 8, [1], [200])])
def test_wide_groups(flint, heads, kv_heads, new, total):
    cache = Cache(new, total, heads, kv_heads, 32)
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)


@pytest.mark.parametrize("longest", [1, 64])
def test_offsets_beyond_32_bits(flint, longest):
    """A cache of 5 * 10^9 values per tensor, of which the last pages are used."""
    cache = Cache([2, 1], [700, 300], 8, 8, 256, longest=longest)
    small, pages = cache.k_pages.shape[0], 40000
    for name in ("k_pages", "v_pages"):
        large = torch.empty(pages, 8, 256, 64, dtype=torch.half, device=DEV)
        large[-small:] = getattr(cache, name)
        setattr(cache, name, large)
    counts = [3, 2]
    for s, n in enumerate(counts):
        cache.table[s, :n] += pages - small
    cache.shape.pages = pages
    cache.store(flint)
    o, lse = cache.attend(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    cache.check(o, lse)


def test_a_captured_step_decodes_on(flint):
    """One captured store and attention, replayed as the sequences grow by a token each time: lengths, tokens and
    the page table change in place between replays."""
    steps, totals = 20, [125, 3, 300]
    final = Cache([steps] * 3, [t + steps for t in totals], 8, 2, 16, longest=1)
    shape = final.shape
    step_shape = PagedShape(3, 3, 8, 2, 64, final.width, final.width, 8 * 64, shape.pages, 16, shape.table_stride, 1)
    qkv = torch.zeros(3, final.width, dtype=torch.half, device=DEV)
    starts = torch.arange(4, dtype=torch.int32, device=DEV)
    lengths = torch.ones(3, dtype=torch.int32, device=DEV)
    table = torch.zeros_like(final.table)
    o, lse = torch.zeros(3, 8 * 64, dtype=torch.half, device=DEV), torch.zeros(8, 3, device=DEV)
    workspace = torch.empty(flint.paged_attention_workspace(step_shape), dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        flint.paged_store(final.k_pages, final.v_pages, qkv[:, 8 * 64:], qkv[:, 10 * 64:], starts, lengths, table, step_shape)
        flint.paged_attention(o, lse, qkv, final.k_pages, final.v_pages, starts, lengths, table, step_shape, SCALE,
                              workspace)
    table.copy_(final.table)
    for i in range(steps):
        lengths.copy_(torch.tensor([t + i + 1 for t in totals], dtype=torch.int32))
        for s in range(3):
            qkv[s] = final.qkv[final.first[s] + i]
        graph.replay()
        torch.cuda.synchronize()
        assert not flint.kernel_fault()
        for s, t in enumerate(totals):
            for h in range(8):
                want = ragged.Head(qkv[s:s + 1, 64 * h:64 * h + 64], final.k[s][:t + i + 1, h // 4],
                                   final.v[s][:t + i + 1, h // 4], t + i, SCALE)
                assert ragged.within(o[s:s + 1, 64 * h:64 * h + 64], want.o, want.o_bound) <= 1
                assert ragged.within(lse[h, s:s + 1], want.lse, ragged.LSE_BOUND) <= 1


def test_a_prompt_in_chunks_and_token_by_token(flint):
    """The chain of a server: a prompt's attention at once, the same through the cache in chunks of
    odd sizes and then single tokens, and the words' probabilities at the end."""
    heads, kv_heads, length = 6, 2, 333
    g = torch.Generator(device=DEV).manual_seed(5)
    width = (heads + 2 * kv_heads) * 64
    qkv = torch.randn(length, width, generator=g, device=DEV).half()
    out = torch.randn(1000, heads * 64, generator=g, device=DEV).half() * 0.05
    starts = torch.tensor([0, length], dtype=torch.int32, device=DEV)
    packed = PackedShape(1, length, heads, kv_heads, 64, width, width, heads * 64)
    parts = qkv[:, :heads * 64], qkv[:, heads * 64:(heads + kv_heads) * 64], qkv[:, (heads + kv_heads) * 64:]
    o, lse = torch.empty(length, heads * 64, dtype=torch.half, device=DEV), torch.empty(heads, length, device=DEV)
    workspace = torch.empty(flint.packed_attention_workspace(packed), dtype=torch.uint8, device=DEV)
    flint.packed_attention_forward(o, lse, *parts, starts, packed, SCALE, workspace)
    pages = [torch.full((24, kv_heads, 16, 64), float("nan"), dtype=torch.half, device=DEV) for _ in range(2)]
    table = torch.randperm(24, generator=g, device=DEV).to(torch.int32)[None, :21].contiguous()
    at, chunks = 0, [130, 7, 64, 99, 1, 1, 17, 1, 1, 12]
    assert sum(chunks) == length
    through = torch.empty_like(o)
    for n in chunks:
        shape = PagedShape(1, n, heads, kv_heads, 64, width, width, heads * 64, 24, 16, 21, n)
        rows = [t[at:at + n] for t in parts]
        ends = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        lengths = torch.tensor([at + n], dtype=torch.int32, device=DEV)
        workspace = torch.empty(flint.paged_attention_workspace(shape), dtype=torch.uint8, device=DEV)
        flint.paged_store(*pages, rows[1], rows[2], ends, lengths, table, shape)
        flint.paged_attention(through[at:at + n], None, rows[0], *pages, ends, lengths, table, shape, SCALE, workspace)
        at += n
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    # Both are within their bounds of the same exact values.
    for h in range(heads):
        head = [t[:, 64 * c:64 * c + 64] for t, c in zip(parts, (h, h // 3, h // 3))]
        want = ragged.Head(*head, 0, SCALE)
        for got in (o, through):
            assert ragged.within(got[:, 64 * h:64 * h + 64], want.o, want.o_bound) <= 1
    # Their logits give the same most likely words but where two are closer than the rounding.
    results = []
    for rows in (o, through):
        logits = torch.empty(length, 1000, dtype=torch.half, device=DEV)
        flint.gemm_nt(logits, rows, out, length, 1000, heads * 64)
        targets = torch.arange(length, device=DEV).to(torch.int32).to(torch.uint16)
        values = [torch.empty(length, device=DEV) for _ in range(3)]
        top = torch.empty(length, 4, device=DEV), torch.empty(length, 4, dtype=torch.uint16, device=DEV)
        flint.token_log_probs(*values, *top, logits, targets, False, length, 1000, 1000, 4)
        torch.cuda.synchronize()
        exact = torch.log_softmax(logits.double(), 1)
        assert (values[0] - exact[torch.arange(length), torch.arange(length)]).abs().max() < 2.0 ** -15
        assert torch.equal(top[1].to(torch.int64)[:, 0], logits.float().argmax(1))
        results.append(top[0])
    # |o| stays below 5 and each logit sums 384 products with |w| around 0.05: 2^-10 * 5 * 0.05 * 384 is above any
    # difference of two roundings.
    assert (results[0] - results[1]).abs().max() < 2.0 ** -10 * 5 * 0.05 * 384
