"""A paged cache of 8 bits: new tokens' keys and values as codes and scales, exactly, and attention over them
against 64 bits."""

import pytest
import torch

import ragged
from eight import BLOCK, Blocks
from flint_b200 import PagedShape

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 0.125


def integers(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Cache:
    """Sequences of total[s] positions, the last new[s] of them this call's; what came before was appended in two
    steps. Unused slots hold any codes, blocks behind a sequence's end a scale of NaN, and table entries behind
    its pages name no page."""

    def __init__(self, new, total, heads, kv_heads, page_size, seed=0, longest=None, gap=0, amplitude=1.0):
        self.new, self.total, self.heads, self.kv_heads, self.size = new, total, heads, kv_heads, page_size
        g = torch.Generator().manual_seed(seed + sum(total) + 7 * heads + page_size)
        self.rows = sum(new) + 2
        self.width = (heads + 2 * kv_heads) * 64 + gap
        qkv = torch.randn(self.rows, self.width, generator=g).mul_(amplitude).half()
        self.first = [0]
        for n in new:
            self.first.append(self.first[-1] + n)
        qkv[self.first[-1]:] = float("nan")
        counts = [-(-t // page_size) for t in total]
        pages = sum(counts) + 3
        order = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((len(new), max([*counts, 1]) + 2), 1 << 30, dtype=torch.int32)
        k_pages, v_pages = (torch.randint(-128, 128, (pages, kv_heads, page_size, 64), generator=g, dtype=torch.int8)
                            for _ in range(2))
        k_scales, v_scales = (torch.full((pages, kv_heads, page_size // BLOCK), float("nan")) for _ in range(2))
        self.blocks = []
        at = 0
        for s, (n, t) in enumerate(zip(new, total)):
            table[s, :counts[s]] = order[at:at + counts[s]]
            at += counts[s]
            old = max(t - n, 0)
            both = []
            for codes, scales in ((k_pages, k_scales), (v_pages, v_scales)):
                blocks = Blocks(kv_heads)
                every = torch.randn(old, kv_heads, 64, generator=g).mul_(amplitude).half()
                blocks.append(every[:old // 3])
                blocks.append(every[old // 3:])
                positions = torch.arange(old)
                codes[table[s].long()[positions // page_size], :, positions % page_size] = blocks.codes.to(torch.int8)
                positions = torch.arange(0, old, BLOCK)
                scales[table[s].long()[positions // page_size], :, positions % page_size // BLOCK] = blocks.scales
                both.append(blocks)
            self.blocks.append(both)
        self.shape = PagedShape(len(new), self.rows, heads, kv_heads, 64, self.width, self.width, heads * 64 + gap, pages,
                                page_size, table.shape[1], longest or max([*new, 1]))
        self.qkv, self.table, self.starts, self.lengths = qkv.to(DEV), table.to(DEV), integers(self.first), integers(total)
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = (t.to(DEV) for t in (k_pages, v_pages, k_scales, v_scales))

    @property
    def arrays(self):
        return self.k_pages, self.v_pages, self.k_scales, self.v_scales

    def fresh(self, s, which):
        n, kept = self.new[s], min(self.new[s], self.total[s])
        rows = self.qkv[self.first[s] + n - kept:self.first[s] + n, (self.heads + which * self.kv_heads) * 64:]
        return rows[:, :self.kv_heads * 64].reshape(kept, self.kv_heads, 64).cpu()

    def append(self):
        """The same on the host."""
        for s, both in enumerate(self.blocks):
            for which, blocks in enumerate(both):
                blocks.append(self.fresh(s, which))

    def store(self, flint, stream=None):
        k, v = self.qkv[:, self.heads * 64:], self.qkv[:, (self.heads + self.kv_heads) * 64:]
        flint.paged8_store(*self.arrays, k, v, self.starts, self.lengths, self.table, self.shape, stream=stream)

    def workspace(self, flint):
        return torch.empty(flint.paged8_attention_workspace(self.shape), dtype=torch.uint8, device=DEV)

    def outputs(self):
        return (torch.full((self.rows, self.shape.o_stride), 7.0, dtype=torch.half, device=DEV),
                torch.full((self.heads, self.rows), 7.0, device=DEV))

    def attend(self, flint, workspace=None, out=None, stream=None, lse=True):
        o, stat = out or self.outputs()
        workspace = self.workspace(flint) if workspace is None else workspace
        flint.paged8_attention(o, stat if lse else None, self.qkv, *self.arrays, self.starts, self.lengths, self.table,
                               self.shape, SCALE, workspace, stream=stream)
        return o, stat

    def check_stored(self):
        """Codes and scales, and everything else as it was (given `before`)."""
        codes = [t.cpu() for t in (self.k_pages, self.v_pages)]
        scales = [t.cpu() for t in (self.k_scales, self.v_scales)]
        table = self.table.cpu().long()
        for s, both in enumerate(self.blocks):
            for which, blocks in enumerate(both):
                positions = torch.arange(blocks.codes.shape[0])
                got = codes[which][table[s][positions // self.size], :, positions % self.size]
                torch.testing.assert_close(got.float(), blocks.codes, rtol=0, atol=0)
                positions = positions[::BLOCK]
                got = scales[which][table[s][positions // self.size], :, positions % self.size // BLOCK]
                torch.testing.assert_close(got, blocks.scales, rtol=0, atol=0, equal_nan=True)

    def check_attention(self, o, lse):
        """o and lse against 64 bits. Probabilities are rounded relative to a row's largest product of one and V's scale, so
        that what underflows there is below 2^-25 of the largest value that V's scales allow."""
        qkv = self.qkv.double()
        for s, (n, t) in enumerate(zip(self.new, self.total)):
            rows = slice(self.first[s], self.first[s] + n)
            k, v = (blocks.values().to(DEV) for blocks in self.blocks[s])
            largest = 127 * self.blocks[s][1].scales.nan_to_num().amax().item() if t else 0.0
            for h in range(self.heads):
                g = h // (self.heads // self.kv_heads)
                head = ragged.Head(qkv[rows, h * 64:(h + 1) * 64], k[:, g], v[:, g], t - n, SCALE)
                bound = head.o_bound + t * ragged.TINY * largest
                assert ragged.within(o[rows, h * 64:(h + 1) * 64], head.o, bound) <= 1.0, (s, h)
                assert ragged.within(lse[h, rows], head.lse, torch.full_like(head.lse, ragged.LSE_BOUND)) <= 1.0, (s, h)
        assert (o[self.first[-1]:] == 7.0).all() and (lse[:, self.first[-1]:] == 7.0).all()
        assert (o[:, self.heads * 64:] == 7.0).all()


@pytest.mark.parametrize("page_size", [16, 32, 128, 1024])
@pytest.mark.parametrize("new, total", [([1], [1]), ([5], [5]), ([1, 1, 1, 1], [1, 16, 17, 700]),
                                        ([3, 0, 40, 1, 0], [17, 9, 300, 129, 0]), ([200], [333]), ([7], [3])])
def test_store(flint, page_size, new, total):
    cache = Cache(new, total, 4, 2, page_size)
    before = [t.clone() for t in cache.arrays]
    cache.store(flint)
    cache.append()
    cache.check_stored()
    # Nothing but the positions of the new tokens' blocks has changed.
    table = cache.table.cpu().long()
    changed = torch.zeros(cache.shape.pages, page_size // BLOCK, dtype=torch.bool)
    for s, (n, t) in enumerate(zip(new, total)):
        blocks = torch.arange(max(t - n, 0) // BLOCK, -(-t // BLOCK)) if n else torch.arange(0)
        changed[table[s][blocks * BLOCK // page_size], blocks % (page_size // BLOCK)] = True
    for old, now in zip(before, cache.arrays):
        old, now = (x.cpu().unflatten(2, (-1, BLOCK)) if x.dim() == 4 else x.cpu() for x in (old, now))
        keep = (~changed)[:, None].expand(-1, 2, -1)
        assert torch.equal(old[keep].nan_to_num(99), now[keep].nan_to_num(99))
    assert not flint.kernel_fault()


def test_a_block_grows_token_by_token(flint):
    """Small, large and equal values, zeros, an infinity that the next block does not see, FP16's smallest number."""
    sizes = [0.0, 1.0, 1.0, 3.0, 0.5, 100.0, 2.0 ** -24, 0.0, 65504.0, 1.0, 0.0, 1.0, 2.0, 3.0, 4.0, 5.0,
             2.0 ** -24, 0.0, 2.0 ** -20, 1e-3, float("inf"), 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0,
             0.0, 0.0, 1.0]
    cache = Cache([1], [1], 2, 2, 32)
    cache.table = integers([[2, 0]])
    cache.shape.table_stride = 2
    kept = [Blocks(2), Blocks(2)]
    for position, size in enumerate(sizes):
        g = torch.Generator(device=DEV).manual_seed(position)
        values = torch.randn(1, 4 * 64, generator=g, device=DEV).clamp(-1, 1).mul(min(size, 65504.0)).half()
        if size == float("inf"):
            values[0, 5] = size
        cache.qkv[0, 128:] = values[0]
        cache.lengths.fill_(position + 1)
        cache.store(flint)
        for which in range(2):
            kept[which].append(values[:, which * 128:(which + 1) * 128].reshape(1, 2, 64))
        for which in range(2):
            positions = torch.arange(position + 1)
            page = torch.tensor([2, 0])[positions // 32]
            got = cache.arrays[which].cpu()[page, :, positions % 32].float()
            torch.testing.assert_close(got, kept[which].codes, rtol=0, atol=0)
            got = cache.arrays[2 + which].cpu()[page[::16], :, positions[::16] % 32 // 16]
            torch.testing.assert_close(got, kept[which].scales, rtol=0, atol=0, equal_nan=True)


NEW = [([1], [1]), ([1], [17]), ([1, 1, 1], [33, 1, 1000]), ([5, 1, 0, 2], [5, 130, 70, 600]), ([40, 300], [40, 500]),
       ([1, 0], [0, 0])]


@pytest.mark.parametrize("new, total", NEW, ids=lambda n: "-".join(map(str, n)))
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (12, 12), (8, 2), (8, 1), (5, 1), (48, 2)])
@pytest.mark.parametrize("page_size", [16, 64, 256])
def test_attention(flint, new, total, heads, kv_heads, page_size):
    cache = Cache(new, total, heads, kv_heads, page_size, gap=8)
    cache.store(flint)
    cache.append()
    cache.check_attention(*cache.attend(flint))
    assert not flint.kernel_fault()


@pytest.mark.parametrize("longest", [1, 2, 5, 17, 1000])
def test_longest_bounds_nothing(flint, longest):
    cache = Cache([1, 70, 3], [400, 200, 2500], 8, 2, 32, longest=longest)
    cache.store(flint)
    cache.append()
    cache.check_attention(*cache.attend(flint))


@pytest.mark.parametrize("amplitude", [1e-4, 30.0])
@pytest.mark.parametrize("longest", [1, 100])
def test_small_and_large_values(flint, amplitude, longest):
    cache = Cache([1, 3], [300, 77], 4, 2, 16, amplitude=amplitude, longest=longest)
    cache.qkv[:, :256] = (cache.qkv[:, :256].float() / amplitude).half()
    cache.store(flint)
    cache.append()
    cache.check_attention(*cache.attend(flint))


@pytest.mark.parametrize("longest", [1, 100])
def test_scales_far_apart(flint, longest):
    """V's blocks of 2^-20 and of 1,000 next to each other, K's as well; and blocks of zeros."""
    cache = Cache([1, 2], [500, 200], 4, 2, 16, longest=longest)
    g = torch.Generator().manual_seed(3)
    for both in cache.blocks:
        for blocks in both:
            blocks.scales *= torch.tensor([2.0 ** -20, 1.0, 1000.0])[torch.randint(0, 3, blocks.scales.shape, generator=g)]
            blocks.scales[2] = 0.0
            blocks.codes[32:48] = 0.0
    for both in cache.blocks:
        both[0].scales.clamp_(max=0.03)
    for s, both in enumerate(cache.blocks):
        for which, blocks in enumerate(both):
            positions = torch.arange(blocks.codes.shape[0])
            cache.arrays[which][cache.table[s].cpu().long()[positions // 16].to(DEV), :, (positions % 16).to(DEV)] = \
                blocks.codes.to(torch.int8).to(DEV)
            cache.arrays[2 + which][cache.table[s].long()[:blocks.scales.shape[0]], :, 0] = blocks.scales.to(DEV)
    cache.store(flint)
    cache.append()
    cache.check_stored()
    cache.check_attention(*cache.attend(flint))


@pytest.mark.parametrize("longest", [1, 64])
@pytest.mark.parametrize("which", [2, 3])
def test_a_scale_that_is_not_a_number(flint, longest, which):
    """Rows that see one of its positions are NaN, and no others."""
    cache = Cache([50, 20], [80, 200], 4, 2, 16, longest=longest)
    cache.store(flint)
    cache.append()
    want = cache.attend(flint)
    cache.arrays[which][cache.table[0, 3], 1] = float("nan")       # positions 48 to 63 of sequence 0, K/V head 1
    o, lse = cache.attend(flint)
    sees = torch.arange(30, 80, device=DEV) >= 48
    assert o[:50, 128:256].isnan().all(1).equal(sees)
    assert lse[2:, :50].isnan().equal(sees.expand(2, -1))
    for got, old, rows in ((o[:50, :128], want[0][:50, :128], slice(None)), (o[50:70], want[0][50:70], slice(None)),
                           (o[:18], want[0][:18], slice(None))):
        assert torch.equal(got[rows], old[rows])


@pytest.mark.parametrize("longest", [1, 64])
def test_tokens_without_a_position(flint, longest):
    cache = Cache([5, 3], [2, 40], 4, 2, 16, longest=longest)
    cache.store(flint)
    cache.append()
    o, lse = cache.attend(flint)
    cache.check_attention(o, lse)
    assert (o[:3, :256] == 0).all() and (lse[:, :3] == float("-inf")).all()


@pytest.mark.parametrize("heads, kv_heads, new, total", [(4, 1, [1], [40000]), (8, 1, [1, 3], [20001, 300]),
                                                         (16, 2, [5, 5], [30000, 7000]), (2, 1, [200], [5000])])
def test_long_caches(flint, heads, kv_heads, new, total):
    cache = Cache(new, total, heads, kv_heads, 128)
    cache.store(flint)
    cache.append()
    cache.check_attention(*cache.attend(flint))


@pytest.mark.parametrize("heads, kv_heads, new, total", [(128, 1, [1, 2], [300, 40]), (64, 1, [1], [129]),
                                                         (40, 1, [3], [70]), (24, 1, [1, 1], [900, 2])])
def test_wide_groups(flint, heads, kv_heads, new, total):
    cache = Cache(new, total, heads, kv_heads, 64)
    cache.store(flint)
    cache.append()
    cache.check_attention(*cache.attend(flint))


@pytest.mark.parametrize("count", [40, 130])
@pytest.mark.parametrize("new", [1, 3, 60])
def test_many_sequences(flint, count, new):
    g = torch.Generator().manual_seed(count)
    total = [int(t) for t in torch.randint(1, 700, (count,), generator=g)]
    cache = Cache([min(new, t) for t in total], total, 4, 2, 32)
    cache.store(flint)
    cache.append()
    cache.check_attention(*cache.attend(flint))


@pytest.mark.parametrize("count", [33, 90, 128, 200])
@pytest.mark.parametrize("longest", [1, 64])
def test_many_sequences_without_tokens_among_them(flint, count, longest):
    g = torch.Generator().manual_seed(count)
    total = [int(t) if t > 0 else 0 for t in torch.randint(-300, 1200, (count,), generator=g)]
    total[count // 2] = 5000
    new = [0 if i % 3 == 1 else min(t, 1 + i % 2) for i, t in enumerate(total)]
    cache = Cache(new, total, 8, 2, 32, longest=longest)
    cache.store(flint)
    cache.append()
    cache.check_attention(*cache.attend(flint))
    assert not flint.kernel_fault()


@pytest.mark.parametrize("longest", [1, 64])
@pytest.mark.parametrize("page", [-1, 1 << 30])
def test_page_numbers_out_of_range_are_reported(flint, longest, page):
    cache = Cache([1, 1], [100, 60], 4, 2, 16, longest=longest)
    cache.store(flint)
    cache.append()
    want = cache.attend(flint)
    flint.kernel_fault()
    cache.table[0, 2] = page
    before = [t.clone() for t in cache.arrays]
    o, lse = cache.attend(flint)
    assert flint.kernel_fault() and not flint.kernel_fault()
    assert torch.equal(o[1], want[0][1])
    cache.table[0, 6] = page          # the new token's
    cache.store(flint)
    assert flint.kernel_fault()
    for old, now in zip(before, cache.arrays):
        assert torch.equal(old.nan_to_num(9), now.nan_to_num(9))


@pytest.mark.parametrize("starts, lengths", [([0, 5, 3], [4, 4]), ([-3, 2, 4], [8, 8]), ([0, 2, 1 << 20], [9, 9]),
                                             ([0, 1, 2], [-5, 1 << 30])])
@pytest.mark.parametrize("longest", [1, 64])
def test_starts_and_lengths_out_of_range_are_reported(flint, starts, lengths, longest):
    cache = Cache([2, 2], [30, 40], 4, 2, 16, longest=longest)
    cache.starts, cache.lengths = integers(starts), integers(lengths)
    cache.table.clamp_(max=cache.shape.pages - 1)
    flint.kernel_fault()
    cache.store(flint)
    cache.attend(flint)
    assert flint.kernel_fault() and not flint.kernel_fault()


@pytest.mark.parametrize("longest", [1, 64])
def test_without_log_sum_exps(flint, longest):
    cache = Cache([1, 2], [3000, 40], 8, 1, 64, longest=longest)
    cache.store(flint)
    want = cache.attend(flint)
    o, lse = cache.attend(flint, lse=False)
    assert torch.equal(o, want[0]) and (lse == 7.0).all()


@pytest.mark.parametrize("heads, kv_heads, new, total", [(12, 12, [1] * 5, [100, 3000, 64, 700, 1]),
                                                         (8, 2, [300, 1], [5000, 40])])
def test_results_repeat_and_replay(flint, heads, kv_heads, new, total):
    cache = Cache(new, total, heads, kv_heads, 64)
    workspace, out = cache.workspace(flint), cache.outputs()
    cache.store(flint)
    want = [t.clone() for t in cache.attend(flint, workspace, out)]
    for _ in range(3):
        workspace.fill_(255)
        for got, old in zip(cache.attend(flint, workspace, out), want):
            assert torch.equal(got, old)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            cache.store(flint)
            cache.attend(flint, workspace, out)
    torch.cuda.current_stream().wait_stream(side)
    for tensor in out:
        tensor.fill_(7.0)
    workspace.fill_(255)
    graph.replay()
    for got, old in zip(out, want):
        assert torch.equal(got, old)


def test_two_streams_at_once(flint):
    caches = [Cache([1] * 8, [2000 + 37 * i + s for i in range(8)], 8, 2, 32, seed=s) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces, outs = [c.workspace(flint) for c in caches], [c.outputs() for c in caches]
    torch.cuda.synchronize()
    for _ in range(20):
        for cache, stream, space, out in zip(caches, streams, spaces, outs):
            cache.store(flint, stream=stream)
            cache.attend(flint, space, out, stream=stream)
    torch.cuda.synchronize()
    for cache, out in zip(caches, outs):
        cache.append()
        cache.check_attention(*out)


@pytest.mark.parametrize("longest", [1, 64])
def test_offsets_beyond_32_bits(flint, longest):
    """Codes of 4.5 GB each, the sequence on their last pages."""
    cache = Cache([1], [100], 2, 2, 64, longest=longest)
    pages = (9 << 29) // (2 * 64 * 64)
    used = cache.table[0, :2].long()
    big = [torch.empty(pages, *t.shape[1:], dtype=t.dtype, device=DEV) for t in cache.arrays]
    cache.table[0, :2] = integers([pages - 1, pages - 2])
    for large, small in zip(big, cache.arrays):
        large[[pages - 1, pages - 2]] = small[used]
    cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales = big
    cache.shape.pages = pages
    cache.store(flint)
    cache.append()
    cache.check_attention(*cache.attend(flint))
    assert not flint.kernel_fault()
