"""Packed attention (sequences of any lengths one behind the other, grouped heads) against 64 bits."""

import pytest
import torch

import ragged
from flint_b200 import PackedShape

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 0.125


class Batch:
    """Inputs of a ragged batch as one matrix of [q | k | v] rows, with rows before the first sequence and
    behind the last one; those hold NaN, which must not reach anything."""

    def __init__(self, lengths, heads, kv_heads, before=0, behind=5, seed=0, extra=0, size=1.0):
        self.lengths, self.heads, self.kv_heads = lengths, heads, kv_heads
        self.rows = before + sum(lengths) + behind
        g = torch.Generator(device=DEV).manual_seed(seed + sum(lengths) + 31 * heads)
        self.width = (heads + 2 * kv_heads) * 64 + extra
        self.qkv = (torch.randn(self.rows, self.width, generator=g, device=DEV) * size).half()
        self.d_o = torch.randn(self.rows, heads * 64, generator=g, device=DEV).half()
        first = [before]
        for n in lengths:
            first.append(first[-1] + n)
        self.first = first
        self.starts = torch.tensor(first, dtype=torch.int32, device=DEV)
        for t in (self.qkv, self.d_o):
            t[:before] = float("nan")
            t[first[-1]:] = float("nan")
        self.shape = PackedShape(len(lengths), self.rows, heads, kv_heads, 64, self.width, self.width, heads * 64)

    def parts(self, rows):
        q, kv = self.heads * 64, self.kv_heads * 64
        return rows[:, :q], rows[:, q:q + kv], rows[:, q + kv:q + 2 * kv]

    def forward(self, flint, stream=None, workspace=None):
        o = torch.full((self.rows, self.heads * 64), 7.0, dtype=torch.half, device=DEV)
        lse = torch.full((self.heads, self.rows), 7.0, device=DEV)
        if workspace is None:
            workspace = torch.full((flint.packed_attention_workspace(self.shape),), 255, dtype=torch.uint8, device=DEV)
        flint.packed_attention_forward(o, lse, *self.parts(self.qkv), self.starts, self.shape, SCALE, workspace,
                                       stream=stream)
        return o, lse

    def backward(self, flint, o, lse, stream=None, workspace=None):
        grads = torch.full_like(self.qkv, 7.0)
        if workspace is None:
            workspace = torch.full((flint.packed_attention_backward_workspace(self.shape),), 255, dtype=torch.uint8,
                                   device=DEV)
        flint.packed_attention_backward(*self.parts(grads), self.d_o, o, lse, *self.parts(self.qkv), self.starts,
                                        self.shape, SCALE, workspace, stream=stream)
        return grads

    def check(self, o, lse, grads=None):
        group = self.heads // self.kv_heads
        q, k, v = self.parts(self.qkv)
        column = lambda t, h: t[:, 64 * h:64 * h + 64]
        for a, b in zip(self.first, self.first[1:]):
            if a == b:
                continue
            for g in range(self.kv_heads):
                dk = dv = dk_bound = dv_bound = 0.0
                for h in range(g * group, (g + 1) * group):
                    want = ragged.Head(column(q, h)[a:b], column(k, g)[a:b], column(v, g)[a:b], 0, SCALE,
                                       None if grads is None else column(self.d_o, h)[a:b])
                    assert ragged.within(column(o, h)[a:b], want.o, want.o_bound) <= 1
                    assert ragged.within(lse[h, a:b], want.lse, ragged.LSE_BOUND) <= 1
                    if grads is None:
                        continue
                    dq = column(self.parts(grads)[0], h)[a:b]
                    assert ragged.within(dq, want.dq, want.dq_bound) <= 1
                    dk, dv = dk + want.dk, dv + want.dv
                    dk_bound, dv_bound = dk_bound + want.dk_bound, dv_bound + want.dv_bound
                if grads is not None:
                    for got, exact, bound in ((self.parts(grads)[1], dk, dk_bound), (self.parts(grads)[2], dv, dv_bound)):
                        bound = bound + ragged.HALF * exact.abs() + ragged.TINY
                        assert ragged.within(column(got, g)[a:b], exact, bound) <= 1
        # Rows of no sequence, and columns of no head, are left as they were.
        outside = torch.ones(self.rows, dtype=torch.bool, device=DEV)
        outside[self.first[0]:self.first[-1]] = False
        assert (o[outside] == 7).all() and (lse[:, outside] == 7).all()
        if grads is not None:
            assert (grads[outside] == 7).all() and (grads[:, (self.heads + 2 * self.kv_heads) * 64:] == 7).all()


LENGTHS = [[1], [2, 1, 1], [37], [64], [65, 63], [128], [129], [127, 1, 128, 255], [0, 5, 0, 64, 300, 0], [1000, 3],
           [513, 129, 257, 31, 8, 1], [1] * 150, [2049]]
HEADS = [(1, 1), (4, 4), (6, 2), (8, 1), (5, 5), (7, 1)]


@pytest.mark.parametrize("lengths", LENGTHS, ids=lambda n: "-".join(map(str, n[:6])))
@pytest.mark.parametrize("heads, kv_heads", HEADS)
def test_forward_and_backward(flint, lengths, heads, kv_heads):
    batch = Batch(lengths, heads, kv_heads, before=3 if len(lengths) > 1 else 0)
    o, lse = batch.forward(flint)
    grads = batch.backward(flint, o, lse)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    batch.check(o, lse, grads)


@pytest.mark.parametrize("lengths, heads, kv_heads", [([700, 350, 1], 128, 1), ([90, 1, 400], 64, 2), ([33] * 40, 96, 3),
                                                      ([1024] * 4, 12, 12), ([3000, 1500], 16, 4), ([5, 3], 1024, 8),
                                                      ([1200, 40, 700], 8, 1), ([130] * 3, 128, 2)])
def test_wide_groups_and_many_items(flint, lengths, heads, kv_heads):
    batch = Batch(lengths, heads, kv_heads, extra=72)
    o, lse = batch.forward(flint)
    grads = batch.backward(flint, o, lse)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    batch.check(o, lse, grads)


@pytest.mark.parametrize("heads, kv_heads", [(12, 12), (8, 1), (6, 2)])
@pytest.mark.parametrize("count, longest", [(3, 1000), (20, 60), (32, 500), (33, 500), (100, 260), (128, 130), (129, 130)])
def test_batches_of_many_short_sequences(flint, count, longest, heads, kv_heads):
    """Tiles of one to eight key tiles, several per CTA, in batches on both sides of what deals them out whole."""
    g = torch.Generator().manual_seed(count + heads)
    lengths = torch.randint(0, longest + 1, (count,), generator=g).tolist()
    lengths[count // 2] = longest
    batch = Batch(lengths, heads, kv_heads, before=9)
    o, lse = batch.forward(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    batch.check(o, lse)


@pytest.mark.parametrize("size", [4.0, 0.01])
def test_large_and_small_scores(flint, size):
    batch = Batch([300, 150, 700], 4, 2, size=size)
    o, lse = batch.forward(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    if size < 1:     # (scores of 16 times the size have 16 times the absolute error that the bounds count)
        batch.check(o, lse)
    else:
        q, k, v = (t.clone() for t in batch.parts(batch.qkv))
        wider = ragged.SCORE
        try:
            ragged.SCORE, ragged.LSE_BOUND = 16 * wider, 16 * wider
            batch.check(o, lse)
        finally:
            ragged.SCORE, ragged.LSE_BOUND = wider, wider


def test_values_of_one_sequence_do_not_reach_another(flint):
    """Infinities and NaN in a sequence's rows change nothing in its neighbours, either direction."""
    clean = Batch([100, 60, 200, 7], 6, 2)
    o, lse = clean.forward(flint)
    grads = clean.backward(flint, o, lse)
    dirty = Batch([100, 60, 200, 7], 6, 2)
    for row, value in ((100, "nan"), (130, "inf"), (159, "-inf"), (360, "nan")):
        dirty.qkv[row] = float(value)
        dirty.d_o[row] = float(value)
    got_o, got_lse = dirty.forward(flint)
    got_grads = dirty.backward(flint, got_o, got_lse)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    for a, b in ((0, 100), (160, 360)):
        assert torch.equal(got_o[a:b], o[a:b]) and torch.equal(got_lse[:, a:b], lse[:, a:b])
        assert torch.equal(got_grads[a:b], grads[a:b])


@pytest.mark.parametrize("keys", [range(0, 1), range(0, 64), range(30, 200), range(128, 129), range(1, 300, 2)], ids=str)
def test_keys_of_minus_infinity_weigh_nothing(flint, keys):
    batch = Batch([260, 40], 4, 2)
    q, k, _ = batch.parts(batch.qkv)
    q.view(batch.rows, 4, 64)[:, :, 5].abs_().add_(0.5)
    for j in keys:
        if j < 260:
            k.view(batch.rows, 2, 64)[j, :, 5] = float("-inf")
    o, lse = batch.forward(flint)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    q, k, v = batch.parts(batch.qkv)
    for h in range(4):
        head = [t[:260, 64 * c:64 * c + 64] for t, c in ((q, h), (k, h // 2), (v, h // 2))]
        scores = head[0].double() @ head[1].double().T * SCALE
        scores = scores.masked_fill(torch.ones_like(scores).triu(1).bool(), float("-inf"))
        counts = (scores > float("-inf")).any(1)
        p = torch.softmax(scores, 1)
        got, want = o[:260, 64 * h:64 * h + 64], p @ head[2].double()
        spread = p @ head[2].double().abs()
        bound = ragged.HALF * want.abs() + (ragged.HALF + ragged.SCORE) * spread + 260 * ragged.TINY * 8
        assert got[~counts].isnan().all()
        assert ragged.within(got[counts], want[counts], bound[counts]) <= 1


def test_nan_in_a_query_or_a_key(flint):
    batch = Batch([200], 2, 1)
    batch.qkv[17, 0] = float("nan")            # query 17 of head 0
    batch.qkv[150, 2 * 64 + 3] = float("nan")  # key 150
    o, _ = batch.forward(flint)
    torch.cuda.synchronize()
    o = o[:200].view(200, 2, 64)
    assert o[17, 0].isnan().all() and o[150:, :].isnan().all()
    assert not o[18:150].isnan().any() and not o[17, 1].isnan().any() and not o[:17].isnan().any()


def test_an_lse_that_is_not_asked_for(flint):
    batch = Batch([77, 200], 4, 4)
    o, lse = batch.forward(flint)
    alone = torch.full_like(o, 7.0)
    workspace = torch.empty(flint.packed_attention_workspace(batch.shape), dtype=torch.uint8, device=DEV)
    flint.packed_attention_forward(alone, None, *batch.parts(batch.qkv), batch.starts, batch.shape, SCALE, workspace)
    torch.cuda.synchronize()
    assert torch.equal(o, alone)


def test_separate_matrices(flint):
    """q, k, v and the outputs in matrices of their own, with their own distances between rows."""
    batch = Batch([190, 1, 64], 6, 3, behind=0)
    q, k, v = (t.contiguous() for t in batch.parts(batch.qkv))
    o = torch.zeros(batch.rows, 6 * 64 + 8, dtype=torch.half, device=DEV)
    d_o = torch.zeros_like(o)
    d_o[:, :6 * 64] = batch.d_o
    lse = torch.zeros(6, batch.rows, device=DEV)
    shape = PackedShape(3, batch.rows, 6, 3, 64, 6 * 64, 3 * 64, 6 * 64 + 8)
    workspace = torch.empty(max(flint.packed_attention_workspace(shape),
                                flint.packed_attention_backward_workspace(shape)), dtype=torch.uint8, device=DEV)
    flint.packed_attention_forward(o, lse, q, k, v, batch.starts, shape, SCALE, workspace)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    flint.packed_attention_backward(dq, dk, dv, d_o, o, lse, q, k, v, batch.starts, shape, SCALE, workspace)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    batch.check(o[:, :6 * 64], lse, torch.cat([dq, dk, dv], 1))
    assert (o[:, 6 * 64:] == 0).all()


def test_results_repeat_bit_for_bit(flint):
    batch = Batch([900, 64, 333, 1024, 5, 700], 12, 4)
    o, lse = batch.forward(flint)
    grads = batch.backward(flint, o, lse)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device=DEV)
    for trial in range(4):
        flush.fill_(trial)
        again_o, again_lse = batch.forward(flint)
        again = batch.backward(flint, again_o, again_lse)
        torch.cuda.synchronize()
        assert not flint.kernel_fault()
        assert torch.equal(o.view(torch.int16), again_o.view(torch.int16)) or trial < 0
        inside = slice(0, batch.first[-1])
        assert torch.equal(lse, again_lse)
        assert torch.equal(grads[inside].view(torch.int16), again[inside].view(torch.int16))


def test_gradients_agree_with_differences(flint):
    """The directional derivative of sum(o * d_o), by central differences in 64 bits."""
    batch = Batch([150, 33], 4, 2, behind=0)
    o, lse = batch.forward(flint)
    grads = batch.backward(flint, o, lse)
    torch.cuda.synchronize()

    def loss(qkv):
        total = 0.0
        for a, b in zip(batch.first, batch.first[1:]):
            for h in range(4):
                part = lambda c: qkv[a:b, 64 * c:64 * c + 64]
                scores = part(h) @ part(4 + h // 2).T * SCALE
                scores = scores.masked_fill(torch.ones_like(scores).triu(1).bool(), float("-inf"))
                total = total + (torch.softmax(scores, 1) @ part(6 + h // 2) *
                                 batch.d_o[a:b, 64 * h:64 * h + 64].double()).sum()
        return total

    x = batch.qkv.double()
    for part in range(3):
        direction = torch.zeros_like(x)
        columns = batch.parts(direction)[part]
        columns.copy_(torch.randn(columns.shape, device=DEV, dtype=torch.float64))
        step = 1e-4
        slope = (loss(x + step * direction) - loss(x - step * direction)) / (2 * step)
        mine = (grads.double() * direction).sum()
        # Each gradient is within about 2^-9 of its size; independent signs add up as a root of squares,
        # of which eight times is allowed.
        allowed = 8 * 2.0 ** -9 * (batch.parts(grads)[part].double() * columns).norm()
        assert abs(slope - mine) <= allowed


def test_captured_and_replayed_on_another_stream(flint):
    batch = Batch([300, 17, 512], 8, 2)
    want_o, want_lse = batch.forward(flint)
    want = batch.backward(flint, want_o, want_lse)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    o, lse = torch.full_like(want_o, 7.0), torch.full_like(want_lse, 7.0)
    grads = torch.full_like(want, 7.0)
    size = max(flint.packed_attention_workspace(batch.shape), flint.packed_attention_backward_workspace(batch.shape))
    workspace = torch.empty(size, dtype=torch.uint8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        flint.packed_attention_forward(o, lse, *batch.parts(batch.qkv), batch.starts, batch.shape, SCALE, workspace)
        flint.packed_attention_backward(*batch.parts(grads), batch.d_o, o, lse, *batch.parts(batch.qkv), batch.starts,
                                        batch.shape, SCALE, workspace)
    for _ in range(3):
        o.fill_(7), lse.fill_(7), grads.fill_(7), workspace.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        assert not flint.kernel_fault()
        inside = slice(0, batch.first[-1])
        assert torch.equal(o, want_o) and torch.equal(lse, want_lse) and torch.equal(grads[inside], want[inside])


def test_offsets_beyond_32_bits(flint):
    """Rows so far apart that the last ones lie beyond 2^32 values, forward and backward."""
    batch = Batch([150, 40], 4, 2, before=0, behind=0)
    wide, before = 65536, 70000
    rows = before + batch.rows
    qkv = torch.empty(rows, wide, dtype=torch.half, device=DEV)
    qkv[before:, :batch.width] = batch.qkv
    grads = torch.empty_like(qkv)
    d_o = torch.zeros(rows, 4 * 64, dtype=torch.half, device=DEV)
    d_o[before:] = batch.d_o
    starts = batch.starts + before
    o, lse = torch.zeros_like(d_o), torch.zeros(4, rows, device=DEV)
    shape = PackedShape(2, rows, 4, 2, 64, wide, wide, 4 * 64)
    workspace = torch.empty(max(flint.packed_attention_workspace(shape),
                                flint.packed_attention_backward_workspace(shape)), dtype=torch.uint8, device=DEV)
    flint.packed_attention_forward(o, lse, *batch.parts(qkv), starts, shape, SCALE, workspace)
    flint.packed_attention_backward(*batch.parts(grads), d_o, o, lse, *batch.parts(qkv), starts, shape, SCALE, workspace)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    batch.check(o[before:], lse[:, before:], grads[before:, :batch.width])


def test_two_calls_at_once(flint):
    """Two batches on two streams, each with its own workspace, again and again."""
    batches = [Batch([700, 33, 1500], 8, 2, seed=1), Batch([2000, 1, 90, 400], 6, 6, seed=2)]
    want, streams, outputs = [], [torch.cuda.Stream() for _ in batches], []
    for batch in batches:
        o, lse = batch.forward(flint)
        want.append((o, lse, batch.backward(flint, o, lse)))
    torch.cuda.synchronize()
    for trial in range(6):
        outputs = []
        for batch, stream in zip(batches, streams):
            with torch.cuda.stream(stream):
                o, lse = batch.forward(flint)
                outputs.append((o, lse, batch.backward(flint, o, lse)))
        torch.cuda.synchronize()
        assert not flint.kernel_fault()
        for got, expected in zip(outputs, want):
            assert torch.equal(got[0], expected[0]) and torch.equal(got[1], expected[1])
            inside = expected[2] == expected[2]
            assert torch.equal(got[2][inside], expected[2][inside])


def test_one_shape_for_other_lengths(flint):
    """A captured call serves other lengths, which it reads from the device: starts may change between replays."""
    batch = Batch([300, 17, 512], 4, 2, behind=0)
    workspace = torch.empty(flint.packed_attention_workspace(batch.shape), dtype=torch.uint8, device=DEV)
    o, lse = torch.empty(batch.rows, 256, dtype=torch.half, device=DEV), torch.empty(4, batch.rows, device=DEV)
    graph = torch.cuda.CUDAGraph()
    flint.packed_attention_forward(o, lse, *batch.parts(batch.qkv), batch.starts, batch.shape, SCALE, workspace)
    with torch.cuda.graph(graph):
        flint.packed_attention_forward(o, lse, *batch.parts(batch.qkv), batch.starts, batch.shape, SCALE, workspace)
    for lengths in ([829, 0, 0], [0, 0, 829], [1, 800, 28], [276, 277, 276]):
        batch.lengths, batch.first = lengths, [0, lengths[0], lengths[0] + lengths[1], 829]
        batch.starts.copy_(torch.tensor(batch.first, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert not flint.kernel_fault()
        batch.check(o, lse)


@pytest.mark.parametrize("starts", [[0, 50, 40, 90], [-5, 10, 20, 90], [0, 30, 60, 1000], [91, 92, 93, 94]])
def test_starts_out_of_range_are_reported(flint, starts):
    batch = Batch([30, 30, 30], 4, 2, behind=0)
    batch.starts.copy_(torch.tensor(starts, dtype=torch.int32))
    o, lse = batch.forward(flint)
    torch.cuda.synchronize()
    assert flint.kernel_fault()
    assert not flint.kernel_fault()
    batch.backward(flint, o, lse)
    torch.cuda.synchronize()
    assert flint.kernel_fault()


@pytest.mark.parametrize("heads, kv_heads", [(2, 2), (4, 1)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_reaches_the_gradients_of_all_its_keys(flint, heads, kv_heads, bad):
    """Whatever column of a step's scores the query has: its row is NaN, and so are dq there and dk and dv of the keys
    that it sees. Other sequences, and keys beyond its block, get nothing of it."""
    for query in (5, 127, *range(192, 208), 299):
        batch = Batch([300, 200], heads, kv_heads, behind=0)
        batch.qkv[query, :64] = bad
        batch.qkv[:300, heads * 64] = 1.0     # (so that an infinite query's scores are infinite or NaN)
        o, lse = batch.forward(flint)
        grads = batch.backward(flint, o, lse)
        torch.cuda.synchronize()
        assert not flint.kernel_fault()
        dq, dk, dv = batch.parts(grads)
        assert o[query, :64].isnan().all() and dq[query, :64].isnan().all()
        assert dk[:query + 1, :64].isnan().all() and dv[:query + 1, :64].isnan().all()
        assert not grads[300:].isnan().any() and not o[300:].isnan().any()
        beyond = (query // 128 + 1) * 128
        assert not dv[beyond:300].isnan().any() and not dk[beyond:300].isnan().any()
        assert not dq[:, 64:].isnan().any() and not o[:, 64:].isnan().any()


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 11])
def test_small_and_large_output_gradients(flint, size):
    batch = Batch([300, 1, 40, 700], 8, 2)
    batch.d_o = (batch.d_o.float() * size).half()
    o, lse = batch.forward(flint)
    grads = batch.backward(flint, o, lse)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    batch.check(o, lse, grads)


def test_two_training_calls_at_once_against_64_bits(flint):
    batches = [Batch([700, 33, 1500], 8, 2, seed=1), Batch([2000, 1, 90, 400], 6, 6, seed=2)]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    for _ in range(2):
        outputs = []
        for batch, stream in zip(batches, streams):
            with torch.cuda.stream(stream):
                o, lse = batch.forward(flint)
                outputs.append((o, lse, batch.backward(flint, o, lse)))
        torch.cuda.synchronize()
        assert not flint.kernel_fault()
        for batch, results in zip(batches, outputs):
            batch.check(*results)


def test_as_many_sequences_as_there_can_be(flint):
    """65,535 sequences of one token or none, a few of them longer."""
    lengths = [i % 2 for i in range(65535)]
    lengths[7], lengths[30000], lengths[65534] = 300, 129, 5
    heads, kv_heads = 4, 2
    batch = Batch([1], heads, kv_heads)
    rows = sum(lengths)
    g = torch.Generator(device=DEV).manual_seed(3)
    batch.qkv = torch.randn(rows, batch.width, generator=g, device=DEV).half()
    batch.d_o = torch.randn(rows, heads * 64, generator=g, device=DEV).half()
    ends = torch.tensor(lengths).cumsum(0)
    batch.starts = torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to(torch.int32).to(DEV)
    batch.rows = rows
    batch.shape = PackedShape(65535, rows, heads, kv_heads, 64, batch.width, batch.width, heads * 64)
    o, lse = batch.forward(flint)
    grads = batch.backward(flint, o, lse)
    torch.cuda.synchronize()
    assert not flint.kernel_fault()
    q, k, v = batch.parts(batch.qkv)
    # One token: p is 1, so o is v and dv the group's sum of d_o; its score has no gradient.
    single = torch.tensor([n == 1 for n in lengths])
    at = (ends - 1)[single].to(DEV)
    spread = lambda t: t.view(rows, kv_heads, 1, 64).expand(-1, -1, 2, -1).reshape(rows, -1)
    assert torch.equal(o[at], spread(v)[at])
    scores = (q.double() * spread(k).double()).view(rows, heads, 64).sum(2).T * SCALE
    assert ((lse.double() - scores)[:, at]).abs().max() <= ragged.LSE_BOUND
    dq, dk, dv = batch.parts(grads)
    summed = batch.d_o.double().view(rows, kv_heads, 2, 64).sum(2).reshape(rows, -1)
    assert ((dv.double() - summed)[at].abs() <= ragged.HALF * summed[at].abs() + 2 * (ragged.HALF + ragged.SCORE) *
            batch.d_o.double().view(rows, kv_heads, 2, 64).abs().sum(2).reshape(rows, -1)[at] + ragged.TINY).all()
    # The longer ones in full.
    for s in (7, 30000, 65534):
        batch.first = [int(ends[s]) - lengths[s], int(ends[s])]
        whole = slice(*batch.first)
        small = Batch([lengths[s]], heads, kv_heads, behind=0)
        small.qkv, small.d_o = batch.qkv[whole], batch.d_o[whole]
        small.check(o[whole], lse[:, whole], grads[whole])
