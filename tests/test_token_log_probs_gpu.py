"""Log-probabilities of given tokens, entropy, alternatives and the logits' gradient, against 64 bits.

Bounds: an exponential is off by 2^-22 of itself and a sum of up to 65,536 of them, in at most 256
sequential FP32 adds per thread and a tree, by 2^-16 of itself in all; so the logarithms are off
by 2^-16 and one rounding of their operands, the entropy by 2^-16 of (1 + itself). In the
gradient that moves p by 2^-16 of itself and log p + entropy by as much in absolute terms; FP16 then rounds once."""

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
SUM = 2.0 ** -16


def make(rows, vocab, cols, fp32, seed=0, spread=2.0, offset=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed + rows + vocab)
    kind = torch.float32 if fp32 else torch.half
    logits = torch.full((rows, cols), float("nan"), dtype=kind, device=DEV)   # padding must not count
    logits[:, :vocab] = (torch.randn(rows, vocab, generator=g, device=DEV) * spread + offset).to(kind)
    targets = torch.randint(0, vocab, (rows,), generator=g, device=DEV).to(torch.int32)
    return logits, targets.to(torch.uint16)


def forward(flint, logits, targets, vocab, top, stream=None):
    rows, cols = logits.shape
    values = [torch.full((rows,), 7.0, device=DEV) for _ in range(3)]
    best = torch.full((rows, top), 7.0, device=DEV), torch.full((rows, top), 7, dtype=torch.uint16, device=DEV)
    flint.token_log_probs(*values, *(best if top else (None, None)), logits, targets, logits.dtype == torch.float32,
                          rows, vocab, cols, top, stream=stream)
    return (*values, *best)


def exact(logits, targets, vocab, top):
    x = logits[:, :vocab].double()
    log_p = torch.log_softmax(x, 1)
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(1)
    t = targets.to(torch.int64).clamp(max=vocab - 1)[:, None]
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return log_p.gather(1, t)[:, 0], entropy, torch.logsumexp(x, 1), log_p.gather(1, order), order


def check(got, want, size):
    rounding = 2.0 ** -22 * size
    assert (got[0] - want[0]).abs().max() <= SUM + rounding
    assert ((got[1] - want[1]).abs() / (1 + want[1])).max() <= SUM + rounding
    assert (got[2] - want[2]).abs().max() <= SUM + rounding
    if got[4].numel():
        assert torch.equal(got[4].to(torch.int64), want[4])
        assert (got[3] - want[3]).abs().max() <= SUM + rounding


SIZES = [(1, 8, 8, 1), (3, 1, 8, 1), (5, 31, 32, 31), (2, 33, 64, 32), (7, 500, 504, 5), (1, 50257, 50304, 20),
         (3, 65536, 65536, 32), (200, 1000, 1000, 0), (300, 777, 1024, 3), (9, 13312, 13312, 20), (2, 26624, 26632, 7),
         (150, 50257, 50304, 5), (301, 53249, 53256, 1), (20, 4096, 4096, 32), (65, 20000, 20000, 8)]


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("rows, vocab, cols, top", SIZES)
def test_forward(flint, rows, vocab, cols, top, fp32):
    logits, targets = make(rows, vocab, cols, fp32)
    got = forward(flint, logits, targets, vocab, top)
    torch.cuda.synchronize()
    check(got, exact(logits, targets, vocab, top), 30)


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("spread, offset", [(0.0, 3.0), (0.01, -7.0), (20.0, 100.0), (30.0, -5000.0), (0.25, 0.0)])
def test_flat_peaked_and_shifted_rows(flint, fp32, spread, offset):
    """Equal logits and many ties (quarter steps below), single words that take everything, large offsets."""
    logits, targets = make(40, 3001, 3008, fp32, spread=spread, offset=offset)
    if spread == 0.25:
        logits[:, :3001] = (logits[:, :3001] * 4).round() / 4
        logits[logits == 0] = -0.0       # equal to +0
        logits[:, 5:700:7] = 0.0
    got = forward(flint, logits, targets, 3001, 20)
    torch.cuda.synchronize()
    check(got, exact(logits, targets, 3001, 20), 4 * 5200 if offset < -100 else 500)


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("vocab", [100, 9000, 50257])
def test_minus_infinity_infinity_and_nan(flint, fp32, vocab):
    cols = (vocab + 7) // 8 * 8
    logits, targets = make(12, vocab, cols, fp32)
    inf = float("inf")
    targets[:] = torch.full((12,), 3, dtype=torch.int32).to(torch.uint16)
    logits[0] = -inf                                    # no token can come
    logits[1, 1:vocab] = -inf                           # one can, and the target cannot
    logits[2, :vocab // 2] = -inf
    logits[3, 17] = inf
    logits[4, 40] = float("nan")
    logits[5, :vocab - 5] = -inf                        # fewer than the alternatives asked for
    logits[6, 40] = -float("nan")
    logits[6, 41] = inf
    got = forward(flint, logits, targets, vocab, 9)
    torch.cuda.synchronize()
    want = exact(logits, targets, vocab, 9)
    usual = [1, 2, 5, 7, 8, 9, 10, 11]
    finite = lambda t: torch.where(t[usual].isinf(), -1e30, t[usual].double())
    for i in range(4):
        assert (finite(got[i]) - finite(want[i])).abs().max() <= 2 * SUM
    for row in (1, 2, 5, 7):
        assert torch.equal(got[4][row].to(torch.int64), want[4][row])
    assert got[1][1] == 0 and got[0][1] == -inf and got[3][1, 0] == 0 and (got[3][1, 1:] == -inf).all()
    assert got[0][0] == -inf and got[1][0] == 0 and got[2][0] == -inf and (got[3][0] == -inf).all()
    assert got[4][0].tolist() == list(range(9))
    for row, first in ((3, [17]), (4, [40]), (6, [40, 41])):
        assert got[0][row].isnan() and got[1][row].isnan() and got[2][row].isnan() and got[3][row].isnan().all()
        assert got[4][row].tolist()[:len(first)] == first


def test_a_target_outside_the_vocabulary_does_not_count(flint):
    logits, targets = make(6, 1000, 1008, False)
    targets[2:4] = torch.tensor([1000, 65535], dtype=torch.int32).to(torch.uint16)
    got = forward(flint, logits, targets, 1000, 2)
    dlogits = torch.full_like(logits, 7.0)
    d = torch.full((6,), 3.0, device=DEV)
    flint.token_log_probs_backward(dlogits, logits, targets, got[2], None, d, None, False, 6, 1000, 1008)
    torch.cuda.synchronize()
    assert (got[0][2:4] == 0).all() and (got[0][[0, 1, 4, 5]] < 0).all()
    assert (dlogits[2:4] == 0).all() and (dlogits[0, :1000] != 0).any()


def test_parts_that_are_not_asked_for(flint):
    logits, targets = make(50, 2000, 2000, True)
    whole = forward(flint, logits, targets, 2000, 5)
    for wanted in ([0], [1], [2], [3], []):
        out = [torch.full_like(t, 7) if i in wanted or (i == 4 and 3 in wanted) else None for i, t in enumerate(whole)]
        flint.token_log_probs(*out, logits, targets if 0 in wanted else None, True, 50, 2000, 2000,
                              5 if 3 in wanted else 0)
        torch.cuda.synchronize()
        for mine, want in zip(out, whole):
            assert mine is None or torch.equal(mine, want)


def gradient(flint, logits, targets, vocab, d_log_probs, d_entropy, in_place=False):
    rows, cols = logits.shape
    _, entropy, lse, *_ = forward(flint, logits, targets, vocab, 0)
    out = logits.clone() if in_place else torch.full_like(logits, 7.0)
    flint.token_log_probs_backward(out, out if in_place else logits, targets, lse, entropy, d_log_probs, d_entropy,
                                   logits.dtype == torch.float32, rows, vocab, cols)
    return out


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("terms", ["both", "log_probs", "entropy"])
@pytest.mark.parametrize("rows, vocab, cols", [(1, 1, 8), (3, 8, 8), (5, 500, 504), (4, 50257, 50304), (300, 777, 1024),
                                               (3, 65536, 65536), (1000, 129, 136)])
def test_gradient(flint, rows, vocab, cols, terms, fp32):
    logits, targets = make(rows, vocab, cols, fp32)
    g = torch.Generator(device=DEV).manual_seed(rows)
    a = torch.randn(rows, generator=g, device=DEV) * 8 if terms != "entropy" else None
    b = torch.randn(rows, generator=g, device=DEV) if terms != "log_probs" else None
    got = gradient(flint, logits, targets, vocab, a, b)
    same = gradient(flint, logits, targets, vocab, a, b, in_place=True)
    torch.cuda.synchronize()
    x = logits[:, :vocab].double().requires_grad_()
    log_p = torch.log_softmax(x, 1)
    t = targets.to(torch.int64)[:, None]
    entropy = -(log_p.exp() * log_p).sum(1)
    zero = torch.zeros(rows, dtype=torch.float64, device=DEV)
    da, db = (zero if d is None else d.double() for d in (a, b))
    want, = torch.autograd.grad((log_p.gather(1, t)[:, 0] * da + entropy * db).sum(), x)
    p, da, db = log_p.exp().detach(), da[:, None].abs(), db[:, None].abs()
    moved = p * (da + db * (1 + log_p.detach().abs() + entropy.detach()[:, None])) * 4 * SUM
    bound = moved + want.abs() * (2.0 ** -23 if fp32 else 2.0 ** -11) + (1e-30 if fp32 else 2.0 ** -25)
    assert ((got[:, :vocab].double() - want).abs() / bound).max() <= 1
    assert (got[:, vocab:] == 0).all()
    assert torch.equal(got, same)


@pytest.mark.parametrize("fp32", [False, True])
def test_gradient_of_tokens_that_cannot_come(flint, fp32):
    logits, targets = make(4, 900, 904, fp32)
    logits[0] = float("-inf")
    logits[1, 100:] = float("-inf")
    logits[2, 5] = float("nan")
    targets[:] = torch.full((4,), 3, dtype=torch.int32).to(torch.uint16)
    d = torch.ones(4, device=DEV)
    got = gradient(flint, logits, targets, 900, d, d)
    torch.cuda.synchronize()
    assert (got[0] == 0).all() and (got[1, 100:] == 0).all() and (got[1, :100] != 0).any()
    assert got[2, :900].isnan().all() and not got[3].isnan().any()


def test_gradient_agrees_with_differences(flint):
    logits, targets = make(30, 400, 400, True)
    g = torch.Generator(device=DEV).manual_seed(9)
    a, b = (torch.randn(30, generator=g, device=DEV) for _ in range(2))
    got = gradient(flint, logits, targets, 400, a, b)
    direction = torch.randn(30, 400, generator=g, device=DEV, dtype=torch.float64)

    def loss(x):
        log_p = torch.log_softmax(x, 1)
        return (log_p.gather(1, targets.to(torch.int64)[:, None])[:, 0] * a - (log_p.exp() * log_p).sum(1) * b).sum()

    step = 1e-5
    slope = (loss(logits.double() + step * direction) - loss(logits.double() - step * direction)) / (2 * step)
    # FP32 gradients with bounds of 2^-14 of their terms, added with independent signs.
    assert abs(slope - (got.double() * direction).sum()) <= 2.0 ** -12 * (got.double() * direction).norm()


@pytest.mark.parametrize("rows, vocab, fp32", [(3, 50257, True), (700, 50257, False), (40, 65536, True)])
def test_results_repeat_and_replay(flint, rows, vocab, fp32):
    cols = (vocab + 7) // 8 * 8
    logits, targets = make(rows, vocab, cols, fp32)
    want = forward(flint, logits, targets, vocab, 20)
    torch.cuda.synchronize()
    again = [torch.zeros_like(t) for t in want]
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        flint.token_log_probs(*again, logits, targets, fp32, rows, vocab, cols, 20)
    for _ in range(3):
        for t in again:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(want, again))


LOWEST = [(1, 8), (3, 8), (31, 16), (100, 8), (1001, 8), (9001, 96), (20001, 8), (50257, 8), (50257, 200)]


def near_the_lowest(rows, vocab):
    """FP16 rows whose logits are minus infinity, the type's lowest value or a few steps of 32 above it."""
    g = torch.Generator(device=DEV).manual_seed(rows * vocab)
    logits = torch.full((rows, (vocab + 7) // 8 * 8), float("nan"), dtype=torch.half, device=DEV)
    steps = torch.randint(0, 16, (rows, vocab), generator=g, device=DEV)
    cannot = torch.rand(rows, vocab, generator=g, device=DEV) < 0.6
    cannot[:, 0] = False
    kind, column = torch.arange(rows, device=DEV)[:, None] % 8, torch.arange(vocab, device=DEV)[None, :]
    middle = column == vocab // 2
    steps = torch.where((kind == 3) | (kind == 4), steps, 0)
    steps = torch.where((kind == 5) & middle, 3, steps)        # -65,408
    steps = torch.where((kind == 6) & middle, 15, steps)       # -65,024
    steps = torch.where((kind == 7) & middle, 17, steps)       # -64,960
    x = (steps * 32 - 65504).double()
    x = torch.where((kind == 1) & ~middle, float("-inf"), x)
    x = torch.where((kind == 2) & (column % 2 == 1), float("-inf"), x)
    x = torch.where(((kind == 4) | ((kind >= 6) & ~middle)) & cannot, float("-inf"), x)
    logits[:, :vocab] = x.half()
    assert torch.equal(logits[:, :vocab].double(), x)
    targets = torch.where(kind[:, 0] % 2 == 0, vocab // 2, 0).to(torch.int32).to(torch.uint16)
    return logits, targets


@pytest.mark.parametrize("vocab, rows", LOWEST)
def test_rows_near_the_types_lowest_value(flint, vocab, rows):
    """Minus infinity stays apart from the lowest finite value, also where that is a row's largest logit. lse
    is rounded to FP32 once more at 65,504, by 2^-9 at most."""
    logits, targets = near_the_lowest(rows, vocab)
    top = min(vocab, 5)
    got = forward(flint, logits, targets, vocab, top)
    torch.cuda.synchronize()
    want = exact(logits, targets, vocab, top)
    for mine, right, bound in ((got[0], want[0], SUM), (got[1], want[1], SUM * (1 + want[1])),
                               (got[2], want[2], SUM + 2.0 ** -9), (got[3], want[3], SUM)):
        assert torch.equal(mine.isinf(), right.isinf())
        off = torch.where(right.isinf(), 0.0, (mine.double() - right).abs())
        # (2^-22 of differences of up to 544, where these are not 0.)
        assert (off <= bound + 2.0 ** -22 * torch.where(right.isinf(), 0.0, right.abs())).all()
    assert torch.equal(got[4].to(torch.int64), want[4])
    assert (got[1][1::8] == 0).all()          # one possible word


@pytest.mark.parametrize("terms", ["both", "log_probs", "entropy"])
@pytest.mark.parametrize("vocab, rows", LOWEST)
def test_gradient_of_rows_near_the_types_lowest_value(flint, vocab, rows, terms):
    """The gradient's p comes from the FP32 lse, which is off by 2^-9 at 65,504: log p by that, and p by that of itself
    (twice as much is allowed below for the square of it)."""
    logits, targets = near_the_lowest(rows, vocab)
    g = torch.Generator(device=DEV).manual_seed(rows)
    a = torch.randn(rows, generator=g, device=DEV) * 8 if terms != "entropy" else None
    b = torch.randn(rows, generator=g, device=DEV) if terms != "log_probs" else None
    got = gradient(flint, logits, targets, vocab, a, b)
    same = gradient(flint, logits, targets, vocab, a, b, in_place=True)
    torch.cuda.synchronize()
    log_p = torch.log_softmax(logits[:, :vocab].double(), 1)
    p = log_p.exp()
    none = log_p.isinf()
    log_p = torch.where(none, 0.0, log_p)
    entropy = -(p * log_p).sum(1, keepdim=True)
    zero = torch.zeros(rows, 1, dtype=torch.float64, device=DEV)
    da, db = (zero if d is None else d.double()[:, None] for d in (a, b))
    at_target = torch.zeros_like(p).scatter_(1, targets.to(torch.int64)[:, None], 1.0)
    want = da * (at_target - p) - db * p * (log_p + entropy)
    moved = p * (da.abs() + db.abs() * (1 + log_p.abs() + entropy)) * 2 * (2.0 ** -9 + 4 * SUM)
    bound = moved + want.abs() * 2.0 ** -11 + 2.0 ** -25
    assert ((got[:, :vocab].double() - want).abs() <= bound).all()
    away = none & (at_target == 0)
    assert (got[:, :vocab][away] == 0).all() and (got[:, vocab:] == 0).all()
    assert torch.equal(got, same)


@pytest.mark.parametrize("rows, vocab, fp32, top", [(400, 51200, False, 5), (310, 51073, False, 0), (300, 51200, True, 32),
                                                    (320, 25600, True, 5), (3, 51200, False, 20)])
def test_rows_at_the_limit_of_two_blocks_on_an_sm(flint, rows, vocab, fp32, top):
    """Slices of 6,385 to 6,400 words of shared memory, several rows to a block."""
    cols = (vocab + 7) // 8 * 8
    logits, targets = make(rows, vocab, cols, fp32)
    got = forward(flint, logits, targets, vocab, top)
    torch.cuda.synchronize()
    check(got, exact(logits, targets, vocab, top), 30)


@pytest.mark.parametrize("vocab, rows", [(1, 4), (3, 4), (100, 8), (9001, 4), (50257, 4), (50257, 200)])
def test_fp32_rows_of_the_types_lowest_value(flint, vocab, rows):
    """All of a row masked with the lowest finite value, some of it with minus infinity, and all but one word."""
    lowest = torch.finfo(torch.float32).min
    logits, targets = make(rows, vocab, (vocab + 7) // 8 * 8, True)
    logits[:, :vocab] = lowest
    logits[1::4, 1:vocab:2] = -float("inf")
    logits[2::4, vocab // 2] = 0.0
    logits[3::4, :vocab // 2] = -float("inf")
    got = forward(flint, logits, targets, vocab, min(vocab, 5))
    torch.cuda.synchronize()
    want = exact(logits, targets, vocab, min(vocab, 5))
    for mine, right in zip(got[:4], want[:4]):
        assert torch.equal(mine.isneginf(), right.float().isneginf()) and not mine.isnan().any()
        off = torch.where(right.float().isneginf(), 0.0, (mine.double() - right).abs())
        # (One rounding of values up to 2^128, or SUM of logarithms.)
        assert (off <= SUM + torch.where(right.isinf(), 0.0, right.abs()) * 2.0 ** -24).all()
    assert torch.equal(got[4].to(torch.int64), want[4])
