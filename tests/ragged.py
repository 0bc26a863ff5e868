"""Attention over ragged batches in 64 bits, straight from the definition, with bounds on what
rounding may do to the library's results.

The bounds count roundings, element by element. Forward: the output rounds to FP16 once (2^-11 of
it), every probability rounds to FP16 before the product with V (2^-11 of it, or 2^-25 of the
largest where it is subnormal), and scores are FP32 sums of 64 products whose error moves a probability
by less than 2^-13 of itself. Backward: the same for P in dV; dS = P (dP - delta) rounds to
FP16 once more, P in it is off by 2^-13, and delta is taken from the rounded o, whose own error is the forward's.
"""

import torch

HALF = 2.0 ** -11      # half a step of FP16, relative
SCORE = 2.0 ** -13     # what the FP32 scores' errors do to a probability, relative
TINY = 2.0 ** -25      # half a step of FP16's subnormals


class Head:
    """One sequence's queries [n, 64] on keys and values [m, 64]; query i sees keys 0 .. before + i."""

    def __init__(self, q, k, v, before, scale, d_o=None):
        q, k, v = (t.double() for t in (q, k, v))
        n, m = q.shape[0], k.shape[0]
        sees = torch.arange(m, device=q.device)[None, :] <= torch.arange(n, device=q.device)[:, None] + before
        scores = (q @ k.T * scale).masked_fill(~sees, float("-inf"))
        self.lse = torch.logsumexp(scores, 1) if m else torch.full((n,), float("-inf"), device=q.device).double()
        nothing = ~sees.any(1) if m else torch.ones(n, dtype=torch.bool, device=q.device)
        p = torch.where(sees, torch.exp(scores - self.lse[:, None]), 0.0)
        p[nothing] = 0.0
        self.o = p @ v
        largest = v.abs().amax() if m else 0.0
        spread = p @ v.abs()
        self.o_bound = HALF * self.o.abs() + (HALF + SCORE) * spread + m * TINY * largest + TINY
        if d_o is None:
            return
        d_o = d_o.double()
        dp = d_o @ v.T
        delta = (d_o * self.o).sum(1, keepdim=True)
        ds = torch.where(sees, p * (dp - delta), 0.0)
        self.dq, self.dk, self.dv = ds @ k * scale, ds.T @ q * scale, p.T @ d_o
        off = torch.where(sees, p * ((HALF + SCORE) * (dp - delta).abs() + 2.0 ** -16 * (d_o.abs() @ v.abs().T)
                                     + (d_o.abs() * self.o_bound).sum(1, keepdim=True)) + TINY, 0.0)
        self.dq_bound = HALF * self.dq.abs() + scale * (off @ k.abs()) + TINY
        # (Without the final rounding: heads that share a key add up first.)
        self.dk_bound = scale * (off.T @ q.abs())
        self.dv_bound = (HALF + SCORE) * (p.T @ d_o.abs()) + n * TINY * d_o.abs().amax()


def within(got, want, bound):
    """The largest error in units of its bound (values that are not finite must agree)."""
    got, want = got.double(), want.double()
    same = (got == want) | (got.isnan() & want.isnan())
    ratio = torch.where(same, 0.0, (got - want).abs() / bound)
    assert not ratio.isnan().any()
    return ratio.max().item() if ratio.numel() else 0.0


LSE_BOUND = 2.0 ** -13   # absolute: the scores' error above, and 2^-22 of values up to 100
