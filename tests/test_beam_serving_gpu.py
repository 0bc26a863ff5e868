"""Beam search over a paged cache of 8 bits, as a server runs it: selection, fork, reserve, copies, storing, attention.

Every step is checked on its own: attention against 64 bits over what every beam's own history of codes should be, and the
selection from the library's logits (another rounding of them could choose another beam)."""

import pytest
import torch

import ragged
from eight import Blocks
from flint_b200 import PageArrays, PagePool, PagedShape
from test_beams_gpu import Step

pytestmark = pytest.mark.gpu
DEV = "cuda"
HEADS, KV, SIZE, VOCAB, SCALE = 4, 2, 16, 200, 0.125
WIDTH = (HEADS + 2 * KV) * 64


@pytest.mark.parametrize("groups, beams, prompt, steps", [(3, 4, 21, 24), (1, 7, 32, 20), (5, 1, 3, 18)])
def test_a_search(flint, groups, beams, prompt, steps):
    g = torch.Generator(device=DEV).manual_seed(groups * 100 + beams)
    rows = groups * beams
    stride = -(-(prompt + steps) // SIZE)
    pool = PagePool(rows, stride, rows * stride, SIZE)
    embedding = torch.randn(VOCAB, WIDTH, generator=g, device=DEV).half()
    head = (torch.randn(HEADS * 64, VOCAB, generator=g, device=DEV) * 0.3).half()
    whole = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=DEV)
    codes = [torch.randint(-128, 128, (pool.pages, KV, SIZE, 64), generator=g, device=DEV, dtype=torch.int8) for _ in range(2)]
    scales = [torch.full((pool.pages, KV, 1), float("nan"), device=DEV) for _ in range(2)]
    copies = PageArrays([*codes, *scales])
    state = [whole(rows, stride), whole(rows), whole(pool.pages)]       # table, lengths, references
    spare = [torch.empty_like(t) for t in state]
    moves, counts = whole(rows, 2), whole(2)
    space = torch.empty(flint.pages_workspace(pool), dtype=torch.uint8, device=DEV)
    select_space = torch.empty(flint.beam_select_workspace(groups, beams), dtype=torch.uint8, device=DEV)
    copied = 0

    def forward(tokens, per_row):
        """tokens int64 [rows * per_row]: stores them and attends; (o, lse, qkv)."""
        qkv = embedding[tokens]
        starts = torch.arange(rows + 1, device=DEV, dtype=torch.int32) * per_row
        shape = PagedShape(rows, rows * per_row, HEADS, KV, 64, WIDTH, WIDTH, HEADS * 64, pool.pages, SIZE, stride, per_row)
        workspace = torch.empty(flint.paged8_attention_workspace(shape), dtype=torch.uint8, device=DEV)
        o = torch.empty(rows * per_row, HEADS * 64, dtype=torch.half, device=DEV)
        lse = torch.empty(HEADS, rows * per_row, device=DEV)
        flint.paged8_store(*codes, *scales, qkv[:, HEADS * 64:], qkv[:, (HEADS + KV) * 64:], starts, state[1], state[0], shape)
        flint.paged8_attention(o, lse, qkv, *codes, *scales, starts, state[1], state[0], shape, SCALE, workspace)
        return o, lse, qkv

    def reserve(n):
        nonlocal copied
        flint.pages_reserve(*state, moves, counts, torch.full((rows,), n, dtype=torch.int32, device=DEV), pool, space)
        flint.pages_copy(copies, moves, counts, rows)
        assert counts[1].item() == 0
        copied += counts[0].item()

    # The prompt, once per row; then beam 0 of each group alone is in use.
    tokens = torch.randint(0, VOCAB, (groups, prompt), generator=g, device=DEV).repeat_interleave(beams, 0)
    reserve(prompt)
    o, lse, qkv = forward(tokens.flatten(), prompt)
    kept = []
    for r in range(rows):
        both = [Blocks(KV), Blocks(KV)]
        for which, blocks in enumerate(both):
            first = (HEADS + which * KV) * 64
            blocks.append(qkv[r * prompt:(r + 1) * prompt, first:first + KV * 64].view(prompt, KV, 64))
        kept.append(both)
    o = o.view(rows, prompt, -1)[:, -1]
    step = Step(groups, beams, VOCAB, None, True, end=5, power=1.0, history=steps + 1)
    step.finished.zero_()
    step.lengths.zero_()
    step.scores = torch.zeros(rows)
    step.scores.view(groups, beams)[:, 1:] = float("-inf")
    for i in range(steps):
        step.logits = (o.float() @ head.float()).cpu()
        out = step.call(flint, workspace=select_space)
        step.check(out)
        step.scores, step.finished, step.lengths = out[0].cpu(), out[3].cpu(), out[4].cpu()
        step.histories = out[5].to(torch.int32).cpu()
        parents = out[1]
        flint.pages_fork(*spare, *state, parents, pool)
        state, spare = spare, state
        reserve(1)
        o, lse, qkv = forward(out[2].to(torch.int64), 1)
        following = []
        for r, parent in enumerate(parents.tolist()):
            both = []
            for which in range(2):
                blocks = Blocks(KV)
                blocks.codes, blocks.scales = kept[parent][which].codes.clone(), kept[parent][which].scales.clone()
                first = (HEADS + which * KV) * 64
                blocks.append(qkv[r:r + 1, first:first + KV * 64].view(1, KV, 64))
                both.append(blocks)
            following.append(both)
            k, v = (blocks.values().to(DEV) for blocks in both)
            for h in range(HEADS):
                one = ragged.Head(qkv[r:r + 1, h * 64:(h + 1) * 64], k[:, h // 2], v[:, h // 2], k.shape[0] - 1, SCALE)
                bound = one.o_bound + k.shape[0] * ragged.TINY * 127 * both[1].scales.amax().item()
                assert ragged.within(o[r:r + 1, h * 64:(h + 1) * 64], one.o, bound) <= 1.0
                assert abs(lse[h, r].item() - one.lse.item()) <= ragged.LSE_BOUND
        kept = following
    # Pages that several hold count as one.
    assert state[1].tolist() == [prompt + steps] * rows
    assert state[2].sum().item() == rows * stride
    assert copied > 0 or beams == 1
    assert not flint.kernel_fault()
