"""How far attention over pages of 8 bits is from 64 bits beside its results' own rounding, as the root of the mean square
over many elements.

With x the result in 64 bits and d what scores, exponentials and sums add to it, the call's result is x + d rounded to FP16, and its mean
square error r^2 + d^2 with r that rounding's. r is 2^-12 / sqrt 3 of x or more. A probability is off by 2^-18.5 of itself (the
polynomial's; the special-function unit's 2^-22), by its score's error (64 FP32 additions of a sum of size 8 or so, 2^-24 each and of either sign: below
2^-17) and by the roundings of its two parts (2^-22): by less than 2^-16. With values of either sign x and d add up in the same way, so
that d is below 2^-16 of x, r^2 + d^2 below (1.006 r)^2. A probability rounded to FP16 once is off by as much as r
relative to itself, which makes it (1.4 r)^2.
"""

import pytest
import torch

import ragged
from test_paged8_gpu import DEV, SCALE, Cache

pytestmark = pytest.mark.gpu
MOST = 1.1


def root_mean_square(errors):
    return torch.cat([e.flatten() for e in errors]).square().mean().sqrt().item()


def against_its_rounding(cache, o):
    """The results' error and their rounding's, over all sequences and heads."""
    qkv, got, least = cache.qkv.double(), [], []
    for s, (n, t) in enumerate(zip(cache.new, cache.total)):
        rows = slice(cache.first[s], cache.first[s] + n)
        k, v = (blocks.values().to(DEV) for blocks in cache.blocks[s])
        for h in range(cache.heads):
            g = h // (cache.heads // cache.kv_heads)
            want = ragged.Head(qkv[rows, h * 64:(h + 1) * 64], k[:, g], v[:, g], t - n, SCALE).o
            got.append(o[rows, h * 64:(h + 1) * 64].double() - want)
            least.append(want.half().double() - want)
    return root_mean_square(got), root_mean_square(least)


@pytest.mark.parametrize("new", [1, 2, 4, 5, 8, 16, 17, 100])      # 4 to 68 rows of a head's group, and a tile in parts
@pytest.mark.parametrize("count, total", [(24, 700), (3, 6000)])
def test_results_are_off_by_their_own_rounding(flint, new, count, total):
    cache = Cache([new] * count, [total - 19 * i for i in range(count - 1)] + [new + 30], 8, 2, 32, seed=new)
    cache.store(flint)
    cache.append()
    got, least = against_its_rounding(cache, cache.attend(flint)[0])
    assert got <= MOST * least, got / least


def put(cache, s, which, block, codes, scale):
    """Sets a block that the sequence has already, on the host and in the cache."""
    blocks, size = cache.blocks[s][which], cache.size
    positions = torch.arange(block * 16, block * 16 + 16)
    blocks.codes[positions], blocks.scales[block] = codes, scale
    page = cache.table[s].cpu().long()[positions // size].to(DEV)
    cache.arrays[which][page, :, (positions % size).to(DEV)] = codes.to(torch.int8).to(DEV)
    cache.arrays[2 + which][page[0], :, block * 16 % size // 16] = scale.to(DEV)


@pytest.mark.parametrize("amplitude", [1e-3, 1e-2, 1.0])
@pytest.mark.parametrize("new", [1, 4, 8, 16, 100])
def test_zeros_cost_other_values_no_accuracy(flint, new, amplitude):
    """Blocks of V that are 0 have no part in a result but their probabilities'. Their weight must not push the others' probabilities
    below what FP16 holds: values of 10^-3 give scales near 2^-15, and products of both that are off by 2^-25 would be by a
    thousandth of themselves and more. (Results near 10^-4 are FP16 numbers of their full precision above 2^-14, and off by 2^-25
    below: both sides have that rounding.)"""
    count = 12
    cache = Cache([new] * count, [new + 48 + 3 * i for i in range(count)], 8, 2, 32, seed=new)
    cache.qkv[:, (cache.heads + cache.kv_heads) * 64:] *= amplitude
    for s in range(count):
        blocks = cache.blocks[s][1]
        for block in range(3):
            put(cache, s, 1, block, blocks.codes[16 * block:16 * block + 16] * (block != 1), blocks.scales[block] * amplitude * (block != 1))
        for block in range(3, blocks.scales.shape[0]):
            blocks.scales[block] *= amplitude
            at = block * 16
            cache.v_scales[cache.table[s, at // 32].long(), :, at % 32 // 16] *= amplitude
    cache.store(flint)
    cache.append()
    cache.check_stored()
    got, least = against_its_rounding(cache, cache.attend(flint)[0])
    assert got <= MOST * least, got / least
