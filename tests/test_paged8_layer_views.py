"""A layer's part of one tensor of all layers' scales: where its size is no multiple of 16 bytes it starts at any multiple of 4."""

import pytest
import torch

from flint_b200 import PageArrays, PagedShape
from test_ragged_refusals import MB, paged, raises
from test_serving_refusals import copy

DEV = "cuda"
AT = [1 * MB, 2 * MB, 3 * MB, 4 * MB, 5 * MB, 5 * MB + 256, 6 * MB, 7 * MB, 8 * MB]


@pytest.mark.parametrize("offset", [0, 4, 8, 12])
def test_arrays_of_odd_sizes(flint, offset):
    """Nothing is said of the array; the next one that is wrong is named."""
    raises(flint, "moves is null", lambda: copy(flint, (MB, 2 * MB + offset), (64, 12), pages=5, moves=None))
    shape = paged(pages=11, kv_heads=1, heads=4)
    for i in (2, 3):
        at = [*AT[:i], AT[i] + offset, *AT[i + 1:6], None, *AT[7:]]
        raises(flint, "starts is null", lambda: flint.paged8_store(*at, shape, stream=0))


@pytest.mark.parametrize("offset", [1, 2, 6])
def test_no_array_starts_within_a_number(flint, offset):
    raises(flint, "an array is not 4-byte aligned", lambda: copy(flint, (MB, 2 * MB + offset), (64, 12), pages=5))
    shape = paged(pages=11, kv_heads=1, heads=4)
    for i, name in ((2, "k_scales"), (3, "v_scales")):
        raises(flint, f"{name} is not 4-byte aligned",
               lambda: flint.paged8_store(*AT[:i], AT[i] + offset, *AT[i + 1:], shape, stream=0))


def test_sizes_of_whole_16_bytes(flint):
    raises(flint, "an array is not 16-byte aligned", lambda: copy(flint, (MB, 2 * MB + 8), (64, 8), pages=4))
    raises(flint, "an array is not 16-byte aligned", lambda: copy(flint, (MB, 2 * MB + 8), (64, 48), pages=5))


@pytest.mark.gpu
@pytest.mark.parametrize("pages, kv_heads, page_size", [(7, 1, 16), (15, 2, 16), (9, 1, 32), (5, 3, 16), (8, 1, 16)])
@pytest.mark.parametrize("longest", [1, 100])
def test_layers_of_one_tensor(flint, pages, kv_heads, page_size, longest):
    """Stored, attended to and copied: the same as in tensors of their own."""
    layers, heads, g = 3, 2 * kv_heads, torch.Generator().manual_seed(pages)
    blocks = page_size // 16
    codes = [torch.randint(-127, 128, (layers, pages, kv_heads, page_size, 64), generator=g, dtype=torch.int8).to(DEV) for _ in range(2)]
    scales = [torch.rand(layers, pages, kv_heads, blocks, generator=g).to(DEV) for _ in range(2)]
    apart = [[t[i].clone() for t in (*codes, *scales)] for i in range(layers)]
    width = (heads + 2 * kv_heads) * 64
    qkv = torch.randn(2, width, generator=g).half().to(DEV)
    shape = PagedShape(2, 2, heads, kv_heads, 64, width, width, heads * 64, pages, page_size, 2, longest)
    starts, lengths, table = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in
                              ([0, 1, 2], [page_size + 5, 9], [[3, 1], [4, 0]]))
    work = torch.empty(flint.paged8_attention_workspace(shape), dtype=torch.uint8, device=DEV)

    def layer(arrays):
        o = torch.empty(2, heads * 64, dtype=torch.half, device=DEV)
        flint.paged8_store(*arrays, qkv[:, heads * 64:], qkv[:, (heads + kv_heads) * 64:], starts, lengths, table, shape)
        flint.paged8_attention(o, None, qkv, *arrays, starts, lengths, table, shape, 0.125, work)
        return o

    moves = torch.tensor([[3, 2], [0, pages - 3 if pages == 5 else pages - 1]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([1 if pages == 5 else 2, 0], dtype=torch.int32, device=DEV)
    views = [[t[i] for t in (*codes, *scales)] for i in range(layers)]
    for here, there in zip(views, apart):
        assert torch.equal(layer(here), layer(there))
    for those in (views, apart):
        flint.pages_copy(PageArrays([t for arrays in those for t in arrays]), moves, counts, 2)
    for here, there in zip(views, apart):
        for a, b in zip(here, there):
            assert torch.equal(a, b)
    assert not flint.kernel_fault()
