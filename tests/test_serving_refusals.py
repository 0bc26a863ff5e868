"""What the 8-bit cache, a cache's pages and beam selection refuse, before any CUDA call."""

import ctypes

import pytest
import torch

import flint_b200
from flint_b200 import PageArrays, PagePool, PagedShape
from test_ragged_refusals import MB, PAGES, ROWS, paged, raises


@pytest.mark.parametrize("changes, text", ROWS + PAGES)
def test_paged8_shapes(flint, changes, text):
    raises(flint, text, lambda: flint.paged8_attention_workspace(paged(**changes)))
    raises(flint, text, lambda: flint.paged8_store(*[MB] * 9, paged(**changes), stream=0))
    raises(flint, text, lambda: flint.paged8_attention(*[MB] * 10, paged(**changes), 0.125, stream=0))


@pytest.mark.parametrize("scale", [0.0, -1.0, float("inf"), float("nan")])
def test_paged8_scales(flint, scale):
    raises(flint, "must be finite and positive", lambda: flint.paged8_attention(*[MB] * 10, paged(), scale, stream=0))


def test_paged8_store_pointers(flint):
    at = [1 * MB, 2 * MB, 3 * MB, 4 * MB, 5 * MB, 5 * MB + 256, 6 * MB, 7 * MB, 8 * MB]
    names = ["k_pages", "v_pages", "k_scales", "v_scales", "k", "v", "starts", "lengths", "page_table"]
    for i, name in enumerate(names):
        raises(flint, f"{name} is null", lambda: flint.paged8_store(*at[:i], None, *at[i + 1:], paged(), stream=0))
        raises(flint, f"{name} is not 16-byte aligned",
               lambda: flint.paged8_store(*at[:i], at[i] + 4, *at[i + 1:], paged(), stream=0))
    for first in range(4):
        for i in range(first + 1, 9):
            if i == 5:
                continue
            moved = list(at)
            moved[first] = at[i]
            raises(flint, "overlap", lambda: flint.paged8_store(*moved, paged(), stream=0))
    raises(flint, "shape is null", lambda: flint.paged8_store(*at, None, stream=0))


def test_nothing_to_do(flint):
    flint.paged8_store(*[None] * 9, paged(rows=0), stream=0)
    flint.paged8_attention(*[None] * 10, paged(sequences=0), 0.125, stream=0)
    none = PagePool(0, 4, 10, 16)
    flint.pages_truncate(*[None] * 4, none, stream=0)
    flint.pages_copy(PageArrays([]), None, None, 5, stream=0)
    flint.beam_select(*[None] * 11, True, 0, 4, 100, 104, stream=0)


POOLS = [(dict(sequences=65536), "sequences (65536) can be up to 65535"),
         (dict(pages=0), "pages (0) must be from 1 to 16777216"),
         (dict(pages=(1 << 24) + 1), "pages (16777217) must be"),
         (dict(page_size=8), "page_size (8) must be a power of two from 16 to 1024"),
         (dict(page_size=24), "page_size (24) must be"),
         (dict(page_size=2048), "page_size (2048) must be"),
         (dict(table_stride=0), "table_stride (0) must be from 1 to 4194304"),
         (dict(table_stride=(1 << 22) + 1), "table_stride (4194305) must be")]


def pool(**changes):
    return PagePool(**{**dict(sequences=4, table_stride=6, pages=20, page_size=16), **changes})


@pytest.mark.parametrize("changes, text", POOLS)
def test_pools(flint, changes, text):
    bad = pool(**changes)
    raises(flint, text, lambda: flint.pages_workspace(bad))
    raises(flint, text, lambda: flint.pages_fork(*[MB] * 7, bad, stream=0))
    raises(flint, text, lambda: flint.pages_reserve(*[MB] * 6, bad, MB, 1 << 40, stream=0))
    raises(flint, text, lambda: flint.pages_truncate(*[MB] * 4, bad, stream=0))
    raises(flint, text, lambda: flint.pages_compact(*[MB] * 7, bad, MB, 1 << 40, stream=0))


CALLS = {"fork": (["next_table", "next_lengths", "next_references", "page_table", "lengths", "references", "parents"], 3),
         "reserve": (["page_table", "lengths", "references", "moves", "counts", "added"], 5),
         "truncate": (["page_table", "lengths", "references", "keep"], 3),
         "compact": (["next_table", "next_references", "moves", "counts", "page_table", "lengths", "references"], 4)}


@pytest.mark.parametrize("name", CALLS)
def test_page_pointers(flint, name):
    names, outputs = CALLS[name]
    spaced = name in ("reserve", "compact")

    def call(at, space=1 << 30, size=1 << 20):
        getattr(flint, f"pages_{name}")(*at, pool(), *([space, size] if spaced else []), stream=0)

    at = [(i + 1) * MB for i in range(len(names))]
    for i, what in enumerate(names):
        raises(flint, f"{what} is null", lambda: call([*at[:i], None, *at[i + 1:]]))
        raises(flint, f"{what} is not 16-byte aligned", lambda: call([*at[:i], at[i] + 8, *at[i + 1:]]))
        for j in range(i):
            if j < outputs:
                raises(flint, "overlap", lambda: call([*at[:i], at[j], *at[i + 1:]]))
    if spaced:
        needed = flint.pages_workspace(pool())
        raises(flint, f"needs {needed} bytes of workspace, given {needed - 1}", lambda: call(at, size=needed - 1))
        raises(flint, "workspace is null", lambda: call(at, space=None))
        raises(flint, "overlap", lambda: call(at, space=at[0]))
    raises(flint, "pool is null", lambda: getattr(flint, f"pages_{name}")(*at, None, *([MB, MB] if spaced else []), stream=0))


def copy(flint, arrays=(1 * MB, 2 * MB), sizes=(64, 128), pages=10, moves=3 * MB, counts=4 * MB, most=5, count=None):
    count = len(arrays) if count is None else count
    flint.call("flint_b200_pages_copy", (ctypes.c_void_p * max(1, len(arrays)))(*arrays),
               (ctypes.c_size_t * max(1, len(sizes)))(*sizes), count, pages, moves, counts, most, stream=0)


@pytest.mark.parametrize("changes, text", [
    (dict(count=129), "count (129) can be up to 128"),
    (dict(pages=(1 << 24) + 1), "pages (16777217)"),
    (dict(most=(1 << 24) + 1), "most_moves (16777217) can be up to"),
    (dict(sizes=(64, 0)), "page_bytes[1] (0) must be a multiple of 4"),
    (dict(sizes=(6, 64)), "page_bytes[0] (6) must be a multiple of 4"),
    (dict(sizes=(64, (1 << 28) + 4)), "page_bytes[1] (268435460) must be"),
    (dict(arrays=(MB, None)), "an array is null"),
    (dict(arrays=(MB, 2 * MB + 4)), "an array is not 16-byte aligned"),
    (dict(arrays=(MB, MB + 512)), "an array and an array overlap"),
    (dict(moves=None), "moves is null"),
    (dict(counts=None), "counts is null"),
    (dict(moves=MB + 16), "an array and moves overlap")])
def test_copies(flint, changes, text):
    raises(flint, text, lambda: copy(flint, **changes))


def test_page_arrays_are_whole():
    with pytest.raises(ValueError, match="expected 4 pages"):
        PageArrays([torch.zeros(4, 8), torch.zeros(5, 8)])
    with pytest.raises(ValueError, match="expected 4 pages"):
        PageArrays([torch.zeros(4, 8).T.contiguous().T])


def select(flint, fp32=True, groups=2, beams=3, vocab=100, cols=104, stride=20, end=5, power=0.0, size=1 << 30, **changes):
    names = ["next_scores", "parents", "tokens", "next_finished", "next_lengths", "next_histories", "logits", "scores",
             "finished", "lengths", "histories"]
    at = {name: (i + 1) * MB for i, name in enumerate(names)}
    at.update(changes)
    flint.beam_select(*[at[n] for n in names], fp32, groups, beams, vocab, cols, stride, end, power, 1 << 30, size, stream=0)


@pytest.mark.parametrize("changes, text", [
    (dict(beams=0), "beams (0) must be from 1 to 32"),
    (dict(beams=33), "beams (33) must be"),
    (dict(groups=1 << 20), "groups (1048576) times beams (3) can be up to 1048576"),
    (dict(cols=100), "cols (100) must be a multiple of 8 from 8 to 65536"),
    (dict(cols=65544), "cols (65544) must be"),
    (dict(vocab=0), "vocab (0) must be from 1 to cols (104)"),
    (dict(vocab=105), "vocab (105) must be"),
    (dict(end=100), "end_token (100) must be -1 or below vocab (100)"),
    (dict(end=-2), "end_token (-2) must be"),
    (dict(power=-0.5), "length_power (-0.5) must be from 0 to 16"),
    (dict(power=16.5), "length_power (16.5) must be"),
    (dict(power=float("nan")), "length_power (nan) must be"),
    (dict(power=float("inf")), "length_power (inf) must be"),
    (dict(finished=None), "finished and next_finished go together"),
    (dict(next_finished=None), "finished and next_finished go together"),
    (dict(finished=None, next_finished=None), "finished and next_finished must be given"),
    (dict(lengths=None), "lengths and next_lengths go together"),
    (dict(lengths=None, next_lengths=None), "lengths and next_lengths must be given"),
    (dict(lengths=None, next_lengths=None, histories=None, next_histories=None, power=1.0), "lengths and next_lengths must be"),
    (dict(histories=None), "histories and next_histories go together"),
    (dict(stride=0), "history_stride (0) must be from 1 to 16777216"),
    (dict(stride=(1 << 24) + 1), "history_stride (16777217) must be")])
def test_beams(flint, changes, text):
    raises(flint, text, lambda: select(flint, **changes))


def test_beam_workspaces(flint):
    raises(flint, "beams (0) must be from 1 to 32", lambda: flint.beam_select_workspace(1, 0))
    raises(flint, "groups (1048577) times", lambda: flint.beam_select_workspace(1048577, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("changes, text", [
    (dict(size=0), "bytes of workspace, given 0"),
    (dict(logits=None), "logits is null"),
    (dict(scores=None), "scores is null"),
    (dict(parents=None), "parents is null"),
    (dict(tokens=3 * MB + 2), "tokens is not 16-byte aligned"),
    (dict(next_scores=7 * MB), "next_scores and logits overlap"),
    (dict(next_histories=11 * MB), "next_histories and histories overlap")])
def test_beam_pointers(flint, changes, text):
    """(The workspace's size depends on the GPU.)"""
    raises(flint, text, lambda: select(flint, **changes))


@pytest.mark.gpu
def test_paged8_attention_pointers(flint):
    names = ["o", "lse", "q", "k_pages", "v_pages", "k_scales", "v_scales", "starts", "lengths", "page_table"]
    at = [(i + 1) * MB for i in range(10)]
    for i, name in enumerate(names):
        if name != "lse":
            raises(flint, f"{name} is null",
                   lambda: flint.paged8_attention(*at[:i], None, *at[i + 1:], paged(), 0.125, 1 << 40, 1 << 40, stream=0))
        if i > 0:
            raises(flint, "overlap", lambda: flint.paged8_attention(at[i], *at[1:], paged(), 0.125, 1 << 40, 1 << 40, stream=0))
    raises(flint, "bytes of workspace, given 0", lambda: flint.paged8_attention(*at, paged(), 0.125, None, stream=0))
