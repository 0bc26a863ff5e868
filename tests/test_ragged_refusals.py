"""What packed attention, the paged cache and token log-probabilities refuse, before any CUDA call."""

import pytest

import flint_b200
from flint_b200 import PackedShape, PagedShape

MB = 1 << 20


def raises(flint, text, call):
    with pytest.raises(flint_b200.FlintError) as error:
        call()
    assert text in str(error.value)
    assert error.value.status == flint_b200.ERROR_INVALID_ARGUMENT


def packed(**changes):
    fields = dict(sequences=2, rows=100, heads=4, kv_heads=2, head_width=64, q_stride=512, kv_stride=512, o_stride=256)
    return PackedShape(**{**fields, **changes})


def paged(**changes):
    fields = dict(sequences=2, rows=100, heads=4, kv_heads=2, head_width=64, q_stride=512, kv_stride=512, o_stride=256,
                  pages=10, page_size=16, table_stride=5, longest=50)
    return PagedShape(**{**fields, **changes})


ROWS = [(dict(sequences=65536), "sequences (65536) can be up to 65535"),
        (dict(rows=(1 << 24) + 1), "rows (16777217) up to 16777216"),
        (dict(heads=0), "heads (0) must be from 1 to 1024"),
        (dict(kv_heads=0), "a multiple of kv_heads (0)"),
        (dict(heads=5), "heads (5) must be from 1 to 1024 and a multiple of kv_heads (2)"),
        (dict(heads=1028, q_stride=1 << 18, o_stride=1 << 18), "heads (1028) must be from 1 to 1024"),
        (dict(heads=129, kv_heads=1, q_stride=1 << 18, o_stride=1 << 18), "up to 128 times it"),
        (dict(head_width=128), "head_width (128) must be 64"),
        (dict(q_stride=248), "q_stride (248) must be a multiple of 8 from 256 to 16777216"),
        (dict(kv_stride=132), "kv_stride (132) must be a multiple of 8 from 128"),
        (dict(o_stride=(1 << 24) + 8), "o_stride (16777224) must be a multiple of 8")]
PAGES = [(dict(page_size=8), "page_size (8) must be a power of two from 16 to 1024"),
         (dict(page_size=48), "page_size (48) must be"),
         (dict(pages=0), "pages (0) must be from 1 to"),
         (dict(pages=1 << 26), "pages (67108864) must be from 1 to 67108863"),
         (dict(table_stride=0), "table_stride (0) must be from 1"),
         (dict(table_stride=1 << 23), "table_stride (8388608) must be from 1 to 4194304"),
         (dict(longest=0), "longest (0) must be from 1 to 16777216")]


def forward(flint, shape, scale=0.125, workspace_bytes=1 << 60, **changes):
    at = dict(o=1 * MB, lse=2 * MB, q=3 * MB, k=3 * MB + 512, v=3 * MB + 768, starts=4 * MB, workspace=1 << 61)
    at.update(changes)
    flint.packed_attention_forward(at["o"], at["lse"], at["q"], at["k"], at["v"], at["starts"], shape, scale,
                                   at["workspace"], workspace_bytes, stream=0)


@pytest.mark.parametrize("changes, text", ROWS)
def test_shapes(flint, changes, text):
    raises(flint, text, lambda: forward(flint, packed(**changes)))
    raises(flint, text, lambda: flint.packed_attention_workspace(packed(**changes)))
    raises(flint, text, lambda: flint.packed_attention_backward_workspace(packed(**changes)))
    raises(flint, text, lambda: flint.paged_attention_workspace(paged(**changes)))
    raises(flint, text, lambda: flint.paged_store(*[MB] * 7, paged(**changes), stream=0))


@pytest.mark.parametrize("changes, text", PAGES)
def test_page_shapes(flint, changes, text):
    raises(flint, text, lambda: flint.paged_attention_workspace(paged(**changes)))
    raises(flint, text, lambda: flint.paged_store(*[MB] * 7, paged(**changes), stream=0))


@pytest.mark.parametrize("scale", [0.0, -1.0, float("inf"), float("nan")])
def test_scales(flint, scale):
    raises(flint, "must be finite and positive", lambda: forward(flint, packed(), scale))


def test_null_shapes(flint):
    raises(flint, "shape is null", lambda: forward(flint, None))
    raises(flint, "shape is null", lambda: flint.paged_store(*[MB] * 7, None, stream=0))


def test_nothing_to_do(flint):
    flint.packed_attention_forward(None, None, None, None, None, None, packed(sequences=0), 0.125, stream=0)
    flint.packed_attention_forward(None, None, None, None, None, None, packed(rows=0), 0.125, stream=0)
    flint.packed_attention_backward(*[None] * 10, packed(rows=0), 0.125, stream=0)
    flint.paged_store(*[None] * 7, paged(rows=0), stream=0)
    flint.paged_attention(*[None] * 8, paged(sequences=0), 0.125, stream=0)
    flint.token_log_probs(None, None, None, None, None, None, None, False, 0, 8, 8, stream=0)
    flint.token_log_probs_backward(None, None, None, None, None, None, None, False, 0, 8, 8, stream=0)


def test_store_pointers(flint):
    at = [1 * MB, 2 * MB, 3 * MB, 3 * MB + 256, 4 * MB, 5 * MB, 6 * MB]
    names = ["k_pages", "v_pages", "k", "v", "starts", "lengths", "page_table"]
    for i, name in enumerate(names):
        raises(flint, f"{name} is null", lambda: flint.paged_store(*at[:i], None, *at[i + 1:], paged(), stream=0))
        raises(flint, f"{name} is not 16-byte aligned",
               lambda: flint.paged_store(*at[:i], at[i] + 4, *at[i + 1:], paged(), stream=0))
    for i in (1, 2, 4, 5, 6):
        raises(flint, f"k_pages and {names[i]} overlap",
               lambda: flint.paged_store(at[i] - 16 if i > 1 else at[i], *at[1:], paged(), stream=0))


def log_probs(flint, rows=4, vocab=100, cols=104, top=3, fp32=False, **changes):
    at = dict(log_probs=1 * MB, entropy=2 * MB, lse=3 * MB, top_log_probs=4 * MB, top_tokens=5 * MB, logits=6 * MB,
              targets=7 * MB)
    at.update(changes)
    flint.token_log_probs(*at.values(), fp32, rows, vocab, cols, top, stream=0)


@pytest.mark.parametrize("changes, text", [
    (dict(cols=100), "cols (100) must be a multiple of 8 from 8 to 65536"),
    (dict(cols=65544), "cols (65544) must be"),
    (dict(vocab=105), "vocab (105) must be from 1 to cols (104)"),
    (dict(vocab=0), "vocab (0) must be"),
    (dict(rows=(1 << 31) + 1), "rows (2147483649) can be up to 2147483648"),
    (dict(top=33), "top (33) can be up to 32"),
    (dict(vocab=2, top=3), "top (3) can be up to 32 and up to vocab (2)"),
    (dict(targets=None), "log_probs and targets go together: targets is null"),
    (dict(log_probs=None), "log_probs and targets go together: log_probs is null"),
    (dict(logits=None), "logits is null"),
    (dict(top_tokens=None), "top_tokens is null"),
    (dict(top_log_probs=None), "top_log_probs is null"),
    (dict(entropy=2 * MB + 4), "entropy is not 16-byte aligned"),
    (dict(lse=2 * MB), "entropy and lse overlap"),
    (dict(top_tokens=6 * MB), "top_tokens and logits overlap")])
def test_log_probs(flint, changes, text):
    raises(flint, text, lambda: log_probs(flint, **changes))


def backward(flint, rows=4, vocab=100, cols=104, **changes):
    at = dict(dlogits=1 * MB, logits=2 * MB, targets=3 * MB, lse=4 * MB, entropy=5 * MB, d_log_probs=6 * MB,
              d_entropy=7 * MB)
    at.update(changes)
    flint.token_log_probs_backward(*at.values(), True, rows, vocab, cols, stream=0)


@pytest.mark.parametrize("changes, text", [
    (dict(cols=12), "cols (12) must be"),
    (dict(vocab=200), "vocab (200) must be"),
    (dict(d_log_probs=None, d_entropy=None), "d_log_probs and d_entropy are both null"),
    (dict(targets=None), "targets is null"),
    (dict(entropy=None), "entropy is null"),
    (dict(lse=None), "lse is null"),
    (dict(dlogits=None), "dlogits is null"),
    (dict(logits=1 * MB + 16), "dlogits and logits overlap"),
    (dict(lse=1 * MB), "dlogits and lse overlap")])
def test_log_probs_backward(flint, changes, text):
    raises(flint, text, lambda: backward(flint, **changes))


def test_kernel_needs_a_workspace(flint):
    """(On a machine without a GPU the workspace's size, which depends on its SMs, is a CUDA error.)"""
    import torch

    if torch.cuda.is_available():
        raises(flint, "bytes of workspace, given 0", lambda: forward(flint, packed(), workspace_bytes=0))
