"""Operators for several continuations of a prompt, as cases that can be timed and checked.

Three operators make up a step of a search that keeps its candidates in a paged cache:

    cache8   new tokens' keys and values stored in a paged cache of 8 bits, with one scale for 16
             positions of a head, and the tokens' attention to all that is in it
    pages    a step's bookkeeping: sequences that continue others' pages and grow by some tokens, with
             the pages that they no longer share copied (fork); or the pages in use moved together (compact)
    beams    the best continuations of each group of beams, over the beams and the vocabulary,
             and the reordered histories

Every case runs in two forms: elementary torch operations, and the library's calls (``own``). Heads
are 64 wide, as everywhere in the library. Lengths and the shape of a search come from a case's
``pattern``, so that a case has the same work whatever the seed of its values.
"""

import math
import random

import numpy as np
import torch

own = False

HEAD = 64
BLOCK = 16                       # positions that share a scale
VOCAB, PADDED = 50257, 50304

_library = []


def _flint():
    if not _library:
        from flint_b200.binding import Flint

        _library.append(Flint())
    return _library[0]


# ---- cases ------------------------------------------------------------------------------------


def listed():
    return [
        # Interactive use: one sequence, one token, GPT-2 124M's heads.
        {"name": "cache8_1x1_1000", "kind": "cache8", "sequences": 1, "new": 1, "longest": 1000, "pattern": 0,
         "heads": 12, "kv_heads": 12, "page_size": 64},
        # A server's decoding step: 64 sequences of very different lengths, grouped heads.
        {"name": "cache8_64x1_8192", "kind": "cache8", "sequences": 64, "new": 1, "longest": 8192, "pattern": 1,
         "heads": 32, "kv_heads": 8, "page_size": 32},
        # A few guessed tokens checked against two long caches.
        {"name": "cache8_2x5_100000", "kind": "cache8", "sequences": 2, "new": 5, "longest": 100000, "pattern": 2,
         "heads": 16, "kv_heads": 2, "page_size": 128},
        # Prompts that are worked off in chunks, some of them next to decoding sequences.
        {"name": "cache8_6x512_4096", "kind": "cache8", "sequences": 6, "new": 512, "longest": 4096, "pattern": 3,
         "heads": 16, "kv_heads": 4, "page_size": 16},
        # One prompt's eight beams on GPT-2 124M's twelve layers, after a step of the search.
        {"name": "pages_fork_1x8", "kind": "fork", "groups": 1, "beams": 8, "longest": 333, "added": 1, "pattern": 8,
         "layers": 12, "kv_heads": 12, "page_size": 16, "bits": 16},
        # A server's: 64 prompts with eight beams each, in a cache of 8 bits.
        {"name": "pages_fork_64x8", "kind": "fork", "groups": 64, "beams": 8, "longest": 2048, "added": 1, "pattern": 5,
         "layers": 12, "kv_heads": 8, "page_size": 32, "bits": 8},
        # Four samples of each of 100 prompts grow by a chunk of tokens.
        {"name": "pages_fork_100x4", "kind": "fork", "groups": 100, "beams": 4, "longest": 1024, "added": 150,
         "pattern": 6, "layers": 12, "kv_heads": 12, "page_size": 64, "bits": 16},
        # A pool that sequences have come to and gone from, half of it free, moved together.
        {"name": "pages_compact_4000", "kind": "compact", "sequences": 100, "longest": 2000, "pattern": 7,
         "layers": 12, "kv_heads": 8, "page_size": 32, "bits": 8},
        # One prompt's four beams, from a decoder's FP32 logits.
        {"name": "beams_1x4_fp32", "kind": "beams", "groups": 1, "beams": 4, "vocab": VOCAB, "cols": PADDED, "fp32": True,
         "length": 50, "power": 0.0, "finished": False, "pattern": 8},
        # A server's step: eight beams for each of 64 prompts, some of them finished.
        {"name": "beams_64x8", "kind": "beams", "groups": 64, "beams": 8, "vocab": VOCAB, "cols": PADDED, "fp32": False,
         "length": 400, "power": 1.0, "finished": True, "pattern": 9},
        # A wide search over FP32 logits.
        {"name": "beams_40x31_fp32", "kind": "beams", "groups": 40, "beams": 31, "vocab": 32001, "cols": 32008,
         "fp32": True, "length": 100, "power": 0.6, "finished": True, "pattern": 10},
        # A corpus is translated offline.
        {"name": "beams_1000x5", "kind": "beams", "groups": 1000, "beams": 5, "vocab": VOCAB, "cols": PADDED,
         "fp32": False, "length": 60, "power": 0.6, "finished": True, "pattern": 11},
    ]


# Query heads and heads of keys and values that they share.
HEADS = [(12, 12), (16, 4), (32, 8), (8, 1), (6, 2), (12, 4), (20, 20), (16, 2)]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    most = max(_cost(case) for case in listed())
    while True:
        kind = rng.choice(["cache8", "cache8", "cache8", "fork", "fork", "compact", "beams", "beams", "beams"])
        heads, kv_heads = rng.choice(HEADS)
        pattern = rng.randrange(1 << 20)
        if kind == "cache8":
            new = rng.choice([1, 1, spread(2, 16), spread(16, 700)])
            case = {"kind": kind, "sequences": spread(1, 64), "new": new, "longest": spread(max(new, 2), 100000),
                    "pattern": pattern, "heads": heads, "kv_heads": kv_heads,
                    "page_size": rng.choice([16, 32, 64, 128, 256])}
        elif kind == "beams":
            vocab = rng.choice([VOCAB, spread(500, 65536)])
            case = {"kind": kind, "groups": spread(1, 1000), "beams": spread(1, 32), "vocab": vocab,
                    "cols": PADDED if vocab == VOCAB else min(65536, (vocab + 7) // 8 * 8 + rng.choice([0, 0, 8, 64])),
                    "fp32": rng.random() < 0.4, "length": spread(1, 1000), "power": rng.choice([0.0, 0.6, 1.0]),
                    "finished": rng.random() < 0.7, "pattern": pattern}
        else:
            case = {"kind": kind, "longest": spread(1, 4096), "pattern": pattern, "layers": rng.choice([1, 6, 12, 24]),
                    "kv_heads": kv_heads, "page_size": rng.choice([16, 32, 64, 128]), "bits": rng.choice([8, 16])}
            if kind == "fork":
                case.update(groups=spread(1, 100), beams=spread(1, 16), added=rng.choice([1, 1, spread(2, 200)]))
            else:
                case.update(sequences=spread(1, 200))
        if _cost(case) <= most and _held(case) < 12e9:
            return case


def _spread_lengths(rng, count, longest):
    """Lengths that spread over the logarithm from a sixteenth of the longest, which is among them."""
    total = [max(1, int(longest * math.exp(-rng.random() * math.log(16)))) for _ in range(count)]
    total[rng.randrange(count)] = longest
    return total


def _lengths(case):
    """(new tokens, tokens in all) of each sequence of a cache8 case."""
    total = _spread_lengths(random.Random(case["pattern"]), case["sequences"], case["longest"])
    new = [min(case["new"], t) for t in total]
    if case["new"] > 16:     # a chunk for most, one token for sequences that are past their prompt
        new = [1 if i % 3 == 2 else n for i, n in enumerate(new)]
    return new, total


def _pairs(case):
    """Pairs of a token and a key that it sees, over all sequences."""
    return sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(*_lengths(case)))


class _Search:
    """The tables of a fork or compact case on the host: `table` [sequences, entries] with -1 where there is
    no page, `lengths`, `references` [pages], and for a fork `parents` and `added`."""

    def __init__(self, case):
        rng, size = random.Random(case["pattern"]), case["page_size"]
        if case["kind"] == "fork":
            groups, beams = case["groups"], case["beams"]
            prompts = _spread_lengths(rng, groups, case["longest"])
            lengths = [p + rng.randrange(1, 65) for p in prompts]      # generated so far
            shared = [p // size for p in prompts]                      # the prompt's whole pages
            added = [case["added"]] * (groups * beams)
        else:
            groups, beams = case["sequences"], 1
            lengths = _spread_lengths(rng, groups, case["longest"])
            shared, added = [0] * groups, []
        most = max(lengths) + (case["added"] if case["kind"] == "fork" else 0)
        self.sequences, self.entries = groups * beams, (most + size - 1) // size
        used = [(length + size - 1) // size for length in lengths]
        count = sum(s + (u - s) * beams for s, u in zip(shared, used))
        if case["kind"] == "fork":
            # Room for what the step can take, and some more.
            room = sum(beams * (1 + (case["added"] + size - 1) // size) for _ in lengths) + 7
        else:
            room = count
        self.pages = count + room
        order = np.random.RandomState(case["pattern"]).permutation(self.pages)[:count]
        self.table = np.full((self.sequences, self.entries), -1, np.int32)
        self.lengths = np.repeat(np.array(lengths, np.int32), beams)
        at = 0
        for g, (s, u) in enumerate(zip(shared, used)):
            self.table[g * beams:(g + 1) * beams, :s] = order[at:at + s]
            at += s
            for b in range(beams):
                self.table[g * beams + b, s:u] = order[at:at + u - s]
                at += u - s
        self.references = np.bincount(self.table[self.table >= 0], minlength=self.pages).astype(np.int32)
        # A beam is mostly continued by itself or by its group's best ones; a group in twenty is over.
        self.parents = np.array([-1 if over else g * beams + min(int(rng.random() ** 2 * beams), beams - 1)
                                 for g in range(groups) for over in [groups > 1 and rng.random() < 0.05]
                                 for _ in range(beams)], np.int32)
        self.added = np.where(self.parents >= 0, np.array(added or [0] * self.sequences, np.int32), 0).astype(np.int32)

    def copies(self, case):
        """Pages that the step copies."""
        if case["kind"] == "compact":
            used = self.references > 0
            return int(used[int(used.sum()):].sum())
        sharers = {}
        for t, parent in enumerate(self.parents):
            if parent >= 0 and self.lengths[parent] % case["page_size"]:
                page = self.table[parent, self.lengths[parent] // case["page_size"]]
                sharers[page] = sharers.get(page, 0) + 1
        return sum(n - 1 for n in sharers.values())


def _page_bytes(case):
    """Bytes of a page of keys or values in one layer, with its scales."""
    values = case["kv_heads"] * case["page_size"] * HEAD
    return values * 2 if case["bits"] == 16 else values + values // (HEAD * BLOCK) * 4


def work(case):
    if case["kind"] == "beams":
        rows, size = case["groups"] * case["beams"], 4 if case["fp32"] else 2
        read = (rows - sum(_finished(case))) * case["vocab"] * size
        return {"bytes": read + rows * (30 + 4 * case["length"]), "flops": 4 * read // size}
    if case["kind"] in ("fork", "compact"):
        search = _Search(case)
        tables = 8 * search.table.size + 8 * search.pages + 16 * search.sequences
        moved = 2 * search.copies(case) * 2 * case["layers"] * _page_bytes(case)
        return {"bytes": tables + moved, "flops": 0}
    new, total = _lengths(case)
    heads, kv_heads = case["heads"], case["kv_heads"]
    tokens = sum(new)
    # New keys and values in, then stored; the whole cache and its scales read; queries in, outputs out.
    cache = sum(total) * kv_heads * HEAD * 2 + sum((t + BLOCK - 1) // BLOCK for t in total) * kv_heads * 8
    fresh = tokens * kv_heads * HEAD * 2 * 3
    return {"bytes": fresh + cache + tokens * heads * (HEAD * 4 + 4), "flops": 4 * HEAD * heads * _pairs(case)}


def _held(case):
    """Bytes of the caches."""
    if case["kind"] == "beams":
        return 0
    if case["kind"] == "cache8":
        return sum(_lengths(case)[1]) * case["kv_heads"] * HEAD * 2
    return _Search(case).pages * 2 * case["layers"] * _page_bytes(case)


def _cost(case):
    needs = work(case)
    plain = 0     # the plain form's intermediate values
    if case["kind"] == "cache8":
        new, total = _lengths(case)
        plain = 12 * case["sequences"] * max(total) * (case["heads"] * max(new) + case["kv_heads"] * HEAD)
    elif case["kind"] == "beams":
        plain = 8 * case["groups"] * case["beams"] * case["vocab"]
    return needs["bytes"] + plain + needs["flops"] / 200


# ---- inputs -----------------------------------------------------------------------------------


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)

    def normal(*shape):
        return torch.randn(*shape, generator=generator, device="cuda")

    state = {"case": dict(case)}
    {"cache8": _prepare_cache8, "fork": _prepare_pages, "compact": _prepare_pages,
     "beams": _prepare_beams}[case["kind"]](case, state, normal, generator)
    return state


def _integers(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache8(shape, normal, generator):
    """Codes and scales as storing FP16 values gives them: a block's largest value is 127 steps."""
    codes = torch.empty(*shape, HEAD, dtype=torch.int8, device="cuda")
    flat = codes.view(-1, HEAD)
    for at in range(0, flat.shape[0], 1 << 20):
        flat[at:at + (1 << 20)] = (normal(*flat[at:at + (1 << 20)].shape) * 36).round().clamp(-127, 127)
    scales = normal(*shape[:-1], shape[-1] // BLOCK).mul(0.3).exp().mul(0.028)
    return codes, scales


def _prepare_cache8(case, state, normal, generator):
    new, total = _lengths(case)
    rows, heads, kv_heads, size = sum(new), case["heads"], case["kv_heads"], case["page_size"]
    # Queries, keys and values as one product makes them: side by side in a token's row.
    width = (heads + 2 * kv_heads) * HEAD
    pages_of = [(t + size - 1) // size for t in total]
    count = sum(pages_of) + 3
    order = torch.randperm(count, generator=generator, device="cuda").to(torch.int32)
    table = torch.zeros(case["sequences"], max(pages_of), dtype=torch.int32, device="cuda")
    first = 0
    for s, n in enumerate(pages_of):
        table[s, :n] = order[first:first + n]
        first += n
    k_pages, k_scales = _cache8((count, kv_heads, size), normal, generator)
    v_pages, v_scales = _cache8((count, kv_heads, size), normal, generator)
    state.update(qkv=normal(rows, width).half(), starts=_integers(np.cumsum([0, *new])), lengths=_integers(total),
                 table=table, longest=max(total), most=max(new), scale=HEAD ** -0.5, k_pages=k_pages,
                 v_pages=v_pages, k_scales=k_scales, v_scales=v_scales,
                 o=torch.empty(rows, heads * HEAD, dtype=torch.float16, device="cuda"),
                 lse=torch.empty(heads, rows, device="cuda"))


def _prepare_pages(case, state, normal, generator):
    search = _Search(case)
    layers, shape = case["layers"], (search.pages, case["kv_heads"], case["page_size"])
    if case["bits"] == 8:
        caches = [torch.empty(layers, *shape, HEAD, dtype=torch.int8, device="cuda") for _ in range(2)]
        caches += [normal(layers, search.pages, case["kv_heads"], case["page_size"] // BLOCK).abs() for _ in range(2)]
    else:
        caches = [torch.empty(layers, *shape, HEAD, dtype=torch.float16, device="cuda") for _ in range(2)]
    for cache in caches[:2]:
        # Whatever is in the pages is copied as it is: whole random bytes, and in FP16 numbers below 2 in size.
        raw = cache.view(torch.int8).view(-1)
        for at in range(0, raw.numel(), 1 << 28):
            raw[at:at + (1 << 28)].random_(-128, 128, generator=generator)
        if case["bits"] == 16:
            cache.view(torch.int16).bitwise_and_(-0x4001)
    state.update(table=_integers(search.table), lengths=_integers(search.lengths),
                 references=_integers(search.references), parents=_integers(search.parents),
                 added=_integers(search.added), caches=caches, layers=[layer for cache in caches for layer in cache])
    most = search.sequences if case["kind"] == "fork" else search.pages // 2
    state.update(next_table=torch.empty_like(state["table"]), next_lengths=torch.empty_like(state["lengths"]),
                 next_references=torch.empty_like(state["references"]),
                 moves=torch.empty(most, 2, dtype=torch.int32, device="cuda"),
                 counts=torch.empty(2, dtype=torch.int32, device="cuda"))


def _finished(case):
    rng = random.Random(case["pattern"])
    return [case["finished"] and rng.random() < 0.15 for _ in range(case["groups"] * case["beams"])]


def _prepare_beams(case, state, normal, generator):
    rows, vocab, cols = case["groups"] * case["beams"], case["vocab"], case["cols"]
    kind = torch.float32 if case["fp32"] else torch.float16
    # Logits as of a trained model: a broad bulk, a common offset, and a few words that stand out.
    # Padded columns are zero, as a padded table gives.
    logits = torch.zeros(rows, cols, dtype=kind, device="cuda")
    for first in range(0, rows, 1024):
        part = normal(min(1024, rows - first), vocab) * 2.0 - 3.0
        picks = torch.randint(0, vocab, (part.shape[0], 8), generator=generator, device="cuda")
        part.scatter_add_(1, picks, normal(part.shape[0], 8).abs() * 4.0 + 2.0)
        logits[first:first + part.shape[0], :vocab] = part.to(kind)
    rng = random.Random(case["pattern"] + 1)
    finished = _finished(case)
    most = case["length"] + 1
    lengths = [rng.randrange(max(1, case["length"] // 2), most) if over else case["length"] for over in finished]
    histories = torch.randint(0, vocab, (rows, most), generator=generator, device="cuda").to(torch.int32)
    state.update(logits=logits, scores=normal(rows).abs().mul(-2.0) - 0.7 * case["length"] ** 0.5,
                 finished=_integers(finished), lengths=_integers(lengths), histories=histories.to(torch.uint16),
                 end=vocab - 1 if case["finished"] else -1,
                 next_scores=torch.empty(rows, device="cuda"), parents=torch.empty(rows, dtype=torch.int32, device="cuda"),
                 tokens=torch.empty(rows, dtype=torch.uint16, device="cuda"),
                 next_finished=torch.empty(rows, dtype=torch.int32, device="cuda"),
                 next_lengths=torch.empty(rows, dtype=torch.int32, device="cuda"),
                 next_histories=torch.zeros(rows, most, dtype=torch.uint16, device="cuda"))


# ---- one pass -----------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"cache8": _own_cache8, "fork": _own_fork, "compact": _own_compact, "beams": _own_beams}[kind](state)
    return {"cache8": _plain_cache8, "fork": _plain_fork, "compact": _plain_compact,
            "beams": _plain_beams}[kind](state)


def _kept(s, name, make):
    """What a program makes once and keeps from call to call: a shape, a workspace."""
    if name not in s:
        s[name] = make()
    return s[name]


def _workspace(s, size):
    return _kept(s, "workspace", lambda: torch.empty(size(), dtype=torch.uint8, device="cuda"))


# 8 bits

def _own_cache8(s):
    from flint_b200.binding import PagedShape

    flint, case = _flint(), s["case"]
    q, k, v = _parts(case, s["qkv"])
    shape = _kept(s, "shape", lambda: PagedShape(
        case["sequences"], s["qkv"].shape[0], case["heads"], case["kv_heads"], HEAD, s["qkv"].shape[1], s["qkv"].shape[1],
        case["heads"] * HEAD, s["k_pages"].shape[0], case["page_size"], s["table"].shape[1], s["most"]))
    workspace = _workspace(s, lambda: flint.paged8_attention_workspace(shape))
    cache = (s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    flint.paged8_store(*cache, k, v, s["starts"], s["lengths"], s["table"], shape)
    flint.paged8_attention(s["o"], s["lse"], q, *cache, s["starts"], s["lengths"], s["table"], shape, s["scale"],
                           workspace)
    return (s["o"], s["lse"], *cache)


def _parts(case, qkv):
    """Views of the queries, keys and values of a matrix of token rows."""
    q, kv = case["heads"] * HEAD, case["kv_heads"] * HEAD
    return qkv[:, :q], qkv[:, q:q + kv], qkv[:, q + kv:]


def _plain_store8(s, pages, scales, fresh):
    """Stores the rows `fresh` [rows, kv heads * 64] in the blocks of 16 positions that they fall into."""
    size, kv_heads, per_page = s["case"]["page_size"], s["case"]["kv_heads"], s["case"]["page_size"] // BLOCK
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    first = lengths - new                                        # position of the first new token
    most = (s["most"] + 2 * BLOCK - 2) // BLOCK                  # blocks that a sequence's new tokens touch
    block = (first // BLOCK)[:, None] + torch.arange(most, device="cuda")
    position = block[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")        # [sequence, block, 16]
    is_new = (position >= first[:, None, None]) & (position < lengths[:, None, None])
    kept = position < first[:, None, None]
    row = (starts[:-1] - first)[:, None, None] + position
    x = fresh[row.clamp(0, fresh.shape[0] - 1)].float().unflatten(3, (kv_heads, HEAD))
    x = torch.where(is_new[..., None, None], x, 0.0)
    page = s["table"].long().gather(1, (block // per_page).clamp(max=s["table"].shape[1] - 1))
    slot = (block % per_page * BLOCK)[:, :, None] + torch.arange(BLOCK, device="cuda")
    codes = pages[page[:, :, None], :, slot].float()             # [sequence, block, 16, kv head, 64]
    before = scales[page, :, block % per_page]                   # [sequence, block, kv head]
    # (A tensor, not a number: torch multiplies by a number's reciprocal, which rounds twice.)
    scale = x.abs().amax((2, 4)) / torch.full((), 127.0, device="cuda")
    scale = torch.where(kept.any(2)[..., None], torch.maximum(before, scale), scale)
    wide = scale[:, :, None, :, None]
    values = torch.where(is_new[..., None, None], x, codes * before[:, :, None, :, None])
    codes = torch.where(wide > 0, (values / wide).round(), 0.0)
    touched = is_new.any(2)
    scales[page[touched], :, (block % per_page)[touched]] = scale[touched]
    write = (is_new | kept) & touched[..., None]
    pages[page[:, :, None].expand_as(slot)[write], :, slot[write]] = codes[write].to(torch.int8)


def _plain_cache8(s):
    case, size = s["case"], s["case"]["page_size"]
    heads, kv_heads, group, sequences = case["heads"], case["kv_heads"], case["heads"] // case["kv_heads"], case["sequences"]
    q, k, v = _parts(case, s["qkv"])
    _plain_store8(s, s["k_pages"], s["k_scales"], k)
    _plain_store8(s, s["v_pages"], s["v_scales"], v)
    # Every sequence is padded to the longest: keys [sequence, kv head, keys, 64], queries [.., new * group, 64].
    table = s["table"].long()
    keys = table.shape[1] * size

    def values(pages, scales):
        x = pages[table].float().unflatten(3, (-1, BLOCK)) * scales[table][..., None, None]
        return x.flatten(3, 4).transpose(1, 2).reshape(sequences, kv_heads, keys, HEAD)

    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    token = torch.arange(s["most"], device="cuda")
    row = (starts[:-1, None] + token).clamp(max=q.shape[0] - 1)
    real = token < new[:, None]
    qs = q[row].float().view(sequences, s["most"], kv_heads, group, HEAD).permute(0, 2, 1, 3, 4)
    scores = torch.matmul(qs.reshape(sequences, kv_heads, -1, HEAD), values(s["k_pages"], s["k_scales"]).transpose(2, 3))
    scores = scores.mul_(s["scale"]).view(sequences, kv_heads, s["most"], group, keys)
    sees = torch.arange(keys, device="cuda") <= ((lengths - new)[:, None] + token)[..., None]
    scores.masked_fill_(~sees[:, None, :, None, :], float("-inf"))
    top = scores.amax(4, keepdim=True)
    weights = scores.sub_(top).exp_()
    total = weights.sum(4, keepdim=True)
    weights /= total
    out = torch.matmul(weights.view(sequences, kv_heads, -1, keys), values(s["v_pages"], s["v_scales"]))
    out = out.view(sequences, kv_heads, s["most"], group, HEAD).permute(0, 2, 1, 3, 4).reshape(sequences, s["most"], -1)
    lse = (top + total.log())[..., 0].permute(0, 2, 1, 3).reshape(sequences, s["most"], heads)
    return (out[real].half(), lse[real].T.contiguous(), s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])


# Pages

def _own_fork(s):
    from flint_b200.binding import PageArrays, PagePool

    flint, case = _flint(), s["case"]
    pool = _kept(s, "pool", lambda: PagePool(*s["table"].shape, s["references"].shape[0], case["page_size"]))
    arrays = _kept(s, "arrays", lambda: PageArrays(s["layers"]))
    workspace = _workspace(s, lambda: flint.pages_workspace(pool))
    flint.pages_fork(s["next_table"], s["next_lengths"], s["next_references"], s["table"], s["lengths"],
                     s["references"], s["parents"], pool)
    flint.pages_reserve(s["next_table"], s["next_lengths"], s["next_references"], s["moves"], s["counts"], s["added"],
                        pool, workspace)
    flint.pages_copy(arrays, s["moves"], s["counts"], s["moves"].shape[0])
    return (s["next_table"], s["next_lengths"], s["next_references"], s["moves"], s["counts"], *s["caches"])


def _own_compact(s):
    from flint_b200.binding import PageArrays, PagePool

    flint, case = _flint(), s["case"]
    pool = _kept(s, "pool", lambda: PagePool(*s["table"].shape, s["references"].shape[0], case["page_size"]))
    arrays = _kept(s, "arrays", lambda: PageArrays(s["layers"]))
    workspace = _workspace(s, lambda: flint.pages_workspace(pool))
    flint.pages_compact(s["next_table"], s["next_references"], s["moves"], s["counts"], s["table"], s["lengths"],
                        s["references"], pool, workspace)
    flint.pages_copy(arrays, s["moves"], s["counts"], s["moves"].shape[0])
    return (s["next_table"], s["next_references"], s["moves"], s["counts"], *s["caches"])


def _used(table, lengths, size):
    """Which entries of a table hold a page."""
    return torch.arange(table.shape[1], device="cuda") < ((lengths + size - 1) // size)[:, None]


def _plain_fork(s):
    size = s["case"]["page_size"]
    table, lengths, parents = s["table"].long(), s["lengths"].long(), s["parents"].long()
    sequences, pages = table.shape[0], s["references"].shape[0]
    # Fork: the parents' tables, and every page's references in the new tables instead of the old ones.
    alive, parent = parents >= 0, parents.clamp(min=0)
    next_lengths = torch.where(alive, lengths[parent], 0)
    used = _used(table, next_lengths, size)
    next_table = torch.where(used, table[parent], -1)
    spare = torch.zeros(pages + 1, dtype=torch.int64, device="cuda")     # its last place takes the entries without a page

    def counted(table, used):
        return spare.scatter_add(0, torch.where(used, table, pages).flatten(), torch.ones_like(table).flatten())

    references = s["references"].long() - (counted(table, _used(table, lengths, size)) - counted(next_table, used))[:pages]
    # Reserve: who writes into a page that another one reads takes a copy, and the one that is left alone keeps it.
    added, sequence = s["added"].long(), torch.arange(sequences, device="cuda")
    grows = (next_lengths % size > 0) & (added > 0)
    last = torch.where(grows, next_table.gather(1, (next_lengths // size).clamp(max=table.shape[1] - 1)[:, None])[:, 0], pages)
    growers = spare.scatter_add(0, last, torch.ones_like(last))
    lowest = torch.full_like(spare, sequences).scatter_reduce(0, last, sequence, "amin")
    keeps = (growers[last] >= torch.cat([references, spare[:1]])[last]) & (lowest[last] == sequence)
    copies = grows & ~keeps
    had = (next_lengths + size - 1) // size
    grown = next_lengths + added
    fresh = torch.arange(table.shape[1], device="cuda")
    fresh = (fresh >= had[:, None]) & (fresh < ((grown + size - 1) // size)[:, None])
    needs = fresh.sum(1) + copies
    before = needs.cumsum(0) - needs
    free = torch.argsort((references != 0).to(torch.int8), stable=True)           # free pages first, in order
    missing = (needs.sum() - (references == 0).sum()).clamp(min=0)
    place = before[:, None] + copies[:, None] + fresh.cumsum(1) - 1
    out = torch.where(fresh, free[place.clamp(0, pages - 1)], next_table)
    to = free[before.clamp(max=pages - 1)]
    at = (next_lengths // size).clamp(max=table.shape[1] - 1)[:, None]
    out.scatter_(1, at, torch.where(copies, to, out.gather(1, at)[:, 0])[:, None])
    taken = spare.scatter_add(0, torch.where(fresh, out, pages).flatten(), fresh.flatten().long())
    taken = taken.scatter_add(0, torch.where(copies, to, pages), copies.long())
    taken = taken.scatter_add(0, torch.where(copies, last, pages), -copies.long())
    enough = missing == 0
    moves = torch.full((sequences + 1, 2), -1, dtype=torch.int64, device="cuda")
    rank = torch.where(copies & enough, copies.cumsum(0) - 1, sequences)
    moves.scatter_(0, rank[:, None].expand(-1, 2), torch.stack([last, to], 1))
    moves = moves[:sequences].to(torch.int32)
    real = moves[moves[:, 0] >= 0].long()
    for cache in s["caches"]:
        cache[:, real[:, 1]] = cache[:, real[:, 0]]
    return (torch.where(enough, out, next_table).to(torch.int32), torch.where(enough, grown, next_lengths).to(torch.int32),
            torch.where(enough, references + taken[:pages], references).to(torch.int32), moves,
            torch.stack([(copies & enough).sum(), missing]).to(torch.int32), *s["caches"])


def _plain_compact(s):
    size, pages, most = s["case"]["page_size"], s["references"].shape[0], s["moves"].shape[0]
    table, references = s["table"].long(), s["references"].long()
    used = references > 0
    count = used.sum()
    page = torch.arange(pages, device="cuda")
    above, holes = used & (page >= count), ~used & (page < count)
    # The i-th used page behind the place where the last one will be goes to the i-th hole before it.
    source, target = (torch.argsort((~which).to(torch.int8), stable=True) for which in (above, holes))
    moved = above.sum()
    which = page < moved
    number = page.scatter(0, source, torch.where(which, target, source))
    moves = torch.where(which[:most, None], torch.stack([source, target], 1)[:most], -1).to(torch.int32)
    real = moves[moves[:, 0] >= 0].long()
    for cache in s["caches"]:
        cache[:, real[:, 1]] = cache[:, real[:, 0]]
    next_references = torch.zeros_like(references).scatter_add(0, number, torch.where(used, references, 0))
    next_table = torch.where(_used(table, s["lengths"].long(), size), number[table.clamp(min=0)], -1)
    return (next_table.to(torch.int32), next_references.to(torch.int32), moves,
            torch.stack([moved, count]).to(torch.int32), *s["caches"])


# Beams

def _own_beams(s):
    flint, case = _flint(), s["case"]
    workspace = _workspace(s, lambda: flint.beam_select_workspace(case["groups"], case["beams"]))
    flint.beam_select(s["next_scores"], s["parents"], s["tokens"], s["next_finished"], s["next_lengths"],
                      s["next_histories"], s["logits"], s["scores"], s["finished"], s["lengths"], s["histories"],
                      case["fp32"], case["groups"], case["beams"], case["vocab"], case["cols"], s["histories"].shape[1],
                      s["end"], case["power"], workspace)
    return (s["next_scores"], s["parents"], s["tokens"], s["next_finished"], s["next_lengths"], s["next_histories"])


def _top(values, count):
    """Places of the `count` largest FP32 values of each row, equal ones in ascending order of place."""
    # FP32 bits as integers of the same order, with the place behind them: no two keys are equal.
    bits = values.contiguous().view(torch.int32).to(torch.int64)
    order = torch.where(bits >= 0, bits, -(bits & 0x7fffffff))
    keys = order * 65536 + (65535 - torch.arange(values.shape[1], device="cuda"))
    return 65535 - (torch.topk(keys, count, dim=1).values & 65535)


def _plain_beams(s):
    case, groups, beams, vocab = s["case"], s["case"]["groups"], s["case"]["beams"], s["case"]["vocab"]
    rows, finished, lengths = groups * beams, s["finished"] > 0, s["lengths"].long()
    # Totals in 64 bits: two beams' continuations can be as close as FP32's rounding of them.
    x = s["logits"][:, :vocab].float()
    top = x.amax(1, keepdim=True)
    lse = top.double() + (x - top).exp().double().sum(1, keepdim=True).log()
    best = _top(x, min(beams, vocab))
    totals = s["scores"].double()[:, None] + (x.gather(1, best).double() - lse)
    # A finished beam goes on as it is, by its end token.
    only = torch.arange(best.shape[1], device="cuda") == 0
    totals = torch.where(finished[:, None], torch.where(only, s["scores"].double()[:, None], float("-inf")), totals)
    best = torch.where(finished[:, None], max(s["end"], 0), best)
    grown = torch.where(finished, lengths, lengths + 1)
    ranks = totals / grown.clamp(min=1).double()[:, None] ** case["power"]
    # A row's candidates are in order already, equal ones by token: a stable sort leaves them so.
    place = torch.sort(ranks.view(groups, -1), dim=1, descending=True, stable=True).indices[:, :beams]
    parents = (place // best.shape[1] + torch.arange(groups, device="cuda")[:, None] * beams).flatten()
    scores, tokens = (t.view(groups, -1).gather(1, place).flatten() for t in (totals, best))
    # Places that no candidate takes: the beam of that place, at minus infinity.
    none = torch.isneginf(scores)
    row = torch.arange(rows, device="cuda")
    parents = torch.where(none, row, parents)
    tokens = torch.where(none, torch.where(finished, max(s["end"], 0), 0), tokens)
    over, at = finished[parents], lengths[parents]
    width = s["histories"].shape[1]
    column = torch.arange(width, device="cuda")
    histories = torch.where(column < at[:, None], s["histories"].to(torch.int32)[parents], 0)
    histories = torch.where((column == at[:, None]) & ~over[:, None], tokens.to(torch.int32)[:, None], histories)
    return (scores.float(), parents.to(torch.int32), tokens.to(torch.int32).to(torch.uint16),
            (over | (tokens == s["end"])).to(torch.int32), torch.where(over, at, at + 1).to(torch.int32),
            histories.to(torch.uint16))


# ---- the same from the definition, in 64 bits -------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "cache8":
        return _exact_cache8(case, s)
    if case["kind"] == "beams":
        return _exact_beams(case, s)
    return _exact_fork(case, s) if case["kind"] == "fork" else _exact_compact(case, s)


def _exact_cache8(case, s):
    heads, kv_heads, size = case["heads"], case["kv_heads"], case["page_size"]
    group = heads // kv_heads
    new, total = _lengths(case)
    rows = sum(new)
    qkv = s["qkv"].view(rows, heads + 2 * kv_heads, HEAD)
    table = s["table"].cpu()
    caches = [(s["k_pages"].clone(), s["k_scales"].clone()), (s["v_pages"].clone(), s["v_scales"].clone())]
    o = torch.empty(rows, heads, HEAD, dtype=torch.float64, device="cuda")
    lse = torch.empty(heads, rows, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, length) in enumerate(zip(new, total)):
        for which, (pages, scales) in enumerate(caches):
            first = heads + which * kv_heads
            position = length - n
            while position < length:
                # One block at a time. A scale is an FP32 number, and so is a value divided by it before it is rounded.
                block, end = position // BLOCK, min(length, (position // BLOCK + 1) * BLOCK)
                page, slot = int(table[i, position // size]), block * BLOCK % size
                fresh = qkv[at + position - (length - n):at + end - (length - n), first:first + kv_heads].double()
                kept = position - block * BLOCK
                scale = (fresh.abs().amax((0, 2)) / 127).float()
                held = pages[page, :, slot:slot + kept].double()
                if kept:
                    old = scales[page, :, slot // BLOCK]
                    scale = torch.where(old > scale, old, scale)
                    held = (held * old.double()[:, None, None]).float().double()
                    held = torch.round((held / scale.double()[:, None, None]).float())
                    pages[page, :, slot:slot + kept] = torch.nan_to_num(held).to(torch.int8)
                codes = torch.round((fresh.transpose(0, 1) / scale.double()[:, None, None]).float())
                pages[page, :, slot + kept:slot + kept + end - position] = torch.nan_to_num(codes).to(torch.int8)
                scales[page, :, slot // BLOCK] = scale
                position = end
        positions = torch.arange(length, device="cuda")
        page, slot = s["table"][i].long()[positions // size], positions % size
        k, v = (pages[page, :, slot].double() * scales[page, :, slot // BLOCK].double()[..., None]
                for pages, scales in caches)                      # [key, kv head, 64]
        sees = positions[None, :] <= positions[length - n:, None]
        for h in range(heads):
            scores = (qkv[at:at + n, h].double() @ k[:, h // group].T * s["scale"]).masked_fill(~sees, float("-inf"))
            lse[h, at:at + n] = torch.logsumexp(scores, 1)
            o[at:at + n, h] = torch.softmax(scores, 1) @ v[:, h // group]
        at += n
    return (o.view(rows, -1), lse, caches[0][0], caches[1][0], caches[0][1].double(), caches[1][1].double())


def _exact_moved(s, moves):
    out = []
    for cache in s["caches"]:
        cache = cache.clone()
        if moves:
            source, target = torch.tensor(moves, device="cuda").T
            cache[:, target] = cache[:, source]
        out.append(cache.double() if cache.dtype == torch.float32 else cache)
    return out


def _exact_fork(case, s):
    size, (sequences, entries) = case["page_size"], s["table"].shape
    old, lengths, parents, added = (s[name].tolist() for name in ("table", "lengths", "parents", "added"))
    references = s["references"].tolist()
    rows, next_lengths = [], []
    for parent in parents:
        rows.append(old[parent][:-(-lengths[parent] // size)] if parent >= 0 else [])
        next_lengths.append(lengths[parent] if parent >= 0 else 0)
    for row, length in zip(old, lengths):
        for page in row[:-(-length // size)]:
            references[page] -= 1
    for row in rows:
        for page in row:
            references[page] += 1
    # Sequences that write into the same partly filled page.
    writers = {}
    for t, (row, length) in enumerate(zip(rows, next_lengths)):
        if length % size and added[t]:
            writers.setdefault(row[-1], []).append(t)
    copying = set()
    for page, those in writers.items():
        copying.update(those if references[page] > len(those) else those[1:])
    free = [page for page, count in enumerate(references) if count == 0]
    needed = len(copying) + sum(-(-(n + a) // size) - -(-n // size) for n, a in zip(next_lengths, added))
    moves, missing = [], max(0, needed - len(free))
    if not missing:
        free = iter(free)
        for t, row in enumerate(rows):
            if t in copying:
                page = next(free)
                moves.append((row[-1], page))
                references[row[-1]] -= 1
                references[page] = 1
                row[-1] = page
            next_lengths[t] += added[t]
            while len(row) < -(-next_lengths[t] // size):
                row.append(next(free))
                references[row[-1]] = 1
    table = [row + [-1] * (entries - len(row)) for row in rows]
    return (_integers(table), _integers(next_lengths), _integers(references),
            _integers(moves + [(-1, -1)] * (sequences - len(moves))), _integers([len(moves), missing]),
            *_exact_moved(s, moves))


def _exact_compact(case, s):
    references, lengths = s["references"].tolist(), s["lengths"].tolist()
    pages, most = len(references), s["moves"].shape[0]
    count = sum(r > 0 for r in references)
    sources = [p for p in range(count, pages) if references[p] > 0]
    holes = [p for p in range(count) if references[p] == 0]
    moves = list(zip(sources, holes))
    number = dict(moves)
    after = [0] * pages
    for page, r in enumerate(references):
        if r > 0:
            after[number.get(page, page)] = r
    table = []
    for row, length in zip(s["table"].tolist(), lengths):
        n = -(-length // case["page_size"])
        table.append([number.get(page, page) for page in row[:n]] + [-1] * (len(row) - n))
    return (_integers(table), _integers(after), _integers(moves + [(-1, -1)] * (most - len(moves))),
            _integers([len(moves), count]), *_exact_moved(s, moves))


def _exact_beams(case, s):
    beams, vocab, end = case["beams"], case["vocab"], s["end"]
    columns = [[] for _ in range(6)]
    for g in range(case["groups"]):
        rows = slice(g * beams, (g + 1) * beams)
        finished, lengths = s["finished"][rows] > 0, s["lengths"][rows]
        scores, histories = s["scores"][rows].double(), s["histories"][rows].to(torch.int32)
        totals = scores[:, None] + torch.log_softmax(s["logits"][rows, :vocab].double(), 1)
        only = torch.full((vocab,), float("-inf"), dtype=torch.float64, device="cuda")
        only[max(end, 0)] = 0.0
        totals = torch.where(finished[:, None], scores[:, None] + only, totals)
        ranks = totals / torch.where(finished, lengths, lengths + 1).double()[:, None] ** case["power"]
        # Equal ones stay in the order of beam and token. (A stable sort of the best by value, and of those equal to the last.)
        flat = ranks.flatten()
        least = torch.topk(flat, beams).values[-1]
        among = (flat >= least).nonzero()[:, 0]
        place = among[torch.sort(flat[among], descending=True, stable=True).indices[:beams]]
        parent, token = place // vocab, place % vocab
        over = finished[parent]
        columns[0].append(totals.flatten()[place])
        columns[1].append((parent + g * beams).to(torch.int32))
        columns[2].append(token.to(torch.int32))
        columns[3].append((over | (token == end)).to(torch.int32))
        at = lengths[parent]
        columns[4].append(torch.where(over, at, at + 1).to(torch.int32))
        own_history = histories[parent]
        column = torch.arange(own_history.shape[1], device="cuda")
        own_history = torch.where(column < at[:, None], own_history, 0)
        own_history = torch.where((column == at[:, None]) & ~over[:, None], token.to(torch.int32)[:, None], own_history)
        columns[5].append(own_history)
    out = [torch.cat(column) for column in columns]
    out[2], out[5] = out[2].to(torch.uint16), out[5].to(torch.uint16)
    return tuple(out)
