"""Operators on prompts of different lengths, as cases that can be timed and checked.

Three operators make up a pass over a ragged batch, from its rows to the probabilities of its tokens:

    packed       causal attention over sequences that lie one behind the other in the rows of a
                 batch, with grouped heads; forward alone (scoring) or with its gradients (training)
    paged        new tokens, one or a chunk of them for each sequence, whose keys and values are
                 stored in the pages of a cache and which then attend to all that is in it
    log_probs    log-probabilities of given tokens with the entropy and the most likely
                 alternatives, alone (serving, scoring) or with the logits' gradient (training)

Every case runs in two forms: elementary torch operations in 32 bits, and the library's calls
(``own``). Heads are 64 wide, as everywhere in the library. Lengths come from a case's ``pattern``,
so that a case has the same work whatever the seed of its values.
"""

import math
import random

import torch

own = False

HEAD = 64
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
        # One short prompt: the smallest call, where latency counts.
        {"name": "packed_forward_1x37", "kind": "packed", "sequences": 1, "longest": 37, "pattern": 0,
         "heads": 12, "kv_heads": 12, "backward": False},
        # A batch of short ragged prompts on GPT-2 124M's heads: scoring.
        {"name": "packed_forward_24x700", "kind": "packed", "sequences": 24, "longest": 700, "pattern": 1,
         "heads": 12, "kv_heads": 12, "backward": False},
        # Sixteen ragged sequences of up to 1,024 tokens in training, one block's attention.
        {"name": "packed_train_16x1024", "kind": "packed", "sequences": 16, "longest": 1024, "pattern": 2,
         "heads": 12, "kv_heads": 12, "backward": True},
        # A few long documents, four query heads to each head of keys and values.
        {"name": "packed_train_5x4096", "kind": "packed", "sequences": 5, "longest": 4096, "pattern": 3,
         "heads": 16, "kv_heads": 4, "backward": True},
        # Interactive use: one sequence, one token, GPT-2 124M's heads.
        {"name": "paged_1x1_1000", "kind": "paged", "sequences": 1, "new": 1, "longest": 1000, "pattern": 0,
         "heads": 12, "kv_heads": 12, "page_size": 64},
        # A server's decoding step: 64 sequences of very different lengths, grouped heads.
        {"name": "paged_64x1_8192", "kind": "paged", "sequences": 64, "new": 1, "longest": 8192, "pattern": 1,
         "heads": 32, "kv_heads": 8, "page_size": 32},
        # A few guessed tokens checked against two long caches.
        {"name": "paged_2x5_100000", "kind": "paged", "sequences": 2, "new": 5, "longest": 100000, "pattern": 2,
         "heads": 16, "kv_heads": 2, "page_size": 128},
        # Prompts that are worked off in chunks, some of them next to decoding sequences.
        {"name": "paged_6x512_4096", "kind": "paged", "sequences": 6, "new": 512, "longest": 4096, "pattern": 3,
         "heads": 16, "kv_heads": 4, "page_size": 16},
        # One decoding sequence's token with twenty alternatives, from a decoder's FP32 logits.
        {"name": "log_probs_1_fp32", "kind": "log_probs", "rows": 1, "vocab": VOCAB, "cols": PADDED,
         "fp32": True, "top": 20, "backward": False},
        # FP32 logits of many sequences.
        {"name": "log_probs_1000_fp32", "kind": "log_probs", "rows": 1000, "vocab": VOCAB, "cols": PADDED,
         "fp32": True, "top": 5, "backward": False},
        # A corpus scored with a model's FP16 logits.
        {"name": "log_probs_8192", "kind": "log_probs", "rows": 8192, "vocab": VOCAB, "cols": PADDED,
         "fp32": False, "top": 5, "backward": False},
        # Training on weighted log-probabilities with an entropy term.
        {"name": "log_probs_train_4096", "kind": "log_probs", "rows": 4096, "vocab": VOCAB, "cols": PADDED,
         "fp32": False, "top": 0, "backward": True},
    ]


# Query heads and heads of keys and values that they share.
HEADS = [(12, 12), (16, 4), (32, 8), (8, 1), (6, 2), (12, 4), (20, 20), (16, 2)]


def draw(rng):
    def spread(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    most = max(_cost(case) for case in listed())
    while True:
        kind = rng.choice(["packed", "packed", "paged", "paged", "log_probs", "log_probs"])
        heads, kv_heads = rng.choice(HEADS)
        if kind == "packed":
            case = {"kind": kind, "sequences": spread(1, 32), "longest": spread(1, 4096),
                    "pattern": rng.randrange(1 << 20), "heads": heads, "kv_heads": kv_heads,
                    "backward": rng.random() < 0.5}
        elif kind == "paged":
            new = rng.choice([1, 1, spread(2, 16), spread(16, 700)])
            case = {"kind": kind, "sequences": spread(1, 64), "new": new, "longest": spread(max(new, 2), 100000),
                    "pattern": rng.randrange(1 << 20), "heads": heads, "kv_heads": kv_heads,
                    "page_size": rng.choice([16, 32, 64, 128, 256])}
        else:
            vocab = rng.choice([VOCAB, spread(500, 65536)])
            case = {"kind": kind, "rows": spread(1, 8192), "vocab": vocab,
                    "cols": PADDED if vocab == VOCAB else min(65536, (vocab + 7) // 8 * 8 + rng.choice([0, 0, 8, 64])),
                    "fp32": rng.random() < 0.4, "top": rng.choice([0, 1, 5, 20, 32]),
                    "backward": rng.random() < 0.4}
        if _cost(case) <= most:
            return case


def _lengths(case):
    """(new tokens, tokens in all) of each sequence. The longest is as long as the case says; the
    others spread over the logarithm from a sixteenth of it, and single tokens are among them."""
    rng = random.Random(case["pattern"])
    count, longest = case["sequences"], case["longest"]
    total = [max(1, int(longest * math.exp(-rng.random() * math.log(16)))) for _ in range(count)]
    total[rng.randrange(count)] = longest
    if case["kind"] == "packed":
        if count > 4:
            total[total.index(min(total))] = 1
        return total, total
    new = [min(case["new"], t) for t in total]
    if case["new"] > 16:     # a chunk for most, one token for sequences that are past their prompt
        new = [1 if i % 3 == 2 else n for i, n in enumerate(new)]
    return new, total


def _visible(case):
    """Pairs of a token and a key that it sees, over all sequences."""
    return sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(*_lengths(case)))


def work(case):
    if case["kind"] == "log_probs":
        rows, cols, size = case["rows"], case["cols"], 4 if case["fp32"] else 2
        read = rows * case["vocab"] * size
        out = rows * (12 + 2 + 6 * case["top"])
        if not case["backward"]:
            return {"bytes": read + out, "flops": 6 * rows * case["vocab"]}
        # The logits, which do not stay on the chip from one direction to the other, and the gradient.
        return {"bytes": 2 * read + rows * cols * size + 2 * out, "flops": 13 * rows * case["vocab"]}
    new, total = _lengths(case)
    heads, kv_heads = case["heads"], case["kv_heads"]
    pairs = _visible(case)
    tokens = sum(new)
    q_bytes, kv_bytes = tokens * heads * HEAD * 2, tokens * kv_heads * HEAD * 2
    if case["kind"] == "paged":
        # New keys and values in, then stored; the whole cache read; queries in, outputs out.
        cache = sum(total) * kv_heads * HEAD * 2 * 2
        return {"bytes": 4 * kv_bytes + cache + 2 * q_bytes + tokens * heads * 4,
                "flops": 4 * HEAD * heads * pairs}
    if not case["backward"]:
        return {"bytes": 2 * q_bytes + 2 * kv_bytes + tokens * heads * 4, "flops": 4 * HEAD * heads * pairs}
    return {"bytes": 6 * q_bytes + 6 * kv_bytes + 2 * tokens * heads * 4, "flops": 14 * HEAD * heads * pairs}


def _cost(case):
    needs = work(case)
    scores = 0 if case["kind"] == "log_probs" else 40 * _visible(case) * case["heads"]   # of the plain form
    return needs["bytes"] + scores + needs["flops"] / 200


# ---- inputs -----------------------------------------------------------------------------------


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)

    def normal(*shape):
        return torch.randn(*shape, generator=generator, device="cuda")

    state = {"case": dict(case)}
    if case["kind"] == "log_probs":
        _prepare_log_probs(case, state, normal, generator)
    else:
        _prepare_attention(case, state, normal, generator)
    return state


def _prepare_log_probs(case, state, normal, generator):
    rows, vocab, cols = case["rows"], case["vocab"], case["cols"]
    kind = torch.float32 if case["fp32"] else torch.float16
    # Logits as of a trained model: a broad bulk, a common offset, and in most rows a few words
    # that stand out, the target often among them. Padded columns are zero, as a padded table gives.
    logits = torch.zeros(rows, cols, dtype=kind, device="cuda")
    for first in range(0, rows, 1024):
        part = normal(min(1024, rows - first), vocab) * 2.0 - 3.0
        picks = torch.randint(0, vocab, (part.shape[0], 4), generator=generator, device="cuda")
        part.scatter_add_(1, picks, normal(part.shape[0], 4).abs() * 4.0 + 2.0)
        logits[first:first + part.shape[0], :vocab] = part.to(kind)
    targets = torch.randint(0, vocab, (rows,), generator=generator, device="cuda")
    likely = logits[:, :vocab].argmax(1)
    targets = torch.where(normal(rows) > 0, likely, targets)
    state.update(logits=logits, targets=targets.to(torch.int32).to(torch.uint16))
    if case["backward"]:
        # Advantages and an entropy weight, divided by the rows and multiplied by a loss scale.
        state.update(d_log_probs=normal(rows) * 8.0, d_entropy=torch.full((rows,), 0.08, device="cuda"))
    if not own:
        return
    state.update(log_probs=torch.empty(rows, device="cuda"), entropy=torch.empty(rows, device="cuda"),
                 lse=torch.empty(rows, device="cuda"),
                 top_log_probs=torch.empty(rows, case["top"], device="cuda"),
                 top_tokens=torch.empty(rows, case["top"], dtype=torch.uint16, device="cuda"))
    if case["backward"]:
        state.update(dlogits=torch.empty_like(logits))


def _prepare_attention(case, state, normal, generator):
    new, total = _lengths(case)
    rows, heads, kv_heads = sum(new), case["heads"], case["kv_heads"]
    # Queries, keys and values as one product makes them: side by side in a token's row.
    width = (heads + 2 * kv_heads) * HEAD
    qkv = normal(rows, width).half()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)

    def integers(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    state.update(qkv=qkv, starts=integers(starts), new=new, total=total, scale=HEAD ** -0.5)
    if case["kind"] == "packed":
        if case["backward"]:
            state.update(d_o=normal(rows, heads * HEAD).half())
    else:
        size = case["page_size"]
        pages_of = [(t + size - 1) // size for t in total]
        count = sum(pages_of) + 3
        order = torch.randperm(count, generator=generator, device="cuda").to(torch.int32)
        table = torch.zeros(case["sequences"], max(pages_of), dtype=torch.int32, device="cuda")
        first = 0
        for s, n in enumerate(pages_of):
            table[s, :n] = order[first:first + n]
            first += n
        pages = [torch.empty(count, kv_heads, size, HEAD, dtype=torch.float16, device="cuda") for _ in range(2)]
        for tensor in pages:
            for at in range(0, count, 1024):
                tensor[at:at + 1024] = normal(*tensor[at:at + 1024].shape).half()
        state.update(k_pages=pages[0], v_pages=pages[1], table=table, lengths=integers(total))
    if not own:
        return
    from flint_b200.binding import PackedShape, PagedShape

    state.update(o=torch.empty(rows, heads * HEAD, dtype=torch.float16, device="cuda"),
                 lse=torch.empty(heads, rows, device="cuda"))
    common = (case["sequences"], rows, heads, kv_heads, HEAD, width, width, heads * HEAD)
    if case["kind"] == "packed":
        shape = PackedShape(*common)
        size = _flint().packed_attention_workspace(shape)
        if case["backward"]:
            state.update(d_qkv=torch.empty_like(qkv))
            size = max(size, _flint().packed_attention_backward_workspace(shape))
    else:
        shape = PagedShape(*common, state["k_pages"].shape[0], case["page_size"], state["table"].shape[1], max(new))
        size = _flint().paged_attention_workspace(shape)
    state.update(shape=shape, workspace=torch.empty(size, dtype=torch.uint8, device="cuda"))


def _parts(case, qkv):
    """Views of the queries, keys and values (or their gradients) of a matrix of token rows."""
    q, kv = case["heads"] * HEAD, case["kv_heads"] * HEAD
    return qkv[:, :q], qkv[:, q:q + kv], qkv[:, q + kv:]


# ---- one pass -----------------------------------------------------------------------------------


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"packed": _own_packed, "paged": _own_paged, "log_probs": _own_log_probs}[kind](state)
    return {"packed": _plain_packed, "paged": _plain_paged, "log_probs": _plain_log_probs}[kind](state)


def _own_packed(s):
    flint = _flint()
    q, k, v = _parts(s["case"], s["qkv"])
    flint.packed_attention_forward(s["o"], s["lse"], q, k, v, s["starts"], s["shape"], s["scale"], s["workspace"])
    if not s["case"]["backward"]:
        return s["o"], s["lse"]
    dq, dk, dv = _parts(s["case"], s["d_qkv"])
    flint.packed_attention_backward(dq, dk, dv, s["d_o"], s["o"], s["lse"], q, k, v, s["starts"], s["shape"],
                                    s["scale"], s["workspace"])
    return s["o"], s["lse"], s["d_qkv"]


def _own_paged(s):
    flint = _flint()
    q, k, v = _parts(s["case"], s["qkv"])
    flint.paged_store(s["k_pages"], s["v_pages"], k, v, s["starts"], s["lengths"], s["table"], s["shape"])
    flint.paged_attention(s["o"], s["lse"], q, s["k_pages"], s["v_pages"], s["starts"], s["lengths"], s["table"],
                          s["shape"], s["scale"], s["workspace"])
    return s["o"], s["lse"], s["k_pages"], s["v_pages"]


def _own_log_probs(s):
    flint, case = _flint(), s["case"]
    rows, vocab, cols, top = case["rows"], case["vocab"], case["cols"], case["top"]
    flint.token_log_probs(s["log_probs"], s["entropy"], s["lse"], s["top_log_probs"] if top else None,
                          s["top_tokens"] if top else None, s["logits"], s["targets"], case["fp32"], rows, vocab,
                          cols, top)
    out = (s["log_probs"], s["entropy"], s["lse"], s["top_log_probs"], s["top_tokens"])
    if not case["backward"]:
        return out
    flint.token_log_probs_backward(s["dlogits"], s["logits"], s["targets"], s["lse"], s["entropy"],
                                   s["d_log_probs"], s["d_entropy"], case["fp32"], rows, vocab, cols)
    return (*out, s["dlogits"])


def _weights(q, k, scale, before):
    """Probabilities and log-sum-exp of queries [kv head, group, n, 64] on keys [kv head, m, 64], the
    first query seeing `before` + 1 of them."""
    n, m = q.shape[2], k.shape[1]
    scores = torch.matmul(q, k.unsqueeze(1).transpose(2, 3)) * scale
    hidden = torch.arange(m, device="cuda")[None, :] > torch.arange(n, device="cuda")[:, None] + before
    scores.masked_fill_(hidden, float("-inf"))
    top = scores.amax(3, keepdim=True)
    weights = scores.sub_(top).exp_()
    total = weights.sum(3, keepdim=True)
    weights /= total
    return weights, (top + total.log()).squeeze(3)


def _grouped(rows, kv_heads):
    """Rows [n, heads * 64] as FP32 [kv head, group, n, 64]."""
    n = rows.shape[0]
    return rows.float().view(n, kv_heads, -1, HEAD).permute(1, 2, 0, 3).contiguous()


def _rows(values):
    """The inverse: [kv head, group, n, 64] as rows [n, heads * 64]."""
    return values.permute(2, 0, 1, 3).reshape(values.shape[2], -1)


def _plain_packed(s):
    case, scale, starts = s["case"], s["scale"], [0]
    for n in s["new"]:
        starts.append(starts[-1] + n)
    q, k, v = _parts(case, s["qkv"])
    kv_heads = case["kv_heads"]
    o, lse, grads = [], [], []
    for a, b in zip(starts, starts[1:]):
        qs = _grouped(q[a:b], kv_heads)
        ks, vs = (t[a:b].float().view(b - a, kv_heads, HEAD).transpose(0, 1).contiguous() for t in (k, v))
        p, stat = _weights(qs, ks, scale, 0)
        out = torch.matmul(p, vs.unsqueeze(1))
        o.append(_rows(out).half())
        lse.append(stat.reshape(-1, b - a))
        if case["backward"]:
            do = _grouped(s["d_o"][a:b], kv_heads)
            dv = torch.matmul(p.transpose(2, 3), do).sum(1, keepdim=True)
            dp = torch.matmul(do, vs.unsqueeze(1).transpose(2, 3))
            ds = dp.sub_((do * out).sum(3, keepdim=True)).mul_(p).mul_(scale)
            dq = torch.matmul(ds, ks.unsqueeze(1))
            dk = torch.matmul(ds.transpose(2, 3), qs).sum(1, keepdim=True)
            grads.append(torch.cat([_rows(dq), _rows(dk), _rows(dv)], 1).half())
    out = (torch.cat(o), torch.cat(lse, 1))
    return (*out, torch.cat(grads)) if case["backward"] else out


def _plain_paged(s):
    case, size = s["case"], s["case"]["page_size"]
    q, k, v = _parts(case, s["qkv"])
    kv_heads = case["kv_heads"]
    at = 0
    o, lse = [], []
    for i, (n, total) in enumerate(zip(s["new"], s["total"])):
        positions = torch.arange(total - n, total, device="cuda")
        page, slot = s["table"][i].long()[positions // size], positions % size
        s["k_pages"][page, :, slot] = k[at:at + n].view(n, kv_heads, HEAD)
        s["v_pages"][page, :, slot] = v[at:at + n].view(n, kv_heads, HEAD)
        used = s["table"][i, :(total + size - 1) // size].long()
        ks, vs = (t[used].transpose(0, 1).reshape(kv_heads, -1, HEAD)[:, :total].float()
                  for t in (s["k_pages"], s["v_pages"]))
        p, stat = _weights(_grouped(q[at:at + n], kv_heads), ks, s["scale"], total - n)
        o.append(_rows(torch.matmul(p, vs.unsqueeze(1))).half())
        lse.append(stat.reshape(-1, n))
        at += n
    return torch.cat(o), torch.cat(lse, 1), s["k_pages"], s["v_pages"]


def _top(values, count):
    """Places of the `count` largest values of each row, equal ones in ascending order of place."""
    # FP32 bits as integers of the same order, with the place behind them: no two keys are equal.
    bits = values.contiguous().view(torch.int32).to(torch.int64)
    order = torch.where(bits >= 0, bits, -(bits & 0x7fffffff))
    keys = order * 65536 + (65535 - torch.arange(values.shape[1], device="cuda"))
    return 65535 - (torch.topk(keys, count, dim=1).values & 65535)


def _plain_log_probs(s):
    case, rows, vocab = s["case"], s["case"]["rows"], s["case"]["vocab"]
    targets = s["targets"].to(torch.int64)
    parts = []
    for first in range(0, rows, 2048):
        x = s["logits"][first:first + 2048, :vocab].float()
        t = targets[first:first + 2048, None]
        top = x.amax(1, keepdim=True)
        shifted = x - top
        e = shifted.exp()
        total = e.sum(1, keepdim=True)
        log_total = total.log()
        entropy = log_total - (e * shifted).sum(1, keepdim=True) / total
        log_prob = shifted.gather(1, t) - log_total
        best = _top(x, case["top"]) if case["top"] else t[:, :0]
        out = [log_prob[:, 0], entropy[:, 0], (top + log_total)[:, 0], shifted.gather(1, best) - log_total,
               best.to(torch.int32).to(torch.uint16)]
        if case["backward"]:
            a, b = (s[name][first:first + 2048, None] for name in ("d_log_probs", "d_entropy"))
            grad = -(e / total) * (a + b * (shifted - log_total + entropy))
            grad.scatter_add_(1, t, a)
            whole = torch.zeros(x.shape[0], case["cols"], dtype=s["logits"].dtype, device="cuda")
            whole[:, :vocab] = grad.to(whole.dtype)
            out.append(whole)
        parts.append(out)
    return tuple(torch.cat(column) for column in zip(*parts))


# ---- the same from the definition, in 64 bits -------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "log_probs":
        return _exact_log_probs(case, s)
    return _exact_attention(case, s)


def _exact_log_probs(case, s):
    vocab, top = case["vocab"], case["top"]
    columns = []
    for first in range(0, case["rows"], 512):
        rows = slice(first, first + 512)
        x = s["logits"][rows, :vocab].double().requires_grad_(case["backward"])
        log_p = torch.log_softmax(x, 1)
        picked = log_p.gather(1, s["targets"][rows].to(torch.int64)[:, None])[:, 0]
        entropy = -(log_p.exp() * log_p).sum(1)
        # A stable sort in descending order leaves equal logits in ascending order of place.
        best = torch.sort(x.detach(), dim=1, descending=True, stable=True).indices[:, :top]
        out = [picked.detach(), entropy.detach(), torch.logsumexp(x.detach(), 1), log_p.detach().gather(1, best),
               best.to(torch.int32).to(torch.uint16)]
        if case["backward"]:
            loss = (picked * s["d_log_probs"][rows].double() + entropy * s["d_entropy"][rows].double()).sum()
            grad, = torch.autograd.grad(loss, x)
            out.append(torch.nn.functional.pad(grad, (0, case["cols"] - vocab)))
        columns.append(out)
    return tuple(torch.cat(column) for column in zip(*columns))


def _exact_attention(case, s):
    new, total = s["new"], s["total"]
    heads, kv_heads, group = case["heads"], case["kv_heads"], case["heads"] // case["kv_heads"]
    rows, paged, backward = sum(new), case["kind"] == "paged", case.get("backward", False)
    qkv = s["qkv"].double().view(rows, heads + 2 * kv_heads, HEAD)
    o = torch.empty(rows, heads, HEAD, dtype=torch.float64, device="cuda")
    lse = torch.empty(heads, rows, dtype=torch.float64, device="cuda")
    d_qkv = torch.zeros_like(qkv)
    if paged:
        caches = [s["k_pages"].clone(), s["v_pages"].clone()]
    at = 0
    for i, (n, length) in enumerate(zip(new, total)):
        here = slice(at, at + n)
        if paged:
            for place, cache in enumerate(caches):
                fresh = s["qkv"].view(rows, -1, HEAD)[here, heads + place * kv_heads:heads + (place + 1) * kv_heads]
                for t in range(n):
                    p = length - n + t
                    cache[s["table"][i, p // case["page_size"]].long(), :, p % case["page_size"]] = fresh[t]
        positions = torch.arange(length, device="cuda")
        sees = positions[None, :] <= positions[length - n:, None]
        for h in range(heads):
            g = h // group
            if paged:
                page = s["table"][i].long()[positions // case["page_size"]]
                k, v = (cache[page, g, positions % case["page_size"]].double() for cache in caches)
            else:
                k, v = qkv[here, heads + g], qkv[here, heads + kv_heads + g]
            leaves = [t.clone().requires_grad_(backward) for t in (qkv[here, h], k, v)]
            scores = (leaves[0] @ leaves[1].T * s["scale"]).masked_fill(~sees, float("-inf"))
            out = torch.softmax(scores, 1) @ leaves[2]
            o[here, h] = out.detach()
            lse[h, here] = torch.logsumexp(scores.detach(), 1)
            if backward:
                d_o = s["d_o"].view(rows, heads, HEAD)[here, h].double()
                dq, dk, dv = torch.autograd.grad(out, leaves, d_o)
                d_qkv[here, h] = dq
                d_qkv[here, heads + g] += dk
                d_qkv[here, heads + kv_heads + g] += dv
        at += n
    out = (o.view(rows, -1), lse)
    if paged:
        return (*out, *caches)
    return (*out, d_qkv.view(rows, -1)) if backward else out
