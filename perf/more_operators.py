"""The cache of keys and values that is held in 8 bits, and the attention that reads it.

* ``write``: ``QuantizedCache.write``: keys and values of new tokens to int8 codes, one scale for each page of 64 tokens and head, and the pages that were
  written to read back (``QuantizedCache.read``), older tokens of theirs among them;
* ``read``: ``QuantizedCache.read``: cached tokens as floats again;
* ``attend``: ``QuantizedCache.attend``: causal attention of the newest tokens over the cache, query heads sharing key heads, for one token of each sequence,
  a few or a whole prompt; with a window, and first tokens that stay visible behind it (sinks), or without.

Sizes: 1 .. 256 sequences of up to 131,072 tokens, 1 .. 16,384 rows, 1 .. 32 key heads, 1 .. 16 query heads to each, widths 32 .. 256, odd ones among them;
float32, float16 and bfloat16 (queries: float16 and bfloat16).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
PAGE = 64
MOST_FLOPS = 5.4e11
MOST_CODES = 1 << 29


def _write(name, sequences, tokens, context, heads, width, kind, ragged):
    return {"name": name, "op": "write", "sequences": sequences, "tokens": tokens, "context": context, "heads": heads, "width": width, "type": kind, "ragged": ragged}


def _attend(name, sequences, tokens, context, heads, group, width, kind, ragged, window=0, sinks=0):
    return {"name": name, "op": "attend", "sequences": sequences, "tokens": tokens, "context": context, "heads": heads, "group": group, "width": width, "type": kind,
            "ragged": ragged, "window": window, "sinks": sinks}


def listed():
    return [
        # one new token of each of 64 requests: latency, and pages that are nearly full
        _write("write_token", 64, 1, 2000, 8, 128, "bf16", True),
        # prompts of several requests, of lengths that end inside pages
        _write("write_prompt", 7, 4096, 4096, 8, 128, "bf16", True),
        # a finished cache handed on to a program that computes in 16 bits
        {"name": "read_all", "op": "read", "sequences": 4, "context": 8192, "heads": 8, "width": 128, "type": "bf16", "ragged": True},
        # heads of an odd width, in full precision
        {"name": "read_odd", "op": "read", "sequences": 3, "context": 1001, "heads": 12, "width": 73, "type": "f32", "ragged": True},
        # one token of one request: latency only
        _attend("token_one", 1, 1, 1000, 8, 4, 128, "bf16", False),
        # one token of each of 64 requests of any length, some places of the batch empty: the cache is read once, nothing else counts
        _attend("token_batch", 64, 1, 8192, 8, 4, 128, "bf16", True),
        # one token behind two very long documents: little to share out but the length
        _attend("token_long", 2, 1, 131072, 4, 8, 128, "f16", False),
        # long conversations through a window, with sinks
        _attend("token_window", 48, 1, 32768, 8, 8, 128, "bf16", True, 4096, 4),
        # a long prompt
        _attend("prompt", 1, 8192, 8192, 8, 4, 128, "bf16", False),
        # short prompts of several requests, heads of an odd width that share nothing
        _attend("prompt_odd", 9, 700, 700, 12, 1, 80, "f16", True),
        # a piece of a prompt behind what is cached of it already
        _attend("prompt_piece", 2, 512, 30000, 8, 4, 128, "bf16", False),
        # a long prompt through a window, with sinks
        _attend("prompt_window", 1, 16384, 16384, 4, 8, 64, "bf16", False, 1024, 16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "attend", "attend"])
    c = {"op": op, "sequences": _log(rng, 1, 256), "heads": _log(rng, 1, 32), "width": rng.choice([64, 128, 128, 128, 256, rng.randint(32, 256)]), "ragged": rng.random() < 0.7}
    c["context"] = _log(rng, 1, 131072)
    if op == "read":
        c["type"] = rng.choice(["f32", "f16", "bf16"])
        most_codes = 1 << 26
    elif op == "write":
        c |= {"tokens": rng.choice([1, _log(rng, 1, 4096)]), "type": rng.choice(["f32", "f16", "bf16", "bf16"])}
        most_codes = 1 << 27
    else:
        c |= {"tokens": rng.choice([1, 1, rng.randint(2, 16), _log(rng, 16, 8192)]), "group": _log(rng, 1, 16), "type": rng.choice(["f16", "bf16", "bf16"])}
        windowed = rng.random() < 0.35
        c |= {"window": _log(rng, 16, 8192) if windowed else 0, "sinks": rng.choice([0, rng.randint(1, 128)]) if windowed else 0}
        most_codes = MOST_CODES
    c["tokens"] = min(c.get("tokens", 1), c["context"])
    if op == "read":
        del c["tokens"]

    def too_much():
        codes = 2 * c["sequences"] * c["context"] * c["heads"] * c["width"]
        rows = c["sequences"] * c.get("tokens", 1)
        return codes > most_codes or rows > 16384 or rows * c["heads"] * c["width"] * c.get("group", 1) > 1 << 26 or (op == "attend" and _flops(c, *_plan(c)) > MOST_FLOPS)

    while too_much():
        if c["sequences"] > 1:
            c["sequences"] //= 2
        elif c["heads"] > 1:
            c["heads"] //= 2
        else:
            c["context"] = max(1, c["context"] // 2)
            if "tokens" in c:
                c["tokens"] = min(max(1, c["tokens"] // 2), c["context"])
    return c


def _plan(case):
    """(tokens that each sequence holds, rows of the call that each has), as a program's scheduler knows them.  In ragged batches one place of sixteen is empty."""
    n, context = case["sequences"], case["context"]
    tokens = context if case["op"] == "read" else case["tokens"]
    rs = np.random.RandomState(1000 * n + context % 997 + tokens)
    lengths, counts = np.full(n, context), np.full(n, tokens)
    if case["ragged"]:
        if tokens > 1:
            counts = rs.randint(tokens // 3, tokens, n) + 1
        before = context - tokens
        lengths = counts + (rs.randint(before // 8, before, n) + 1 if before else 0)
        lengths = np.minimum(lengths, context)
        counts = np.minimum(counts, lengths)
        lengths[13::16] = 0
        if tokens > 1:
            counts[13::16] = 0
    return lengths.astype(np.int64), (lengths if case["op"] == "read" else counts).astype(np.int64)


def _begun(lengths, counts):
    """Where the first page that a write touches begins."""
    return np.maximum(0, lengths - counts) // PAGE * PAGE


def _starts(counts):
    return np.concatenate([[0], np.cumsum(counts)])


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads, width, op = case["heads"], case["width"], case["op"]
    lengths, counts = _plan(case)
    n = int(counts.sum())
    pages = (lengths + PAGE - 1) // PAGE
    pool = int(pages.sum()) + 5
    s = {"case": case, "lengths_known": lengths, "counts_known": counts}
    # pages wherever there was room, -1 where a sequence has none
    places = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = np.full((len(lengths), max(1, int(pages.max()))), -1, np.int64)
    for i, (a, b) in enumerate(zip(_starts(pages)[:-1], _starts(pages)[1:])):
        table[i, : b - a] = np.arange(a, b)
    at = torch.from_numpy(table).cuda()
    s["table"] = torch.where(at >= 0, places[at.clamp(min=0)], -1).contiguous()
    s["lengths"] = torch.from_numpy(lengths).to("cuda", torch.int32)
    s["offsets"] = torch.from_numpy(_starts(counts)).cuda() if len(set(counts.tolist())) > 1 else None
    # keys have a few large columns, as rotated ones do; whatever the pages hold behind the tokens is of other requests
    columns = 1.0 + 5.0 * (torch.rand(heads, 1, width, generator=g, device="cuda") < 0.03)
    for name in ("key", "value"):
        codes, scales = torch.empty(pool, heads, PAGE, width, dtype=torch.int8, device="cuda"), torch.empty(pool, heads, device="cuda")
        step = max(1, (1 << 26) // (heads * PAGE * width))
        for a in range(0, pool, step):
            x = _normal(g, min(step, pool - a), heads, PAGE, width)
            x *= columns if name == "key" else torch.exp(0.5 * _normal(g, x.shape[0], heads, 1, 1))
            scale = x.abs().amax((2, 3)) / 127.0
            scales[a : a + step], codes[a : a + step] = scale, torch.round(x / scale[:, :, None, None]).clamp(-127, 127).to(torch.int8)
        s[name + "_codes"], s[name + "_scales"] = codes, scales
    if op == "write":
        rows = _normal(g, n, 2, heads, width)  # parts of one projection's rows
        rows[:, 0] *= columns[:, 0]
        rows = rows.to(TYPES[case["type"]])
        s["keys"], s["values"] = rows[:, 0], rows[:, 1]
        begun = _begun(lengths, counts)
        s["back"] = int((lengths - begun).sum())
        s["back_offsets"] = torch.from_numpy(_starts(lengths - begun)).cuda()
        s["back_known"] = lengths - begun
    elif op == "attend":
        s["queries"] = (1.5 * _normal(g, n, heads * case["group"], width)).to(TYPES[case["type"]])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    parts = [s[name + "_" + kind] for name in ("key", "value") for kind in ("codes", "scales")]
    if own:
        import vq_b200 as vq

        s["cache"] = vq.QuantizedCache.from_parts(*parts)
        for name in ("key", "value"):
            del s[name + "_codes"], s[name + "_scales"]
    elif case["op"] == "write":
        # a page more, for what has no place
        for name in ("key", "value"):
            for kind in ("codes", "scales"):
                part = s[name + "_" + kind]
                s[name + "_" + kind] = torch.cat([part, torch.zeros_like(part[:1])])
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------
def _rows_of(s, offsets, counts, n):
    """(sequence, position) of each of n rows: a sequence's rows are its last tokens."""
    at, lengths = torch.arange(n, device="cuda"), s["lengths"].long()
    if offsets is None:
        each = n // len(counts)
        return at // each, at % each + lengths[at // each] - each
    sequence = torch.searchsorted(offsets[1:], at, right=True)
    return sequence, at - offsets[sequence + 1] + lengths[sequence]


def _plain_read(s, offsets, counts, n):
    sequence, position = _rows_of(s, offsets, counts, n)
    there = position >= 0
    position = position.clamp(min=0)
    page = s["table"][sequence, position // PAGE].long()
    found = []
    for name in ("key", "value"):
        x = s[name + "_codes"][page, :, position % PAGE].float() * s[name + "_scales"][page][:, :, None] * there[:, None, None]
        found.append(x.to(TYPES[s["case"]["type"]]))
    return found


def _plain_write(s):
    counts, lengths, table = s["counts_known"], s["lengths"].long(), s["table"]
    each = torch.from_numpy(counts).cuda() if s["offsets"] is None else s["offsets"][1:] - s["offsets"][:-1]
    starts = s["offsets"][:-1] if s["offsets"] is not None else torch.arange(len(counts), device="cuda") * int(counts[0])
    first = lengths - each
    most = (int(counts.max()) + PAGE - 2) // PAGE + 1  # pages that a sequence's rows may fall into
    position = ((first // PAGE)[:, None] + torch.arange(most, device="cuda"))[:, :, None] * PAGE + torch.arange(PAGE, device="cuda")
    row = position - first[:, None, None]
    written = (position >= 0) & (row >= 0) & (row < each[:, None, None])  # sequences x pages x slots
    kept = (row < 0) & (first[:, None, None] >= 0)
    row = torch.where(written, row + starts[:, None, None], 0).flatten()
    touched = written.any(-1)
    column = torch.where(touched, position[:, :, 0] // PAGE, 0)
    spare = s["key_codes"].shape[0] - 1
    page = torch.where(touched, table.gather(1, column).long(), spare).flatten()
    written, kept = written.flatten(0, 1), kept.flatten(0, 1)
    for name in ("key", "value"):
        x = s[name + "s"][row].double().unflatten(0, (-1, PAGE)) * written[:, :, None, None]  # pages x slots x heads x width
        old = torch.where(written[:, 0, None], 0.0, s[name + "_scales"][page])  # (a page begun anew)
        largest = x.abs().amax((1, 3))
        scale = torch.where(largest > 0, (largest / 127.0).float().clamp_min(2.0**-126), 0.0)
        scale = torch.maximum(scale, old)
        held = torch.where(scale > 0, scale, 1.0).double()[:, None, :, None]
        before = s[name + "_codes"][page].permute(0, 2, 1, 3).double() * old.double()[:, None, :, None]
        codes = torch.round(torch.where(written[:, :, None, None], x, before * kept[:, :, None, None]) / held)
        s[name + "_codes"][page], s[name + "_scales"][page] = codes.to(torch.int8).permute(0, 2, 1, 3), scale
    return _plain_read(s, s["back_offsets"], s["back_known"], s["back"])


def _plain_attend(s):
    case, queries = s["case"], s["queries"]
    heads, group, width, window, sinks = case["heads"], case["group"], case["width"], case["window"], case["sinks"]
    y = torch.zeros_like(queries)
    for i, (start, length, count) in enumerate(zip(_starts(s["counts_known"]).tolist(), s["lengths_known"].tolist(), s["counts_known"].tolist())):
        if length == 0 or count == 0:
            continue
        page = s["table"][i, : (length + PAGE - 1) // PAGE].long()
        keys, values = ((s[n + "_codes"][page].float() * s[n + "_scales"][page][:, :, None, None]).transpose(1, 2).flatten(0, 1)[:length].permute(1, 0, 2) for n in ("key", "value"))
        q = queries[start : start + count].float().view(count, heads, group, width).transpose(0, 1)  # heads x rows x group x width
        step = max(1, (1 << 28) // (heads * group * min(length, (window or length) + sinks + 1024)))
        for a in range(0, count, step):
            b = min(a + step, count)
            low, high = length - count + a, length - count + b  # positions of the rows
            begin = max(0, low - window + 1) if window else 0
            seen = torch.cat([torch.arange(min(sinks, begin), device="cuda"), torch.arange(begin, high, device="cuda")])
            position = torch.arange(low, high, device="cuda")[:, None]
            visible = seen <= position
            if window:
                visible &= (seen > position - window) | (seen < sinks)
            some = slice(begin, high) if begin == 0 or not sinks else seen
            scores = (q[:, a:b].reshape(heads, -1, width) @ keys[:, some].mT) * width**-0.5
            scores = scores.view(heads, b - a, group, -1).masked_fill(~visible[:, None, :], -math.inf)
            p = torch.exp(scores - scores.amax(-1, keepdim=True))
            z = (p.flatten(1, 2) @ values[:, some]).view(heads, b - a, group, width) / p.sum(-1, keepdim=True)
            y[start + a : start + b] = z.transpose(0, 1).flatten(1, 2).to(y.dtype)
    return y


# ---- the framework's calls --------------------------------------------------------------------------------------
def _own(s):
    case, cache = s["case"], s["cache"]
    if case["op"] == "attend":
        return cache.attend(s["queries"], s["table"], s["lengths"], offsets=s["offsets"], window=case["window"] or None, sinks=case["sinks"])
    kind = TYPES[case["type"]]
    if case["op"] == "read":
        return cache.read(s["table"], s["lengths"], int(s["counts_known"].sum()), offsets=s["offsets"], dtype=kind)
    cache.write(s["keys"], s["values"], s["table"], s["lengths"], offsets=s["offsets"])
    return cache.read(s["table"], s["lengths"], s["back"], offsets=s["back_offsets"], dtype=kind)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "attend":
        return _plain_attend(state)
    return _plain_write(state) if op == "write" else _plain_read(state, state["offsets"], state["counts_known"], int(state["counts_known"].sum()))


def _pairs(case, lengths, counts):
    """Visible pairs of a query token and a cached one, and the cached tokens that any query sees."""
    window, sinks, pairs, seen = case["window"], case["sinks"], 0, 0
    for length, count in zip(lengths.tolist(), counts.tolist()):
        if length == 0 or count == 0:
            continue
        p = np.arange(length - count, length, dtype=np.int64)
        begin = np.maximum(0, p - window + 1) if window else np.zeros_like(p)
        pairs += int((p + 1 - begin + np.minimum(sinks, begin)).sum())
        seen += length - int(begin[0]) + min(sinks, int(begin[0]))
    return pairs, seen


def _flops(case, lengths, counts):
    return 4 * case["width"] * case["heads"] * case["group"] * _pairs(case, lengths, counts)[0]


def work(case):
    lengths, counts = _plan(case)
    size, values = BYTES[case["type"]], case["heads"] * case["width"]
    if case["op"] == "attend":
        seen = _pairs(case, lengths, counts)[1]
        nbytes = 2 * size * int(counts.sum()) * values * case["group"] + 2 * seen * values + 8 * case["heads"] * (seen // PAGE + 1)
        return {"bytes": nbytes, "flops": _flops(case, lengths, counts)}
    if case["op"] == "read":
        n = int(counts.sum())
        return {"bytes": 2 * n * values * (1 + size), "flops": 2 * n * values}
    n, back = int(counts.sum()), int((lengths - _begun(lengths, counts)).sum())
    # new tokens in, the pages' codes out (those of older tokens in), and what is read back
    return {"bytes": 2 * values * (n * (size + 1) + (back - n) + back * size), "flops": 2 * values * (3 * n + back)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------
def _exact_read(s, codes_of, begins):
    """Tokens begins[i] .. lengths[i] - 1 of every sequence, one behind the other."""
    found = []
    for name in ("key", "value"):
        rows = []
        for i, length in enumerate(s["lengths_known"].tolist()):
            for j in range(begins[i] // PAGE, (length + PAGE - 1) // PAGE):
                codes, scales = codes_of(name, int(s["places"][i, j]))
                x = (codes.double() * scales.double()[:, None, None]).transpose(0, 1)
                rows.append(x[max(0, begins[i] - j * PAGE) : length - j * PAGE])
        found.append(torch.cat(rows))
    return found


def exact(case, seed):
    s = _inputs(case, seed)
    s["places"] = s["table"].cpu().numpy()
    lengths, counts = s["lengths_known"].tolist(), s["counts_known"].tolist()
    if case["op"] == "read":
        return _exact_read(s, lambda name, p: (s[name + "_codes"][p], s[name + "_scales"][p]), [0] * len(lengths))
    if case["op"] == "write":
        done, start = {}, 0
        for i, (length, count) in enumerate(zip(lengths, counts)):
            if length == 0:
                start += count
                continue
            first = length - count
            for j in range(first // PAGE, (length + PAGE - 1) // PAGE):
                p, a, b = int(s["places"][i, j]), max(first - j * PAGE, 0), min(length - j * PAGE, PAGE)
                for name in ("key", "value"):
                    begin = start + j * PAGE + a - first
                    new = s[name + "s"][begin : begin + b - a].double().transpose(0, 1)  # heads x tokens x width
                    step = (new.abs().amax((1, 2)) / 127.0).clamp_min(2.0**-126).float().double()
                    old_codes = s[name + "_codes"][p].double()
                    values = torch.zeros_like(old_codes)
                    if a > 0:
                        before = s[name + "_scales"][p].double()
                        step = torch.maximum(step, before)
                        values[:, :a] = old_codes[:, :a] * before[:, None, None]
                    values[:, a:b] = new
                    done[name, p] = torch.round(values / step[:, None, None]), step
            start += count
        return _exact_read(s, lambda name, p: done[name, p], _begun(s["lengths_known"], s["counts_known"]).tolist())
    heads, group, width, window, sinks = case["heads"], case["group"], case["width"], case["window"], case["sinks"]
    y = torch.zeros(s["queries"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for i, (length, count) in enumerate(zip(lengths, counts)):
        for h in range(heads if length and count else 0):
            pages = s["places"][i, : -(-length // PAGE)].tolist()
            k, v = ((s[n + "_codes"][pages, h].double() * s[n + "_scales"][pages, h].double()[:, None, None]).reshape(-1, width)[:length] for n in ("key", "value"))
            step = max(1, (1 << 26) // (group * length))
            for a in range(0, count, step):
                b = min(a + step, count)
                q = s["queries"][start + a : start + b, h * group : (h + 1) * group].double()
                p = torch.arange(length - count + a, length - count + b, device="cuda")[:, None, None]
                j = torch.arange(length, device="cuda")
                hidden = (j > p) | ((j <= p - window) & (j >= sinks)) if window else j > p
                scores = torch.einsum("rgd,jd->rgj", q, k) / math.sqrt(width)
                y[start + a : start + b, h * group : (h + 1) * group] = torch.softmax(scores.masked_fill(hidden, -math.inf), -1) @ v
        start += count
    return y
