"""Keys and values written as 8-bit codes, read back and attended to, against the same in 64 bits.

Tolerances.  Codes, scales and what is read back are the definition's, bit for bit.  Attention: a score is a sum of `width` products in f32, off by at most
(width + 8) 2^-23 of the products' magnitudes (tensor cores may cut off where others round), and that much of itself is what e^score is off, with 2^-21 for the exponential and 2^-22 of
the scores' distance from the largest for its argument; e^(S - m) s_v is an f16 number of the row's largest, which is between 1/2 and 1: its eleven bits are off by half a step, eps / 2 =
2^-11 of it, or, below 2^-14, by half of 2^-24, which is 2^-24 of the largest; sums over n tokens are off by (n + 64) 2^-23 of their magnitudes.  The result's own rounding is half a step of its type."""
import math
import threading

import numpy as np
import pytest

import vq_b200 as vq

pytestmark = pytest.mark.gpu
PAGE = 64


def torch_():
    import torch
    return torch


def gen(seed):
    return torch_().Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, dtype="float32"):
    torch = torch_()
    return torch.randn(shape, generator=gen(seed), device="cuda").to(getattr(torch, dtype))


class Model:
    """The cache by its definition, in 64 bits on the CPU."""

    def __init__(self, pages, heads, width):
        self.codes = np.zeros((2, pages, heads, PAGE, width))
        self.scales = np.zeros((2, pages, heads))
        self.known = np.zeros((pages, PAGE), bool)  # tokens that somebody wrote

    def write(self, keys, values, table, lengths, offsets):
        for b in range(len(lengths)):
            count = offsets[b + 1] - offsets[b]
            first = int(lengths[b]) - count
            for page_at in range(max(first, 0) // PAGE, (max(int(lengths[b]), 0) + PAGE - 1) // PAGE):
                lo, hi = max(first, page_at * PAGE, 0), min(int(lengths[b]), (page_at + 1) * PAGE)
                if lo >= hi or page_at >= table.shape[1] or not 0 <= table[b, page_at] < self.codes.shape[1]:
                    continue
                p, a, e, row = table[b, page_at], lo % PAGE, hi - page_at * PAGE, offsets[b] + lo - first
                for which, x in enumerate((keys, values)):
                    new = x[row : row + e - a].transpose(1, 0, 2)
                    with np.errstate(all="ignore"):
                        largest = np.abs(new).max((1, 2))
                        s = np.where(largest > 0, np.maximum((largest.astype(np.float32) / np.float32(127)).astype(np.float32), np.float32(2.0**-126)), np.float32(0)).astype(np.float64)
                        s = np.where(np.isfinite(largest), s, np.nan)
                        old = np.zeros_like(s) if a == 0 else self.scales[which, p]
                        s = np.maximum(s, old)  # (NaN wins)
                        div = np.where(s > 0, s, 1.0)[:, None, None]
                        kept = np.rint(self.codes[which, p, :, :a] * old[:, None, None] / div)
                        self.codes[which, p, :, :a] = np.where(np.isnan(s)[:, None, None], self.codes[which, p, :, :a], kept)
                        self.codes[which, p, :, a:e] = np.where((s > 0)[:, None, None], np.rint(new / div), 0.0)
                    self.scales[which, p] = s
                if a == 0:
                    self.known[p] = False
                self.known[p, a:e] = True

    def values(self, which, p, t):
        return self.codes[which, p, :, t] * self.scales[which, p][:, None]


def check_cache(cache, model, tokens=True):
    known = model.known[:, None, :, None]
    for which, (codes, scales) in enumerate(((cache.key_codes, cache.key_scales), (cache.value_codes, cache.value_scales))):
        touched = model.known.any(1)
        assert np.array_equal(scales[touched].astype(np.float64), model.scales[which][touched], equal_nan=True)
        fine = known & ~np.isnan(model.scales[which])[:, :, None, None]
        assert np.array_equal(np.where(fine, codes, 0), np.where(fine, model.codes[which], 0)), (which, int((np.where(fine, codes, 0) != np.where(fine, model.codes[which], 0)).sum()))


def starts(counts):
    return np.concatenate([[0], np.cumsum(counts)]).astype(np.int64)


def device(a):
    torch = torch_()
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def some_cache(seed, lengths, heads, width, columns=None, spare=3, garbage=True):
    """A cache of random codes and a table of scattered pages."""
    torch = torch_()
    pages = [max(0, -(-int(v) // PAGE)) for v in lengths]
    pool = sum(pages) + spare
    rs = np.random.RandomState(seed)
    place = rs.permutation(pool)
    columns = max(pages + [1]) if columns is None else columns
    table, at = np.full((len(lengths), columns), -1, np.int32), 0
    for b, n in enumerate(pages):
        table[b, : min(n, columns)] = place[at : at + n][:columns]
        at += n
    g = gen(seed)
    parts = []
    for _ in range(2):
        codes = (42 * torch.randn(pool, heads, PAGE, width, generator=g, device="cuda")).clamp(-128, 127).round().to(torch.int8)
        scales = torch.exp(0.7 * torch.randn(pool, heads, generator=g, device="cuda")) / 42
        parts += [codes, scales]
    return vq.QuantizedCache.from_parts(*parts), parts, table


def attend64(parts, queries, table, lengths, offsets, scale=None, window=None, sinks=0):
    """(result, limit of its error) in 64 bits; nan limits nothing.  Rows of no sequence: 0."""
    torch = torch_()
    kc, ks, vc, vs = (p.double() for p in parts)
    pool, heads, _, width = kc.shape
    n, qheads = queries.shape[:2]
    group = qheads // heads
    scale = width**-0.5 if scale is None else scale
    y, limit = (torch.zeros(queries.shape, dtype=torch.float64, device="cuda") for _ in range(2))
    for b in range(len(lengths)):
        r0, r1 = int(offsets[b]), int(offsets[b + 1])
        length = max(int(lengths[b]), 0)
        keys = min(length, table.shape[1] * PAGE)
        if r1 <= r0 or keys == 0:
            continue
        j = torch.arange(keys, device="cuda")
        page = torch.from_numpy(table[b].astype(np.int64)).cuda()[j // PAGE]
        there = (page >= 0) & (page < pool)
        page = torch.where(there, page, 0)
        k = kc[page, :, j % PAGE] * ks[page][:, :, None]  # tokens x heads x width
        v, sv = vc[page, :, j % PAGE] * vs[page][:, :, None], vs[page]
        k, v, sv = (torch.where(there.view(-1, *[1] * (t.dim() - 1)), t, torch.zeros_like(t)) for t in (k, v, sv))
        position = torch.arange(length - (r1 - r0), length, device="cuda")[:, None]
        seen = there & (j <= position)
        if window:
            seen &= (j > position - window) | (j < sinks)
        for h in range(heads):
            x = queries[r0:r1, h * group : (h + 1) * group].double()
            S = torch.einsum("rgd,jd->rgj", x, k[:, h]) * scale
            A = torch.einsum("rgd,jd->rgj", x.abs(), k[:, h].abs()) * abs(scale)
            mask = seen[:, None, :]
            S, A = torch.where(mask, S, -math.inf), torch.where(mask, A, 0.0)
            m = S.amax(-1, keepdim=True)
            p = torch.where(mask, torch.exp(S - torch.where(m == -math.inf, 0.0, m)), 0.0)
            l = p.sum(-1, keepdim=True)
            empty = l == 0
            p = torch.where(empty, 0.0, p / torch.where(empty, 1.0, l))
            vh = torch.where(seen.any(0)[:, None], v[:, h], 0.0)
            z = p @ vh
            far = torch.where(mask, (S - m).abs(), 0.0)
            eps = p * (2.0**-11 + 2.0**-21 + (width + 8) * 2.0**-23 * A + 2.0**-22 * far + (keys + 64) * 2.0**-23)
            small = (p * sv[:, h].abs()).amax(-1, keepdim=True) * 2.0**-24 * 128 * keys  # weights off by 2^-24 of the largest, times codes
            y[r0:r1, h * group : (h + 1) * group] = z
            limit[r0:r1, h * group : (h + 1) * group] = eps @ vh.abs() + z.abs() * eps.sum(-1, keepdim=True) + small
    return y, limit


def check(y, want, limit):
    torch = torch_()
    info = torch.finfo(y.dtype)
    off = (y.double() - want).abs()
    tiny = {torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}[y.dtype]
    bad = ~(off <= limit + (want.abs() + limit) * info.eps / 2 + tiny) & ~(torch.isnan(y) & torch.isnan(want))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {y[bad][0]} for {want[bad][0]} (limit {limit[bad][0]:.3e}, off {off[bad][0]:.3e})"


# ---- writing ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,width", [(1, 1), (2, 128), (3, 73), (1, 256), (2, 32), (5, 7)])
def test_prompts_then_tokens_are_the_definitions(heads, width, dtype):
    """Prompts, pieces and single tokens, of sequences that begin anywhere in a page, in pages that held something else."""
    torch = torch_()
    lengths, pool = np.array([0, 3, 64, 130, 65, 200]), 24
    cache, model = vq.QuantizedCache.empty(pool, heads, width), Model(pool, heads, width)
    table = np.random.RandomState(3).permutation(pool).reshape(6, 4).astype(np.int32)
    for step, counts in enumerate(([0, 3, 64, 130, 65, 200], [1] * 6, [1, 2, 63, 0, 1, 5], [1] * 6, [70, 0, 0, 1, 61, 0])):
        counts = np.array(counts)
        lengths = counts.copy() if step == 0 else lengths + counts
        x = normal(10 * step + width, int(counts.sum()), 2, heads, width) * 1.7**step
        if step == 3:
            x *= 0.01  # (nothing grows)
        x = x.to(getattr(torch, dtype))
        offsets = starts(counts)
        given = None if len(set(counts)) == 1 else device(offsets)
        cache.write(x[:, 0], x[:, 1], device(table), device(lengths.astype(np.int32)), offsets=given)
        wide = x.double().cpu().numpy()
        model.write(wide[:, 0], wide[:, 1], table, lengths, offsets)
        check_cache(cache, model)
    # a request's pages given to another one
    counts = np.array([0, 0, 0, 0, 10, 0])
    lengths = np.array([0, 0, 0, 0, 10, 0])
    x = normal(99, 10, 2, heads, width, dtype=dtype) * 0.125
    cache.write(x[:, 0], x[:, 1], device(table), device(lengths.astype(np.int32)), offsets=device(starts(counts)))
    wide = x.double().cpu().numpy()
    model.write(wide[:, 0], wide[:, 1], table, lengths, starts(counts))
    check_cache(cache, model)


def test_quotients_next_to_halves_are_the_real_ones():
    """Values that are halves of the scale, and scales that grow by a little: where a reciprocal would go the wrong way."""
    torch = torch_()
    cache, model = vq.QuantizedCache.empty(2, 1, 256), Model(2, 1, 256)
    s = np.float32(0.1) / np.float32(127)
    x = ((np.arange(64 * 256).reshape(64, 1, 256) % 255 - 127) * 0.5 * np.float64(s)).astype(np.float32)
    x[0, 0, 0] = 0.1
    table = np.array([[1]], np.int32)
    first = torch.from_numpy(x[:40]).cuda()
    cache.write(first, first, device(table), device(np.array([40], np.int32)))
    model.write(x[:40].astype(np.float64), x[:40].astype(np.float64), table, [40], [0, 40])
    check_cache(cache, model)
    for i in range(40, 50):
        x[i, 0, 3] = np.float32(0.1) * np.float32(1 + (i - 39) * 0.013)
        one = torch.from_numpy(x[i : i + 1]).cuda()
        cache.write(one, one, device(table), device(np.array([i + 1], np.int32)))
        model.write(x[i : i + 1].astype(np.float64), x[i : i + 1].astype(np.float64), table, [i + 1], [0, 1])
        check_cache(cache, model)


def test_zeros_small_numbers_infinities_and_nan():
    torch = torch_()
    cache, model = vq.QuantizedCache.empty(4, 2, 16), Model(4, 2, 16)
    table = np.array([[2], [0], [3], [1]], np.int32)
    x = normal(1, 4 * 3, 2, 16)
    x[0:3] = 0
    x[3:6] *= 2.0**-126
    x[7, 1, 3] = math.inf
    x[10, 0, 5] = math.nan
    lengths = np.full(4, 3, np.int32)

    def both(x, lengths, count):
        cache.write(x, x, device(table), device(lengths))
        wide = x.double().cpu().numpy()
        model.write(wide, wide, table, lengths, starts([count] * 4))
        check_cache(cache, model)

    both(x, lengths, 3)
    assert np.isnan(cache.key_scales[3, 1]) and not np.isnan(cache.key_scales[3, 0]) and np.isnan(cache.key_scales[1, 0]) and cache.key_scales[2].tolist() == [0, 0]
    both(normal(2, 4, 2, 16), lengths + 1, 1)  # NaN stays
    assert np.isnan(cache.key_scales[3, 1])
    both(normal(3, 8, 2, 16), np.full(4, 2, np.int32), 2)  # until the page begins anew
    assert np.isfinite(cache.key_scales).all()


def test_tokens_that_are_not_there_are_not_written():
    torch = torch_()
    heads, width, pool = 2, 40, 6
    cache, parts, _ = some_cache(5, [0], heads, width, spare=pool)
    before = [cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales]
    x = normal(4, 6 * 3, heads, width)
    # an empty place, more rows than tokens, no page, pages that the cache does not have, a token behind the table
    table = np.array([[0, 1], [2, 1], [-1, 1], [pool, 1], [-(2**31), 2**31 - 1], [3, -1]], np.int32)
    lengths = np.array([0, 2, 30, 30, 70, 130], np.int32)
    cache.write(x, x, device(table), device(lengths))
    after = [cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales]
    model = Model(pool, heads, width)
    model.write(x.double().cpu().numpy(), x.double().cpu().numpy(), table, lengths, starts([3] * 6))
    assert model.known.sum() == 2 and model.known[2, :2].all()
    check_cache(cache, model)
    for a, b in zip(before, after):
        assert np.array_equal(np.delete(a, 2, 0), np.delete(b, 2, 0))


def test_rows_and_heads_of_any_distance():
    torch = torch_()
    heads, width, n = 3, 72, 70
    x = normal(8, n, 2 * heads + 1, width + 8)
    layouts = [x[:, 1 : 1 + heads, :width], x[:, heads + 1 :, 5 : 5 + width].contiguous(), normal(9, heads, n, width).transpose(0, 1), normal(9, n, heads, width + 1)[:, :, 1:],
               normal(10, n, heads, 2 * width)[:, :, ::2], normal(11, n, 1, width).expand(n, heads, width)]
    table, lengths = np.array([[0, 1]], np.int32), np.array([n], np.int32)
    for i, k in enumerate(layouts):
        for v in (layouts[(i + 1) % len(layouts)], k):
            cache, model = vq.QuantizedCache.empty(2, heads, width), Model(2, heads, width)
            cache.write(k, v, device(table), device(lengths))
            model.write(k.double().cpu().numpy(), v.double().cpu().numpy(), table, lengths, [0, n])
            check_cache(cache, model)


# ---- reading ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("heads,width", [(1, 1), (2, 128), (3, 73), (1, 256)])
def test_read_gives_codes_times_scales(heads, width, dtype):
    torch = torch_()
    lengths, counts = np.array([130, 0, 64, 5, 200, 1]), np.array([130, 0, 10, 7, 65, 1])
    cache, parts, table = some_cache(2, lengths, heads, width)
    parts[1][table[0, 0]], parts[3][table[0, 1]] = math.nan, 0.0
    cache = vq.QuantizedCache.from_parts(*parts)
    table[4, 1] = -1
    offsets = 2 + starts(counts)  # rows 0, 1 and the last three belong to nobody
    n = int(offsets[-1]) + 3
    got = cache.read(device(table), device(lengths.astype(np.int32)), n, offsets=device(offsets), dtype=getattr(torch, dtype))
    codes, scales = [parts[0].cpu(), parts[2].cpu()], [parts[1].cpu(), parts[3].cpu()]
    for which in range(2):
        want = torch.zeros(n, heads, width, dtype=torch.float32)
        for b in range(len(lengths)):
            for i in range(counts[b]):
                j = lengths[b] - counts[b] + i
                p = table[b, j // PAGE] if j >= 0 else -1
                if p >= 0:
                    want[offsets[b] + i] = codes[which][p, :, j % PAGE].float() * scales[which][p][:, None]
        want = want.to(getattr(torch, dtype))
        assert torch.equal(torch.nan_to_num(got[which].cpu(), 123.0), torch.nan_to_num(want, 123.0))


def test_parts_come_back_as_they_were_given():
    torch = torch_()
    cache, parts, _ = some_cache(7, [200], 3, 33)
    parts[1][0, 0], parts[1][0, 1], parts[3][1, 2] = -1.0, math.inf, 0.0
    again = vq.QuantizedCache.from_parts(*parts)
    assert np.array_equal(again.key_codes, parts[0].cpu().numpy()) and np.array_equal(again.value_codes, parts[2].cpu().numpy())
    scales = parts[1].cpu().numpy().copy()
    scales[0, :2] = np.nan
    assert np.array_equal(again.key_scales, scales, equal_nan=True) and np.array_equal(again.value_scales, parts[3].cpu().numpy())
    other = vq.QuantizedCache.from_parts(again.key_codes, again.key_scales, again.value_codes, again.value_scales)
    assert np.array_equal(other.value_codes, again.value_codes) and again.shape() == (parts[0].shape[0], 3, 33)


# ---- attention -------------------------------------------------------------------------------------------------
def attend_case(seed, lengths, counts, heads, group, width, dtype="bfloat16", rest=(0, 0), sharp=1.0, **how):
    torch = torch_()
    lengths, counts = np.array(lengths), np.array(counts)
    cache, parts, table = some_cache(seed, lengths, heads, width)
    offsets = rest[0] + starts(counts)
    n = int(offsets[-1]) + rest[1]
    x = (sharp * normal(seed + 1, n, heads * group, width)).to(getattr(torch, dtype))
    given = None if len(set(counts)) == 1 and rest == (0, 0) else device(offsets)
    y = cache.attend(x, device(table), device(lengths.astype(np.int32)), offsets=given, **how)
    assert y.dtype == x.dtype and y.shape == x.shape
    check(y, *attend64(parts, x, table, lengths, offsets, **how))
    return cache, parts, table, x, y


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads,group,width", [(1, 1, 1), (2, 4, 128), (1, 8, 64), (3, 1, 73), (2, 5, 256), (1, 16, 32), (1, 17, 80), (1, 40, 96), (2, 3, 160), (1, 2, 192), (1, 7, 224)])
def test_one_token_of_each_sequence(heads, group, width, dtype):
    attend_case(1, [1, 64, 65, 0, 1000, 63, 127, 2, 128, 333], [1] * 10, heads, group, width, dtype)


@pytest.mark.parametrize("length", [1, 2, 63, 64, 65, 128, 255, 256, 257, 511, 513, 1024, 4097, 20_000])
def test_one_token_of_one_sequence(length):
    attend_case(length, [length], [1], 2, 4, 128)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("heads,group,width", [(2, 4, 128), (1, 1, 64), (1, 3, 80), (1, 8, 256), (2, 2, 40), (1, 5, 96)])
def test_rows_of_any_number(heads, group, width, dtype):
    attend_case(4, [300, 64, 130, 1, 70, 0, 500, 33, 200], [300, 1, 17, 1, 64, 0, 129, 33, 5], heads, group, width, dtype, rest=(3, 2))


@pytest.mark.parametrize("tokens", [1, 2, 3, 15, 16, 17, 31, 32, 33, 64, 100, 127, 128, 129, 256, 300, 513])
def test_prompts(tokens):
    attend_case(tokens, [tokens], [tokens], 1, 2, 128)
    attend_case(tokens, [tokens + 1000, tokens + 77], [tokens] * 2, 2, 1, 64)


def test_a_long_prompt():
    attend_case(6, [2500], [2500], 2, 4, 128)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 64), (65, 3), (100, 130), (128, 0), (5000, 7), (2**31 - 1, 2**31 - 1), (2**40, 0), (300, 1000)])
@pytest.mark.parametrize("width", [64, 128])
def test_windows_with_sinks(window, sinks, width):
    attend_case(9, [700, 3, 64, 1025, 200], [1] * 5, 1, 4, width, window=window, sinks=sinks)
    attend_case(9, [700, 3, 64, 1025, 200], [300, 3, 40, 1, 129], 2, 1, width, window=window, sinks=sinks)


def test_scales_of_scores():
    for scale in (0.0, 1.0, -0.3, 1e-20):
        attend_case(11, [300, 90], [1, 1], 2, 2, 64, scale=scale)
        attend_case(11, [300, 90], [200, 20], 2, 2, 64, scale=scale)


def test_sharp_scores():
    """All weight on one token or another, far apart from tile to tile."""
    for sharp in (30.0, 300.0):
        attend_case(12, [1000, 400], [1, 1], 2, 4, 128, sharp=sharp)
        attend_case(12, [1000, 400], [600, 400], 1, 4, 128, sharp=sharp)


@pytest.mark.parametrize("counts", [[1, 1, 1], [200, 40, 100]])
def test_scales_far_apart(counts):
    """Pages whose scales differ by 2^40 and more, zeros among them."""
    torch = torch_()
    lengths = np.array([500, 190, 100])
    _, parts, table = some_cache(13, lengths, 2, 128)
    g = gen(14)
    parts[1] *= torch.exp(3 * torch.randn(parts[1].shape, generator=g, device="cuda"))
    parts[3] *= torch.exp2(torch.randint(-45, 45, parts[3].shape, generator=g, device="cuda").float())
    parts[3][table[0, 1]], parts[1][table[0, 2]] = 0.0, 0.0
    parts[3][table[2, 0]] = 2.0**-126
    cache = vq.QuantizedCache.from_parts(*parts)
    offsets = starts(counts)
    for dtype in ("bfloat16", "float16"):
        x = normal(15, int(offsets[-1]), 8, 128, dtype=dtype)
        y = cache.attend(x, device(table), device(lengths.astype(np.int32)), offsets=device(offsets))
        want, limit = attend64(parts, x, table, lengths, offsets)
        top = torch.finfo(y.dtype).max * 0.99
        fine = want.abs() + limit < top
        check(torch.where(fine, y, 0), torch.where(fine, want, 0.0), torch.where(fine, limit, 0.0))


def test_queries_of_any_size():
    """Queries whose scores would leave f16 or be 0 in it."""
    torch = torch_()
    lengths = np.array([200, 70])
    for size, dtype in ((2.0**-30, "bfloat16"), (2.0**60, "bfloat16"), (2.0**-20, "float16"), (60000.0, "float16"), (2.0**-120, "bfloat16")):
        for counts in ([1, 1], [150, 70]):
            cache, parts, table = some_cache(16, lengths, 1, 64)
            offsets = starts(counts)
            x = (normal(17, int(offsets[-1]), 4, 64).clamp(-1, 1) * size).to(getattr(torch, dtype))
            scale = 0.3 / size
            y = cache.attend(x, device(table), device(lengths.astype(np.int32)), offsets=device(offsets), scale=scale)
            check(y, *attend64(parts, x, table, lengths, offsets, scale=scale))


@pytest.mark.parametrize("counts", [[1] * 5, [65, 20, 130, 1, 30]])
def test_tokens_that_are_not_there_are_not_seen(counts):
    torch = torch_()
    lengths = np.array([70, 400, 130, 0, 10])
    cache, parts, table = some_cache(18, [70, 400, 130, 64, 64], 2, 64)
    table[1, 0], table[1, 3], table[2, 1], table[2, 2] = -1, 10**6, -(2**31), 2**31 - 1
    lengths[4] = -5
    offsets = starts(counts)
    x = normal(19, int(offsets[-1]), 4, 64, dtype="bfloat16")
    for how in ({}, {"window": 64, "sinks": 3}):
        y = cache.attend(x, device(table), device(lengths.astype(np.int32)), offsets=device(offsets), **how)
        check(y, *attend64(parts, x, table, lengths, offsets, **how))
        assert (y[offsets[3] :] == 0).all()
    # a table that has fewer columns than the tokens
    for columns in (0, 1, 2):
        y = cache.attend(x, device(table)[:, :columns], device(lengths.astype(np.int32)), offsets=device(offsets))
        check(y, *attend64(parts, x, table[:, :columns], lengths, offsets))


@pytest.mark.parametrize("counts", [[1, 1], [100, 100]])
@pytest.mark.parametrize("which", [1, 3])
def test_nan_stays_where_it_is_seen(counts, which):
    """Rows that see a page of NaN are NaN; rows in front of it, behind their window, and other heads are not."""
    torch = torch_()
    lengths = np.array([200, 250])
    _, parts, table = some_cache(20, lengths, 2, 64)
    parts[which][table[0, 2], 1] = math.nan  # tokens 128 .. 191 of sequence 0
    parts[which][table[1, 3], 0] = math.nan  # 192 .. 249 of sequence 1
    spare = parts[0].shape[0] - 1
    cache = vq.QuantizedCache.from_parts(*parts)
    offsets = starts(counts)
    x = normal(21, int(offsets[-1]), 4, 64, dtype="bfloat16")
    for window, sinks in ((None, 0), (5, 0), (5, 130)):
        y = cache.attend(x, device(table), device(lengths.astype(np.int32)), offsets=device(offsets), window=window, sinks=sinks)
        for b in range(2):
            position = np.arange(lengths[b] - counts[b], lengths[b])
            lo, hi, head = ((128, 192, 1), (192, 250, 0))[b]
            seen = np.array([any(lo <= j < hi and (window is None or j > p - window or j < sinks) for j in range(p + 1)) for p in position])
            nan = torch.isnan(y[offsets[b] : offsets[b + 1]]).cpu().numpy()
            assert (nan[:, 2 * head : 2 * head + 2] == seen[:, None, None]).all()
            assert not nan[:, 2 - 2 * head : 4 - 2 * head].any()


@pytest.mark.parametrize("tokens", [1, 90])
def test_infinite_and_nan_queries_make_their_rows_nan_and_no_others(tokens):
    torch = torch_()
    lengths = np.array([150, 90])
    cache, parts, table = some_cache(22, lengths, 1, 64)
    x = normal(23, 2 * tokens, 4, 64, dtype="float16")
    x[0, 1, 3], x[tokens, 2, 63] = math.inf, math.nan
    y = cache.attend(x, device(table), device(lengths.astype(np.int32)))
    nan = torch.isnan(y).any(-1).cpu()
    assert nan[0].tolist() == [False, True, False, False] and nan[tokens].tolist() == [False, False, True, False] and int(nan.sum()) == 2
    assert torch.isnan(y[0, 1]).all()


@pytest.mark.parametrize("tokens", [1, 5, 140])
def test_rows_heads_and_results_of_any_distance(tokens):
    torch = torch_()
    lengths = np.array([150, 300])
    heads, width, n = 4, 72, 2 * tokens
    cache, parts, table = some_cache(24, lengths, 2, width)
    wide = device(np.concatenate([table, table], 1))[:, : table.shape[1]]
    for x in (normal(25, n, heads + 2, width + 8, dtype="float16")[:, 1:5, 8:], normal(26, heads, n, width, dtype="float16").transpose(0, 1),
              normal(27, n, heads, width + 3, dtype="float16")[:, :, 3:], normal(28, n, heads, 2 * width, dtype="float16")[:, :, ::2]):
        want, limit = attend64(parts, x, table, lengths, starts([tokens] * 2))
        room = torch.full((n, heads + 1, width + 5), 7.0, dtype=torch.float16, device="cuda")
        turned = torch.full((heads, n + 1, width), 7.0, dtype=torch.float16, device="cuda")
        for out in (None, room[:, 1:, 3 : 3 + width], turned[:, :n].transpose(0, 1)):
            y = cache.attend(x, wide, device(lengths.astype(np.int32)), out=out)
            assert out is None or y is out
            check(y, want, limit)
        assert (room[:, 0] == 7).all() and (room[:, 1:, :3] == 7).all() and (room[:, 1:, 3 + width :] == 7).all() and (turned[:, n] == 7).all()


@pytest.mark.parametrize("counts", [[1, 1, 1], [50, 1, 70]])
def test_rows_of_no_sequence(counts):
    torch = torch_()
    lengths = np.array([64, 0, 100])
    cache, parts, table = some_cache(29, lengths, 1, 64)
    offsets = 4 + starts(counts)
    n = int(offsets[-1]) + 3
    x = normal(30, n, 2, 64, dtype="bfloat16")
    y = cache.attend(x, device(table), device(lengths.astype(np.int32)), offsets=device(offsets))
    assert (y[:4] == 0).all() and (y[n - 3 :] == 0).all()
    out = torch.full_like(y, 5.0)
    cache.attend(x, device(table), device(lengths.astype(np.int32)), offsets=device(offsets), out=out)
    assert (out[:4] == 5).all() and (out[n - 3 :] == 5).all() and torch.equal(out[4 : n - 3], y[4 : n - 3])


def test_the_same_call_gives_the_same_bits():
    torch = torch_()
    for lengths, counts in (([9000, 50, 3000], [1, 1, 1]), ([900, 50, 300], [600, 50, 2])):
        cache, parts, table, x, y = attend_case(31, lengths, counts, 2, 4, 128)
        for _ in range(3):
            assert torch.equal(y, cache.attend(x, device(table), device(np.array(lengths, np.int32)), offsets=device(starts(counts))))


def test_offsets_of_any_kind_stay_in_bounds():
    """Offsets that do not ascend: no result is promised, but nothing outside the rows is written and the next call is right."""
    torch = torch_()
    cache, parts, table = some_cache(32, [500, 300, 200, 100], 1, 64)
    lengths = device(np.array([500, 300, 200, 100], np.int32))
    room = torch.full((300, 4, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    x = normal(33, 200, 4, 64, dtype="bfloat16")
    for offsets in ([0, 150, 100, 200, 200], [200, 100, 50, 20, 0], [-5, 10, 2**40, 200, 7], [300, 400, 500, 600, 700]):
        cache.attend(x, device(table), lengths, offsets=device(np.array(offsets, np.int64)), out=room[50:250])
        cache.read(device(table), lengths, 200, offsets=device(np.array(offsets, np.int64)))
    assert (room[:50] == 3).all() and (room[250:] == 3).all()
    right = np.array([0, 50, 100, 150, 200])
    check(cache.attend(x, device(table), lengths, offsets=device(right)), *attend64(parts, x, table, [500, 300, 200, 100], right))


def test_many_sequences():
    rs = np.random.RandomState(5)
    lengths = rs.randint(0, 300, 700)
    attend_case(34, lengths, [1] * 700, 1, 4, 64)
    counts = np.minimum(lengths, rs.choice([0, 1, 1, 3, 40], 700))
    attend_case(35, lengths, counts, 1, 2, 64)


@pytest.mark.parametrize("heads,group,tokens", [(2, 1, 100), (4, 2, 128), (3, 1, 64), (8, 2, 33)])
def test_many_short_prompts(heads, group, tokens):
    """More tiles than SMs, none of which has more than two pages."""
    torch = torch_()
    lengths = np.random.RandomState(tokens).randint(tokens, 129, 150)
    attend_case(36, lengths, [tokens] * 150, heads, group, 64)
    counts = np.random.RandomState(7).randint(0, tokens + 1, 150)
    attend_case(37, lengths, counts, heads, group, 128, rest=(1, 1))


def test_without_tensor_cores():
    """VQB_NO_TENSOR=1, in a process of its own: the same results, by other sums."""
    import os
    import subprocess
    import sys
    code = """
import numpy as np, torch
from tests import test_gpu_cache as t
t.attend_case(41, [300, 0, 64], [1, 1, 1], 2, 4, 72)
t.attend_case(42, [300, 5, 200], [120, 5, 33], 1, 3, 128, "float16", rest=(2, 1), window=50, sinks=3)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, env={**os.environ, "VQB_NO_TENSOR": "1"}, timeout=120)


# ---- together --------------------------------------------------------------------------------------------------
def run_together(step_of, tokens=70, seed=40):
    """A prompt, then single tokens, each of which writes and attends: (results, what they should be, limits)."""
    torch = torch_()
    heads, group, width, sequences = 2, 3, 80, 4
    prompt = np.array([100, 0, 63, 7])
    pool = 16
    cache, model = vq.QuantizedCache.empty(pool, heads, width), Model(pool, heads, width)
    table = np.random.RandomState(seed).permutation(pool).reshape(4, 4).astype(np.int32)
    lengths = prompt.copy()
    on_gpu = device(table)
    found = []
    for step in range(tokens):
        counts = prompt if step == 0 else np.ones(4, int)
        lengths = lengths + (0 if step == 0 else 1)
        offsets = starts(counts)
        rows = normal(seed + step, int(counts.sum()), heads * group + 2 * heads, width, dtype="bfloat16")
        q, k, v = rows[:, : heads * group], rows[:, heads * group : heads * (group + 1)], rows[:, heads * (group + 1) :]
        y = step_of(cache, q, k, v, on_gpu, device(lengths.astype(np.int32)), device(offsets) if step == 0 else None)
        wide = k.double().cpu().numpy(), v.double().cpu().numpy()
        model.write(*wide, table, lengths, offsets)
        if step % 23 == 0 or step == tokens - 1:
            parts = [torch.from_numpy(a.copy()).cuda() for a in (model.codes[0], model.scales[0], model.codes[1], model.scales[1])]
            found.append((y.clone(), *attend64(parts, q, table, lengths, offsets)))
    check_cache(cache, model)
    return found


def test_a_run_of_steps():
    def step(cache, q, k, v, table, lengths, offsets):
        cache.write(k, v, table, lengths, offsets=offsets)
        return cache.attend(q, table, lengths, offsets=offsets)

    for y, want, limit in run_together(step):
        check(y, want, limit)


def test_a_captured_step_is_replayed_with_new_tokens():
    """One graph of a step, its inputs and lengths changed in place."""
    torch = torch_()
    held = {}

    def step(cache, q, k, v, table, lengths, offsets):
        if offsets is not None:
            cache.write(k, v, table, lengths, offsets=offsets)
            return cache.attend(q, table, lengths, offsets=offsets)
        if "graph" not in held:
            held["in"] = [q.contiguous(), k.contiguous(), v.contiguous(), lengths.clone()]
            held["out"] = torch.empty_like(held["in"][0])
            side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
                cache.write(held["in"][1], held["in"][2], table, held["in"][3])
                cache.attend(held["in"][0], table, held["in"][3], out=held["out"])
            held["graph"], held["table"] = g, table
        for to, new in zip(held["in"], (q, k, v, lengths)):
            to.copy_(new)
        held["graph"].replay()
        return held["out"]

    for y, want, limit in run_together(step):
        check(y, want, limit)
    torch.cuda.synchronize()
    held.clear()


def test_two_captured_graphs_take_turns():
    torch = torch_()
    graphs = []
    for seed, lengths, counts in ((50, [9000, 40], [1, 1]), (51, [3000, 700], [1, 1]), (52, [300, 200], [128, 128])):
        cache, parts, table = some_cache(seed, lengths, 2, 128)
        x, out = normal(seed, sum(counts), 8, 128, dtype="bfloat16"), torch.empty(sum(counts), 8, 128, dtype=torch.bfloat16, device="cuda")
        t, n = device(table), device(np.array(lengths, np.int32))
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            cache.attend(x, t, n, out=out)
        graphs.append((g, cache, x, t, n, out, attend64(parts, x, table, lengths, starts(counts))))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for stream, (g, *_, out, _) in zip(streams, graphs):
            out.zero_()
        torch.cuda.synchronize()
        for stream, (g, *_) in zip(streams, graphs):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for g, *_, out, want in graphs:
            check(out, *want)
    graphs.clear()


def test_calls_on_other_streams_follow_each_other():
    torch = torch_()
    cache, parts, table = some_cache(53, [8000, 5000], 2, 128)
    t, n = device(table), device(np.array([8000, 5000], np.int32))
    x = normal(54, 2, 8, 128, dtype="float16")
    k = normal(55, 2, 2, 128, dtype="float16")
    model = Model(parts[0].shape[0], 2, 128)
    for which in range(2):
        model.codes[which], model.scales[which] = parts[2 * which].cpu().numpy(), parts[2 * which + 1].cpu().numpy()
    model.write(k.double().cpu().numpy(), k.double().cpu().numpy(), table, [8000, 5000], [0, 1, 2])
    now = [torch.from_numpy(a.copy()).cuda() for a in (model.codes[0], model.scales[0], model.codes[1], model.scales[1])]
    want = attend64(now, x, table, [8000, 5000], [0, 1, 2])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    with torch.cuda.stream(streams[0]):
        cache.write(k, k, t, n)
    results = []
    for s in streams[1:]:
        with torch.cuda.stream(s):
            results.append(cache.attend(x, t, n))
    torch.cuda.synchronize()
    for y in results:
        check(y, *want)


def test_threads():
    torch = torch_()
    work = []
    for seed in range(4):
        lengths = [3000 + 100 * seed, 10]
        cache, parts, table = some_cache(seed, lengths, 1, 64)
        x = normal(seed, 2, 4, 64, dtype="bfloat16")
        work.append((cache, x, device(table), device(np.array(lengths, np.int32)), attend64(parts, x, table, lengths, [0, 1, 2]), []))
    torch.cuda.synchronize()

    def go(cache, x, t, n, want, found):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                found.append(cache.attend(x, t, n))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=go, args=w) for w in work]
    [t.start() for t in threads]
    [t.join() for t in threads]
    for *_, want, found in work:
        assert len(found) == 20
        for y in found:
            check(y, *want)


def test_host_memory():
    torch = torch_()
    lengths, counts = np.array([100, 3, 70], np.int32), np.array([100, 3, 70])
    table = np.array([[0, 1], [2, -1], [3, 4]], np.int32)
    x = normal(60, 173, 2, 48).cpu().numpy()
    cache, model = vq.QuantizedCache.empty(5, 2, 48), Model(5, 2, 48)
    cache.write(x, x[::-1], table, lengths, offsets=starts(counts))
    model.write(x.astype(np.float64), x[::-1].astype(np.float64), table, lengths, starts(counts))
    check_cache(cache, model)
    k, v = cache.read(table, lengths, 173, offsets=starts(counts))
    assert isinstance(k, np.ndarray) and k.dtype == np.float32
    gk, gv = cache.read(device(table), device(lengths), 173, offsets=device(starts(counts)))
    assert np.array_equal(k, gk.cpu().numpy()) and np.array_equal(v, gv.cpu().numpy())
    q = normal(61, 173, 4, 48, dtype="float16")
    y = cache.attend(q.cpu().numpy(), table, lengths.tolist(), offsets=starts(counts).tolist())
    assert isinstance(y, np.ndarray) and y.dtype == np.float16
    assert np.array_equal(y, cache.attend(q, device(table), device(lengths), offsets=device(starts(counts))).cpu().numpy())
    room = np.full((173, 5, 48), 9, np.float16)
    cache.attend(q.cpu().numpy(), table, lengths, offsets=starts(counts), out=room[:, :4])
    assert np.array_equal(room[:, :4], y) and (room[:, 4] == 9).all()
    mixed = cache.attend(q, table, lengths, offsets=starts(counts))  # rows on the GPU, the rest not
    assert np.array_equal(mixed.cpu().numpy(), y)


def test_refusals():
    torch = torch_()
    cache, parts, table = some_cache(70, [100], 2, 64)
    t, n = device(table), device(np.array([100], np.int32))
    q = normal(71, 1, 4, 64, dtype="bfloat16")
    k = normal(72, 1, 2, 64, dtype="bfloat16")
    with pytest.raises(vq.DimensionMismatch, match="expected 64, got 32"):
        cache.attend(q[:, :, :32], t, n)
    with pytest.raises(vq.InvalidParameter, match="multiple of the cache's heads"):
        cache.attend(q[:, :3], t, n)
    with pytest.raises(vq.BackendError, match="f16 or bf16"):
        cache.attend(q.float(), t, n)
    with pytest.raises(vq.InvalidParameter, match="finite"):
        cache.attend(q, t, n, scale=math.nan)
    with pytest.raises(vq.InvalidParameter, match="offsets are needed"):
        cache.attend(normal(1, 3, 4, 64, dtype="bfloat16"), t.expand(2, -1).contiguous(), n.expand(2).contiguous())
    with pytest.raises(vq.InvalidParameter, match="ascend"):
        cache.attend(q, t, n, offsets=[0, 5])
    with pytest.raises(vq.DimensionMismatch, match="expected 2, got 4"):
        cache.write(q, q, t, n)
    with pytest.raises(ValueError, match="int32"):
        cache.attend(q, t.long(), n)
    with pytest.raises(ValueError, match="same shape and type"):
        cache.write(k, k.float(), t, n)
    with pytest.raises(ValueError, match="requires a gradient"):
        cache.attend(q.float().requires_grad_().half(), t, n)
    with pytest.raises(ValueError, match="out must be"):
        cache.attend(q, t, n, out=torch.empty(1, 4, 64, device="cuda"))
    with pytest.raises(vq.BackendError, match="256 values"):
        vq.QuantizedCache.empty(1, 1, 257)
    with pytest.raises(vq.EmptyInput):
        vq.QuantizedCache.empty(0, 1, 64)
    with pytest.raises(vq.EmptyInput):
        cache.attend(q[:0], t[:0], n[:0])
    assert cache.attend(q[:0], t, n).shape == (0, 4, 64)
    cache.write(k[:0], k[:0], t, n)
    assert cache.read(t, n, 0)[0].shape == (0, 2, 64)
    with pytest.raises(vq.BackendError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            try:
                cache.attend(q, table, n)
            finally:
                torch.zeros(1, device="cuda")


def test_results_are_on_the_caches_device_whatever_the_current_stream_is():
    torch = torch_()
    cache, parts, table = some_cache(73, [500], 1, 64)
    x = normal(74, 1, 4, 64, dtype="bfloat16")
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        y = cache.attend(x, device(table), device(np.array([500], np.int32)))
        torch.cuda.current_stream().synchronize()
    check(y, *attend64(parts, x, table, [500], [0, 1]))
