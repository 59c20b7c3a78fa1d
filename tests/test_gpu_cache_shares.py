"""Attention over caches long enough that every block's share has many pages, ends inside tiles and spans several: every token counts once, with its own page's scales.

Made so that sums are exact.  Scores are whole numbers of powers of two (the scores' scale times log2(e) is 1 in f32), value scales are powers of two, so weights are powers of two,
also as f16 numbers; codes of values are small, and all weights times codes of a row together are below 2^24 of the smallest of them: no sum of any of them is rounded.  What is left is
the exponential's own error below the line, 2^-22 of each term, the rounding of at most 400 additions there (a share has some 100 pages, a row some 50 parts), 400 x 2^-24, and the
quotient: less than 2^-14 together.  A page that is missed, taken twice or weighed with another one's scale changes
most of a row's values by 1 % and more (of texts of 150,000 tokens), a single token by 2^-10."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest

import vq_b200 as vq
from tests.test_gpu_cache import PAGE, device, gen, starts, torch_

pytestmark = pytest.mark.gpu

SCALE = float(np.float32(math.log(2.0)))
assert np.float32(SCALE) * np.float32(1.44269504088896341) == np.float32(1.0)


def exact_case(seed, lengths, counts, heads, group, width, dtype="float16", window=None, sinks=0, missing=0.05, more_columns=0):
    torch = torch_()
    g = gen(seed)
    lengths, counts = np.array(lengths), np.array(counts)
    pages = [-(-int(v) // PAGE) for v in lengths]
    pool = sum(pages) + 3
    rs = np.random.RandomState(seed)
    place, at = rs.permutation(pool), 0
    table = np.full((len(lengths), max(pages) + more_columns), -1, np.int32)
    for b, n in enumerate(pages):
        table[b, :n] = np.where(rs.rand(n) < missing, -1, place[at : at + n])
        at += n
    if more_columns:  # what a server's table holds behind the tokens
        for b, n in enumerate(pages):
            table[b, n:] = rs.randint(0, pool, table.shape[1] - n)
    kc = torch.randint(-100, 100, (pool, heads, PAGE, width), generator=g, device="cuda", dtype=torch.int8)
    kc[..., 0] = torch.randint(0, 2, kc.shape[:3], generator=g, device="cuda", dtype=torch.int8)
    vc = torch.randint(-3, 4, (pool, heads, PAGE, width), generator=g, device="cuda", dtype=torch.int8)
    ks, vs = (torch.exp2(torch.randint(0, top, (pool, heads), generator=g, device="cuda").float()) for top in (2, 4))
    nan_head = heads - 1  # of the first sequence: a page of NaN
    vs[next(int(p) for p in table[0, pages[0] // 2 :] if p >= 0), nan_head] = math.nan
    cache = vq.QuantizedCache.from_parts(kc, ks, vc, vs)
    offsets = starts(counts)
    x = torch.zeros(int(offsets[-1]), heads * group, width, device="cuda", dtype=getattr(torch, dtype))
    x[..., 0] = torch.randint(0, 3, x.shape[:2], generator=g, device="cuda").to(x.dtype)
    given = None if len(set(counts)) == 1 else device(offsets)
    y = cache.attend(x, device(table), device(lengths.astype(np.int32)), offsets=given, scale=SCALE, window=window, sinks=sinks)
    info = torch.finfo(y.dtype)
    for b in range(len(lengths)):
        r0, r1, n = int(offsets[b]), int(offsets[b + 1]), int(lengths[b])
        j = torch.arange(n, device="cuda")
        page = torch.from_numpy(table[b].astype(np.int64)).cuda()[j // PAGE]
        there, slot = page >= 0, j % PAGE
        page = page.clamp(min=0)
        position = torch.arange(n - (r1 - r0), n, device="cuda")[:, None]
        seen = there & (j <= position)
        if window:
            seen &= (j > position - window) | (j < sinks)
        for h in range(heads):
            rows = y[r0:r1, h * group : (h + 1) * group]
            nan = (seen & torch.isnan(vs[page, h])).any(-1)
            assert torch.isnan(rows[nan]).all() and not torch.isnan(rows[~nan]).any()
            s = x[r0:r1, h * group : (h + 1) * group, :1].double() * (kc[page, h, slot, 0].double() * ks[page, h].double())  # rows x group x tokens
            p = torch.where(seen[:, None], torch.exp2(s), 0.0)
            v = vc[page, h, slot].double()
            w = p * vs[page, h].double().nan_to_num()
            empty = p.sum(-1, keepdim=True) == 0
            assert (w @ v.abs()).max() < 2.0**24
            want = torch.where(empty, 0.0, (w @ v) / torch.where(empty, 1.0, p.sum(-1, keepdim=True)))
            off = (rows.double() - want).abs()
            # (a result below the type's normal numbers is rounded to a multiple of the smallest one: by half of that, 2^-25 for f16, at most)
            bad = ~(off <= want.abs() * (info.eps / 2 + 2.0**-14) + info.smallest_normal * info.eps / 2) & ~nan[:, None, None]
            assert not bad.any(), f"sequence {b} head {h}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: {rows[bad][0]} for {want[bad][0]}"


LONG = [150_001, 30_000, 99_999, 140_007]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("how", [{}, {"window": 90_000, "sinks": 1000}], ids=["all", "window"])
@pytest.mark.parametrize("group,width", [(1, 32), (8, 40)])
def test_single_tokens_behind_very_long_texts(group, width, how, dtype):
    """Without a window some 180 pages a share of the 3 x 148 blocks, 45 a warp: what a warp looks ahead for, 32 pages at a time, is renewed."""
    exact_case(1, LONG, [1] * 4, 12, group, width, dtype, **how)


@pytest.mark.parametrize("group", [1, 8])
def test_a_few_tokens_behind_very_long_texts(group):
    exact_case(2, LONG, [2] * 4, 10, group, 32)  # sixteen rows a tile
    exact_case(3, LONG, [4, 1, 3, 2], 10, group, 32)


@pytest.mark.parametrize("width", [32, 96, 200])
def test_single_tokens_of_a_large_batch(width):
    """Shares that end inside tiles and have several."""
    lengths = np.random.RandomState(4).randint(1, 6000, 64)
    exact_case(4, lengths, [1] * 64, 8, 4, width)


@pytest.mark.parametrize("how", [{}, {"window": 20_000, "sinks": 100}], ids=["all", "window"])
@pytest.mark.parametrize("counts,group,width,dtype", [([256, 100, 300], 1, 32, "float16"), ([100, 100, 100], 2, 32, "bfloat16"), ([200, 40, 130], 1, 96, "float16"), ([130, 34, 70], 1, 200, "float16"),
                                                      ([256, 1, 20], 3, 64, "float16")], ids=str)
def test_pieces_of_prompts_behind_long_texts(counts, group, width, dtype, how):
    """Shares of 50 to 200 pages, one a step: what is looked ahead for, 32 at a time, is renewed."""
    exact_case(5, [60_001, 30_000, 44_444], counts, 8 if width < 200 else 4, group, width, dtype, **how)


@pytest.mark.parametrize("columns", [1, 100, 2000])
def test_tables_wider_than_their_tokens_need(columns):
    """As in a captured step, whose table is as wide as the longest text allowed; what is behind the tokens is of other requests."""
    exact_case(6, [1000], [1], 8, 4, 64, more_columns=columns)
    exact_case(7, [1000, 130, 64], [1] * 3, 2, 8, 64, more_columns=columns)
    exact_case(8, [700, 5, 333], [700, 5, 333], 2, 1, 80, more_columns=columns)
    exact_case(9, [300] * 3, [64] * 3, 2, 1, 64, more_columns=columns)


def test_odd_pages_without_tensor_cores():
    """Pages that are not there, NaN, infinite queries, scales far apart and offsets out of order, on the CUDA cores."""
    code = """
from tests import test_gpu_cache as t, test_gpu_cache_shares as s
t.test_tokens_that_are_not_there_are_not_seen([1] * 5)
t.test_tokens_that_are_not_there_are_not_seen([65, 20, 130, 1, 30])
for which in (1, 3):
    t.test_nan_stays_where_it_is_seen([100, 100], which)
t.test_infinite_and_nan_queries_make_their_rows_nan_and_no_others(90)
t.test_scales_far_apart([200, 40, 100])
t.test_rows_of_no_sequence([50, 1, 70])
t.test_rows_heads_and_results_of_any_distance(5)
t.test_offsets_of_any_kind_stay_in_bounds()
s.exact_case(10, [1500, 70], [1, 1], 2, 2, 48)
s.exact_case(11, [500, 70], [90, 3], 2, 2, 48, window=100, sinks=9, more_columns=5)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, env={**os.environ, "VQB_NO_TENSOR": "1"}, timeout=300)
