"""Attention over pages whose values have a scale of 0 and codes that are not 0: their tokens count below the line, and add nothing above it.

Tolerances are those of tests/test_gpu_cache.py; where all values of a row are 0 its result is 0, exactly."""
import os
import subprocess
import sys

import numpy as np
import pytest

import vq_b200 as vq
from tests.test_gpu_cache import attend64, check, device, normal, some_cache, starts, torch_

pytestmark = pytest.mark.gpu

LENGTHS = np.array([960, 70, 330, 200])  # (fifteen pages: several for each warp)


def zero_case(seed, counts, heads, group, width, dtype="bfloat16", **how):
    """Pages in front, in the middle and at the end of a sequence, all pages of one, and pages of one head."""
    torch = torch_()
    _, parts, table = some_cache(seed, LENGTHS, heads, width)
    parts[1][:] = 1 / 42  # equal scales of keys: no page has all of the weight
    for page in (table[0, 0], table[0, 4], table[0, 9], table[0, 14], table[1, 0], table[1, 1], table[2, 5], table[2, 1]):
        parts[3][page] = 0.0
    parts[3][table[3, 2], heads - 1] = 0.0
    cache = vq.QuantizedCache.from_parts(*parts)
    offsets = starts(counts)
    x = normal(seed + 1, int(offsets[-1]), heads * group, width, dtype=dtype)
    given = None if len(set(counts)) == 1 else device(offsets)
    y = cache.attend(x, device(table), device(LENGTHS.astype(np.int32)), offsets=given, **how)
    check(y, *attend64(parts, x, table, LENGTHS, offsets, **how))
    assert (y[offsets[1] : offsets[2]] == 0).all()


@pytest.mark.parametrize("how", [{}, {"window": 100, "sinks": 5}], ids=["all", "window"])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [5, 5, 5, 5], [70, 70, 70, 70], [400, 1, 130, 9]], ids=str)
@pytest.mark.parametrize("heads,group,width,dtype", [(2, 4, 128, "bfloat16"), (1, 3, 73, "float16"), (2, 1, 64, "bfloat16"), (1, 2, 256, "float16")])
def test_values_of_scale_0_add_nothing_whatever_their_codes(heads, group, width, dtype, counts, how):
    zero_case(61, counts, heads, group, width, dtype, **how)


def test_values_of_scale_0_without_tensor_cores():
    code = """
from tests import test_gpu_cache_scales as t
t.zero_case(62, [1, 1, 1, 1], 2, 2, 72)
t.zero_case(63, [300, 1, 130, 9], 1, 3, 128, "float16", window=100, sinks=5)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    subprocess.run([sys.executable, "-c", code], check=True, cwd=root, env={**os.environ, "VQB_NO_TENSOR": "1"}, timeout=120)


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [70, 70, 70, 70]], ids=str)
def test_an_infinite_query_over_values_of_scale_0_is_not_taken_for_0(counts):
    """0 times a weight that is NaN is NaN, as in the rows that see other values."""
    torch = torch_()
    _, parts, table = some_cache(64, LENGTHS, 1, 64)
    parts[3][:] = 0.0
    cache = vq.QuantizedCache.from_parts(*parts)
    x = normal(65, sum(counts), 2, 64, dtype="float16")
    x[0, 1, 3] = float("inf")
    y = cache.attend(x, device(table), device(LENGTHS.astype(np.int32)))
    assert torch.isnan(y[0, 1]).all() and (y[0, 0] == 0).all() and (y[1:] == 0).all()
