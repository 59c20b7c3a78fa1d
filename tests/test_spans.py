"""Distances of rows and heads that the calls on 8-bit codes and on a cache take: by the library's own rule, compiled and run without a GPU, and at the C ABI."""
import os
import subprocess

import numpy as np
import pytest

import vq_b200 as vq
from vq_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rules(tmp_path):
    exe = os.path.join(str(tmp_path), "test_spans")
    subprocess.check_call(["/usr/bin/g++", "-std=c++17", "-O1", "-Wall", "-o", exe, os.path.join(ROOT, "tests", "cpp", "test_spans.cpp")])
    res = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=60)
    assert res.returncode == 0, res.stdout.decode()


@pytest.mark.gpu
@pytest.mark.parametrize("n,ld", [(2**23 + 1, 2**40), (2**24 + 1, 2**40), (2, 2**63)])
def test_rows_too_far_apart_are_refused_before_anything_is_read(n, ld):
    """Host memory, as anything else would be the caller's own lie: none of it is touched."""
    lib, cache = _lib.load(), vq.QuantizedCache.empty(1, 1, 4)
    x, y = np.zeros(4, np.float16), np.full(4, 7, np.float16)
    table, lengths = np.zeros((1, 1), np.int32), np.ones(1, np.int32)
    sequences = table.ctypes.data, 1, 1, 1, lengths.ctypes.data, None
    assert lib.vqb_cache_write(cache._h, x.ctypes.data, ld, 4, x.ctypes.data, 4, 4, 1, n, 1, 4, *sequences) == 90
    assert lib.vqb_cache_write(cache._h, x.ctypes.data, 4, 4, x.ctypes.data, ld, 4, 1, n, 1, 4, *sequences) == 90
    assert lib.vqb_cache_attend(cache._h, x.ctypes.data, 1, n, 1, 4, ld, 4, *sequences, 1.0, 0, 0, y.ctypes.data, 4, 4, 0) == 90
    assert lib.vqb_cache_attend(cache._h, x.ctypes.data, 1, n, 1, 4, 4, 4, *sequences, 1.0, 0, 0, y.ctypes.data, ld, 4, 0) == 90
    assert (y == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("ld", [2**63, 2**59, 2**64 - 4])
def test_rows_of_products_too_far_apart_are_refused(ld):
    """Two rows in host memory: what they span would have come out as a few bytes."""
    lib, m = _lib.load(), vq.QuantizedMatrix.fit(np.ones((4, 4), np.float32), gradient=True)
    x, codes, scales, y = np.zeros((2, 4), np.float16), np.zeros((2, 4), np.int8), np.ones(2, np.float32), np.full((2, 4), 7, np.float16)
    at = [v.ctypes.data for v in (x, codes, scales, y)]
    ctx = m._ctx.handle
    assert lib.vqb_row_quantize(ctx, at[0], 1, 2, 4, ld, at[1], 4, at[2]) == 90
    assert lib.vqb_row_quantize(ctx, at[0], 1, 2, 4, 4, at[1], ld, at[2]) == 90
    assert lib.vqb_qmat_product(m._h, at[0], 1, 2, 4, ld, None, None, at[3], 1, 4, 0) == 90
    assert lib.vqb_qmat_product(m._h, at[0], 1, 2, 4, 4, None, None, at[3], 1, ld, 0) == 90
    assert lib.vqb_qmat_product_codes(m._h, at[1], ld, at[2], 2, 4, None, None, at[3], 1, 4, 0) == 90
    assert lib.vqb_qmat_product_codes(m._h, at[1], 4, at[2], 2, 4, None, None, at[3], 1, ld, 0) == 90
    assert lib.vqb_qmat_input_gradient(m._h, at[0], 1, 2, 4, ld, None, at[3], 4, 0) == 90
    assert lib.vqb_qmat_input_gradient(m._h, at[0], 1, 2, 4, 4, None, at[3], ld, 0) == 90
    assert (y == 7).all()
    assert lib.vqb_qmat_product(m._h, at[0], 1, 1, 4, ld, None, None, at[3], 1, ld, 0) == 0 and (y[0] == 0).all()  # (one row: no distance)


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 40])
def test_heads_far_apart_are_taken(count):
    """More than 2^28 values from head to head: what a head behind a head of 2^21 rows of 128 values has."""
    import torch
    from tests.test_gpu_cache import attend64, check, device, normal, some_cache
    lengths = np.array([200])
    cache, parts, table = some_cache(90, lengths, 2, 128)
    apart = 2**28 + 128
    room = torch.zeros(apart + count * 128, dtype=torch.float16, device="cuda")
    far = torch.as_strided(room, (count, 2, 128), (128, apart, 1))
    x = normal(91, count, 2, 128, dtype="float16")
    far.copy_(x)
    n, t = device(lengths.astype(np.int32)), device(table)
    out = torch.as_strided(torch.zeros_like(room), (count, 2, 128), (128, apart, 1))
    check(cache.attend(far, t, n, out=out), *attend64(parts, x, table, lengths, [0, count]))
    same = vq.QuantizedCache.from_parts(*parts)
    cache.write(far, far, t, n)
    same.write(x, x, t, n)
    for a, b in zip(cache.read(t, n, 200), same.read(t, n, 200)):
        assert torch.equal(a, b)
