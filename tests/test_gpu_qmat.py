"""Rows quantized to 8 bits with a scale each, products of codes, grouped products and gradients, against the same in 64 bits.

Tolerances: the sums of products of codes are exact; the steps behind them (to f32, times the row's scale, times the channel's, plus the bias)
round four times, by at most 2^-24 of |sum s t| + |bias| each; the result's own rounding is half a step of its type."""
import numpy as np
import pytest

import vq_b200 as vq

pytestmark = pytest.mark.gpu
TINY = {"float32": 2.0**-149, "float16": 2.0**-24, "bfloat16": 2.0**-133}


def torch_():
    import torch
    return torch


def gen(seed):
    return torch_().Generator(device="cuda").manual_seed(seed)


def normal(seed, *shape, dtype="float32", scale=1.0):
    torch = torch_()
    return (scale * torch.randn(shape, generator=gen(seed), device="cuda")).to(getattr(torch, dtype))


def codes64(x):
    """(codes, scales) of rows by the definition, in 64 bits; the scales as float32 numbers."""
    torch = torch_()
    x = x.double()
    a = x.abs().amax(-1) if x.shape[-1] else x.new_zeros(x.shape[:-1])
    s = torch.where(a > 0, (a / 127).float().clamp_min(2.0**-126).double(), a)
    ok = torch.isfinite(a)
    s = torch.where(ok, s, torch.nan)
    q = torch.where(((a > 0) & ok)[..., None], torch.round(x / s[..., None]), 0.0)
    return q, s


def groups_of(offsets, n, groups):
    """The group of each row, -1 for none."""
    g = np.full(n, -1)
    if offsets is None:
        return np.zeros(n, int)
    for i in range(groups):
        g[offsets[i]:offsets[i + 1]] = i
    return g


def product64(q, s, wq, ws, bias=None, offsets=None):
    """(result, magnitude that the rounding goes by, rows of a group); wq: groups x outputs x inputs, all in 64 bits"""
    torch = torch_()
    g = torch.from_numpy(groups_of(offsets, q.shape[0], wq.shape[0])).to(q.device)
    y = q.new_zeros(q.shape[0], wq.shape[1])
    b = torch.zeros_like(y)
    for i in range(wq.shape[0]):
        rows = g == i
        y[rows] = (q[rows] @ wq[i].T) * s[rows, None] * ws[i]
        if bias is not None:
            b[rows] = bias.double().reshape(wq.shape[0], -1)[i]
    return y + b, y.abs() + b.abs(), g >= 0


def check(y, want, size, extra=0.0):
    torch = torch_()
    step = torch.finfo(y.dtype).eps / 2
    name = str(y.dtype)[6:]
    limit = 4 * 2.0**-24 * size + step * want.abs() * (1 + 2.0**-20) + TINY[name] + extra
    top = torch.finfo(y.dtype).max
    off = (y.double() - want).abs()
    bad = ~(off <= limit) & ~(torch.isnan(y) & torch.isnan(want)) & ~(want.abs() > top * (1 - step))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, first at {bad.nonzero()[0].tolist()}: {y[bad][0]} for {want[bad][0]} (limit {limit[bad][0]:.3e})"


# ---- rows ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,dim", [(1, 1), (1, 4096), (5, 7), (33, 15), (64, 16), (257, 129), (9, 1001), (40, 1024), (6, 2049), (3, 8192), (2, 40_001)])
def test_rows_are_the_definitions(n, dim, dtype):
    torch = torch_()
    x = normal(n + dim, n, dim, dtype=dtype)
    x[::3] *= 100.0
    q, s = vq.RowQuantizer.fit().quantize(x)
    want_q, want_s = codes64(x)
    assert q.dtype is torch.int8 and s.dtype is torch.float32
    assert torch.equal(s.double(), want_s) and torch.equal(q.double(), want_q)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_quotients_that_are_halves_go_to_even(dtype):
    """127 as the largest value makes the scale 1; halves are then halves, and their neighbours are not."""
    torch = torch_()
    x = (torch.arange(-253, 254, device="cuda") / 2.0).to(getattr(torch, dtype))
    if dtype == "float32":
        x = torch.cat([x, torch.nextafter(x, x + 1), torch.nextafter(x, x - 1), x.new_tensor([127.0])])
        x = x[x.abs() <= 127]
    x = torch.cat([x, x.new_tensor([127.0])])
    rows = torch.stack([x, x * 2.0**-20 if dtype != "float16" else x * 0.5, -x])
    q, s = vq.RowQuantizer.fit().quantize(rows)
    want_q, want_s = codes64(rows)
    assert torch.equal(s.double(), want_s) and torch.equal(q.double(), want_q)


def test_scales_of_many_sizes():
    """Random quotients next to halves: x = (h + 1/2) s nudged by single steps, s any float32."""
    torch = torch_()
    a = torch.exp(40 * torch.randn(4000, 1, generator=gen(5), device="cuda")).clamp(1e-30, 1e30)
    s = (a.double() / 127).float()
    h = torch.randint(-126, 126, (4000, 64), generator=gen(6), device="cuda") + 0.5
    x = (h.double() * s.double()).float()
    x = torch.where(torch.rand(4000, 64, generator=gen(7), device="cuda") < 0.5, torch.nextafter(x, torch.zeros_like(x)), x)
    x = torch.cat([x, a], 1)
    q, got = vq.RowQuantizer.fit().quantize(x)
    want_q, want_s = codes64(x)
    assert torch.equal(got.double(), want_s) and torch.equal(q.double(), want_q)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("dim", [5, 64, 2999])
def test_rows_of_zeros_and_rows_that_are_not_finite(dim, dtype):
    torch = torch_()
    x = normal(3, 8, dim, dtype=dtype)
    x[1] = 0
    x[2] = -0.0
    x[3, dim // 2] = float("inf")
    x[4, dim - 1] = float("-inf")
    x[5, 0] = float("nan")
    x[6] = torch.finfo(x.dtype).max
    x[7] = torch.finfo(x.dtype).smallest_normal / 256 if dtype != "float16" else 2.0**-24
    q, s = vq.RowQuantizer.fit().quantize(x)
    want_q, want_s = codes64(x)
    assert torch.equal(q.double(), want_q)
    assert torch.equal(torch.isnan(s), torch.tensor([0, 0, 0, 1, 1, 1, 0, 0], device="cuda").bool())
    assert torch.equal(s.double()[[0, 1, 2, 6, 7]], want_s[[0, 1, 2, 6, 7]])


def test_rows_apart_and_unaligned():
    torch = torch_()
    whole = normal(9, 50, 1000, dtype="bfloat16")
    for view in (whole[:, 8:520], whole[:, 1:600], whole[::2, 3:4], whole[:, ::2], whole.T[:70], whole[7:8, 9:]):
        q, s = vq.RowQuantizer.fit().quantize(view)
        want_q, want_s = codes64(view)
        assert torch.equal(s.double(), want_s) and torch.equal(q.double(), want_q)


def test_rows_in_host_memory_and_single_vectors():
    x = np.random.default_rng(3).normal(size=(20, 77)).astype(np.float32)
    rq = vq.RowQuantizer.fit()
    q, s = rq.quantize(x)
    want_q, want_s = codes64(torch_().from_numpy(x))
    assert isinstance(q, np.ndarray) and q.dtype == np.int8 and np.array_equal(q, want_q.numpy()) and np.array_equal(s, want_s.numpy().astype(np.float32))
    q1, s1 = rq.quantize(x[3])
    assert q1.shape == (77,) and s1.shape == () and np.array_equal(q1, q[3]) and s1 == s[3]
    h = x.astype(np.float16)
    assert np.array_equal(rq.quantize(h)[0], codes64(torch_().from_numpy(h))[0].numpy())


# ---- products --------------------------------------------------------------------------------------------------
def matrix64(w, gradient=False):
    q, s = codes64(w)
    return vq.QuantizedMatrix.fit(w, gradient=gradient), q.reshape(-1, *q.shape[-2:]), s.reshape(-1, s.shape[-1])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,inputs,outputs", [(1, 1, 1), (1, 4096, 4096), (2, 100, 129), (8, 1000, 300), (9, 512, 257), (16, 2048, 128), (17, 33, 127), (31, 16, 700), (33, 129, 128),
                                              (64, 4096, 1000), (65, 640, 512), (255, 127, 5), (256, 256, 256), (257, 384, 130), (300, 1001, 515), (513, 96, 1030),
                                              (1030, 2047, 1281), (5000, 17, 33)])
def test_products(n, inputs, outputs, dtype):
    torch = torch_()
    x, w = normal(n, n, inputs, dtype=dtype), normal(inputs, outputs, inputs, scale=inputs**-0.5)
    m, wq, ws = matrix64(w)
    bias = normal(7, outputs) if n % 2 else None
    y = m.product(x, bias)
    assert y.dtype is x.dtype and tuple(y.shape) == (n, outputs)
    want, size, _ = product64(*codes64(x), wq, ws, bias)
    check(y, want, size)
    assert np.array_equal(m.codes, wq[0].cpu().numpy()) and np.array_equal(m.scales, ws[0].float().cpu().numpy())


@pytest.mark.parametrize("n,inputs,outputs", [(1, 4096, 14336), (2, 8200, 9001), (3, 16400, 5000), (8, 1030, 20_011), (16, 4096, 14336), (16, 9000, 3000), (5, 520, 40_000), (4, 64, 150_000)])
def test_products_of_few_rows_with_large_matrices(n, inputs, outputs):
    """Every block has many pieces of the matrix: more than it has room for at a time."""
    torch = torch_()
    x = normal(n, n, inputs, dtype="bfloat16")
    m, wq, ws = matrix64(normal(inputs, outputs, inputs, scale=inputs**-0.5))
    want, size, _ = product64(*codes64(x), wq, ws)
    for _ in range(3):
        check(m.product(x), want, size)


@pytest.mark.parametrize("dtype", ["float32", "float16"])
@pytest.mark.parametrize("n,inputs,outputs", [(64, 4096, 4096), (33, 5000, 700), (100, 8190, 1030), (300, 8192, 256), (17, 130, 257), (250, 1000, 100), (20, 40_000, 130)])
def test_products_of_few_tiles_with_wide_matrices(n, inputs, outputs, dtype):
    """Too few tiles for the SMs: several of them take a part of the width each.  The gradient's way too: outputs and inputs change places."""
    x = normal(n, n, inputs, dtype=dtype)
    m, wq, ws = matrix64(normal(inputs, outputs, inputs, scale=inputs**-0.5))
    bias = normal(1, outputs)
    want, size, _ = product64(*codes64(x), wq, ws, bias)
    check(m.product(x, bias), want, size)
    if dtype == "float16":
        m, wq, ws = matrix64(normal(inputs, inputs, outputs, scale=0.02), gradient=True)
        want, size, extra, _ = gradient_limits(x, wq, ws)
        check(m.input_gradient(x), want, size, extra)


@pytest.mark.parametrize("out", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,inputs,outputs", [(1, 160, 96), (12, 1000, 300), (40, 97, 64), (700, 513, 200)])
def test_products_of_codes_up_to_the_largest(n, inputs, outputs, out):
    """All codes -128: the largest sums that there are."""
    torch = torch_()
    q = torch.randint(-128, 128, (n, inputs), generator=gen(1), device="cuda", dtype=torch.int8)
    wq = torch.randint(-128, 128, (outputs, inputs), generator=gen(2), device="cuda", dtype=torch.int8)
    q[0], wq[0] = -128, -128
    s, t = normal(3, n).abs() * 1e-3, normal(4, outputs) * 1e-3
    m = vq.QuantizedMatrix.from_parts(wq, t)
    y = m.product_of_codes(q, s, dtype=getattr(torch, out))
    want, size, _ = product64(q.double(), s.double(), wq.double()[None], t.double()[None])
    assert y.dtype is getattr(torch, out)
    check(y, want, size)
    single = m.product_of_codes(q[0], s[0], dtype=getattr(torch, out))
    check(single, want[0], size[0])


def test_the_widest_sums_stay_in_32_bits():
    torch = torch_()
    width = 131071
    q = torch.full((3, width), -128, dtype=torch.int8, device="cuda")
    wq = torch.full((2, width), -128, dtype=torch.int8, device="cuda")
    wq[1] = 127
    one = torch.ones(3, device="cuda")
    y = vq.QuantizedMatrix.from_parts(wq, one[:2]).product_of_codes(q, one)
    assert y.tolist() == [[float(np.float32(16384 * width)), float(np.float32(-128 * 127 * width))]] * 3


GROUPED = [
    # n, inputs, outputs, counts (the rest belongs to nobody), rows in front
    (7, 64, 100, [0, 3, 0, 4], 0),
    (1, 32, 17, [0, 0, 1], 0),
    (10, 100, 129, [0, 0, 0], 4),
    (300, 200, 140, [1, 0, 70, 33, 31, 32, 64, 0], 5),
    (1500, 129, 300, [600, 257, 0, 256, 255, 1], 0),
    (64, 1024, 256, [1] * 64, 0),
    (400, 48, 65, [3] * 100, 50),
]


def offsets_of(counts, front):
    return np.concatenate([[front], front + np.cumsum(counts)]).astype(np.int64)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,inputs,outputs,counts,front", GROUPED)
def test_grouped_products(n, inputs, outputs, counts, front, dtype):
    torch = torch_()
    groups = len(counts)
    x, w = normal(n, n, inputs, dtype=dtype), normal(4, groups, outputs, inputs, scale=inputs**-0.5)
    m, wq, ws = matrix64(w)
    off = offsets_of(counts, front)
    bias = normal(8, groups, outputs) if n % 2 == 0 else None
    want, size, within = product64(*codes64(x), wq, ws, bias, off)
    y = m.product(x, bias, offsets=torch.from_numpy(off).cuda())
    check(y[within], want[within], size[within])
    assert not y[~within].any(), "rows of no group"
    out = torch.full_like(y, 5.0)
    again = m.product(x, bias, offsets=off, out=out)  # (offsets from the host; rows of no group stay)
    assert again is out and torch.equal(out[within], y[within]) and bool((out[~within] == 5.0).all())
    q, s = vq.RowQuantizer.fit().quantize(x)
    assert torch.equal(m.product_of_codes(q, s, bias, offsets=torch.from_numpy(off).cuda(), dtype=x.dtype), y)


def test_rows_apart_and_results_apart():
    torch = torch_()
    whole = normal(2, 70, 700, dtype="float16")
    x = whole[:, 3:403]
    m, wq, ws = matrix64(normal(3, 90, 400, scale=0.05))
    want, size, _ = product64(*codes64(x), wq, ws)
    room = torch.full((70, 200), 9.0, device="cuda", dtype=torch.float16)
    y = m.product(x, out=room[:, 50:140])
    check(y, want, size)
    assert bool((room[:, :50] == 9).all()) and bool((room[:, 140:] == 9).all())
    check(m.product(x[5], out=room[0, 10:100]), want[5], size[5])


@pytest.mark.parametrize("n", [1, 20, 300])
def test_rows_that_are_zero_or_not_finite_keep_to_themselves(n):
    torch = torch_()
    x = normal(1, n + 4, 200)
    x[0], x[1, 5], x[2, 7] = 0, float("inf"), float("nan")
    m, wq, ws = matrix64(normal(2, 150, 200))
    bias = normal(3, 150)
    y = m.product(x, bias)
    want, size, _ = product64(*codes64(x), wq, ws, bias)
    assert torch.equal(y[0], bias) and bool(torch.isnan(y[1:3]).all()) and not torch.isnan(y[3:]).any()
    check(y, want, size)


def test_a_channel_that_is_not_finite_is_not_a_number():
    torch = torch_()
    w = normal(2, 140, 64)
    w[7, 3], w[130] = float("nan"), 0.0
    y = vq.QuantizedMatrix.fit(w).product(normal(1, 40, 64))
    assert bool(torch.isnan(y[:, 7]).all()) and not y[:, 130].any() and int(torch.isnan(y).any(0).sum()) == 1


def test_products_in_host_memory():
    rng = np.random.default_rng(1)
    x, w = rng.normal(size=(50, 90)).astype(np.float32), rng.normal(size=(3, 40, 90)).astype(np.float32)
    m, torch = vq.QuantizedMatrix.fit(w), torch_()
    off = np.array([2, 12, 12, 45])
    want, size, within = product64(*codes64(torch.from_numpy(x)), *(codes64(torch.from_numpy(w))), None, off)
    y = m.product(x, offsets=off)
    assert isinstance(y, np.ndarray) and y.dtype == np.float32
    check(torch.from_numpy(y), want, size)
    room = np.full((50, 60), 3.0, np.float16)
    got = m.product(x, offsets=off, out=room[:, 10:50])
    check(torch.from_numpy(got[2:45]), want[2:45], size[2:45])
    assert (room[:2] == 3).all() and (room[45:] == 3).all() and (room[:, :10] == 3).all() and (room[:, 50:] == 3).all()


def test_no_rows():
    torch = torch_()
    m = vq.QuantizedMatrix.fit(normal(1, 30, 20), gradient=True)
    assert tuple(m.product(normal(1, 0, 20)).shape) == (0, 30)
    assert tuple(m.input_gradient(normal(1, 0, 30, dtype="float16")).shape) == (0, 20)
    q, s = vq.RowQuantizer.fit().quantize(normal(1, 0, 20))
    assert tuple(q.shape) == (0, 20) and tuple(s.shape) == (0,)
    assert tuple(m.product_of_codes(q, s).shape) == (0, 30)


# ---- gradients -------------------------------------------------------------------------------------------------
def gradient_limits(dy, wq, ws, offsets=None):
    """(gradient, size for the rounding, what the 16256 steps may be off by): each u = dy t is off by half a step, by 16256 2^-23 of one for the quotient and by
    16256 2^-24 for u itself."""
    torch = torch_()
    g = torch.from_numpy(groups_of(offsets, dy.shape[0], wq.shape[0])).to(dy.device)
    dx, extra, size = (dy.new_zeros(dy.shape[0], wq.shape[2], dtype=torch.float64) for _ in range(3))
    for i in range(wq.shape[0]):
        rows = g == i
        u = dy[rows].double() * ws[i]
        step = u.abs().amax(-1, keepdim=True) / 16256 if u.numel() else u.sum(-1, keepdim=True)
        dx[rows], size[rows] = u @ wq[i], u.abs() @ wq[i].abs()
        extra[rows] = step * (0.5 + 16256 * (2.0**-23 + 2.0**-24)) * wq[i].abs().sum(0)
    return dx, size, extra, g >= 0


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,inputs,outputs", [(1, 1, 1), (1, 300, 200), (3, 129, 1000), (33, 64, 64), (64, 700, 129), (129, 128, 256), (300, 1001, 515), (1000, 257, 96)])
def test_gradients(n, inputs, outputs, dtype):
    dy, w = normal(n, n, outputs, dtype=dtype, scale=0.01), normal(inputs, outputs, inputs, scale=inputs**-0.5)
    dy[::4] *= 30.0
    m, wq, ws = matrix64(w, gradient=True)
    dx = m.input_gradient(dy)
    want, size, extra, _ = gradient_limits(dy, wq, ws)
    assert dx.dtype is dy.dtype and tuple(dx.shape) == (n, inputs)
    check(dx, want, size, extra)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("n,inputs,outputs,counts,front", GROUPED)
def test_grouped_gradients(n, inputs, outputs, counts, front, dtype):
    torch = torch_()
    groups = len(counts)
    dy, w = normal(n, n, outputs, dtype=dtype), normal(4, groups, outputs, inputs, scale=inputs**-0.5)
    m, wq, ws = matrix64(w, gradient=True)
    off = offsets_of(counts, front)
    want, size, extra, within = gradient_limits(dy, wq, ws, off)
    dx = m.input_gradient(dy, offsets=torch.from_numpy(off).cuda())
    check(dx[within], want[within], size[within], extra[within])
    assert not dx[~within].any()
    out = torch.full_like(dx, 5.0)
    m.input_gradient(dy, offsets=off, out=out)
    assert torch.equal(out[within], dx[within]) and bool((out[~within] == 5.0).all())


def test_gradient_is_the_products_difference():
    """Rows on the grid of their scale: a step of one code changes the product by that step times the channel's values, and the gradient says so."""
    torch = torch_()
    n, inputs, outputs = 6, 40, 70
    m, wq, ws = matrix64(normal(2, outputs, inputs), gradient=True)
    x = torch.randint(-100, 100, (n, inputs), generator=gen(1), device="cuda").float()
    x[:, 0] = 127.0
    dy = torch.ones(n, outputs, device="cuda", dtype=torch.float16)
    dy[:, ::3] = -0.5
    dx = m.input_gradient(dy)
    base = m.product(x).double()
    _, size, extra, _ = gradient_limits(dy, wq, ws)
    for k in range(1, inputs):
        there = x.clone()
        there[:, k] += 1.0
        difference = ((m.product(there).double() - base) * dy.double()).sum(1)
        # 2 x 70 values of the products, each rounded four times relative to at most |sum s t|
        products = 8 * 2.0**-24 * ((x.double().abs() + 1) @ (wq[0].abs().T * ws[0])).sum(1)
        check(dx[:, k], difference, size[:, k], extra[:, k] + products)


def test_gradient_of_rows_of_zeros_and_rows_that_are_not_finite():
    torch = torch_()
    m, wq, ws = matrix64(normal(2, 100, 50), gradient=True)
    dy = normal(1, 5, 100, dtype="bfloat16")
    dy[0], dy[1, 3], dy[2, 99] = 0, float("inf"), float("nan")
    dx = m.input_gradient(dy)
    want, size, extra, _ = gradient_limits(dy[3:], wq, ws)
    assert not dx[0].any() and bool(torch.isnan(dx[1:3]).all())
    check(dx[3:], want, size, extra)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,dim", [(14_300, 4096), (7_300, 8192), (14_209, 4104), (7_111, 6160), (70_000, 128), (33_001, 515), (20_000, 1000), (9_000, 2048), (1_100, 16400)])
def test_many_wide_rows_are_the_definitions(n, dim, dtype):
    """Enough of them that bytes under way count: fewer threads a row, with more of it each."""
    torch = torch_()
    x = normal(n, n, dim, dtype=dtype)
    x[5], x[n - 1, 3], x[n // 2, 0] = 0, float("nan"), float("inf")
    q, s = vq.RowQuantizer.fit().quantize(x)
    for part in torch.arange(n, device="cuda").split(2048):
        want_q, want_s = codes64(x[part])
        assert torch.equal(q[part].double(), want_q) and torch.equal(torch.nan_to_num(s[part], nan=-1.0).double(), torch.nan_to_num(want_s, nan=-1.0))


def test_as_many_groups_as_there_may_be():
    torch = torch_()
    counts = [(7 * g) % 5 for g in range(1024)]
    n = sum(counts) + 9
    off = offsets_of(counts, 4)
    x, w = normal(1, n, 48, dtype="bfloat16"), normal(2, 1024, 40, 48, scale=0.1)
    m, wq, ws = matrix64(w, gradient=True)
    y = m.product(x, offsets=torch.from_numpy(off).cuda())
    want, size, within = product64(*codes64(x), wq, ws, None, off)
    check(y[within], want[within], size[within])
    assert not y[~within].any()
    dy = normal(3, n, 40, dtype="bfloat16")
    want, size, extra, within = gradient_limits(dy, wq, ws, off)
    check(m.input_gradient(dy, offsets=off)[within], want[within], size[within], extra[within])


def test_one_group_with_offsets_takes_some_of_the_rows():
    torch = torch_()
    x = normal(1, 50, 64, dtype="float16")
    m, wq, ws = matrix64(normal(2, 30, 64))
    off = np.array([7, 33])
    want, size, within = product64(*codes64(x), wq, ws, None, off)
    y = m.product(x, offsets=off)
    check(y[within], want[within], size[within])
    assert not y[~within].any()
