"""Input gradients of rows that have a few large entries among many small ones, as the gradient of a softmax has, against the same in 64 bits.

Tolerances go by each row's result: half a step of its type, and what the arithmetic in front may lose.  u = dy t is a f32 product (2^-24 of it), comes to whole steps, 127 2^16 of which are
its row's largest, by a reciprocal (2^-24) and a product (2^-25 at most, as 127 2^16 < 2^23), and half a step is lost there; three whole-number sums are joined and scaled in f32
(six roundings of 2^-24 relative to the sum of magnitudes)."""
import pytest

import vq_b200 as vq
from tests.test_gpu_qmat import codes64, gen, normal, torch_

pytestmark = pytest.mark.gpu
STEPS = 127 * 2**16


def limits(dy, wq, ws):
    """(gradient, what the arithmetic in front of the result's rounding may be off by) in 64 bits"""
    u = dy.double() * ws
    step = u.abs().amax(-1, keepdim=True) / STEPS
    return u @ wq, 0.5 * step * wq.abs().sum(0) + 8.5 * 2.0**-24 * (u.abs() @ wq.abs())


def softmax_rows(n, outputs, spread, dtype):
    torch = torch_()
    p = torch.softmax(spread * torch.randn(n, outputs, generator=gen(n), device="cuda"), -1)
    p[torch.arange(n, device="cuda"), torch.randint(0, outputs, (n,), generator=gen(2), device="cuda")] -= 1.0
    return (p * 512.0).to(getattr(torch, dtype))  # (a loss times 512, so that binary16 holds the small ones)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("mean", [0.0, 0.1, 0.3])
@pytest.mark.parametrize("n,outputs", [(24, 32_000), (70, 128_256)])
def test_softmax_rows_keep_their_small_entries(n, outputs, mean, dtype):
    torch = torch_()
    inputs = 96
    w = normal(3, outputs, inputs) + mean
    wq, ws = codes64(w)
    dy = softmax_rows(n, outputs, 1.5, dtype)
    dx = vq.QuantizedMatrix.fit(w, gradient=True).input_gradient(dy)
    want, off = limits(dy, wq, ws)
    size = want.norm(dim=1)
    assert bool((off.norm(dim=1) <= 2.0**-6 * size).all())  # (at the worst; half a step has either sign)
    got = (dx.double() - want).norm(dim=1)
    assert bool((got <= torch.finfo(dx.dtype).eps / 2 * size + off.norm(dim=1)).all())
    # errors of either sign: what is lost of each entry is next to independent, so four of its standard deviations (half a step / sqrt 3, and 2^-24 of u) are not left
    u = dy.double() * ws
    steps = u.abs().amax(-1, keepdim=True) / STEPS
    spread = ((0.5 * steps) ** 2 / 3 * (wq**2).sum(0) + (8.5 * 2.0**-24) ** 2 * (u**2 @ wq**2)).sqrt()
    assert bool((got <= torch.finfo(dx.dtype).eps / 2 * size + 4 * spread.norm(dim=1)).all())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n,inputs,outputs", [(1, 1, 1), (3, 129, 1000), (33, 65, 64), (40, 130, 4100), (65, 700, 129), (129, 128, 256), (300, 1001, 515), (1000, 257, 96), (5000, 40, 33), (700, 3000, 300), (5, 64, 20_001)])
def test_gradients_are_the_definitions_to_their_own_rounding(n, inputs, outputs, dtype):
    torch = torch_()
    dy = normal(n, n, outputs, dtype=dtype, scale=0.01)
    dy[:, ::7] *= 2.0**-9
    dy[::3, outputs // 2] *= 200.0
    w = normal(inputs, outputs, inputs, scale=inputs**-0.5)
    wq, ws = codes64(w)
    dx = vq.QuantizedMatrix.fit(w, gradient=True).input_gradient(dy)
    want, off = limits(dy, wq, ws)
    tiny = 2.0**-24 if dtype == "float16" else 2.0**-133
    limit = torch.finfo(dx.dtype).eps / 2 * want.abs() * (1 + 2.0**-12) + off + tiny
    bad = ~((dx.double() - want).abs() <= limit)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("counts,front", [([33, 0, 31, 64, 65, 1, 0, 200, 32, 96], 3), ([1] * 40, 0), ([70, 20], 9)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_groups_of_any_rows(counts, front, dtype):
    """Tiles of one to sixty-four rows, the last of a group in front of the next one's."""
    torch = torch_()
    import numpy as np
    off = np.concatenate([[front], front + np.cumsum(counts)])
    n, outputs, inputs = int(off[-1]) + 5, 290, 300
    dy = softmax_rows(n, outputs, 3.0, dtype)
    w = normal(5, len(counts), outputs, inputs) + 0.2
    wq, ws = codes64(w)
    dx = vq.QuantizedMatrix.fit(w, gradient=True).input_gradient(dy, offsets=torch.from_numpy(off).cuda())
    tiny = 2.0**-24 if dtype == "float16" else 2.0**-133
    for g, (a, b) in enumerate(zip(off[:-1], off[1:])):
        want, lost = limits(dy[a:b], wq[g], ws[g])
        assert bool(((dx[a:b].double() - want).abs() <= torch.finfo(dx.dtype).eps / 2 * want.abs() * (1 + 2.0**-12) + lost + tiny).all()), g
    assert not dx[:front].any() and not dx[n - 5:].any()


@pytest.mark.parametrize("groups", [492, 493, 494, 495])
def test_as_many_groups_as_leave_room_for_five_stages_and_more(groups):
    torch = torch_()
    outputs, inputs = 700, 40  # (six stages' worth of width)
    w = normal(5, groups, outputs, inputs)
    wq, ws = codes64(w)
    off = torch.arange(groups + 1, device="cuda") * 3
    dy = softmax_rows(3 * groups, outputs, 1.0, "bfloat16")
    dx = vq.QuantizedMatrix.fit(w, gradient=True).input_gradient(dy, offsets=off)
    for g in range(0, groups, 41):
        want, lost = limits(dy[3 * g:3 * g + 3], wq[g], ws[g])
        assert bool(((dx[3 * g:3 * g + 3].double() - want).abs() <= 2.0**-8 * want.abs() * (1 + 2.0**-12) + lost).all()), g


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_the_widest_sums_of_digits_stay_in_32_bits(dtype):
    """131071 outputs of code -128, all but one with both last digits -128: 32640 = 65536 - 256 128 - 128 steps."""
    torch = torch_()
    outputs, part = 131071, 32640 / STEPS
    codes = torch.full((outputs, 2), -128, dtype=torch.int8, device="cuda")
    codes[:, 1] = 127
    scales = torch.full((outputs,), part, device="cuda")
    scales[77] = 1.0
    m = vq.QuantizedMatrix.from_parts(codes, scales, gradient=True)
    dx = m.input_gradient(torch.ones(3, outputs, device="cuda", dtype=getattr(torch, dtype)) / 1024)
    total = (1.0 + (outputs - 1) * part) / 1024
    want = torch.tensor([[-128.0 * total, 127.0 * total]] * 3, dtype=torch.float64, device="cuda")
    assert bool(((dx.double() - want).abs() <= want.abs() * (torch.finfo(dx.dtype).eps / 2 + 2.0**-18)).all())
