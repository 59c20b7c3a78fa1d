"""Operands in host memory beside rows on the GPU: read by the end of the call whatever kind of memory they are in, and refused while a graph is captured."""
import ctypes as C
import gc

import numpy as np
import pytest

import vq_b200 as vq
from tests.test_gpu_qmat import normal, torch_

pytestmark = pytest.mark.gpu
N, INPUTS, OUTPUTS, GROUPS = 300, 256, 200, 3


@pytest.fixture(autouse=True)
def collected():
    """A graph that the collector finds inside a capture would end the capture."""
    gc.collect()
    gc.disable()
    yield
    gc.enable()
    gc.collect()


def operands(pinned, first):
    """(offsets, bias, scales); another set for the second `first`."""
    torch = torch_()
    offsets = torch.tensor([0, 10, 150, 300] if first else [0, 250, 260, 300])
    bias = normal(11 if first else 12, GROUPS, OUTPUTS).cpu()
    scales = normal(13 if first else 14, N).abs().cpu()
    return [t.pin_memory() if pinned else t for t in (offsets, bias, scales)]


@pytest.mark.parametrize("pinned", [False, True])
def test_operands_are_read_by_the_end_of_the_call(pinned):
    torch = torch_()
    m = vq.QuantizedMatrix.fit(normal(1, GROUPS, OUTPUTS, INPUTS), gradient=True)
    x, dy = normal(2, N, INPUTS, dtype="bfloat16"), normal(3, N, OUTPUTS, dtype="bfloat16")
    codes, _ = vq.RowQuantizer.fit().quantize(x)
    on_gpu = [t.cuda() for t in operands(False, True)]
    large, busy = vq.QuantizedMatrix.fit(normal(4, 8192, 8192)), normal(5, 8192, 8192, dtype="bfloat16")

    def calls(offsets, bias, scales):
        return m.product(x, bias, offsets=offsets), m.product_of_codes(codes, scales, bias, offsets=offsets), m.input_gradient(dy, offsets=offsets)

    want = calls(*on_gpu)
    for _ in range(5):
        given, others = operands(pinned, True), operands(False, False)
        torch.cuda.synchronize()
        for _ in range(10):  # (a few ms that the copies are behind)
            large.product(busy)
        got = calls(*given)
        for a, b in zip(given, others):
            a.copy_(b)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("n", [40, 5000])
def test_rows_in_page_locked_memory_are_read_by_the_end_of_the_call(n, ctx):
    """Through the C interface, which takes rows in host memory and results on the GPU."""
    torch = torch_()
    m = vq.QuantizedMatrix.fit(normal(1, OUTPUTS, INPUTS), ctx=ctx)
    x = normal(2, n, INPUTS)
    want = m.product(x)
    large, busy = vq.QuantizedMatrix.fit(normal(4, 8192, 8192), ctx=ctx), normal(5, 8192, 8192, dtype="bfloat16")
    y = torch.empty_like(want)
    for _ in range(3):
        given = x.cpu().pin_memory()
        torch.cuda.synchronize()
        for _ in range(10):
            large.product(busy)
        assert ctx._L.vqb_qmat_product(m._h, C.c_void_p(given.data_ptr()), 0, n, INPUTS, INPUTS, None, None, C.c_void_p(y.data_ptr()), 0, OUTPUTS, 0) == 0
        given.zero_()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("pinned", [False, True])
def test_operands_in_host_memory_are_not_captured(pinned):
    torch = torch_()
    m, one = vq.QuantizedMatrix.fit(normal(1, GROUPS, OUTPUTS, INPUTS), gradient=True), vq.QuantizedMatrix.fit(normal(6, OUTPUTS, INPUTS))
    x, dy = normal(2, N, INPUTS, dtype="bfloat16"), normal(3, N, OUTPUTS, dtype="bfloat16")
    codes, scales = vq.RowQuantizer.fit().quantize(x)
    offsets, bias, host_scales = operands(pinned, True)
    there, bias_there = offsets.cuda(), bias.cuda()
    want = m.product(x, bias_there, offsets=there)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for name, call in [("offsets", lambda: m.product(x, offsets=offsets)), ("bias", lambda: m.product(x, bias, offsets=there)), ("bias", lambda: one.product(x, bias[0])),
                           ("scales", lambda: one.product_of_codes(codes, host_scales)), ("offsets", lambda: m.input_gradient(dy, offsets=offsets))]:
            with pytest.raises(vq.BackendError, match=name + " is in host memory"):
                call()
        y = m.product(x, bias_there, offsets=there)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_rows_and_results_in_host_memory_are_not_captured(ctx):
    torch = torch_()
    m = vq.QuantizedMatrix.fit(normal(1, OUTPUTS, INPUTS), gradient=True, ctx=ctx)
    x = normal(2, N, INPUTS)
    want = m.product(x)
    host_x, host_y, host_q, host_s = np.zeros((N, INPUTS), np.float32), np.zeros((N, OUTPUTS), np.float32), np.zeros((N, INPUTS), np.int8), np.zeros(N, np.float32)
    q, s, y = torch.empty(N, INPUTS, dtype=torch.int8, device="cuda"), torch.empty(N, device="cuda"), torch.empty_like(want)
    there, here = (lambda t: C.c_void_p(t.data_ptr())), (lambda a: C.c_void_p(a.ctypes.data))
    graph = torch.cuda.CUDAGraph()
    lib, h = ctx._L, ctx.handle
    with torch.cuda.graph(graph):
        z = m.product(x)  # (the context is on the captured stream)
        assert lib.vqb_qmat_product(m._h, here(host_x), 0, N, INPUTS, INPUTS, None, None, there(y), 0, OUTPUTS, 0) == 103
        assert lib.vqb_qmat_product(m._h, there(x), 0, N, INPUTS, INPUTS, None, None, here(host_y), 0, OUTPUTS, 0) == 103
        assert lib.vqb_row_quantize(h, here(host_x), 0, N, INPUTS, INPUTS, there(q), INPUTS, there(s)) == 103
        assert lib.vqb_row_quantize(h, there(x), 0, N, INPUTS, INPUTS, here(host_q), INPUTS, there(s)) == 103
        assert lib.vqb_row_quantize(h, there(x), 0, N, INPUTS, INPUTS, there(q), INPUTS, here(host_s)) == 103
        assert lib.vqb_qmat_parts(m._h, here(np.zeros((OUTPUTS, INPUTS), np.int8)), None) == 103
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, want) and torch.equal(m.product(x), want)


@pytest.mark.parametrize("pinned", [False, True])
def test_a_matrix_of_weights_in_host_memory_is_refused_ahead_of_their_copy(pinned, ctx):
    torch = torch_()
    m, x = vq.QuantizedMatrix.fit(normal(1, OUTPUTS, INPUTS), ctx=ctx), normal(2, N, INPUTS)
    want = m.product(x)
    w, codes, scales = torch.zeros(64, 64), torch.zeros(64, 64, dtype=torch.int8), torch.zeros(64)
    if pinned:
        w, codes, scales = w.pin_memory(), codes.pin_memory(), scales.pin_memory()
    there = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    graph, made = torch.cuda.CUDAGraph(), C.c_void_p()
    with torch.cuda.graph(graph):
        y = m.product(x)  # (the context is on the captured stream)
        before = ctx.alloc_count()
        assert ctx._L.vqb_qmat_fit(ctx.handle, there(w), 0, 1, 64, 64, 0, C.byref(made)) == 103 and not made
        assert ctx._L.vqb_qmat_from_parts(ctx.handle, there(codes), there(scales), 1, 64, 64, 1, C.byref(made)) == 103 and not made
        assert ctx.alloc_count() == before, "memory was asked for inside the capture"
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(m.product(x), want)
