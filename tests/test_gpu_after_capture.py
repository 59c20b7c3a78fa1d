"""Calls on the stream of a captured one, after the capture, while work of another stream from before it is still running."""
import gc

import numpy as np
import pytest

import vq_b200 as vq
from tests.test_gpu_qmat import normal, torch_

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def collected():
    """A graph that the collector finds inside a capture would end the capture."""
    gc.collect()
    gc.disable()
    yield
    gc.enable()
    gc.collect()


def captured_on(stream, call):
    """The graph of a call, captured without waiting for the device (as torch.cuda.graph does)."""
    torch = torch_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        graph.capture_begin()
        result = call()
        graph.capture_end()
    return graph, result


def test_a_matrix_that_another_stream_still_reads_is_dropped_and_its_memory_used_again():
    torch = torch_()
    n, width = 2048, 8192
    small, rows = vq.QuantizedMatrix.fit(normal(1, 64, 128)), normal(2, 40, 128)
    want_small = small.product(rows)
    x = normal(3, n, width, dtype="bfloat16")
    weights, other = normal(4, width, width, dtype="bfloat16"), normal(5, width, width, dtype="bfloat16")
    m = vq.QuantizedMatrix.fit(weights)
    want, want_other = m.product(x), vq.QuantizedMatrix.fit(other).product(x)
    user, stream = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        m = vq.QuantizedMatrix.fit(weights)
        torch.cuda.synchronize()
        with torch.cuda.stream(user):
            got = [m.product(x) for _ in range(20)]
        graph, y = captured_on(stream, lambda: small.product(rows))
        with torch.cuda.stream(stream):
            del m
            again = vq.QuantizedMatrix.fit(other)
            z = again.product(x)
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got) and torch.equal(z, want_other) and torch.equal(y, want_small)


def test_a_matrix_dropped_inside_the_capture_goes_back_after_the_work_of_another_stream():
    torch = torch_()
    n, width = 2048, 8192
    small, rows = vq.QuantizedMatrix.fit(normal(1, 64, 128)), normal(2, 40, 128)
    x = normal(3, n, width, dtype="bfloat16")
    weights, other = normal(4, width, width, dtype="bfloat16"), normal(5, width, width, dtype="bfloat16")
    want = vq.QuantizedMatrix.fit(weights).product(x)
    user, stream = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        held = [vq.QuantizedMatrix.fit(weights)]
        torch.cuda.synchronize()
        with torch.cuda.stream(user):
            got = [held[0].product(x) for _ in range(20)]
        graph, _ = captured_on(stream, lambda: (small.product(rows), held.clear()))
        with torch.cuda.stream(stream):
            small.product(rows)
            vq.QuantizedMatrix.fit(other)
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got)


def test_the_scratch_that_another_stream_still_uses():
    torch = torch_()
    from vq_b200 import synth
    books = [synth.uniform01(16 * 256, 8, 3 + i).reshape(16, 256, 8) for i in range(2)]
    a, b = (vq.ProductQuantizer.from_codebooks(c, vq.Distance.Euclidean) for c in books)
    x = torch.from_numpy(synth.uniform01(300_000, 128, 9)).cuda()
    few = x[:5_000].contiguous()
    m, rows = vq.QuantizedMatrix.fit(normal(1, 64, 128)), normal(2, 40, 128)
    want_a, want_b, want_y = a.quantize(x, return_codes=True)[1].clone(), b.quantize(few, return_codes=True)[1].clone(), m.product(rows).clone()
    first, stream = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        torch.cuda.synchronize()
        with torch.cuda.stream(first):
            got = [a.quantize(x, return_codes=True)[1] for _ in range(3)]
        graph, y = captured_on(stream, lambda: m.product(rows))
        with torch.cuda.stream(stream):
            other = b.quantize(few, return_codes=True)[1]
            graph.replay()
        with torch.cuda.stream(first):
            got.append(a.quantize(x, return_codes=True)[1])
        torch.cuda.synchronize()
        assert all(torch.equal(g, want_a) for g in got) and torch.equal(other, want_b) and torch.equal(y, want_y)
    assert np.array_equal(m.codes.shape, (64, 128))
