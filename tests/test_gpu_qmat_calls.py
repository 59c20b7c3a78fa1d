"""RowQuantizer and QuantizedMatrix as programs call them: refusals, streams, captured graphs, threads, contexts, the operators one after the other."""
import ctypes as C
import threading

import numpy as np
import pytest

import vq_b200 as vq
from tests.test_gpu_qmat import check, codes64, gen, gradient_limits, matrix64, normal, offsets_of, product64, torch_

pytestmark = pytest.mark.gpu


# ---- refusals --------------------------------------------------------------------------------------------------
def test_sizes_that_do_not_fit():
    torch = torch_()
    m = vq.QuantizedMatrix.fit(normal(1, 30, 20))
    with pytest.raises(vq.DimensionMismatch, match="expected 20, got 21"):
        m.product(normal(1, 4, 21))
    q, s = vq.RowQuantizer.fit().quantize(normal(1, 4, 21))
    with pytest.raises(vq.DimensionMismatch):
        m.product_of_codes(q, s)
    with pytest.raises(ValueError, match="scales must have shape"):
        m.product_of_codes(q[:, :20], s[:3])
    with pytest.raises(ValueError, match="bias must have shape"):
        m.product(normal(1, 4, 20), normal(1, 31))
    with pytest.raises(ValueError, match="must be int8"):
        m.product_of_codes(q.float(), s)
    with pytest.raises(vq.InvalidParameter, match="without its gradient"):
        m.input_gradient(normal(1, 4, 30, dtype="float16"))
    m = vq.QuantizedMatrix.fit(normal(1, 30, 20), gradient=True)
    with pytest.raises(vq.DimensionMismatch, match="expected 30, got 20"):
        m.input_gradient(normal(1, 4, 20, dtype="float16"))
    with pytest.raises(vq.BackendError, match="f16 or bf16"):
        m.input_gradient(normal(1, 4, 30))
    with pytest.raises(ValueError, match="dy's dtype"):
        m.input_gradient(normal(1, 4, 30, dtype="float16"), out=torch.empty(4, 20, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="out must be"):
        m.product(normal(1, 4, 20), out=torch.empty(4, 29, device="cuda"))
    with pytest.raises(ValueError, match="out must be"):
        m.product(normal(1, 4, 20), out=np.empty((4, 30), np.float32))
    with pytest.raises(ValueError, match="another dtype"):
        m.product(normal(1, 4, 20), dtype=torch.float16, out=torch.empty(4, 30, device="cuda"))


def test_groups_that_do_not_fit():
    m = vq.QuantizedMatrix.fit(normal(1, 3, 30, 20))
    x = normal(1, 10, 20)
    with pytest.raises(ValueError, match="needs offsets"):
        m.product(x)
    with pytest.raises(ValueError, match="offsets must have shape"):
        m.product(x, offsets=[0, 5, 10])
    for bad in ([0, 5, 4, 10], [-1, 2, 3, 4], [0, 1, 2, 11]):
        with pytest.raises(vq.InvalidParameter, match="ascend"):
            m.product(x, offsets=bad)
    with pytest.raises(vq.EmptyInput):
        vq.QuantizedMatrix.fit(np.zeros((0, 4), np.float32))
    with pytest.raises(vq.EmptyInput):
        vq.QuantizedMatrix.fit(np.zeros((3, 0, 4), np.float32))
    with pytest.raises(vq.EmptyInput):
        vq.RowQuantizer.fit().quantize(np.zeros((3, 0), np.float32))


def test_limits():
    torch = torch_()
    with pytest.raises(vq.BackendError, match="131071 inputs"):
        vq.QuantizedMatrix.from_parts(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"))
    with pytest.raises(vq.BackendError, match="131071 outputs"):
        vq.QuantizedMatrix.from_parts(torch.zeros(131072, 1, dtype=torch.int8, device="cuda"), torch.ones(131072, device="cuda"), gradient=True)
    with pytest.raises(vq.BackendError, match="1024 groups"):
        vq.QuantizedMatrix.from_parts(torch.zeros(1025, 1, 1, dtype=torch.int8, device="cuda"), torch.ones(1025, 1, device="cuda"))


def test_pointers_that_are_not_aligned_to_their_values(ctx):
    torch = torch_()
    m = vq.QuantizedMatrix.fit(normal(1, 30, 20), ctx=ctx)
    x, y = torch.zeros(1000, device="cuda"), torch.zeros(1000, device="cuda")
    lib, h = ctx._L, m._h
    p = lambda t, b=0: C.c_void_p(t.data_ptr() + b)  # noqa: E731
    assert lib.vqb_qmat_product(h, p(x, 2), 0, 4, 20, 20, None, None, p(y), 0, 30, 0) == 90
    assert lib.vqb_qmat_product(h, p(x, 1), 2, 4, 20, 20, None, None, p(y), 0, 30, 0) == 90
    assert lib.vqb_qmat_product(h, p(x), 0, 4, 20, 20, None, None, p(y, 2), 0, 30, 0) == 90
    assert lib.vqb_qmat_product(h, p(x), 0, 4, 20, 20, None, p(y, 2), p(y), 0, 30, 0) == 90
    assert lib.vqb_qmat_product(h, p(x), 3, 4, 20, 20, None, None, p(y), 0, 30, 0) == 90
    assert lib.vqb_qmat_product(h, p(x), 0, 4, 20, 19, None, None, p(y), 0, 30, 0) == 90
    assert lib.vqb_qmat_product(h, p(x), 0, 4, 20, 20, None, None, p(y), 0, 29, 0) == 90
    assert lib.vqb_qmat_product(h, p(x), 0, 4, 20, 20, None, None, p(y), 0, 30, 8) == 90
    assert lib.vqb_qmat_product(h, p(x), 0, 4, 20, 20, p(y, 4), None, p(y), 0, 30, 0) == 90
    assert lib.vqb_row_quantize(ctx.handle, p(x), 0, 4, 20, 20, p(y), 19, p(y)) == 90
    assert lib.vqb_row_quantize(ctx.handle, p(x), 0, 1 << 30, 20, 20, p(y), 20, p(y)) == 103
    torch.cuda.synchronize()
    assert not y.any()


@pytest.mark.parametrize("bad", [[-5, 10**9, 3, 7], [40, 30, 20, 10], [0, 40, 0, 40], [2**62, -(2**62), 2**62, 0]])
def test_offsets_on_the_gpu_that_do_not_ascend_touch_nothing_else(bad):
    torch = torch_()
    m, wq, ws = matrix64(normal(1, 3, 30, 40), gradient=True)
    x = normal(1, 40, 40, dtype="float16")
    room = torch.full((60, 40), 7.0, device="cuda", dtype=torch.float16)
    m.product(x, offsets=torch.tensor(bad, device="cuda"), out=room[10:50, :30])
    m.input_gradient(x[:, :30], offsets=torch.tensor(bad, device="cuda"), out=room[10:50])
    torch.cuda.synchronize()
    assert bool((room[:10] == 7).all()) and bool((room[50:] == 7).all())
    off = np.array([0, 10, 20, 40])  # (and the next call is right)
    want, size, _ = product64(*codes64(x), wq, ws, None, off)
    check(m.product(x, offsets=off), want, size)


# ---- one after the other ---------------------------------------------------------------------------------------
def test_experts_of_tokens_and_back():
    """Tokens are quantized once, gathered by expert, go through two products with experts' matrices and a dense one, and the gradient comes back."""
    torch = torch_()
    n, width, hidden, experts = 200, 96, 160, 6
    x = normal(1, n, width, dtype="bfloat16")
    expert = torch.randint(0, experts, (n,), generator=gen(2), device="cuda")
    order = torch.argsort(expert, stable=True)
    off = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.bincount(expert, minlength=experts).cumsum(0)])
    up, down, head = normal(3, experts, hidden, width, scale=0.1), normal(4, experts, width, hidden, scale=0.1), normal(5, 300, width, scale=0.1)
    (u, uq, us), (d, dq, ds), (h, hq, hs) = matrix64(up, True), matrix64(down, True), matrix64(head, True)
    q, s = vq.RowQuantizer.fit().quantize(x)
    a = u.product_of_codes(q[order], s[order], offsets=off, dtype=torch.bfloat16)
    b = d.product(torch.relu(a), offsets=off)
    y = torch.empty_like(b)
    y[order] = b
    logits = h.product(y, dtype=torch.float32)
    o = off.cpu().numpy()
    q64, s64 = codes64(x)
    want, size, _ = product64(q64[order], s64[order], uq, us, None, o)
    check(a, want, size)
    want, size, _ = product64(*codes64(torch.relu(a)), dq, ds, None, o)
    check(b, want, size)
    want, size, _ = product64(*codes64(y), hq, hs)
    check(logits, want, size)
    dlogits = normal(6, n, 300, dtype="bfloat16")
    dy = h.input_gradient(dlogits)
    want, size, extra, _ = gradient_limits(dlogits, hq, hs)
    check(dy, want, size, extra)
    da = d.input_gradient(dy[order], offsets=off) * (a > 0)
    dx = u.input_gradient(da, offsets=off)
    want, size, extra, _ = gradient_limits(da, uq, us, o)
    check(dx, want, size, extra)


def test_the_same_call_gives_the_same_bits():
    torch = torch_()
    for n, k, o in [(1, 4096, 4096), (16, 1000, 4096), (64, 4096, 512), (700, 500, 300)]:
        m = vq.QuantizedMatrix.fit(normal(1, o, k), gradient=True)
        x, dy = normal(2, n, k, dtype="bfloat16"), normal(3, n, o, dtype="bfloat16")
        y, dx = m.product(x), m.input_gradient(dy)
        for _ in range(5):
            assert torch.equal(m.product(x), y) and torch.equal(m.input_gradient(dy), dx)


def test_plain_kernels_agree_with_the_tensor_cores():
    """VQB_NO_TENSOR=1 is read when a context is made."""
    import os
    torch = torch_()
    os.environ["VQB_NO_TENSOR"] = "1"
    try:
        plain = vq.Context(0)
    finally:
        del os.environ["VQB_NO_TENSOR"]
    w, off = normal(1, 4, 200, 130), offsets_of([50, 0, 120, 33], 3)
    a, b = vq.QuantizedMatrix.fit(w, gradient=True), vq.QuantizedMatrix.fit(w, gradient=True, ctx=plain)
    x, dy = normal(2, 210, 130, dtype="float16"), normal(3, 210, 200, dtype="float16")
    assert np.array_equal(a.codes, b.codes) and np.array_equal(a.scales, b.scales)
    assert torch.equal(a.product(x, offsets=off), b.product(x, offsets=off))
    assert torch.equal(a.input_gradient(dy, offsets=off), b.input_gradient(dy, offsets=off))


# ---- streams, graphs, threads, contexts ------------------------------------------------------------------------
def calls(seed, n, k, o, groups=0):
    torch = torch_()
    w = normal(seed, *((groups, o, k) if groups else (o, k)))
    m = vq.QuantizedMatrix.fit(w, gradient=True)
    x, dy = normal(seed + 1, n, k, dtype="bfloat16"), normal(seed + 2, n, o, dtype="bfloat16")
    off = torch.from_numpy(np.linspace(0, n, groups + 1).astype(np.int64)).cuda() if groups else None
    return lambda: (m.product(x, offsets=off), m.input_gradient(dy, offsets=off), *vq.RowQuantizer.fit().quantize(x)), (x, dy)


SHAPES = [(1, 2048, 512, 0), (12, 500, 640, 0), (80, 4096, 300, 0), (900, 333, 450, 0), (300, 256, 200, 5)]


@pytest.mark.parametrize("shape", SHAPES)
def test_captured_calls_replay_with_new_values(shape):
    torch = torch_()
    call, (x, dy) = calls(1, *shape)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in (5, 6):
        x.copy_(normal(seed, *x.shape)), dy.copy_(normal(seed + 9, *dy.shape))
        want = [t.clone() for t in call()]
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_graphs_and_eager_calls_side_by_side():
    torch = torch_()
    made = [calls(10 * i, *SHAPES[i]) for i in range(5)]
    want = [[t.clone() for t in call()] for call, _ in made]
    graphs, outs = [], []
    for call, _ in made[1:4]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call())
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    eager = []
    for _ in range(30):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[3]):
            eager.append([c() for c, _ in (made[0], made[4])])
    torch.cuda.synchronize()
    for got, w in zip(outs, want[1:4]):
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    for first, last in eager:
        assert all(torch.equal(a, b) for a, b in zip((*first, *last), (*want[0], *want[4])))


def test_calls_follow_what_wrote_their_rows_and_what_reads_their_results():
    """No waiting in between: on a side stream, rows are written by the kernel directly before and results read by the one directly after."""
    torch = torch_()
    m, wq, ws = matrix64(normal(1, 700, 512))
    side = torch.cuda.Stream()
    src = [normal(20 + i, 256, 512, dtype="bfloat16") for i in range(4)]
    want = [m.product(s) for s in src]
    x, y = torch.empty_like(src[0]), torch.empty_like(want[0])
    got = []
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for i in range(40):
            x.copy_(src[i % 4])
            m.product(x, out=y)
            got.append(y.clone())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 4]) for i, g in enumerate(got))


def test_a_matrix_made_on_one_stream_is_used_on_another_and_dropped():
    torch = torch_()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x = normal(1, 64, 1024, dtype="float16")
    for i in range(6):
        w = normal(30 + i, 512, 1024)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            m = vq.QuantizedMatrix.fit(w)
        with torch.cuda.stream(b):
            y = m.product(x)
            del m
        torch.cuda.synchronize()
        want, size, _ = product64(*codes64(x), *(t[None] for t in codes64(w)))
        check(y, want, size)


def test_a_matrix_is_not_made_inside_a_capture():
    torch = torch_()
    w, x = normal(1, 40, 64), normal(2, 20, 64)
    m = vq.QuantizedMatrix.fit(w)
    want = m.product(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(vq.BackendError, match="captured"):
            vq.QuantizedMatrix.fit(w)
        y = m.product(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_threads_and_contexts():
    torch = torch_()
    other = vq.Context(0)
    w = normal(1, 300, 700)
    ms = [vq.QuantizedMatrix.fit(w, gradient=True), vq.QuantizedMatrix.fit(w, gradient=True, ctx=other)]
    xs = [normal(40 + i, n, 700, dtype="float16") for i, n in enumerate((1, 9, 130, 600))]
    dys = [normal(50 + i, n, 300, dtype="float16") for i, n in enumerate((1, 9, 130, 600))]
    want = [(ms[0].product(x), ms[0].input_gradient(dy)) for x, dy in zip(xs, dys)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                m = ms[i % 2]
                y, dx = m.product(xs[i]), m.input_gradient(dys[i])
                torch.cuda.current_stream().synchronize()
                if not (torch.equal(y, want[i][0]) and torch.equal(dx, want[i][1])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong


def test_the_other_quantizers_beside_products():
    """One context's scratch, tensor memory and streams, used in turn."""
    torch = torch_()
    from vq_b200 import synth
    pq = vq.ProductQuantizer.from_codebooks(synth.uniform01(16 * 256, 8, 3).reshape(16, 256, 8), vq.Distance.Euclidean)
    rows = torch.from_numpy(synth.uniform01(20_000, 128, 9)).cuda()
    m = vq.QuantizedMatrix.fit(normal(1, 512, 128), gradient=True)
    codes, y, dx = pq.quantize(rows, return_codes=True)[1].clone(), m.product(rows), m.input_gradient(normal(2, 500, 512, dtype="bfloat16"))
    for _ in range(10):
        c2, y2, d2 = pq.quantize(rows, return_codes=True)[1], m.product(rows), m.input_gradient(normal(2, 500, 512, dtype="bfloat16"))
        assert torch.equal(c2, codes) and torch.equal(y2, y) and torch.equal(d2, dx)


# ---- large ones ------------------------------------------------------------------------------------------------
def test_results_beyond_32_bits():
    """2.4e9 results; the last rows are where they belong."""
    torch = torch_()
    n, k, o = 40_003, 32, 60_000
    x, w = normal(1, n, k, dtype="bfloat16"), normal(2, o, k)
    m, wq, ws = matrix64(w)
    y = m.product(x)
    pick = torch.tensor([0, 1, 255, 256, 35_791, 35_792, n - 2, n - 1], device="cuda")
    q, s = codes64(x[pick])
    want, size, _ = product64(q, s, wq, ws)
    check(y[pick], want, size)


@pytest.mark.parametrize("lowest", [-15000, 0])
def test_rows_beyond_32_bits(lowest):
    """Any bits (negative ones: nearly every row holds a NaN), and finite values."""
    torch = torch_()
    n, k = 1_100_000, 2048
    x = torch.empty(n, k, device="cuda", dtype=torch.bfloat16)
    x.view(torch.int16).random_(lowest, 15000, generator=gen(1))
    q, s = vq.RowQuantizer.fit().quantize(x)
    for at in (0, n // 2 - 1, n - 300):
        want_q, want_s = codes64(x[at:at + 300])
        assert torch.equal(q[at:at + 300].double(), want_q) and torch.equal(torch.nan_to_num(s[at:at + 300].double(), -1.0), torch.nan_to_num(want_s, -1.0))


def test_work_from_before_a_captured_call_is_waited_for_after_it():
    """A long call on one stream, a captured one, and a call on a third stream, which uses the first one's scratch."""
    torch = torch_()
    from vq_b200 import synth
    books = [synth.uniform01(16 * 256, 8, 3 + i).reshape(16, 256, 8) for i in range(2)]
    a, b = (vq.ProductQuantizer.from_codebooks(c, vq.Distance.Euclidean) for c in books)
    x = torch.from_numpy(synth.uniform01(300_000, 128, 9)).cuda()
    small = x[:5_000].contiguous()
    m, rows = vq.QuantizedMatrix.fit(normal(1, 64, 128)), normal(2, 40, 128)
    want_a, want_b, want_y = a.quantize(x, return_codes=True)[1].clone(), b.quantize(small, return_codes=True)[1].clone(), m.product(rows).clone()
    first, third = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        got = []
        with torch.cuda.stream(first):
            got.append(a.quantize(x, return_codes=True)[1])
            got.append(a.quantize(x, return_codes=True)[1])
        capture = torch.cuda.Stream()
        with torch.cuda.stream(capture):
            graph.capture_begin()
            y = m.product(rows)
            graph.capture_end()
        with torch.cuda.stream(third):
            got.append(b.quantize(small, return_codes=True)[1])
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want_a) and torch.equal(got[1], want_a) and torch.equal(got[2], want_b) and torch.equal(y, want_y)


def test_a_matrix_dropped_inside_a_capture_leaves_the_capture_alone():
    """As a garbage collector may do it: its memory goes back after the capture."""
    torch = torch_()
    w, x = normal(1, 4096, 4096), normal(2, 20, 4096)
    keep = vq.QuantizedMatrix.fit(normal(3, 40, 4096))
    want = keep.product(x)
    for _ in range(20):
        drop = vq.QuantizedMatrix.fit(w, gradient=True)
        drop.product(x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = keep.product(x)
            del drop
            z = keep.product(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(z, want) and torch.equal(keep.product(x), want)
