"""vqb_qmat_parts to memory on the GPU: the copy may still be waiting when the matrix is dropped on another stream."""
import ctypes as C

import pytest

import vq_b200 as vq
from tests.test_gpu_qmat import normal, torch_

pytestmark = pytest.mark.gpu


def test_codes_that_are_still_being_copied_when_the_matrix_is_dropped(ctx):
    torch = torch_()
    weights, other = normal(1, 2048, 4100), normal(2, 2048, 4100)
    want = torch.from_numpy(vq.QuantizedMatrix.fit(weights, ctx=ctx).codes).cuda()
    user, stream = torch.cuda.Stream(), torch.cuda.Stream()
    busy = normal(3, 8192, 8192, dtype="bfloat16")
    codes = torch.empty_like(want)
    for _ in range(4):
        m = vq.QuantizedMatrix.fit(weights, ctx=ctx)
        torch.cuda.synchronize()
        ctx.synchronize()
        with torch.cuda.stream(user):
            for _ in range(6):
                busy @ busy
            ctx.set_stream(user.cuda_stream)
            assert ctx._L.vqb_qmat_parts(m._h, C.c_void_p(codes.data_ptr()), None) == 0
        ctx.set_stream(stream.cuda_stream)
        del m
        with torch.cuda.stream(stream):
            vq.QuantizedMatrix.fit(other, ctx=ctx)
        torch.cuda.synchronize()
        assert torch.equal(codes, want)
    ctx.set_stream(None)
