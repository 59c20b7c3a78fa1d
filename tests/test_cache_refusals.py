"""What QuantizedCache refuses, and how it takes its arguments, before anything reaches the GPU."""
import types

import numpy as np
import pytest

import vq_b200 as vq
from tests.test_overlapped_launches import _functions, _taken_for_invariant
from vq_b200 import _lib

HERE = types.SimpleNamespace(device=0)


def test_null_handles_are_rejected():
    lib = _lib.load()
    assert lib.vqb_cache_create(None, 1, 1, 1, None) == 90
    assert lib.vqb_cache_from_parts(None, None, None, None, None, 1, 1, 1, None) == 90
    assert lib.vqb_cache_shape(None, None, None, None) == 90
    assert lib.vqb_cache_parts(None, None, None, None, None) == 90
    assert lib.vqb_cache_write(None, None, 0, 0, None, 0, 0, 0, 0, 0, 0, None, 0, 0, 0, None, None) == 90
    assert lib.vqb_cache_read(None, None, None, 0, 0, None, 0, 0, 0, None, None) == 90
    assert lib.vqb_cache_attend(None, None, 0, 0, 0, 0, 0, 0, None, 0, 0, 0, None, None, 1.0, 0, 0, None, 0, 0, 0) == 90
    assert lib.vqb_cache_destroy(None) == 0


def heads(*shape, dtype=np.float32):
    return vq._Heads(np.zeros(shape, dtype), HERE, "queries")


def test_rows_of_heads():
    x = heads(3, 4, 5)
    assert (x.n, x.heads, x.dim, x.ld, x.head_ld, x.type) == (3, 4, 5, 20, 5, 0)
    assert heads(3, 4, 5, dtype=np.float64).type == 0 and heads(3, 4, 5, dtype=np.float16).type == 1
    for shape in ((3, 4), (3,), (1, 2, 3, 4)):
        with pytest.raises(ValueError, match="rows x heads x width"):
            heads(*shape)


def test_strided_rows_are_taken_as_they_are(monkeypatch):
    import torch
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 0, raising=False)
    whole = torch.zeros(6, 9, 16, dtype=torch.float16)

    def seen(t):
        x = vq._Heads(t, HERE, "queries")
        return x.ptr - t.data_ptr(), x.ld, x.head_ld

    assert seen(whole[:, 2:5]) == (0, 144, 16)
    assert seen(whole[:, :, 4:12]) == (0, 144, 16)
    assert seen(whole.transpose(0, 1)) == (0, 16, 144)
    assert seen(whole[:, 3:4, 8:]) == (0, 144, 8)  # one head: the next one is nowhere
    for t in (whole[:, :, ::2], whole[:1, :1].expand(4, 3, 16), torch.as_strided(whole, (3, 3, 16), (16, 16, 1))):
        shift, ld, head_ld = seen(t)
        assert shift != 0 and (ld, head_ld) == (t.shape[1] * t.shape[2], t.shape[2])
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        seen(whole.double())
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 1)
    with pytest.raises(ValueError, match="cuda:1"):
        seen(whole)


def test_rows_that_ask_for_a_gradient():
    import torch
    x = torch.zeros(2, 3, 4, requires_grad=True)
    with pytest.raises(ValueError, match="keys requires a gradient"):
        vq._Heads(x, HERE, "keys")
    with torch.no_grad():
        assert vq._Heads(x, HERE, "keys").n == 2


@pytest.mark.parametrize("out", [np.zeros((3, 4, 5), np.float32), np.zeros((3, 4, 6), np.float16), np.zeros((3, 4, 10), np.float16)[:, :, ::2], np.zeros((5, 4, 3), np.float16).T,
                                 np.broadcast_to(np.zeros((1, 4, 5), np.float16), (3, 4, 5)), np.zeros((3, 4, 5), ">f2"), [0.0]])
def test_results_of_another_form(out):
    with pytest.raises(ValueError, match="out must be"):
        vq._heads_result(heads(3, 4, 5, dtype=np.float16), out)


def test_results():
    x = heads(3, 4, 5, dtype=np.float16)
    room = np.zeros((3, 6, 9), np.float16)
    a, ptr, ld, head_ld = vq._heads_result(x, room[:, 1:5, 2:7])
    assert (ptr, ld, head_ld) == (room.ctypes.data + 2 * 11, 54, 9)
    a, ptr, ld, head_ld = vq._heads_result(x, np.zeros((4, 3, 5), np.float16).transpose(1, 0, 2))
    assert (ld, head_ld) == (5, 15)
    assert vq._heads_result(x, None)[0].shape == (3, 4, 5)


def test_tables_and_lengths():
    x = heads(3, 4, 5)
    a, _, shape, ld = vq._numbers([[1, 2, 3], [4, 5, -1]], x, "table", 2)
    assert a.dtype == np.int32 and shape == (2, 3) and ld == 3
    assert vq._numbers(np.zeros((0, 3), np.int64), x, "table", 2)[2] == (0, 3)
    with pytest.raises(ValueError, match="whole numbers"):
        vq._numbers(np.zeros((2, 3)), x, "table", 2)
    with pytest.raises(ValueError, match="32 bits"):
        vq._numbers([2**31], x, "lengths", 1)
    with pytest.raises(ValueError, match="sequences x columns"):
        vq._numbers([1, 2], x, "table", 2)
    with pytest.raises(ValueError, match="one number a sequence"):
        vq._numbers([[1, 2]], x, "lengths", 1)


def test_tables_on_the_gpu(monkeypatch):
    import torch
    x = heads(3, 4, 5)
    x.cuda, x.keep = True, torch.zeros(1)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    wide = torch.zeros(4, 10, dtype=torch.int32)
    v, ptr, shape, ld = vq._numbers(wide[:, 2:7], x, "table", 2)
    assert ptr == wide.data_ptr() + 8 and tuple(shape) == (4, 5) and ld == 10
    v, ptr, shape, ld = vq._numbers(wide[:1, :3].expand(4, 3), x, "table", 2)
    assert ld == 3 and v.is_contiguous()
    assert vq._numbers(wide[:, ::2], x, "table", 2)[3] == 5
    with pytest.raises(ValueError, match="int32"):
        vq._numbers(wide.long(), x, "table", 2)


def test_kernels_on_the_cache_wait_before_they_read_and_take_nothing_for_invariant():
    """They may start before the kernel in front of them ends; one that left without waiting would let the next one start before the work in front of both has ended."""
    seen = set()
    for name, params, body in _functions():
        if "cache_is_there();" in body:
            seen.add(name)
            assert not _taken_for_invariant(params, body), name
            assert "return;" not in body[: body.index("cache_is_there();")], name
    assert {"cache_write_kernel", "cache_read_kernel", "cache_pages_kernel"} <= seen
