"""What RowQuantizer and QuantizedMatrix refuse before anything reaches the GPU."""
import types

import numpy as np
import pytest

import vq_b200 as vq
from vq_b200 import _lib

HERE = types.SimpleNamespace(device=0)


def test_null_handles_are_rejected():
    lib = _lib.load()
    assert lib.vqb_row_quantize(None, None, 0, 0, 1, 1, None, 1, None) == 90
    assert lib.vqb_qmat_fit(None, None, 0, 1, 1, 1, 0, None) == 90
    assert lib.vqb_qmat_from_parts(None, None, None, 1, 1, 1, 0, None) == 90
    assert lib.vqb_qmat_shape(None, None, None, None) == 90
    assert lib.vqb_qmat_parts(None, None, None) == 90
    assert lib.vqb_qmat_product(None, None, 0, 0, 0, 0, None, None, None, 0, 0, 0) == 90
    assert lib.vqb_qmat_product_codes(None, None, 0, None, 0, 0, None, None, None, 0, 0, 0) == 90
    assert lib.vqb_qmat_input_gradient(None, None, 1, 0, 0, 0, None, None, 0, 0) == 90
    assert lib.vqb_qmat_destroy(None) == 0


def rows(*shape):
    return vq._Values(np.zeros(shape, np.float32), HERE)


def test_rows():
    assert (rows(3, 5).n, rows(3, 5).dim, rows(5).single) == (3, 5, True)
    with pytest.raises(ValueError, match="vector or a matrix"):
        rows(2, 3, 4)
    with pytest.raises(ValueError, match="must be int8"):
        vq._Values(np.zeros((2, 3), np.uint8), HERE, "codes", integers=True)
    assert vq._Values(np.zeros((2, 3)), HERE).type == 0  # (float64 becomes float32)
    assert vq._Values(np.zeros((2, 3), np.float16), HERE).type == 1


def test_rows_on_another_device(monkeypatch):
    import torch
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda self: 1)
    with pytest.raises(ValueError, match="cuda:1"):
        vq._Values(torch.zeros(2, 3), HERE)


@pytest.mark.parametrize("out", [np.zeros((3, 7), np.float32), np.zeros((3, 6), np.float64), np.zeros((3, 6), np.int8), np.zeros((6, 3), np.float32).T, np.zeros((3, 12), np.float32)[:, ::2],
                                 np.broadcast_to(np.zeros(6, np.float32), (3, 6)), [0.0] * 18])
def test_results_of_another_form(out):
    with pytest.raises((ValueError, AttributeError)):
        vq._result(rows(3, 5), 6, None, out)


def test_results():
    room = np.zeros((3, 9), np.float16)
    a, ptr, kind, ld = vq._result(rows(3, 5), 6, None, room[:, 2:8])
    assert (kind, ld, ptr) == (1, 9, room.ctypes.data + 4)
    assert vq._result(rows(3, 5), 6, np.float16, None)[0].shape == (3, 6)
    with pytest.raises(ValueError, match="another dtype"):
        vq._result(rows(3, 5), 6, np.float32, room[:, :6])
    for name in ("bfloat16", "float64", "int8"):
        with pytest.raises(ValueError, match="not offered"):
            vq._result(rows(3, 5), 6, name, None)


def test_what_goes_with_the_rows():
    x = rows(3, 5)
    with pytest.raises(ValueError, match="offsets must have shape"):
        vq._beside(np.zeros(4), x, "int64", (3,), "offsets")
    with pytest.raises(ValueError, match="bias must have shape"):
        vq._beside(np.zeros((2, 5)), x, "float32", (5,), "bias")
    v, _ = vq._beside([1, 2, 3], x, "int64", (3,), "offsets")
    assert v.dtype == np.int64


def test_weights():
    for w in (np.zeros(4, np.float32), np.zeros((1, 2, 3, 4), np.float32), [[1.0]]):
        with pytest.raises(ValueError, match="outputs x inputs"):
            vq.QuantizedMatrix._flat(w)
    flat, (groups, outputs) = vq.QuantizedMatrix._flat(np.zeros((2, 3, 4), np.float32))
    assert flat.shape == (6, 4) and (groups, outputs) == (2, 3)
    assert vq.QuantizedMatrix._flat(np.zeros((2, 0, 4), np.float32))[0].shape == (0, 4)
