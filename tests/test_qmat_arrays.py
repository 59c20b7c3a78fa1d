"""Arrays of other byte orders and types than the library's.  No GPU is reached."""
import types

import numpy as np
import pytest

import vq_b200 as vq

HERE = types.SimpleNamespace(device=0)


@pytest.mark.parametrize("dtype,kind", [(">f4", 0), ("<f4", 0), (">f2", 1), ("<f2", 1), (">f8", 0)])
def test_rows_of_any_byte_order_keep_their_values(dtype, kind):
    x = np.array([[1.0, -2.5, 3.0], [0.25, 100.0, -7.0]])
    v = vq._Values(x.astype(dtype), HERE)
    assert np.array_equal(v.keep, x) and v.keep.dtype == (np.float32, np.float16)[kind] and v.type == kind


@pytest.mark.parametrize("dtype", [">f4", ">f2"])
def test_results_are_not_written_into_arrays_of_another_byte_order(dtype):
    x = vq._Values(np.zeros((3, 5), np.float32), HERE)
    with pytest.raises(ValueError, match="out must be"):
        vq._result(x, 6, None, np.zeros((3, 6), dtype))


@pytest.mark.parametrize("offsets", [[0.0, 2.5, 4.0], np.array([0.0, 2.0, 4.0]), np.array([False, True, True]), "torch"], ids=["list", "floats", "truth values", "torch"])
def test_offsets_that_are_not_whole_numbers_are_refused(offsets):
    if isinstance(offsets, str):
        import torch
        offsets = torch.tensor([0.0, 2.0, 4.0])
    x = vq._Values(np.zeros((4, 5), np.float32), HERE)
    with pytest.raises(ValueError, match="offsets must be whole numbers"):
        vq._beside(offsets, x, "int64", (3,), "offsets")


@pytest.mark.parametrize("dtype", [np.int64, np.int32, np.uint8, ">i8"])
def test_offsets_of_any_whole_type_are_taken(dtype):
    x = vq._Values(np.zeros((4, 5), np.float32), HERE)
    v, _ = vq._beside(np.array([0, 2, 4], dtype), x, "int64", (3,), "offsets")
    assert v.dtype == np.int64 and v.tolist() == [0, 2, 4]


def test_offsets_on_the_gpu_that_are_not_whole_numbers_are_refused(monkeypatch):
    import torch
    x = vq._Values(np.zeros((4, 5), np.float32), HERE)
    x.cuda, x.keep = True, torch.zeros(1)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    with pytest.raises(ValueError, match="offsets must be whole numbers"):
        vq._beside(torch.tensor([0.0, 2.5, 4.0]), x, "int64", (3,), "offsets")
    v, _ = vq._beside(torch.tensor([0, 2, 4], dtype=torch.int32), x, "int64", (3,), "offsets")
    assert v.dtype is torch.int64
