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
