"""Products record nothing for automatic differentiation: whatever requires a gradient is refused rather than losing it.  No GPU is reached but
by the last test, which trains as the class's description says."""
import types

import pytest
import torch

import vq_b200 as vq


class Reached(Exception):
    pass


def matrix():
    def reached(*_):
        raise Reached

    m = vq.QuantizedMatrix.__new__(vq.QuantizedMatrix)
    library = types.SimpleNamespace(vqb_qmat_product=None, vqb_qmat_product_codes=None, vqb_qmat_input_gradient=None)
    m._h, m._ctx, m._grouped, m._shape, m._call = None, types.SimpleNamespace(device=0, _L=library), False, (1, 4, 6), reached
    return m


ROWS, BIAS, CODES, SCALES, DY = torch.zeros(3, 6), torch.zeros(4), torch.zeros(3, 6, dtype=torch.int8), torch.ones(3), torch.zeros(3, 4, dtype=torch.float16)


def recorded(t):
    return t.clone().requires_grad_()


CALLS = {
    "rows": lambda m: m.product(recorded(ROWS)),
    "rows behind others": lambda m: m.product(recorded(ROWS) * 2.0),
    "bias": lambda m: m.product(ROWS, recorded(BIAS)),
    "out": lambda m: m.product(ROWS, out=recorded(torch.zeros(3, 4))),
    "scales": lambda m: m.product_of_codes(CODES, recorded(SCALES)),
    "bias of codes": lambda m: m.product_of_codes(CODES, SCALES, recorded(BIAS)),
    "dy": lambda m: m.input_gradient(recorded(DY)),
}


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS.keys())
def test_what_requires_a_gradient_is_refused(call):
    with pytest.raises(ValueError, match="requires a gradient.*detach"):
        call(matrix())


@pytest.mark.parametrize("name", ["rows", "rows behind others", "bias", "scales", "bias of codes", "dy"])
def test_nothing_is_refused_where_nothing_is_recorded(name):
    with torch.no_grad(), pytest.raises(Reached):
        CALLS[name](matrix())


def test_what_requires_none_is_taken():
    m = matrix()
    for call in (lambda: m.product(ROWS, BIAS), lambda: m.product(recorded(ROWS).detach()), lambda: m.product_of_codes(CODES, SCALES, BIAS), lambda: m.input_gradient(DY)):
        with pytest.raises(Reached):
            call()


@pytest.mark.gpu
def test_rows_in_front_of_a_matrix_are_trained_through_a_function():
    m = vq.QuantizedMatrix.fit(torch.randn(40, 24, device="cuda"), gradient=True)

    class Through(torch.autograd.Function):
        @staticmethod
        def forward(ctx, rows):
            return m.product(rows)

        @staticmethod
        def backward(ctx, dy):
            return m.input_gradient(dy)

    leaf = torch.randn(9, 24, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(ValueError, match="requires a gradient"):
        m.product(leaf)
    y = Through.apply(leaf * 2.0)
    dy = torch.randn_like(y)
    y.backward(dy)
    assert torch.equal(y, m.product(leaf.detach() * 2.0)) and torch.equal(leaf.grad, m.input_gradient(dy) * 2.0)
