"""Operands that carry a tangent (torch's forward mode) are refused: the result would have none, and nobody would be told."""
import types

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward

import vq_b200 as vq
from tests.test_qmat_recorded import BIAS, CODES, DY, ROWS, SCALES, Reached, matrix


def dual(t):
    return forward.make_dual(t.clone(), torch.ones_like(t))


CALLS = {
    "rows": lambda m: m.product(dual(ROWS)),
    "rows behind others": lambda m: m.product(dual(ROWS) * 2.0),
    "bias": lambda m: m.product(ROWS, dual(BIAS)),
    "out": lambda m: m.product(ROWS, out=dual(torch.zeros(3, 4))),
    "scales": lambda m: m.product_of_codes(CODES, dual(SCALES)),
    "bias of codes": lambda m: m.product_of_codes(CODES, SCALES, dual(BIAS)),
    "dy": lambda m: m.input_gradient(dual(DY)),
    "keys": lambda m: vq._Heads(dual(torch.zeros(2, 3, 4)), types.SimpleNamespace(device=0), "keys"),
}


@pytest.mark.parametrize("recording", [True, False])
@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS.keys())
def test_what_carries_a_tangent_is_refused(call, recording):
    """Whether gradients are recorded or not: torch.no_grad does not end forward mode."""
    with forward.dual_level(), torch.set_grad_enabled(recording), pytest.raises(ValueError, match="carries a tangent.*detach"):
        call(matrix())


def test_what_carries_none_is_taken():
    m = matrix()
    with forward.dual_level():
        for call in (lambda: m.product(ROWS, BIAS), lambda: m.product(dual(ROWS).detach()), lambda: m.product(ROWS.numpy()), lambda: m.product_of_codes(CODES, SCALES, BIAS),
                     lambda: m.input_gradient(DY)):
            with pytest.raises(Reached):
                call()
        assert vq._Heads(dual(torch.zeros(2, 3, 4)).detach(), types.SimpleNamespace(device=0), "keys").n == 2


def test_nothing_is_refused_in_a_function_of_ones_own():
    """The forward method of a torch.autograd.Function that has a jvp sees its operands without tangents."""
    class Through(torch.autograd.Function):
        @staticmethod
        def forward(ctx, rows):
            with pytest.raises(Reached):
                matrix().product(rows)
            return rows.clone()

        @staticmethod
        def jvp(ctx, tangent):
            return 3 * tangent

    with forward.dual_level():
        assert (forward.unpack_dual(Through.apply(dual(ROWS))).tangent == 3).all()


@pytest.mark.gpu
def test_calls_on_a_cache():
    cache = vq.QuantizedCache.empty(1, 1, 8)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    x = torch.ones(1, 1, 8, dtype=torch.float16, device="cuda")
    with forward.dual_level():
        for call in (lambda: cache.attend(dual(x), table, lengths), lambda: cache.attend(x, table, lengths, out=dual(x)), lambda: cache.write(dual(x), x, table, lengths),
                     lambda: cache.write(x, dual(x), table, lengths)):
            with pytest.raises(ValueError, match="carries a tangent"):
                call()
        cache.write(x, x, table, lengths)
        assert torch.equal(cache.attend(x, table, lengths), x)
    assert torch.equal(cache.attend(x, table, lengths), x)
    with pytest.raises((ValueError, RuntimeError)):
        torch.func.jvp(lambda q: cache.attend(q, table, lengths), (x,), (x,))
