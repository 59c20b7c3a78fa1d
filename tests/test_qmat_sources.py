"""Kernels of the products may start before the kernel in front of them ends: nothing that one may have written is read as memory that stays the same for
as long as the kernel is there (__ldg, const __restrict__).  Read from the sources."""
from tests.test_overlapped_launches import _functions, _taken_for_invariant


def test_rows_are_not_taken_for_invariant():
    seen = set()
    for name, params, body in _functions():
        if "rows_are_there();" in body:
            seen.add(name)
            assert not _taken_for_invariant(params, body), name
    assert seen == {"quantize_rows_kernel", "product_tc_kernel", "product_few_kernel"}


def test_every_way_out_of_such_a_kernel_is_behind_the_wait():
    """A kernel that ends without waiting would let the next one start before the work in front of both has ended."""
    for name, _, body in _functions():
        if "rows_are_there();" in body and name != "product_tc_kernel":
            first = body.index("rows_are_there();")
            assert "return;" not in body[:first], name
