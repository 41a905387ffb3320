"""Sizes at the edge of what the feed-forward operators address: refused on the host, before anything is launched."""
import ctypes

import pytest

P = ctypes.c_void_p(256)
F32, BF16 = 0, 1
WIDE = (1 << 21) - 1
MOST_ROWS = 1 << 38


def lib():
    from fpn import _lib
    return _lib.load()


def said():
    return lib().fpn_last_error_string().decode()


@pytest.mark.parametrize("rows", [MOST_ROWS + 1, 1 << 39, 1 << 40, (1 << 40) + 1, (1 << 62) + 1])
def test_rows_whose_workspace_would_pass_64_bits_are_refused(rows):
    """At 2^40 rows of 2^21 - 1 floats dg and du alone are 2^64 bytes: a size that wrapped to next to nothing, and a call
    that took such a workspace for enough."""
    L = lib()
    for t in (F32, BF16):
        for size in (L.fpn_dense_workspace_bytes(t, rows, 8, WIDE, 1), L.fpn_dense_grad_workspace_bytes(t, rows, 8, WIDE, 2, 0),
                     L.fpn_gated_workspace_bytes(t, rows, 8, WIDE, 0), L.fpn_gated_grad_workspace_bytes(t, rows, 8, WIDE, 0, 1)):
            assert size == 0 and "rows" in said()
        code = L.fpn_gated_grad(t, rows, 8, WIDE, 0, P, WIDE, None, 0, 0, P, 8, P, WIDE, P, WIDE, 0, P, P, WIDE, 2, None, 8, None, None,
                                WIDE, P, P, P, 1 << 50, None)
        assert code == -3 and "rows" in said()
        code = L.fpn_dense_grad(t, rows, 8, WIDE, P, WIDE, P, 8, P, WIDE, 0, P, WIDE, 2, None, 8, None, WIDE, P, P, 1 << 50, None)
        assert code == -3 and "rows" in said()


@pytest.mark.parametrize("t,size", [(F32, 4), (BF16, 2)])
def test_workspaces_of_the_largest_sizes_are_whole(t, size):
    """Up to the bound no sum of a workspace's parts wraps: it holds dg and du, dh, and the copies of ragged operands."""
    L = lib()
    for rows in (MOST_ROWS, MOST_ROWS // 2 + 1):
        d = rows * WIDE * size
        assert L.fpn_dense_grad_workspace_bytes(t, rows, WIDE, WIDE, 2, 1) >= d
        assert L.fpn_dense_grad_workspace_bytes(t, rows, WIDE, WIDE, 0, 0) >= 2 * d                     # copies of x and dy
        assert L.fpn_gated_grad_workspace_bytes(t, rows, WIDE, WIDE, 0, 1) >= 2 * d
        least = 2 * d + rows * WIDE * 4 + 2 * d                                                          # and of x and dy
        assert least < 1 << 64
        assert L.fpn_gated_grad_workspace_bytes(t, rows, WIDE, WIDE, WIDE, 0) >= least
        need = L.fpn_gated_grad_workspace_bytes(t, rows, WIDE, WIDE, WIDE, 1)
        code = L.fpn_gated_grad(t, rows, WIDE, WIDE, WIDE, P, WIDE, P, WIDE, 0, P, WIDE, P, WIDE, P, WIDE, 0, P, P, WIDE, 2, P, WIDE, P, P,
                                WIDE, P, P, P, need - 1, None)
        assert code == -1 and "workspace" in said()


ROWS = 1 << 34
CALLS = {
    # ragged rows, so that copies would be made first; activations and biases, so that dpre and its sums would
    "dense": lambda L, t: L.fpn_dense(t, ROWS, 515, 259, P, 515, P, 259, 0, P, 2, None, 0, P, 259, P, 259, P, 1 << 60, None),
    "dense_grad": lambda L, t: L.fpn_dense_grad(t, ROWS, 515, 259, P, 259, P, 515, P, 259, 0, P, 259, 2, P, 515, P, 259, P, P, 1 << 60, None),
    "dense_grad, no activation": lambda L, t: L.fpn_dense_grad(t, ROWS, 515, 259, P, 259, P, 515, P, 259, 0, None, 0, 0, P, 515, P, 259, P, P,
                                                               1 << 60, None),
    "dense_grad, held (out,in)": lambda L, t: L.fpn_dense_grad(t, ROWS, 512, 256, P, 256, P, 512, P, 512, 1, P, 256, 2, P, 512, P, 512, P, P,
                                                               1 << 60, None),
    "gated": lambda L, t: L.fpn_gated(t, ROWS, 515, 259, P, 515, P, 259, P, 259, 0, P, P, 2, P, 259, P, P, 259, P, 1 << 60, None),
    "gated_grad": lambda L, t: L.fpn_gated_grad(t, ROWS, 515, 259, 0, P, 259, None, 0, 0, P, 515, P, 259, P, 259, 0, P, P, 259, 2, P, 515, P, P,
                                                259, P, P, P, 1 << 60, None),
    "gated_grad, down projection only": lambda L, t: L.fpn_gated_grad(t, ROWS, 515, 259, 131, P, 131, P, 131, 0, P, 515, P, 259, P, 259, 0, P, P,
                                                                      259, 2, None, 0, None, None, 0, P, P, P, 1 << 60, None),
    "gated_grad, whole rows": lambda L, t: L.fpn_gated_grad(t, ROWS, 512, 256, 128, P, 128, P, 128, 0, P, 512, P, 256, P, 256, 0, P, P, 256, 2, P,
                                                            512, P, P, 256, P, P, P, 1 << 60, None),
}


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("call", list(CALLS))
def test_a_product_beyond_one_launch_is_refused_before_any_launch(call, t):
    """Also where copies, dpre or another product come before it.  (Without a device a launch fails with another code.)"""
    assert CALLS[call](lib(), t) == -3, said()
    assert "workgroups" in said()
