"""Which schedules of coefficients are taken, without a GPU: the C ABI looks at them before any HIP call, and a call on no matrices
makes none."""
import ctypes as C

import pytest


def take(*rows):
    from nerf_amd import _lib
    flat = [v for r in rows for v in r]
    rc = _lib.lib.nerfx_orthogonalize(None, 0, 0, (C.c_float * len(flat))(*flat), len(rows), 1e-7, None, 0, None)
    return rc, _lib.lib.nerfx_last_error()


@pytest.mark.parametrize("rows", [
    [(0.01, 0.0, 0.0)] * 5,                     # 1e-8 of X is left before the last step: below what its halves hold
    [(0.1, 0.9, 0.0)] * 5,                      # 1 stays 1, a singular value of 0.03 goes down to 3e-6
    [(0.0, 1.0, 0.0)] * 2,                      # cubes
    [(3.0, 0.0, 0.0)] * 2 + [(0.01, 0.0, 0.0), (1.0, 0.0, 0.0)],
])
def test_schedules_that_shrink_are_refused(rows):
    rc, text = take(*rows)
    assert rc == -1 and b"shrink" in text, text


@pytest.mark.parametrize("rows", [
    [(3.4445, -4.7750, 2.0315)] * 32, [(1.5, -0.5, 0.0)] * 32, [(4.0, -7.0, 3.2), (3.0, -4.0, 2.0), (1.875, -1.25, 0.375)],
    [(3.0, 0.0, 0.0)] * 3, [(1.0, -1.0, 0.0)] * 5,
    [(0.01, 0.0, 0.0)], [(0.0, 1.0, 0.0)],      # one step: the result is the caller's own number
    [(1.0, 0.0, 0.0)] * 4 + [(1e-6, 0.0, 0.0)],
])
def test_schedules_that_are_taken(rows):
    assert take(*rows)[0] == 0, take(*rows)[1]
