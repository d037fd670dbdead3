"""Bounds of the 8-bit cache's tests and workspaces, on the CPU."""
import numpy as np
import pytest

import kv8_reference as ref


def test_check_rows_takes_no_nan():
    """A NaN compares false either way: it has to count as outside its bound."""
    want, tol = np.ones((2, 3)), np.full((2, 3), 1e-3)
    ref.check_rows(want.astype(np.float32), want, tol)
    ref.check_rows(want + 1e-3 * 0.99, want, tol)
    for at in ((0, 0), (1, 2)):
        for i in range(3):
            a = [want.astype(np.float32), want.copy(), tol.copy()]
            a[i][at] = np.nan
            with pytest.raises(AssertionError):
                ref.check_rows(*a)
    with pytest.raises(AssertionError):
        ref.check_rows(want + 2e-3, want, tol)
    with pytest.raises(AssertionError):
        ref.check_rows(np.full((2, 3), np.inf), want, tol)
