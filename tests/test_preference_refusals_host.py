"""What the preference loss's C entry points refuse about the statistics for the backward pass, before anything is launched."""
import ctypes

from repdl_amd import _lib

A = ctypes.c_void_p(0x7F0000000000)  # never dereferenced: every call below ends on the host, at the missing workspace at the latest


def call(row_stats, coef, steps=3):
    return _lib.lib().repdl_hip_preference_loss_ws(A, A, None, A, A, row_stats, coef, 2, steps, 10, 10 * steps, 10, 0.1, 0.0, -100, 0, None, 0, None)


def test_row_stats_and_coef_go_together():
    assert call(A, A) == -3 and call(None, None) == -3
    assert call(A, None) == -1 and call(None, A) == -1
    assert _lib.lib().repdl_hip_preference_loss(A, A, None, A, A, A, None, 2, 3, 10, 30, 10, 0.1, 0.0, -100, 0, None) == -1
    assert call(None, A, steps=0) == -3  # (no rows: their statistics are an empty tensor, which may be NULL)
    assert call(A, None, steps=0) == -1
