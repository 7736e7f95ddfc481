"""The C entries of K10 refuse what a launch cannot hold, before one is made (so without a GPU)."""
import pytest

from nextou_amd import _lib


@pytest.mark.parametrize("dtype,K", [(0, 1000), (1, 1000), (2, 300), (1, 301)])
@pytest.mark.parametrize("P,N", [(1 << 30, 8), (1 << 31, 9), (1 << 32, 40)])
def test_one_row_for_more_points_than_a_launch_holds(dtype, K, P, N):
    """ldx = 0 reads one row of x for all points: nothing but the launch bounds their number"""
    L = _lib.lib()
    rc = L.nextou_linear_act_fwd(4096, 8192, None, None, 1 << 20, None, P, N, K, 1, 0, 0, N, dtype, 0, 0, 0.0, None)
    assert rc == -1 and b"one launch" in L.nextou_last_error()
