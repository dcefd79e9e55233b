"""Moves and forks of pages whose lists name what is not there."""
import numpy as np
import pytest

from test_gpu_pages import SIZES, Pools

pytestmark = pytest.mark.gpu


def test_entries_without_a_page_keep_their_value(pkg, torch_dev):
    """A table's places without a page (-1, and numbers beyond the pools) are not renamed by a move from there, which is not made."""
    P = Pools(pkg, torch_dev, SIZES, 20, 4, 9)
    P.table[0, 3:] = -1
    P.table[2, :2] = 20
    P.table[3, 5] = 1 << 30
    bufs, t = P.snapshot()
    m = P.up([(-1, 3), (7, 8), (20, 9), (1 << 30, 1)])
    pkg.check(pkg.lib.cmlb200_pages_copy(P.p, m.data_ptr(), 4, None))
    P.torch.cuda.synchronize()
    P.check(P.copied(bufs, [(7, 8)]), np.where(t == 7, 8, t))


def test_forks_of_more_pages_than_numbers_reach(pkg, torch_dev):
    """One more than the largest number of shared pages would be a negative one."""
    P = Pools(pkg, torch_dev, SIZES, 60, 8, 12)
    bufs, t = P.snapshot()
    f = P.up([(0, 1, 2 ** 31 - 1, 5), (0, 2, 2 ** 31 - 1, -1), (0, 3, 12, 5)])
    pkg.check(pkg.lib.cmlb200_pages_fork(P.p, f.data_ptr(), 3, None))
    P.torch.cuda.synchronize()
    P.check(bufs, t)
