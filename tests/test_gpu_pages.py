"""Copies, moves and forks of pages in several pools at once."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Pools:
    """Pools of pages whose sizes and strides have little in common, in one buffer with room between them."""

    def __init__(self, pkg, dev, sizes, pages, slots, table_ld, seed=0):
        import torch
        self.torch, self.pkg, self.dev, self.sizes, self.pages = torch, pkg, dev, sizes, pages
        r = np.random.default_rng(seed)
        self.bufs = [torch.from_numpy(r.integers(0, 256, pages * stride + 64, dtype=np.uint8)).to(dev) for _, stride, _ in sizes]
        self.desc = torch.tensor([[b.data_ptr() + off, stride, n] for b, (n, stride, off) in zip(self.bufs, sizes)], dtype=torch.int64, device=dev)
        self.table = torch.from_numpy(r.integers(0, pages, (slots, table_ld)).astype(np.int32)).to(dev)
        self.p = pkg.Pages(pools=len(sizes), pool=self.desc.data_ptr(), most=max(n for n, _, _ in sizes), pages=pages, table=self.table.data_ptr(), slots=slots, table_ld=table_ld)

    def snapshot(self):
        return [b.cpu().numpy().copy() for b in self.bufs], self.table.cpu().numpy().copy()

    def copied(self, bufs, pairs):
        out = [b.copy() for b in bufs]
        for b, o, (n, stride, off) in zip(bufs, out, self.sizes):
            for f, t in pairs:
                o[off + t * stride:off + t * stride + n] = b[off + f * stride:off + f * stride + n]
        return out

    def check(self, bufs, table):
        got, t = self.snapshot()
        assert all(np.array_equal(a, b) for a, b in zip(got, bufs))
        assert np.array_equal(t, table)

    def up(self, rows):
        return self.torch.tensor(rows, dtype=self.torch.int32, device=self.dev)


# bytes, stride, offset of the first page: 16-byte, 4-byte and single-byte copies, a page of several pieces
SIZES = [(16384, 16384, 0), (40000, 40016, 16), (64, 64, 0), (4, 12, 4), (7, 9, 1), (33, 48, 0)]


@pytest.mark.parametrize("moves", [1, 3, 40])
@pytest.mark.parametrize("table", [True, False])
def test_moves(pkg, torch_dev, moves, table):
    P = Pools(pkg, torch_dev, SIZES, 100, 7, 33, seed=moves)
    ids = np.random.default_rng(moves).permutation(100)
    pairs = sorted(zip(ids[:moves].tolist(), ids[50:50 + moves].tolist()))
    bufs, t = P.snapshot()
    if not table:
        P.p.table = None
    m = P.up(pairs)
    for _ in range(2):                                 # sources are left as they are: the same moves change nothing more
        pkg.check(pkg.lib.cmlb200_pages_copy(P.p, m.data_ptr(), moves, None))
        P.torch.cuda.synchronize()
        name = dict(pairs) if table else {}
        P.check(P.copied(bufs, pairs), np.vectorize(lambda i: name.get(i, i))(t).astype(np.int32))


def test_moves_that_name_no_page_are_not_made(pkg, torch_dev):
    P = Pools(pkg, torch_dev, SIZES, 20, 2, 5)
    bufs, t = P.snapshot()
    pairs = [(-1, 3), (2, 2), (4, 20), (5, -3), (7, 8), (20, 9), (1 << 30, 1)]
    m = P.up(pairs)
    pkg.check(pkg.lib.cmlb200_pages_copy(P.p, m.data_ptr(), len(pairs), None))
    P.torch.cuda.synchronize()
    P.check(P.copied(bufs, [(7, 8)]), np.where(t == 7, 8, t))


def test_a_table_alone_and_many_small_moves(pkg, torch_dev):
    P = Pools(pkg, torch_dev, [(4, 4, 0)], 5000, 40, 300)
    bufs, t = P.snapshot()
    ids = np.random.default_rng(0).permutation(5000)
    pairs = sorted(zip(ids[:2000].tolist(), ids[2000:4000].tolist()))
    name = np.arange(5000)
    name[[a for a, _ in pairs]] = [b for _, b in pairs]
    m = P.up(pairs)
    P.p.pools = 0
    pkg.check(pkg.lib.cmlb200_pages_copy(P.p, m.data_ptr(), len(pairs), None))
    P.torch.cuda.synchronize()
    P.check(bufs, name[t].astype(np.int32))


@pytest.mark.parametrize("pools", [13, 16])
def test_many_moves_in_many_pools(pkg, torch_dev, pools):
    """So many pages that a CTA takes several pools; their number and pages of several pieces do not divide evenly."""
    sizes = [[(64, 64, 0), (20000, 20016, 16), (36, 48, 4)][k % 3] for k in range(pools)]
    P = Pools(pkg, torch_dev, sizes, 1700, 9, 50, seed=pools)
    ids = np.random.default_rng(pools).permutation(1700)
    pairs = sorted(zip(ids[:800].tolist(), ids[800:1600].tolist()))
    bufs, t = P.snapshot()
    name = np.arange(1700)
    name[[a for a, _ in pairs]] = [b for _, b in pairs]
    m = P.up(pairs)
    pkg.check(pkg.lib.cmlb200_pages_copy(P.p, m.data_ptr(), len(pairs), None))
    P.torch.cuda.synchronize()
    P.check(P.copied(bufs, pairs), name[t].astype(np.int32))


def test_forks(pkg, torch_dev):
    P = Pools(pkg, torch_dev, SIZES, 60, 8, 12)
    bufs, t = P.snapshot()
    used = sorted(set(t[[0, 1, 5]].ravel().tolist()))
    free = [i for i in range(60) if i not in used]
    forks = [(0, 2, 5, free[0]), (0, 3, 5, free[1]), (1, 4, 12, -1), (5, 6, 0, free[2]), (5, 7, 0, -1)]
    want = t.copy()
    pairs = []
    for a, b, n, own in forks:
        want[b, :n] = t[a, :n]
        if own >= 0:
            want[b, n] = own
            pairs.append((t[a, n], own))
    f = P.up(forks)
    side = P.torch.cuda.Stream()
    P.torch.cuda.synchronize()
    pkg.check(pkg.lib.cmlb200_pages_fork(P.p, f.data_ptr(), len(forks), side.cuda_stream))
    P.torch.cuda.synchronize()
    P.check(P.copied(bufs, pairs), want)


def test_forks_that_cannot_be_are_not_made(pkg, torch_dev):
    P = Pools(pkg, torch_dev, SIZES, 60, 8, 12)
    bufs, t = P.snapshot()
    forks = [(0, 8, 1, -1), (-1, 2, 1, -1), (3, 3, 1, -1), (0, 1, 13, -1), (0, 4, 12, 5), (0, 5, 1, 60), (0, 6, -1, -1)]
    f = P.up(forks)
    pkg.check(pkg.lib.cmlb200_pages_fork(P.p, f.data_ptr(), len(forks), None))
    P.torch.cuda.synchronize()
    P.check(bufs, t)


def test_captured_moves(pkg, torch_dev):
    import torch
    P = Pools(pkg, torch_dev, SIZES, 30, 2, 6)
    m = P.up([(3, 4), (9, 1)])
    pkg.check(pkg.lib.cmlb200_pages_copy(P.p, m.data_ptr(), 2, None))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.check(pkg.lib.cmlb200_pages_copy(P.p, m.data_ptr(), 2, torch.cuda.current_stream().cuda_stream))
    bufs, t = P.snapshot()
    m.copy_(P.up([(5, 6), (10, 11)]))
    graph.replay()
    torch.cuda.synchronize()
    P.check(P.copied(bufs, [(5, 6), (10, 11)]), np.where(t == 5, 6, np.where(t == 10, 11, t)))
