"""A row's results do not depend on how many rows there are, nor on the tile, the turn or the kernel that it falls to."""
import pytest

from test_gpu_dense8 import Weight, glu, linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,cols,bias,cap", [(209, 333, True, 0.0), (4096, 512, True, 0.0), (1000, 4096, True, 30.0), (700, 1501, False, 5.0), (129, 40000, True, 0.0)])
def test_products(pkg, torch_dev, rows, cols, bias, cap, form):
    import torch
    g = torch.Generator().manual_seed(rows + cols)
    x = torch.randn(300, cols, generator=g).to(getattr(torch, form)).to(torch_dev)
    w = Weight(pkg, torch, torch_dev, rows, cols, cols, bias=bias, cap=cap)
    whole = linear(pkg, torch, w, x)
    for m in (1, 2, 4, 5, 8, 9, 12, 16, 17, 31, 64, 100, 257):
        at = (37 * m) % (300 - m)
        assert (linear(pkg, torch, w, x[at:at + m]) == whole[at:at + m]).all(), m


@pytest.mark.parametrize("act", [0, 1, 3])
@pytest.mark.parametrize("ff,cols", [(100, 300), (1003, 777), (333, 9000)])
def test_gated_products(pkg, torch_dev, ff, cols, act):
    import torch
    g = torch.Generator().manual_seed(ff + cols)
    x = torch.randn(300, cols, generator=g).to(torch.bfloat16).to(torch_dev)
    w = Weight(pkg, torch, torch_dev, 2 * (-(-ff // 16) * 16), cols, ff, ff=ff)
    whole = glu(pkg, torch, w, x, act)
    for m in (1, 2, 7, 8, 9, 16, 17, 40, 100, 257):
        at = (41 * m) % (300 - m)
        assert (glu(pkg, torch, w, x[at:at + m], act) == whole[at:at + m]).all(), m
