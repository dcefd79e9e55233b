"""Products whose CTAs go through several tiles: accumulators and rings that run on from one tile into the next."""
import pytest

from test_gpu_dense8 import Weight, check_glu, check_linear, glu, linear

pytestmark = pytest.mark.gpu

# rows of x, of the weight, columns. Pairs of CTAs with 1.7 to 4.9 tiles each, tiles of one to 20 stages
PAIRS = [(4096, 4096, 256), (1000, 8192, 1024), (2100, 9000, 300), (300, 30000, 100), (129, 32000, 200), (700, 20000, 500), (17, 32000, 1500), (1300, 4000, 5000), (4000, 2048, 1800)]
# single CTAs with 1.7 to 3 tiles
SINGLE = [(3517, 2618, 360), (1081, 7530, 50), (40, 32000, 64), (1097, 7430, 175)]
# clusters of two that share a tile's columns
TWO = [(32, 6250, 1964), (28, 8254, 2167), (180, 4265, 4423)]
# up to 16 rows: more tiles of 16 weight rows than two CTAs an SM, rows quantised by the CTAs and brought as codes
FEW = [(1, 9000, 700), (3, 12000, 700), (8, 20000, 300), (5, 6000, 5000), (8, 5000, 4000), (12, 9000, 500), (16, 20000, 900)]


@pytest.mark.parametrize("m,rows,cols", PAIRS + SINGLE + TWO + FEW)
def test_products(pkg, torch_dev, m, rows, cols):
    import torch
    g = torch.Generator().manual_seed(m + rows + cols)
    x = torch.randn(m, cols, generator=g).to(torch.bfloat16).to(torch_dev)
    w = Weight(pkg, torch, torch_dev, rows, cols, m * 3 + rows + cols, bias=True, cap=20.0 if m % 2 else 0.0)
    got = linear(pkg, torch, w, x)
    check_linear(w, x.double().cpu().numpy(), got)
    assert (linear(pkg, torch, w, x) == got).all()


# more tiles of 16 gate and 16 up rows than SMs, and the same forms as above
@pytest.mark.parametrize("m,ff,cols,act", [(1, 5000, 300, 3), (1, 4000, 2000, 0), (8, 3000, 300, 1), (8, 2600, 4000, 0), (12, 5000, 500, 0), (16, 6001, 333, 1), (1000, 4096, 300, 0), (2100, 4512, 130, 1), (40, 16000, 64, 0),
                                           (1081, 3765, 50, 1), (60, 3100, 1700, 0)])
def test_gated_products(pkg, torch_dev, m, ff, cols, act):
    import torch
    g = torch.Generator().manual_seed(m + ff + cols)
    x = torch.randn(m, cols, generator=g).to(torch.bfloat16).to(torch_dev)
    w = Weight(pkg, torch, torch_dev, 2 * (-(-ff // 16) * 16), cols, ff, ff=ff)
    got = glu(pkg, torch, w, x, act)
    check_glu(w, x.double().cpu().numpy(), act, got)
    assert (glu(pkg, torch, w, x, act) == got).all()


def test_tiles_one_call_after_another(pkg, torch_dev):
    """Calls of different forms in one stream, each with several tiles a CTA: what one leaves in shared or tensor memory is nothing to the next."""
    import torch
    g = torch.Generator().manual_seed(7)
    cases = []
    for m, rows, cols in ((1000, 8192, 300), (40, 32000, 64), (12, 9000, 500), (32, 6250, 1964)):
        w, x = Weight(pkg, torch, torch_dev, rows, cols, rows, bias=True), torch.randn(m, cols, generator=g).to(torch.bfloat16).to(torch_dev)
        cases.append((w, x, linear(pkg, torch, w, x), torch.empty(m, rows, device=torch_dev), torch.empty(pkg.lib.cmlb200_dense8_work_bytes(m, rows, cols), dtype=torch.uint8, device=torch_dev)))
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        for w, x, want, y, work in cases:
            pkg.check(pkg.lib.cmlb200_linear_dense8(w.handle, x.data_ptr(), pkg.DT_BF16, x.shape[1], x.shape[0], y.data_ptr(), y.shape[1], work.data_ptr(), stream.cuda_stream))
    torch.cuda.synchronize()
    for w, x, want, y, work in cases:
        assert (y.double().cpu().numpy() == want).all()
