"""Calls over 8-bit caches whose lists have places that are nothing."""
import numpy as np
import pytest

from test_gpu_cache8 import FORMS, Layer

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,kv_heads,rows", [(8, 2, 150), (32, 8, 1300), (12, 4, 2600)])
def test_tiles_without_rows(pkg, torch_dev, form, heads, kv_heads, rows):
    """A list of a fixed length, as a captured call has, of which the last places, and one in the middle, are empty."""
    import torch
    L = Layer(pkg, torch_dev, form, heads, kv_heads, 64, 64, slots=2, tokens=rows)
    x = torch.from_numpy(L.fresh_rows(rows)).to(torch_dev)
    pos, slot = torch.arange(rows, dtype=torch.int32, device=torch_dev), torch.zeros(rows, dtype=torch.int32, device=torch_dev)
    pkg.check(pkg.lib.cmlb200_qk_norm_append(L.a, x.data_ptr(), L.ld, pos.data_ptr(), slot.data_ptr(), rows, None))
    tiles, none, out = [[k, min(64, rows - k), 0, k] for k in range(0, rows, 64)], [0, 0, 0, 0], []
    for some in (tiles, tiles[:1] + [none] + tiles[1:] + [none, none]):
        t, y = torch.tensor(some, dtype=torch.int32, device=torch_dev), torch.full((rows + 1, heads * 64), 7.0, dtype=torch.bfloat16, device=torch_dev)
        pkg.check(pkg.lib.cmlb200_attention_tiles(L.a, x.data_ptr(), L.ld, t.data_ptr(), len(some), y.data_ptr(), heads * 64, None))
        torch.cuda.synchronize()
        out.append(y.float().cpu().numpy())
    # (as many CTAs share a tile's keys as there are tiles for: few tiles more may be summed in another order)
    assert np.abs(out[0] - out[1]).max() <= (0 if rows > 1000 else 2.0 ** -7 * np.abs(out[0]).max()) and (out[1][rows] == 7).all() and np.isfinite(out[1]).all()
