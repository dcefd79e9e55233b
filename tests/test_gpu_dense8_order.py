"""Weights quantised and multiplied by on one stream, with nothing in between: a product reads its weight in front of the wait for the launch before it."""
import pytest

pytestmark = pytest.mark.gpu


class Calls:
    def __init__(self, pkg, torch, dev, m, rows, cols, gated):
        g = torch.Generator().manual_seed(m + rows)
        self.pkg, self.m, self.rows, self.cols, self.gated = pkg, m, rows, cols, gated
        ld = -(-cols // 128) * 128
        self.sources = [(torch.randn(rows, cols, generator=g) * 0.05).to(torch.bfloat16).to(dev) for _ in range(2)]
        self.x = torch.randn(m, cols, generator=g).to(torch.bfloat16).to(dev)
        self.codes, self.scale = torch.zeros(-(-rows // 16) * 16, ld, dtype=torch.int8, device=dev), torch.zeros(rows, device=dev)
        self.w = pkg.Dense8(rows=rows, cols=cols, ld=ld, w=self.codes.data_ptr(), scale=self.scale.data_ptr())
        self.work = torch.empty(pkg.lib.cmlb200_dense8_work_bytes(m, rows, cols), dtype=torch.uint8, device=dev)
        self.out = torch.empty(m, rows // 2, dtype=torch.bfloat16, device=dev) if gated else torch.empty(m, rows, device=dev)
        torch.cuda.synchronize()

    def quantize(self, i, stream):
        s = self.sources[i]
        self.pkg.check(self.pkg.lib.cmlb200_quantize_rows(s.data_ptr(), self.pkg.DT_BF16, self.cols, self.rows, self.cols, self.codes.data_ptr(), self.codes.shape[1], self.scale.data_ptr(), stream))

    def multiply(self, stream, out=None):
        out, L = self.out if out is None else out, self.pkg.lib
        if self.gated:
            self.pkg.check(L.cmlb200_linear_dense8_glu(self.w, self.x.data_ptr(), self.pkg.DT_BF16, self.cols, self.m, self.rows // 2, 0, out.data_ptr(), out.shape[1], self.work.data_ptr(), stream))
        else:
            self.pkg.check(L.cmlb200_linear_dense8(self.w, self.x.data_ptr(), self.pkg.DT_BF16, self.cols, self.m, out.data_ptr(), out.shape[1], self.work.data_ptr(), stream))


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,rows,cols", [(1, 4096, 4096), (1, 11008, 4096), (12, 4096, 4096), (40, 4096, 2048), (77, 11008, 4096), (600, 8192, 1024), (1, 64, 128), (40, 64, 128), (30, 448, 9000)])
def test_quantised_then_multiplied(pkg, torch_dev, m, rows, cols, gated):
    import torch
    c = Calls(pkg, torch, torch_dev, m, rows, cols, gated)
    stream, want = torch.cuda.Stream(), []
    for i in range(2):
        c.quantize(i, stream.cuda_stream)
        torch.cuda.synchronize()
        c.multiply(stream.cuda_stream)
        torch.cuda.synchronize()
        want.append(c.out.clone())
    assert not torch.equal(*want)
    outs = [torch.empty_like(c.out) for _ in range(24)]
    torch.cuda.synchronize()
    for k, out in enumerate(outs):
        c.quantize(k % 2, stream.cuda_stream)
        c.multiply(stream.cuda_stream, out)
        if k % 3 == 0:                                  # (the second product's codes' launch lies between it and the weight's)
            c.multiply(stream.cuda_stream, out)
    torch.cuda.synchronize()
    for k, out in enumerate(outs):
        assert torch.equal(out, want[k % 2]), k
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        for k, out in enumerate(outs):
            c.quantize(k % 2, torch.cuda.current_stream().cuda_stream)
            c.multiply(torch.cuda.current_stream().cuda_stream, out)
    for _ in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for k, out in enumerate(outs):
            assert torch.equal(out, want[k % 2]), k
