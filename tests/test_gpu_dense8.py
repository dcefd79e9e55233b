"""Rows quantised to int8 and products over them against 64 bits."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

TINY = 127 * 2.0 ** -126
FORMS = ["float32", "bfloat16", "float16"]


def code_of(pkg, torch, x):
    return {torch.float32: pkg.DT_F32, torch.bfloat16: pkg.DT_BF16, torch.float16: pkg.DT_F16}[x.dtype]


def wide(torch, x, extra, lead=0):
    """x as a view of a wider tensor whose rows begin at element `lead`, NaN around it."""
    t = torch.full((x.shape[0], lead + x.shape[1] + extra), float("nan"), dtype=x.dtype, device=x.device)
    t[:, lead:lead + x.shape[1]] = x
    return t[:, lead:lead + x.shape[1]]


def quantize(pkg, torch, x, pad=0, stream=None):
    rows, cols = x.shape
    ldq = -(-cols // 128) * 128 + pad
    q = torch.full((rows + 1, ldq), 99, dtype=torch.int8, device=x.device)
    s = torch.full((rows + 1,), 77.0, device=x.device)
    torch.cuda.synchronize()
    pkg.check(pkg.lib.cmlb200_quantize_rows(x.data_ptr(), code_of(pkg, torch, x), x.stride(0), rows, cols, q.data_ptr(), ldq, s.data_ptr(), stream), "quantize_rows")
    torch.cuda.synchronize()
    filled = -(-cols // 128) * 128
    assert (q[rows] == 99).all() and s[rows] == 77.0 and (q[:rows, filled:] == 99).all() and (q[:rows, cols:filled] == 0).all()
    return q[:rows, :cols].cpu().numpy(), s[:rows].cpu().numpy()


def want_codes(x):
    """Codes and scales by the definition in 64 bits, and how far the quotient is from a tie."""
    x = np.asarray(x, np.float64)
    a = np.maximum(np.abs(x).max(1), TINY)[:, None]
    t = 127 * x / a
    return np.rint(t), (a / 127)[:, 0], np.abs(np.abs(t - np.floor(t)) - 0.5)


def check_codes(q, s, x, form):
    want, scale, tie = want_codes(x)
    # fp32: 127 v and the quotient are rounded, half a unit of 2^-24 each of up to 127
    sure = np.ones_like(tie, bool) if form != "float32" else tie > 127 * 2 * 2.0 ** -24
    assert (q[sure] == want[sure]).all() and (np.abs(q - want) <= 1).all()
    assert (np.abs(s - scale) <= scale * 2.0 ** -24).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (2, 15), (5, 16), (1, 17), (7, 127), (2, 128), (3, 129), (300, 200), (4, 4096), (301, 4097), (2, 16384), (1, 32768), (2, 33001), (300, 8200), (1, 131071)])
def test_rows(pkg, torch_dev, form, rows, cols):
    import torch
    g = torch.Generator().manual_seed(rows * 7919 + cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(torch.randn(rows, 1, generator=g) * 3)).clamp(-60000, 60000).to(getattr(torch, form)).to(torch_dev)
    for extra, lead, pad in ((0, 0, 0), (3, 0, 128), (16, 1, 0), (8, 8, 256)):
        y = wide(torch, x, extra, lead) if extra else x
        q, s = quantize(pkg, torch, y, pad)
        check_codes(q, s, x.double().cpu().numpy(), form)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rows,cols", [(593, 777), (600, 4097), (1100, 2050), (2500, 130), (1200, 9000), (7000, 33)])
def test_many_rows(pkg, torch_dev, form, rows, cols):
    """CTAs of several rows, in every number of warps."""
    test_rows(pkg, torch_dev, form, rows, cols)


@pytest.mark.parametrize("form", FORMS)
def test_ties_and_ends(pkg, torch_dev, form):
    """Ties that a scale rounded to 32 bits would miss; zeros; the smallest and largest numbers; rows that are not numbers."""
    import torch
    t = getattr(torch, form)
    k = torch.arange(0, 128).double()
    rows = [k / 127 * 127, (k + 0.5).clamp_max(127), 2 * k + 1, (2 * k + 1) * 3, k * 0, k * 0 - 0.0]
    rows += [torch.where(k == 5, 254.0, (2 * k + 1)), torch.where(k == 5, 2.0 ** -3, 2.0 ** -4), torch.where(k == 5, 3.0, 1.5), torch.where(k == 0, 7.0, 3.5)]
    fi = torch.finfo(t)
    rows += [torch.where(k == 9, fi.max, fi.max / 2), torch.where(k == 9, -fi.max, k), k * fi.smallest_normal / 64, torch.where(k < 60, fi.smallest_normal * fi.eps, 0.0)]
    x = torch.stack(rows).to(t).to(torch_dev)
    q, s = quantize(pkg, torch, x)
    check_codes(q, s, x.double().cpu().numpy(), form)
    assert q.min() >= -127
    bad = torch.randn(6, 300, device=torch_dev).to(t)
    bad[1, 299], bad[2, 0], bad[4, 150] = float("nan"), float("inf"), float("-inf")
    q, s = quantize(pkg, torch, bad)
    assert np.isnan(s[[1, 2, 4]]).all() and (q[[1, 2, 4]] == 0).all()
    ok = [0, 3, 5]
    check_codes(q[ok], s[ok], bad.double().cpu().numpy()[ok], form)


@pytest.mark.parametrize("form", ["bfloat16", "float16"])
def test_every_largest_number(pkg, torch_dev, form):
    """Rows whose largest number has every mantissa, multiples of 127 among them, and numbers that meet its ties or come next to them."""
    import torch
    t = getattr(torch, form)
    bits = 8 if form == "bfloat16" else 11
    rows = []
    for m in range(1 << (bits - 1), 1 << bits):
        a = float(m)
        k = torch.arange(0, 128).double()
        near = ((k + 0.5) * a / 127).to(t).double().clamp_max(a)           # the numbers around every tie
        rows.append(torch.cat([near, (near * (1 + 2.0 ** -bits)).to(t).double().clamp_max(a), (near * (1 - 2.0 ** -bits)).to(t).double(), torch.tensor([a, a / 2, a / 4, -a / 2])]))
    x = torch.stack(rows)
    for scale in (1.0, 2.0 ** -6, 2.0 ** 4 if form == "float16" else 2.0 ** 100, 2.0 ** -14 if form == "float16" else 2.0 ** -130):
        y = (x * scale).to(t).to(torch_dev)
        q, s = quantize(pkg, torch, y)
        check_codes(q, s, y.double().cpu().numpy(), form)
        q, s = quantize(pkg, torch, y[:200])                              # (few rows: the other shape of CTAs)
        check_codes(q, s, y[:200].double().cpu().numpy(), form)


class Weight:
    """A quantised weight with codes of its own; `half`: gate and up rows in turns of 16."""

    def __init__(self, pkg, torch, dev, rows, cols, seed, bias=False, cap=0.0, pad=0, ff=0):
        g = torch.Generator().manual_seed(seed)
        padded, ld = -(-rows // 16) * 16, -(-cols // 128) * 128 + pad
        codes = torch.zeros(padded, ld, dtype=torch.int8)
        codes[:rows, :cols] = torch.randint(-127, 128, (rows, cols), generator=g, dtype=torch.int8)
        scale = torch.zeros(padded)
        scale[:rows] = torch.exp(torch.randn(rows, generator=g)) * 0.01
        if ff:
            place = torch.arange(rows)
            dead = (place // 32) * 16 + place % 16 >= ff
            codes[:rows][dead], scale[:rows][dead] = 0, 0.0
        self.codes, self.scale = codes.to(dev), scale.to(dev)
        self.bias = (torch.randn(rows, generator=g) * 3).to(dev) if bias else None
        self.w, self.s = codes[:rows, :cols].double().numpy(), scale[:rows].double().numpy()
        self.b = self.bias.double().cpu().numpy() if bias else 0.0
        self.handle = pkg.Dense8(rows=rows, cols=cols, ld=ld, w=self.codes.data_ptr(), scale=self.scale.data_ptr(), bias=self.bias.data_ptr() if bias else None, cap=cap)
        self.cap, self.rows, self.cols, self.ff = cap, rows, cols, ff


def status(pkg):
    st = C.c_int(-1)
    pkg.check(pkg.lib.cmlb200_dense8_status(C.byref(st), 1), "dense8_status")
    return st.value


def work_for(pkg, torch, dev, m, w):
    return torch.full((pkg.lib.cmlb200_dense8_work_bytes(m, w.rows, w.cols),), 171, dtype=torch.uint8, device=dev)


def linear(pkg, torch, w, x, pad=0, stream=None, work=None):
    m = x.shape[0]
    y = torch.full((m + 1, w.rows + pad), 55.0, device=x.device)
    work = work_for(pkg, torch, x.device, m, w) if work is None else work
    torch.cuda.synchronize()
    pkg.check(pkg.lib.cmlb200_linear_dense8(w.handle, x.data_ptr(), code_of(pkg, torch, x), x.stride(0), m, y.data_ptr(), y.stride(0), work.data_ptr(), stream), "linear_dense8")
    torch.cuda.synchronize()
    assert status(pkg) == 0 and (y[m] == 55.0).all() and (y[:, w.rows:] == 55.0).all()
    return y[:m, :w.rows].double().cpu().numpy()


def glu(pkg, torch, w, x, act, pad=0, stream=None):
    m = x.shape[0]
    f = torch.full((m + 1, w.ff + pad), 55.0, dtype=torch.bfloat16, device=x.device)
    work = work_for(pkg, torch, x.device, m, w)
    torch.cuda.synchronize()
    pkg.check(pkg.lib.cmlb200_linear_dense8_glu(w.handle, x.data_ptr(), code_of(pkg, torch, x), x.stride(0), m, w.ff, act, f.data_ptr(), f.stride(0), work.data_ptr(), stream), "linear_dense8_glu")
    torch.cuda.synchronize()
    assert status(pkg) == 0 and (f[m] == 55.0).all() and (f[:, w.ff:] == 55.0).all()
    return f[:m, :w.ff].double().cpu().numpy()


def product(w, x):
    """In 64 bits from the codes: the sums are whole numbers below 2^31."""
    q, s, _ = want_codes(x)
    return (q @ w.w.T) * s[:, None] * w.s


def check_linear(w, x, got):
    """The sum as fp32, both scales' product, x's scale and the products: five roundings of half a unit; the bias one more. The cap: tanh within 2 units and a quotient, a product, and
    what the argument's error makes (a slope of 1 at most)."""
    y = product(w, x)
    want = y + w.b
    slack = 5 * 2.0 ** -24 * np.abs(y) + 2.0 ** -24 * np.abs(want)
    if w.cap:
        want = w.cap * np.tanh(want / w.cap)
        slack = slack + 8 * 2.0 ** -24 * np.abs(want)
    assert (np.abs(got - want) <= slack * 1.01 + 1e-37).all(), (np.abs(got - want) / (slack + 1e-30)).max()


SIZES = [(1, 1, 1), (1, 16, 128), (1, 17, 129), (2, 33, 64), (8, 100, 200), (9, 64, 256), (16, 48, 1000), (17, 130, 384), (31, 257, 515), (32, 4096, 512), (33, 128, 128), (33, 1, 1), (64, 300, 1100),
         (65, 129, 640), (100, 1003, 777), (128, 256, 256), (129, 257, 129), (257, 70, 4100), (300, 2051, 300), (513, 600, 130), (1, 5000, 11008), (4, 300, 40000), (40, 64, 40000), (2100, 1031, 257),
         (200, 5000, 600), (1000, 4096, 1000)]


@pytest.mark.parametrize("m,rows,cols", SIZES)
def test_linear(pkg, torch_dev, m, rows, cols):
    import torch
    g = torch.Generator().manual_seed(m * 31 + rows * 7 + cols)
    x = torch.randn(m, cols, generator=g).to(torch.bfloat16).to(torch_dev)
    w = Weight(pkg, torch, torch_dev, rows, cols, m + rows + cols, bias=rows % 2 == 1, cap=20.0 if cols % 2 else 0.0)
    check_linear(w, x.double().cpu().numpy(), linear(pkg, torch, w, x))


@pytest.mark.parametrize("m", [1, 3, 12, 30, 70, 300])
@pytest.mark.parametrize("form", FORMS)
def test_linear_strides(pkg, torch_dev, m, form):
    """Rows and results inside wider tensors, aligned and not, a weight with a wider stride, every type of x. fp32 rows are whole numbers, whose codes have no ties but exact ones."""
    import torch
    g = torch.Generator().manual_seed(m)
    x = torch.randint(-500, 501, (m, 333), generator=g)
    x[:, 7] = 127 * 4
    x = x.to(getattr(torch, form)).to(torch_dev)
    w = Weight(pkg, torch, torch_dev, 209, 333, m, bias=True, pad=128)
    for extra, lead, pad in ((3, 0, 0), (16, 8, 5), (19, 1, 64)):
        check_linear(w, x.double().cpu().numpy(), linear(pkg, torch, w, wide(torch, x, extra, lead), pad))


ACTS = [0, 1, 3]


def check_glu(w, x, act, got):
    """bf16: half a step of the result (2^-8). Before it, in fp32: the products' five roundings on either side, the exponential of an argument that is off by its own roundings (a few 2^-23 of it)
    and the quotient: 2^-18 of the result for arguments up to 2^4 or 2^-22 times the argument beyond that; the error function's approximation is off by 1.5e-7 of z u / 2; results below
    the smallest normal number may be 0."""
    y = product(w, x).reshape(len(x), -1, 2, 16)
    z, u = y[:, :, 0].reshape(len(x), -1)[:, :w.ff], y[:, :, 1].reshape(len(x), -1)[:, :w.ff]
    if act == 0:
        arg = z
    elif act == 1:
        arg = 2 * np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)
    if act == 3:
        from math import erf
        a = 0.5 * z * (1 + np.vectorize(erf)(z / np.sqrt(2)))
        near = 2e-7 * np.abs(z * u) + 2.0 ** -18 * np.abs(z * u) * np.exp(-z * z / 2) * (1 + z * z)
    else:
        a = z * np.exp(np.minimum(arg, 0)) / (1 + np.exp(-np.abs(arg)))
        # (an exponential that overflows: sigmoid is then below 2^-126)
        near = np.abs(a * u) * (2.0 ** -18 + 2.0 ** -21 * np.abs(arg)) + np.abs(z * u) * 2.0 ** -125
    want = a * u
    assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + near * 1.01 + 2.0 ** -126).all(), (np.abs(got - want) - 2.0 ** -8 * np.abs(want)).max()


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,ff,cols", [(1, 1, 1), (1, 16, 128), (2, 17, 100), (8, 100, 300), (13, 48, 257), (32, 333, 1000), (33, 16, 128), (50, 15, 129), (100, 501, 777), (129, 128, 256), (300, 1003, 130), (700, 64, 64)])
def test_glu(pkg, torch_dev, m, ff, cols, act):
    import torch
    g = torch.Generator().manual_seed(m + ff + cols + act)
    x = torch.randn(m, cols, generator=g).to(torch.bfloat16).to(torch_dev)
    w = Weight(pkg, torch, torch_dev, 2 * (-(-ff // 16) * 16), cols, ff, ff=ff)
    check_glu(w, x.double().cpu().numpy(), act, glu(pkg, torch, w, x, act))
    check_glu(w, x.double().cpu().numpy(), act, glu(pkg, torch, w, wide(torch, x, 5, 1), act, pad=7))


@pytest.mark.parametrize("m", [5, 90])
def test_rows_that_are_not_numbers(pkg, torch_dev, m):
    """NaN and infinities stay in their own rows; a row of zeros is 0 (or the bias)."""
    import torch
    x = torch.randn(m, 200, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(torch_dev)
    x[1, 3], x[2, 199], x[4] = float("nan"), float("inf"), 0.0
    w = Weight(pkg, torch, torch_dev, 100, 200, 3, bias=True)
    y = linear(pkg, torch, w, x)
    assert np.isnan(y[[1, 2]]).all() and (y[4] == w.b).all()
    ok = [i for i in range(m) if i not in (1, 2)]
    check_linear(w, x.double().cpu().numpy()[ok], y[ok])
    w = Weight(pkg, torch, torch_dev, 128, 200, 4, ff=64)
    f = glu(pkg, torch, w, x, 0)
    assert np.isnan(f[[1, 2]]).all() and (f[4] == 0).all()
    check_glu(w, x.double().cpu().numpy()[ok], 0, f[ok])


@pytest.mark.parametrize("m", [1, 20, 200])
def test_largest_sums(pkg, torch_dev, m):
    """Every product at its largest and of one sign: 131,071 columns of 127 * 127 (and -128 in the weight) fit 32 bits."""
    import torch
    x = torch.full((m, 131071), 3.0, dtype=torch.bfloat16, device=torch_dev)
    w = Weight(pkg, torch, torch_dev, 20, 131071, 1)
    w.codes[:, :131071] = -128
    w.codes[5, :131071] = 127
    w.w = w.codes[:20, :131071].double().cpu().numpy()
    check_linear(w, x.double().cpu().numpy(), linear(pkg, torch, w, x))


@pytest.mark.parametrize("m", [2, 150])
def test_streams_and_graphs(pkg, torch_dev, m):
    """Two streams at once with workspaces of their own, a captured call replayed over other rows, and the same result every time."""
    import torch
    w = Weight(pkg, torch, torch_dev, 1000, 600, 9)
    xs = [torch.randn(m, 600, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).to(torch_dev) for i in range(2)]
    want = [linear(pkg, torch, w, x) for x in xs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs, works = [torch.empty(m, 1000, device=torch_dev) for _ in range(2)], [work_for(pkg, torch, torch_dev, m, w) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, y, k, st in zip(xs, outs, works, streams):
            pkg.check(pkg.lib.cmlb200_linear_dense8(w.handle, x.data_ptr(), pkg.DT_BF16, 600, m, y.data_ptr(), 1000, k.data_ptr(), st.cuda_stream), "linear_dense8")
    torch.cuda.synchronize()
    for y, v in zip(outs, want):
        assert (y.double().cpu().numpy() == v).all()
    x, y = xs[0].clone(), outs[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(2):
            pkg.check(pkg.lib.cmlb200_linear_dense8(w.handle, x.data_ptr(), pkg.DT_BF16, 600, m, y.data_ptr(), 1000, works[0].data_ptr(), torch.cuda.current_stream().cuda_stream), "linear_dense8")
    for i in (1, 0, 1):
        x.copy_(xs[i])
        y.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert (y.double().cpu().numpy() == want[i]).all()


CAPTURED_FIRST = """
import ctypes, sys
sys.path.insert(0, {root!r})
import torch
import __graft_entry__ as entry
pkg = entry.load_package()
m, n, k = {m}, 300, 500
x, codes, scale = torch.ones(m, k, device="cuda", dtype=torch.bfloat16), torch.ones(304, 512, device="cuda", dtype=torch.int8), torch.ones(304, device="cuda")
codes[:, k:] = 0
y, work = torch.zeros(m, n, device="cuda"), torch.zeros(pkg.lib.cmlb200_dense8_work_bytes(m, n, k), device="cuda", dtype=torch.uint8)
w = pkg.Dense8(rows=n, cols=k, ld=512, w=codes.data_ptr(), scale=scale.data_ptr())
torch.cuda.synchronize()
g, status = torch.cuda.CUDAGraph(), ctypes.c_int(-1)
with torch.cuda.graph(g):
    pkg.check(pkg.lib.cmlb200_linear_dense8(w, x.data_ptr(), pkg.DT_BF16, k, m, y.data_ptr(), n, work.data_ptr(), torch.cuda.current_stream().cuda_stream), "linear_dense8")
    pkg.check(pkg.lib.cmlb200_dense8_status(ctypes.byref(status), 0))
assert status.value == 0
g.replay()
torch.cuda.synchronize()
assert ((y - k).abs() <= 5 * 2.0 ** -24 * k).all(), y
print("fine")
"""


@pytest.mark.parametrize("m", [1, 12, 40, 600])
def test_captured_before_anything_else_ran(m):
    """The first call of a process is one that is being captured."""
    import subprocess
    import sys
    from pathlib import Path
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST.format(root=str(Path(__file__).resolve().parents[1]), m=m)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
