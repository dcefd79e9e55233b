"""Log probabilities, entropy and alternatives of rows of logits against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def call(pkg, torch, x, tokens, top, ld=None, what="tei", stream=None):
    """x: device rows [rows, vocab] of a wider tensor; returns numpy arrays."""
    rows, vocab = x.shape
    dt = {torch.float32: pkg.DT_F32, torch.bfloat16: pkg.DT_BF16, torch.float16: pkg.DT_F16}[x.dtype]
    lp, en = (torch.full((rows,), 77.0, device=x.device) for _ in range(2))
    ids = torch.full((rows, max(top, 1)), -7, dtype=torch.int32, device=x.device)
    best = torch.full((rows, max(top, 1)), 77.0, device=x.device)
    tk = torch.as_tensor(tokens, dtype=torch.int32, device=x.device)
    torch.cuda.synchronize()
    t, e, i = ("t" in what), ("e" in what), ("i" in what)
    pkg.check(pkg.lib.cmlb200_token_scores(x.data_ptr(), dt, x.stride(0), rows, vocab, tk.data_ptr() if t else None, top, lp.data_ptr() if t else None, en.data_ptr() if e else None,
                                           ids.data_ptr() if i and top else None, best.data_ptr() if top else None, stream), "token_scores")
    torch.cuda.synchronize()
    return lp.cpu().numpy(), en.cpu().numpy(), ids.cpu().numpy()[:, :top], best.cpu().numpy()[:, :top]


def want(x, tokens, top):
    """The same in 64 bits, by the definition."""
    x = x.astype(np.float64)
    lp, en, ids, best = [], [], [], []
    for row, t in zip(x, tokens):
        if np.isnan(row).any() or np.isposinf(row).any():
            m, z, h = 0.0, np.nan, np.nan
        elif np.isneginf(row).all():
            m, z, h = 0.0, 0.0, 0.0
        else:
            m = row.max()                              # (x - m) - ln S: x - (m + ln S) would lose ln S beside the lowest number of a type
            z = np.log(np.exp(row - m).sum())
            p = np.exp(row - m - z)
            h = -(p[p > 0] * np.log(p[p > 0])).sum()
        lp.append((row[t] - m) - z if 0 <= t < len(row) else (np.nan if np.isnan(z) else -np.inf))
        en.append(h)
        clean = np.where(np.isnan(row), -np.inf, row)
        order = np.argsort(-clean, kind="stable")[:top]
        ok = clean[order] > -np.inf
        ids.append(np.where(ok, order, -1))
        best.append(np.where(ok, (row[order] - m) - z, -np.inf))
    return np.array(lp), np.array(en), np.array(ids).reshape(len(x), top), np.array(best).reshape(len(x), top)


def compare(got, ref, vocab):
    """fp32: ln S of a sum of up to `vocab` terms that are each off by a few parts in 2^23 (exponential, its argument, partial sums), and the
    roundings of x - m, ln and the difference: 16 half steps of the result and 2^-20 absolute."""
    for g, w, whole in zip(got, ref, (False, False, True, False)):
        if whole:
            assert np.array_equal(g, w)
            continue
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(np.isinf(g), np.isinf(w)), (g, w)
        ok = np.isfinite(w)
        assert (np.abs(g[ok] - w[ok]) <= 16 * 2.0 ** -24 * np.abs(w[ok]) + 2.0 ** -20).all(), np.abs(g[ok] - w[ok]).max()


TYPES = ["float32", "bfloat16", "float16"]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 2), (3, 7, 5), (1, 32000, 5), (2, 32001, 32), (5, 100003, 20), (300, 1000, 3), (700, 509, 0), (33, 4099, 1), (1, 262144, 32), (9, 65536, 20)])
def test_sizes(pkg, torch_dev, dtype, rows, vocab, top):
    import torch
    g = torch.Generator(device=torch_dev).manual_seed(rows + vocab)
    wide = torch.full((rows, vocab + 13), float("nan"), device=torch_dev, dtype=getattr(torch, dtype))
    wide[:, 3:3 + vocab] = torch.randn(rows, vocab, generator=g, device=torch_dev) * 3 - 1
    x = wide[:, 3:3 + vocab]                           # rows that begin and end anywhere
    tokens = np.random.default_rng(vocab).integers(0, vocab, rows)
    got, ref = call(pkg, torch, x, tokens, top), want(x.float().cpu().numpy(), tokens, top)
    compare(got, ref, vocab)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [11, 5000, 70001])
def test_rows_of_special_values(pkg, torch_dev, dtype, vocab):
    import torch
    r = np.random.default_rng(1)
    x = r.standard_normal((14, vocab)).astype(np.float32)
    x[0] = -np.inf                                     # nothing can come
    x[1, :] = -np.inf; x[1, vocab // 2] = 3            # one token alone
    x[2] = 0                                           # all alike
    x[3, vocab - 1] = np.nan
    x[4, 1] = np.inf
    x[5] = np.where(np.arange(vocab) % 3, x[5], -np.inf)
    x[6] = np.finfo(np.float32 if dtype == "float32" else np.float16).min; x[6, 5] = 0    # masked by the type's lowest value
    x[7] = np.finfo(np.float32 if dtype == "float32" else np.float16).min
    x[8] = np.sort(x[8])                               # the largest last, close together
    x[9] = np.sort(x[9])[::-1]
    x[10, :] = np.nan
    x[11] = -0.0; x[11, ::2] = 0.0                     # the two zeros tie
    x[12] = np.where(np.arange(vocab) < 3, 5.0, -np.inf)       # fewer than are asked for
    x[13] *= 30
    d = torch.from_numpy(np.ascontiguousarray(x)).to(torch_dev).to(getattr(torch, dtype))
    x = d.float().cpu().numpy()
    tokens = r.integers(0, vocab, len(x))
    tokens[1], tokens[9], tokens[13] = vocab // 2, -1, vocab
    top = min(9, vocab)
    compare(call(pkg, torch, d, tokens, top), want(x, tokens, top), vocab)


@pytest.mark.parametrize("stride", [4 * 512, 8 * 512, 4])
def test_large_values_that_crowd_in_few_threads(pkg, torch_dev, stride):
    """The likeliest tokens all lie in the pieces of a few threads, more of them than there is room for."""
    import torch
    rows, vocab = 400, 200000                          # one CTA a row
    x = torch.randn(rows, vocab, generator=torch.Generator(device=torch_dev).manual_seed(3), device=torch_dev)
    for i in range(12):
        x[:, i * 4:: stride] += 20
    tokens = np.arange(rows)
    compare([v[:4] for v in call(pkg, torch, x, tokens, 32)], want(x[:4].cpu().numpy(), tokens[:4], 32), vocab)
    y = x[:1].contiguous()
    compare(call(pkg, torch, y, tokens[:1], 32), want(y.cpu().numpy(), tokens[:1], 32), vocab)


def test_outputs_one_by_one(pkg, torch_dev):
    import torch
    x = torch.randn(4, 1003, device=torch_dev)
    tokens = [1, 2, 3, 1002]
    full, ref = call(pkg, torch, x, tokens, 4), want(x.cpu().numpy(), tokens, 4)
    compare(full, ref, 1003)
    for what in ("t", "e", "te"):
        lp, en, _, _ = call(pkg, torch, x, tokens, 0, what=what)
        assert np.array_equal(lp, full[0] if "t" in what else np.full(4, 77, np.float32)) and np.array_equal(en, full[1] if "e" in what else np.full(4, 77, np.float32))
    lp, en, ids, best = call(pkg, torch, x, tokens, 4, what="")
    assert (lp == 77).all() and (en == 77).all() and (ids == -7).all() and np.array_equal(best, full[3])


def test_streams_and_graphs(pkg, torch_dev):
    import torch
    x = torch.randn(3, 5001, device=torch_dev)
    side = torch.cuda.Stream()
    a = call(pkg, torch, x, [1, 2, 3], 5, stream=side.cuda_stream)
    out = [torch.zeros(3, device=torch_dev), torch.zeros(3, device=torch_dev), torch.zeros(3, 5, dtype=torch.int32, device=torch_dev), torch.zeros(3, 5, device=torch_dev)]
    tk = torch.tensor([1, 2, 3], dtype=torch.int32, device=torch_dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pkg.check(pkg.lib.cmlb200_token_scores(x.data_ptr(), pkg.DT_F32, 5001, 3, 5001, tk.data_ptr(), 5, *(o.data_ptr() for o in out), torch.cuda.current_stream().cuda_stream))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(out, a))
        x.copy_(torch.randn(3, 5001, device=torch_dev))
        a = call(pkg, torch, x, [1, 2, 3], 5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab,top", [(3, 2), (1000, 32), (5003, 1), (16383, 0)])
def test_many_short_rows(pkg, torch_dev, dtype, vocab, top):
    """Enough rows that each is read by few threads; some of special values among them."""
    import torch
    x = torch.randn(900, vocab, generator=torch.Generator(device=torch_dev).manual_seed(vocab), device=torch_dev) * 2
    x[10] = -float("inf")
    x[20, ::2] = -float("inf")
    x[30, 1] = float("nan")
    x[40] = 0
    x = x.to(getattr(torch, dtype))
    tokens = np.random.default_rng(vocab).integers(0, vocab, 900)
    compare(call(pkg, torch, x, tokens, top), want(x.float().cpu().numpy(), tokens, top), vocab)


@pytest.mark.parametrize("rows", [1, 900])
def test_logits_far_from_zero(pkg, torch_dev, rows):
    """The result knows differences alone. An exponent is off by a rounding of itself, wherever the row lies; numbers whose products overflow included."""
    import torch
    vocab = 4099
    x = np.random.default_rng(rows).standard_normal((rows, vocab)).astype(np.float32)
    for r, shift in zip(range(rows), [9000.0] * (rows == 1) or np.tile([5e4, -5e4, 1e6, -3e6, 0.0], rows)):
        x[r] += np.float32(shift)
    if rows > 1:
        x[50] = np.float32(-3.4e38); x[50, 7] = np.float32(-1e37)
        x[51] = np.float32(3e38); x[51, ::3] = np.float32(2.9e38)
        x[52, ::5] = np.float32(-2e38)
        x[53] = np.linspace(-1e38, 1e38, vocab, dtype=np.float32)
        x[54] = np.sort(x[54]); x[54, 4000:] += np.float32(100)
        x[55] = np.linspace(-50, 50, vocab, dtype=np.float32)             # the reference moves all the way
    tokens = np.random.default_rng(5).integers(0, vocab, rows)
    got, ref = call(pkg, torch, torch.from_numpy(x).to(torch_dev), tokens, 7), want(x, tokens, 7)
    compare(got, ref, vocab)
