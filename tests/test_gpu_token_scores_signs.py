"""Token scores at the ends of their range: a certain token has exactly 0, nothing is more than certain, and few values far apart keep their digits."""
import numpy as np
import pytest

from test_gpu_token_scores import TYPES, call, want

pytestmark = pytest.mark.gpu
SIZES = [(1, 1), (7, 5), (300, 5000), (900, 1003), (3, 70001), (700, 32000)]


def rows_of(torch, dev, x, dtype):
    d = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(dev).to(getattr(torch, dtype))
    return d, d.float().cpu().numpy()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("masked", ["never", "lowest"])
def test_a_certain_token(pkg, torch_dev, dtype, rows, vocab, masked):
    import torch
    r = np.random.default_rng(rows + vocab)
    x = np.full((rows, vocab), -np.inf if masked == "never" else np.finfo(np.float32 if dtype == "float32" else np.float16).min, np.float32)
    at = r.integers(0, vocab, rows)
    x[np.arange(rows), at] = r.standard_normal(rows) * np.exp2(r.uniform(-8, 12, rows))
    d, _ = rows_of(torch, torch_dev, x, dtype)
    lp, en, ids, best = call(pkg, torch, d, at, 1)
    assert (lp == 0).all() and (en == 0).all() and np.array_equal(ids[:, 0], at) and (best == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("steep", [0.01, 1, 8, 60])
def test_nothing_is_more_than_certain(pkg, torch_dev, dtype, rows, vocab, steep):
    import torch
    r = np.random.default_rng(rows + vocab)
    x = r.standard_normal((rows, vocab)) * steep + r.uniform(-50, 50, (rows, 1))
    x[r.random(x.shape) < 0.3] = -np.inf
    x[::2, -1] = 75 + steep                            # one token nearly certain, met last
    d, x = rows_of(torch, torch_dev, x, dtype)
    top = min(5, vocab)
    lp, en, ids, best = call(pkg, torch, d, x.argmax(1), top)
    assert (lp <= 0).all() and (en >= 0).all() and (best <= 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [40, 5000, 70001])
@pytest.mark.parametrize("order", [1, -1])
def test_few_values_apart(pkg, torch_dev, dtype, vocab, order):
    """Two to four values that one thread or several meet, the largest first or last, 0.1 to 8 apart.

    A term below the largest is off by four exponentials at most (its own, and those that bring it to another reference: 2^-22 each) and the rounding of its exponent,
    below 5 2^-22 of itself all together: call that f. With p the largest value's share and d the distances from it, ln S is then off by f (1 - p), and the entropy,
    ln S + sum p d, by f (1 - p + 2 sum p d). Beside that, four values are three additions, each rounded by 2^-24 of a sum of which the largest term is p: 3 2^-24 in ln S. (The
    first form of this bound had 2^-23, two of them: -9, -14.625, -16.5 and -23.375 in one thread's pieces took 2.1.) In the entropy there are as many of Q's terms, which
    are up to 1.45 ln 2 times as large while the reference is below the largest value by 1 at most, and the sum's again in bringing Q to that: 9 2^-24; where it is not
    below, 2^-22 (next test). Both are rounded, and the value's distance from the largest is (2^-24 each): 2^-23 of themselves."""
    import torch
    r = np.random.default_rng(vocab)
    rows = 600
    x = np.full((rows, vocab), -np.inf)
    for i in range(rows):
        n = 2 + i % 3
        at = np.sort(r.choice(vocab, n, replace=False)) if i % 2 else r.integers(0, vocab % 4096 or 1) + np.arange(n) * 4096     # (pieces of one thread)
        at = at[at < vocab]
        x[i, at] = r.uniform(-20, 20) + order * np.cumsum(r.uniform(0.1, 8, len(at)))
    d, x = rows_of(torch, torch_dev, x, dtype)
    got, ref = call(pkg, torch, d, x.argmax(1), 4), want(x, x.argmax(1), 4)
    assert np.array_equal(got[2], ref[2])
    p = np.exp(x.astype(np.float64) - x.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    terms, spread = 5 * 2.0 ** -22 * (1 - p.max(1)), 5 * 2.0 ** -21 * np.where(p > 0, p * np.minimum(x.max(1, keepdims=True) - x, 1e9), 0).sum(1)
    for g, w, few in ((got[0], ref[0], 3 * 2.0 ** -24 + terms), (got[1], ref[1], 9 * 2.0 ** -24 + terms + spread), (got[3], ref[3], (3 * 2.0 ** -24 + terms)[:, None])):
        ok = np.isfinite(w)
        with np.errstate(invalid="ignore"):
            off = np.abs(g - w)
        assert np.array_equal(np.isfinite(g), ok) and (off <= few + 2.0 ** -23 * np.abs(w))[ok].all(), off[ok].max()


@pytest.mark.parametrize("order", [1, -1])
def test_values_five_to_six_apart(pkg, torch_dev, order):
    """Two values of one thread: the smaller one's share is below 0.0067, so what is left of the above is an addition (2^-24) and the result's rounding."""
    import torch
    r = np.random.default_rng(5)
    x = np.full((2000, 9000), -np.inf, np.float32)
    at = r.integers(0, 904, 2000)
    x[np.arange(2000), at] = r.uniform(-20, 20, 2000)
    x[np.arange(2000), at + 4096] = x[np.arange(2000), at] + order * r.uniform(5, 6, 2000).astype(np.float32)
    got, ref = call(pkg, torch, torch.from_numpy(x).to(torch_dev), x.argmax(1), 1), want(x, x.argmax(1), 1)
    assert np.abs(got[0] - ref[0]).max() <= 2.0 ** -22 and np.abs(got[1] - ref[1]).max() <= 2.0 ** -22 and (got[0] <= 0).all() and (got[1] >= 0).all()


def test_tokens_outside_the_vocabulary(pkg, torch_dev):
    """-inf in any row, those of NaN and of nothing among them."""
    import torch
    x = torch.randn(6, 77, device=torch_dev)
    x[1, 5], x[2, 6], x[3] = float("nan"), float("inf"), -float("inf")
    for bad in (-1, 77, 2 ** 31 - 1, -2 ** 31):
        lp, en, _, _ = call(pkg, torch, x, [bad] * 6, 0)
        assert np.isneginf(lp).all() and np.isnan(en[1:3]).all() and en[3] == 0 and np.isfinite(en[[0, 4, 5]]).all()
