"""8-bit caches whose groups' scales lie far apart: what a row cannot see, and what its softmax passes over, must not cost the rest its bits."""
import numpy as np
import pytest

import cache8_oracle as co
from test_gpu_cache8 import FORMS, Layer

pytestmark = pytest.mark.gpu


def reference(L, x, pos, slot):
    """Outputs of the rows x of one sequence, whose keys and values are in L.seqs, and how far results may be off.

    A score is off by at most d = (2^-11 + 2^-18) sum |q k| scale (queries are fp16) + 2^-18, a weight by the factor e^(2 d), and weights are rounded to fp16 (2^-11 of
    themselves) where they are normal numbers. They are held in units in which the largest weight times its group's value scale is at least 2^7, and a subnormal
    number is off by at most 2^-25: so a key's product is off by 2^-32 of that largest one times its code, at most FULL. fp32 sums: 2^-16 of the sum of
    weight * |value|. The result is bf16 (2^-8)."""
    q, _ = L.queries_and_keys(x, pos)
    ks, vs = L.seqs[slot]
    k, v, scales = ks.held()[:, :, :L.D], vs.held()[:, :, :L.V], np.repeat(vs.scales, co.GROUP, 0)[:len(vs.codes)]
    want, tol = np.zeros((len(x), L.H, L.V)), np.zeros((len(x), L.H, L.V))
    see, back = np.array([co.visible(p, len(k), L.window, L.keep, L.chunk) for p in pos]), pos[:, None] - np.arange(len(k))
    for h in range(L.H):
        g = h // (L.H // L.G)
        s = q[:, h] @ k[:, g].T * L.scale - (L.slopes[h] * back if L.slopes is not None else 0.0)
        e = np.where(see, np.exp(np.minimum(s - np.where(see, s, -np.inf).max(1, keepdims=True), 0.0)), 0.0)
        e /= e.sum(1, keepdims=True)
        want[:, h] = e @ v[:, g]
        reach = np.where(see, np.abs(q[:, h]) @ np.abs(k[:, g]).T * L.scale, 0.0).max(1, keepdims=True)
        d = reach * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -18
        floor = 2.0 ** -32 * co.FULL[L.form] * see.sum(1, keepdims=True) * (e * scales[:, g]).max(1, keepdims=True)
        tol[:, h] = 2.0 ** -8 * np.abs(want[:, h]) + (np.expm1(2 * d) + 2.0 ** -11 + 2.0 ** -16) * (e @ np.abs(v[:, g])) * (1 + 2.0 ** -8) + floor + 1e-37
    return want.reshape(len(x), -1), tol.reshape(len(x), -1)


def run(L, slot, x, check=True):
    """Rows of one sequence through the kernels; checks every output."""
    n, had = len(x), len(L.seqs[slot][0].codes)
    pos = had + np.arange(n)
    _, k = L.queries_and_keys(x, pos)
    v = x[:, (L.H + L.G) * L.D:L.width].reshape(n, L.G, L.V)
    for seq, y in zip(L.seqs[slot], (k, v)):
        seq.append(np.concatenate([y, np.zeros(y.shape[:2] + (seq.codes.shape[2] - y.shape[2],))], 2))
    got = L.device(x, pos, np.full(n, slot), [(slot, n)], int(n == 1), {slot: had})
    if not check:
        return got
    want, tol = reference(L, x, pos, slot)
    off = np.abs(got - want) / tol
    assert np.isfinite(got).all() and off.max() <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape), got.flat[off.argmax()], want.flat[off.argmax()])
    return got


def sized(L, n, size):
    """Rows whose values have the sizes `size`; keys are small, so weights are alike."""
    x = L.rng.standard_normal((n, L.ld)).astype(np.float32)
    x[:, (L.H + L.G) * L.D:L.width] *= np.asarray(size, np.float32)[:, None]
    return x


# heads, key/value heads, tokens in front that make the tiles of a portion many or few
FEW, MANY = (8, 2, 70), (32, 8, 1250)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("far", [24, 33, 46])
@pytest.mark.parametrize("what", [{}, dict(slopes=True), dict(window=40)])
@pytest.mark.parametrize("tiles", [FEW, MANY])
def test_later_tokens_are_larger(pkg, torch_dev, form, far, what, tiles):
    """A portion whose last tokens have values 2^far times the first ones': rows see none of what comes behind them."""
    heads, kv_heads, n = tiles
    L = Layer(pkg, torch_dev, form, heads, kv_heads, 64, 64, slots=1, tokens=1400, **what)
    size = np.full(n, 2.0 ** (14 - far))
    size[-20:] = 2.0 ** 14
    if n > 100:
        size[30::64] = 2.0 ** 14                       # in the middle of every tile; behind it rows see a large value among small ones
    run(L, 0, sized(L, n, size))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("tiles", [FEW, MANY])
def test_tokens_in_front_of_the_window_are_larger(pkg, torch_dev, form, tiles):
    heads, kv_heads, n = tiles
    L = Layer(pkg, torch_dev, form, heads, kv_heads, 64, 64, slots=1, tokens=1400, window=17)
    size = np.full(n, 2.0 ** -20)
    size[:16] = 2.0 ** 14
    run(L, 0, sized(L, n, size))
    for _ in range(3):
        run(L, 0, sized(L, 1, [2.0 ** -20]))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,kv_heads,rows", [(8, 2, 40), (32, 8, 1230)])
def test_groups_between_kept_tokens_and_window(pkg, torch_dev, form, heads, kv_heads, rows):
    """Pages that a sequence has let go of belong to somebody else: their scales and codes make no difference, not even one of a bit."""
    import torch
    L = Layer(pkg, torch_dev, form, heads, kv_heads, 64, 64, slots=1, tokens=1700, window=48, keep=5)
    run(L, 0, sized(L, 330, np.full(330, 2.0 ** -6)))
    state = [t.clone() for t in (L.k, L.v, L.ks, L.vs)]
    x, had = sized(L, rows, np.full(rows, 2.0 ** -6)), 330
    pos, given_back, seen = had + np.arange(rows), L.table[0, 1:(had - 47) // 16], []
    for scale, code in ((2.0 ** -20, 0), (2.0 ** 10, 100), (float("nan"), 0x7F)):                # (the last: what nothing may read)
        for t, s in zip((L.k, L.v, L.ks, L.vs), state):
            t.copy_(s)
        for t, y in ((L.k, code), (L.v, code), (L.ks, scale), (L.vs, scale)):
            t[torch.from_numpy(given_back.astype(np.int64)).to(torch_dev)] = y
        seen.append(L.device(x, pos, np.zeros(rows), [(0, rows)], 0, {0: had}))
        assert np.isfinite(seen[-1]).all()
    assert all(np.array_equal(seen[0], s) for s in seen[1:])


def steered(L, n, group, far):
    """Keys of `group` meet the queries of all rows, the others oppose them; values elsewhere are 2^far times as large."""
    x = sized(L, n, np.where(np.arange(n) // 16 == group, 2.0 ** (14 - far), 2.0 ** 14))
    d = L.rng.standard_normal(L.D)
    H, G, D = L.H, L.G, L.D
    x[:, :H * D] = np.tile(d, H) * (1 + 0.05 * L.rng.standard_normal((n, H * D)))
    side = np.where(np.arange(n) // 16 == group, 1.0, -1.0)[:, None]
    x[:, H * D:(H + G) * D] = np.tile(d, G) * side * (1 + 0.05 * L.rng.standard_normal((n, G * D)))
    return x


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("far", [10, 24, 40])
@pytest.mark.parametrize("group", [0, 2])
@pytest.mark.parametrize("tiles", [FEW, MANY])
def test_softmax_passes_over_large_values(pkg, torch_dev, form, far, group, tiles):
    """All of a row's softmax is on keys with small values; large ones are in sight and weigh e^-90 or less."""
    heads, kv_heads, n = tiles
    L = Layer(pkg, torch_dev, form, heads, kv_heads, 64, 64, slots=1, tokens=1400, scale=0.75)
    run(L, 0, steered(L, n, group, far))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("far", [10, 24, 40])
@pytest.mark.parametrize("dim,heads,kv_heads,tokens", [(64, 4, 2, 70), (128, 32, 8, 300), (128, 16, 1, 70), (256, 4, 1, 600), (64, 20, 1, 70), (16, 320, 320, 300), (64, 160, 160, 300)])
def test_decoded_tokens_pass_over_large_values(pkg, torch_dev, form, far, dim, heads, kv_heads, tokens):
    """The same for one row, of few and many heads: a group a warp, and several, the one that counts behind the others."""
    L = Layer(pkg, torch_dev, form, heads, kv_heads, dim, dim, slots=1, tokens=700, scale=48.0 / dim)
    x = steered(L, tokens + 3, tokens // 16 - 1, far)
    run(L, 0, x[:tokens], check=False)
    for i in range(3):
        run(L, 0, x[tokens + i:tokens + i + 1])


@pytest.mark.parametrize("form", FORMS)
def test_decoded_tokens_behind_values_of_all_sizes(pkg, torch_dev, form):
    """Groups from 1e-30 to 1e4 in no order, weights alike and steep."""
    L = Layer(pkg, torch_dev, form, 12, 2, 128, 96, slots=1, tokens=900)
    run(L, 0, sized(L, 800, np.exp(np.repeat(L.rng.uniform(-69, 9, 50), 16))), check=False)
    for s in (1, 1, 30, 300):
        x = sized(L, 1, [1e-12])
        x[:, :L.H * L.D] *= s
        run(L, 0, x)


@pytest.mark.parametrize("form,heads,kv_heads,dim,vdim,what", [("i8", 15, 5, 80, 64, {}), ("e4m3", 25, 5, 64, 128, dict(slopes=True)), ("i8", 36, 3, 72, 40, dict(gate="head")),
                                                               ("e4m3", 24, 8, 13, 24, dict(window=100)), ("i8", 28, 4, 96, 96, dict(kav=True)), ("e4m3", 36, 3, 128, 80, dict(gate="wide")),
                                                               ("i8", 40, 5, 33, 65, dict(gate="wide", sink="own")), ("e4m3", 15, 5, 128, 128, dict(chunk=200, keep=9))])
def test_portions_of_many_tiles_of_other_shapes(pkg, torch_dev, form, heads, kv_heads, dim, vdim, what):
    """Groups of 3, 5, 7, 8 and 12 query heads, key and value sizes that differ and are no multiple of 16, where tiles are many."""
    rows = 64 * -(-148 // (kv_heads * -(-(heads // kv_heads) // 4))) - 9       # as many tiles as a B200 has SMs, or just more
    L = Layer(pkg, torch_dev, form, heads, kv_heads, dim, vdim, slots=2, tokens=rows + 60, spread=0.5, **what)
    L.step([(0, 40), (1, 3)])
    L.step([(0, rows), (1, 2)])
    L.check_cache()
