"""Drafts kept and tokens drawn where 32 bits would say otherwise: what 64 bits say comes out."""
import numpy as np
import pytest

import drafts_oracle
from test_gpu_verify import Batch

pytestmark = pytest.mark.gpu


def waits32(words):
    """-ln(1 - v) with v and 1 - v rounded to 32 bits in turn."""
    v = words.astype(np.float32) * np.float32(2.0 ** -32) + np.float32(2.0 ** -33)
    return -np.log(np.maximum(np.float32(1) - v, np.float32(2.0 ** -33)).astype(np.float64))


# keys that have a number v within 2^-17 of 1 among their first 4,096
NEAR_ONE = [4696, 13070, 21403, 21990, 22905, 25665, 32240, 33139, 33309, 37904, 39075, 53892, 57338, 60827, 76520, 76839, 78455, 80362, 85055, 95149, 96227, 96505, 109109, 121855, 131714,
            133384, 134145, 139776, 144082, 148116]


def test_waits_of_numbers_next_to_one(pkg, torch_dev):
    """The longest waits are as exact as the others: of two tokens that come out within a few thousandths, the one that 64 bits prefer is drawn."""
    import torch
    vocab, near_one = 4096, []
    for key in NEAR_ONE:                               # the token, and how far a 32-bit 1 - v moves the logarithm of its wait
        words = drafts_oracle.philox(key, np.arange(1024), 0).reshape(-1)
        j = int(np.argmax(words))
        near_one.append((key, j, float(np.log(waits32(words[j:j + 1])[0] / -np.log1p(-(float(words[j]) + 0.5) / 2.0 ** 32)))))
    assert min(abs(f[2]) for f in near_one) > 0.008 and max(abs(f[2]) for f in near_one) > 0.2
    b = Batch(torch, torch_dev, [0] * len(near_one), vocab, 5)
    b.key = np.array([f[0] for f in near_one], np.uint64)
    x = np.full((len(near_one), vocab), -60.0)
    other = []
    for s, (key, j, off) in enumerate(near_one):
        z = np.log(drafts_oracle.waits(key, vocab))
        k = (j + 1717) % vocab
        other.append(k)
        # logarithms of weights over waits: `off / 2` apart, where a wait that is off by e^off changes places
        x[s, j], x[s, k] = z[j] + off / 2, z[k]
    b.target[:] = torch.from_numpy(x).float()
    got, x = b.call(pkg), b.target.double().cpu().numpy()
    for s, (key, j, off) in enumerate(near_one):
        z = x[s] - np.log(drafts_oracle.waits(key, vocab))
        assert int(np.argmax(z)) == (j if off > 0 else other[s])
        assert got[1][s] == int(np.argmax(z)), (s, off, got[1][s])


def first_coins(keys):
    """u of the first draft, for many keys at once: Philox4x32-10 at counter (0, 1, 0, 0)."""
    u64 = np.uint64
    mask, sh = u64(0xFFFFFFFF), u64(32)
    a, b, c, d = (np.full(keys.shape, x, u64) for x in (0, 1, 0, 0))
    k0, k1 = keys & mask, keys >> sh
    for _ in range(10):
        p, q = a * u64(0xD2511F53), c * u64(0xCD9E8D57)
        a, b, c, d = (q >> sh) ^ b ^ k0, q & mask, (p >> sh) ^ d ^ k1, p & mask
        k0, k1 = (k0 + u64(0x9E3779B9)) & mask, (k1 + u64(0xBB67AE85)) & mask
    return a.astype(np.float64) / 2.0 ** 32


@pytest.fixture(scope="module")
def pool():
    """A few million keys by their first coins."""
    keys = np.random.default_rng(8).integers(0, 2 ** 64, 1 << 22, dtype=np.uint64)
    assert np.array_equal(first_coins(keys[:50]), [drafts_oracle.coins(int(k), 1)[0] for k in keys[:50]])
    u = first_coins(keys)
    order = np.argsort(u)
    return u[order], keys[order]


@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.5])
@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("form,vocab,lead", [("float32", 32000, 0), ("float32", 100003, 1), ("float32", 37, 0), ("bfloat16", 32000, 3), ("float16", 5001, 0)])
def test_coins_next_to_the_chance(pkg, torch_dev, pool, form, vocab, lead, drafter, temperature):
    """Random numbers right below and right above the one at which a draft is turned down: sums of exponentials that hold 32 bits would take one for the other."""
    import torch
    n = 64
    b = Batch(torch, torch_dev, [1] * n, vocab, vocab + n, form, drafter, (temperature,), gap=0.3, lead=lead)
    x = b.target.double().cpu().numpy()
    d = b.draft.double().cpu().numpy() if drafter else None
    t, u, keys = float(b.t[0]), *pool
    want, close = [], 0
    for s in range(n):
        j = int(np.argsort(x[2 * s])[-1 - s % 5])       # a likely token that the drafter finds likelier, so that a coin decides
        b.tokens[s] = j
        p = drafts_oracle.chances(x[2 * s], t)[j]
        q = drafts_oracle.chances(d[s], t)[j] if drafter else 1.0
        i = int(np.searchsorted(u, p / q)) - (s % 2)
        if not 0 <= i < len(u):
            i = 0                                        # (p above q: kept, whatever u is)
        b.key[s] = keys[i]
        assert abs(u[i] * q - p) > 1e-12 * p             # (as far as 64 bits are sure)
        close += abs(u[i] * q - p) < 2e-6 * p
        want.append(int(u[i] * q < p))
    assert (close > n // 8 or not drafter) and 0 < sum(want) < n          # (without a drafter coins of small chances lie further apart)
    got = b.call(pkg)
    assert got[0].tolist() == want
    again = b.call(pkg)
    assert (got == again).all()


def test_every_draft_is_close(pkg, torch_dev, pool):
    """A run of drafts whose chances are exactly the coins of certain words is decided one after another."""
    import torch
    vocab, n = 64, 40
    b = Batch(torch, torch_dev, [n, 3, n], vocab, 4)
    x = b.target.double().cpu().numpy()
    key = [int(k) for k in b.key]
    # two tokens, p of the draft next to the coin: p = 1 / (1 + e^-z), the nearest 32-bit z and the ones beside it
    rows, drafts, kept = [], [], []
    for s, count in enumerate(b.counts):
        u = drafts_oracle.coins(key[s], count)
        done = None
        for i in range(count):
            z = np.float32(np.log(u[i] / (1 - u[i])))
            stop_here = (s, i) in ((0, 37), (1, 1), (2, 33))
            for step in range(-3, 4):                    # the lowest that is kept, or the highest that is not
                y = z
                for _ in range(abs(step)):
                    y = np.nextafter(y, np.float32(np.inf if step > 0 else -np.inf))
                p = 1.0 / (1.0 + np.exp(-float(y)))
                if (u[i] < p) != stop_here and not stop_here:
                    break
                if stop_here and not u[i] < p:
                    chosen = y
            y = chosen if stop_here else y
            row = np.full(vocab, -np.inf)
            row[3], row[9] = float(y), 0.0
            rows.append(row)
            drafts.append(3)
            if done is None and not u[i] < 1.0 / (1.0 + np.exp(-float(y))):
                done = i
        rows.append(x[0])
        kept.append(count if done is None else done)
    b.draft = None
    b.tokens = np.array(drafts, np.int32)
    b.target[:] = torch.from_numpy(np.array(rows)).float()
    assert kept == [37, 1, 33]
    assert b.call(pkg)[0].tolist() == kept


@pytest.mark.parametrize("temperature", [1.0, 0.7])
@pytest.mark.parametrize("vocab,lead", [(3001, 0), (40001, 1), (7, 0)])
@pytest.mark.parametrize("gap", [1e-2, 1e-4, 2e-6])
def test_little_is_left_of_the_difference(pkg, torch_dev, gap, vocab, lead, temperature):
    """A drafter whose chances are nearly the target's: p - q loses its digits in 32 bits, and the token drawn is still the one that 64 bits give. Drafts outside the vocabulary are always turned down."""
    import torch
    n = 48
    b = Batch(torch, torch_dev, [1] * n, vocab, vocab + int(1e7 * gap), "float32", True, (temperature,), gap=gap, lead=lead)
    b.tokens[:] = -1
    got, want = b.call(pkg), b.want()
    x, d = b.target.double().cpu().numpy(), b.draft.double().cpu().numpy()
    for s in range(n):
        p, q = drafts_oracle.chances(x[2 * s], float(b.t[0])), drafts_oracle.chances(d[s], float(b.t[0]))
        with np.errstate(divide="ignore"):
            z = np.log(np.maximum(p - q, 0)) - np.log(drafts_oracle.waits(int(b.key[s]), vocab))
        top = np.sort(z)[-2:]
        assert top[1] - top[0] > 1e-8                    # (64 bits: 2^-53 of p, of a difference of some 1e-7 p)
        assert (got[0][s], got[1][s]) == (0, int(np.argmax(z))) == want[s][:2], (s, got[:, s], want[s])


@pytest.mark.parametrize("form", ["float32", "bfloat16"])
def test_nothing_is_left_of_the_difference(pkg, torch_dev, form):
    """The target's own distribution as the drafter's, from the same logits and from shifted ones: the token is drawn from p."""
    import torch
    n, vocab = 40, 2003
    b = Batch(torch, torch_dev, [1] * n, vocab, 3, form, True)
    b.target.copy_((b.target.float() * 16).round() / 16)
    b.draft.copy_(b.target[::2].float() + (torch.arange(n, device=torch_dev) % 3 * 0.5)[:, None])
    assert torch.equal(b.draft.float() - b.target[::2].float(), (torch.arange(n, device=torch_dev) % 3 * 0.5)[:, None].expand(n, vocab))
    b.tokens[:] = vocab
    got, x = b.call(pkg), b.target.double().cpu().numpy()
    for s in range(n):
        z = np.log(drafts_oracle.chances(x[2 * s], 1.0)) - np.log(drafts_oracle.waits(int(b.key[s]), vocab))
        assert (got[0][s], got[1][s]) == (0, int(np.argmax(z)))


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("vocab,at", [(4, (0, 1, 2)), (4, (0, 1, 2, 3)), (9, (4, 5, 6, 7, 8)), (5000, (0, 1, 2049, 2051)), (40000, (12, 13, 2060, 2061, 4108, 4109)), (300, tuple(range(300)))])
def test_many_close_calls(pkg, torch_dev, vocab, at, drafter):
    """As many tokens as come out nearly equal, however many of them one thread looks at: alone, or as what a drafter's even chances leave."""
    import torch
    n = 200
    b = Batch(torch, torch_dev, [1 if drafter else 0] * n, vocab, 81, "float32", drafter)
    rng, at = np.random.default_rng(vocab), list(at)
    step = 2 if drafter else 1
    for s in range(n):
        row = np.full(vocab, -40.0)
        row[at] = np.log(drafts_oracle.waits(int(b.key[s]), vocab))[at] + rng.normal(size=len(at)) * 2e-6
        b.target[step * s] = torch.from_numpy(row).float()
    if drafter:                                          # q half of p, so that p - q is p / 2 there
        b.tokens[:] = -1
        p = torch.softmax(b.target[::2].double(), 1)
        b.draft.copy_(torch.cat([p[:, :-1] / 2, p[:, -1:] / 2 + 0.5], 1).log().clamp_min(-60).float())
    got = b.call(pkg)
    x, d = b.target.double().cpu().numpy(), b.draft.double().cpu().numpy() if drafter else None
    for s in range(n):
        w = drafts_oracle.chances(x[step * s], 1.0)
        if drafter:
            w = np.maximum(w - drafts_oracle.chances(d[s], 1.0), 0)
        with np.errstate(divide="ignore"):
            z = np.log(w) - np.log(drafts_oracle.waits(int(b.key[s]), vocab))
        top = np.sort(z)[-2:]
        if top[1] - top[0] > 1e-12:
            assert (got[0][s], got[1][s]) == (0, int(np.argmax(z))), (s, np.sort(z)[-4:] - z.max(), z[got[1][s]] - z.max())


def admissible(b, s, kept):
    """Tokens that may follow sequence s's first `kept` drafts where 64 bits are sure to 1e-12 of p: one, but for differences of nearly equal chances."""
    f, n, t = b.first[s], b.counts[s], float(b.t[s])
    x, wait = b.target[f + kept].double().cpu().numpy(), np.log(drafts_oracle.waits(int(b.key[s]), b.vocab))
    if not t >= drafts_oracle.GREEDY:
        return {int(np.argmax(x))}
    p = drafts_oracle.chances(x, t)
    with np.errstate(divide="ignore"):
        plain = int(np.argmax(np.log(p) - wait))
        if kept == n:
            return {plain}
        if b.draft is None:
            j = int(b.tokens[f - s + kept])
            w = np.where(np.arange(b.vocab) == j, 0.0, p) if 0 <= j < b.vocab else p
            return {int(np.argmax(np.log(w) - wait)) if w.max() > 0 else plain}
        q = drafts_oracle.chances(b.draft[f - s + kept].double().cpu().numpy(), t)
        sure, most = np.log(np.maximum(p - q - 1e-12 * p, 0)) - wait, np.log(np.maximum(p - q + 1e-12 * p, 0)) - wait
    fine = {int(j) for j in np.flatnonzero((most >= sure.max()) & (most > -np.inf))}
    return fine if sure.max() > -np.inf else fine | {plain}


@pytest.mark.parametrize("form", ["float32", "bfloat16"])
@pytest.mark.parametrize("spread,temperature", [(0.0, 1.0), (0.01, 1.0), (30.0, 1.0), (300.0, 1.0), (2.0, 0.01), (2.0, 1e-4), (2.0, 100.0), (2.0, 1.0), (2.0, 9e-6)])
@pytest.mark.parametrize("drafter,gap", [(True, 0.2), (True, 1e-3), (False, 0.2)])
def test_every_sequence(pkg, torch_dev, spread, temperature, drafter, gap, form):
    """Flat and steep distributions, drafters near and far, some drafts from outside: all sequences as 64 bits have them, close calls among them."""
    import torch
    b = Batch(torch, torch_dev, [3, 0, 1, 2, 1] * 40, 3001, 18, form, drafter, (temperature,), gap * max(spread, 1e-3), spread)
    b.tokens[::7] = -1
    got, want, several = b.call(pkg), b.want(), 0
    for s, w in enumerate(want):
        fine = admissible(b, s, w[0])
        several += len(fine) > 1
        assert got[0][s] == w[0] and got[1][s] in fine, (s, got[:, s], w, fine)
    assert several <= 0.05 * len(want) or temperature / max(spread, 1e-3) < 0.1      # (steep: one token has all of p and of q, as far as 64 bits go)


@pytest.mark.parametrize("offset", [4096.0, 1e6, -1e30])
def test_every_sequence_far_from_zero(pkg, torch_dev, offset):
    import torch
    b = Batch(torch, torch_dev, [2, 0, 1] * 30, 2000, 72, gap=0.3)
    b.target += offset
    b.draft -= offset / 4
    got, want = b.call(pkg), b.want()
    for s, w in enumerate(want):
        assert (got[0][s], got[1][s]) == w[:2], (s, got[:, s], w)


@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("form,vocab,rise", [("float32", 200003, 1.0), ("float32", 200003, 60.0), ("float32", 1 << 20, 3.0), ("float16", 300000, 40.0), ("float32", 70000, -200.0), ("float32", 70000, 20000.0)])
def test_rows_that_rise(pkg, torch_dev, form, vocab, rise, drafter):
    """Every group of tokens has a larger logit than those in front of it: references change as often as they may."""
    import torch
    counts = [1, 0, 2] * 8
    b = Batch(torch, torch_dev, counts, vocab, 90, form, drafter, (1.0, 0.8))
    line = torch.linspace(0, rise, vocab, device=torch_dev)
    b.target[:] = (line + 0.01 * b.target.float()).to(b.target.dtype)
    if drafter:
        b.draft[:] = (line.flip(0) * 0.5 + 0.01 * b.draft.float()).to(b.draft.dtype)
    b.tokens[1::3] = -1
    got, want = b.call(pkg), b.want()
    for s, w in enumerate(want):
        assert got[0][s] == w[0] and got[1][s] in admissible(b, s, w[0]), (s, got[:, s], w)
