"""Verification of drafted tokens in 64 bits, sequence by sequence, from its definition."""
import numpy as np

GREEDY = 1e-5


def philox(key, c0, c1):
    """Philox4x32-10 (Salmon and others 2011) at counters (c0, c1, 0, 0): [len(c0), 4] words."""
    u64 = np.uint64
    mask, sh = u64(0xFFFFFFFF), u64(32)
    a = np.asarray(c0, u64)
    b, c, d = np.full(a.shape, c1, u64), np.zeros(a.shape, u64), np.zeros(a.shape, u64)
    k0, k1 = int(key) & 0xFFFFFFFF, (int(key) >> 32) & 0xFFFFFFFF
    for _ in range(10):
        p, q = a * u64(0xD2511F53), c * u64(0xCD9E8D57)
        a, b, c, d = (q >> sh) ^ b ^ u64(k0), q & mask, (p >> sh) ^ d ^ u64(k1), p & mask
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack([a, b, c, d], -1)


def waits(key, vocab):
    """The exponentials of all tokens."""
    w = philox(key, np.arange((vocab + 3) // 4), 0).reshape(-1)[:vocab].astype(np.float64)
    return -np.log1p(-(w + 0.5) / 2.0 ** 32)


def coins(key, n):
    return philox(key, np.arange((n + 3) // 4), 1).reshape(-1)[:n].astype(np.float64) / 2.0 ** 32 if n else np.zeros(0)


def chances(row, t):
    """softmax, or None where the row holds no distribution."""
    row = np.asarray(row, np.float64)
    if np.isnan(row).any() or np.isposinf(row).any() or np.isneginf(row).all():
        return None
    e = np.exp((row - row.max()) / t)
    return e / e.sum()


def verify(target, drafts, drafter, t, key):
    """target [n + 1, vocab], drafts [n], drafter [n, vocab] or None. Returns kept, token, and whether rounding in 32 bits could have said otherwise."""
    vocab, n, unsure = target.shape[1], len(drafts), False
    if not t >= GREEDY:
        for i in range(n + 1):
            row = target[i]
            if np.isnan(row).any() or np.isposinf(row).any() or np.isneginf(row).all():
                return i, -1, False
            best = int(np.argmax(row))
            if i == n or best != drafts[i]:
                return i, best, False
    u, i, q, p = coins(key, n), 0, None, chances(target[0], t)
    while i < n:
        if p is None:
            return i, -1, unsure
        d, q = drafts[i], None
        inside = 0 <= d < vocab
        if drafter is not None:
            q = chances(drafter[i], t)
        qd = (q[d] if q is not None else 1.0) if inside else None
        if inside:
            unsure |= bool(abs(u[i] * qd - p[d]) <= 1e-5 * p[d])
        if not inside or not u[i] * qd < p[d]:
            break
        i += 1
        p, q = chances(target[i], t), None
    if p is None:
        return i, -1, unsure
    w = p
    if i < n:
        if q is not None:
            w = np.maximum(p - q, 0.0)
        elif 0 <= drafts[i] < vocab:
            w = np.where(np.arange(vocab) == drafts[i], 0.0, p)
        if not w.max() > 0:
            w, q = p, None
    with np.errstate(divide="ignore"):
        z = np.log(w) - np.log(waits(key, vocab))
        # what 32 bits' rounding of p and q moves a logarithm of p - q by
        blur = 1e-6 + (4e-7 * p / np.maximum(w, 1e-300) if i < n and q is not None else 0.0)
    best = int(np.argmax(z))
    rivals = (z + blur >= z[best] - (blur[best] if np.ndim(blur) else blur)) & (w > 0)
    rivals[best] = False
    return i, best, unsure or bool(rivals.any())
