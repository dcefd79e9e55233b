"""An 8-bit paged cache and attention over it in numpy and 64 bits: groups of 16 tokens of a head share a power-of-two scale."""
import numpy as np

FULL = {"i8": 127.0, "e4m3": 448.0}
GROUP = 16


def round_codes(x, form):
    """The nearest numbers that codes stand for, ties to even; |x| is at most FULL."""
    x = np.asarray(x, np.float64)
    if form == "i8":
        return np.rint(x)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -60))), -6) - 3)      # three bits behind the leading one, subnormals below 2^-6
    return np.rint(x / step) * step


def scale_for(most, form):
    s = 2.0 ** -126
    if most <= 0:
        return s
    s = max(s, 2.0 ** np.ceil(np.log2(most / FULL[form])))
    while s / 2 * FULL[form] >= most and s / 2 >= 2.0 ** -126:
        s /= 2
    while s * FULL[form] < most:
        s *= 2
    return s


class Sequence:
    """Keys (or values) of one sequence: codes [n, heads, width] in units of scales [groups, heads]."""

    def __init__(self, heads, width, form):
        self.form, self.heads = form, heads
        self.codes = np.zeros((0, heads, width))
        self.scales = np.zeros((0, heads))

    def append(self, x):
        x = np.asarray(x, np.float64)
        x = np.clip(np.where(np.isnan(x), 0.0, x), -65504, 65504)
        at = 0
        while at < len(x):
            n = len(self.codes)
            off = n % GROUP
            part = x[at:at + GROUP - off]
            if off == 0:
                self.scales = np.concatenate([self.scales, np.zeros((1, self.heads))])
            fresh = np.zeros(part.shape)
            for h in range(self.heads):
                s = scale_for(np.abs(part[:, h]).max(), self.form)
                if off:
                    was = self.scales[-1, h]
                    s = max(s, was)
                    if s != was:
                        self.codes[n - off:, h] = round_codes(self.codes[n - off:, h] * (was / s), self.form)
                self.scales[-1, h] = s
                fresh[:, h] = round_codes(part[:, h] / s, self.form)
            self.codes = np.concatenate([self.codes, fresh])
            at += len(part)

    def held(self):
        return self.codes * np.repeat(self.scales, GROUP, 0)[:len(self.codes), :, None]


def visible(p, n, window=0, keep=0, chunk=0):
    """Which of keys 0 .. n - 1 the row at position p sees."""
    j = np.arange(n)
    first = p // chunk * chunk if chunk > 0 else (p - window + 1 if window > 0 else 0)
    return (j <= p) & ((j >= first) | (j < keep))


def attend(q, pos, k, v, scale, slopes=None, sinks=None, window=0, keep=0, chunk=0):
    """q [n, heads, dim] at positions pos over k, v [keys, kv heads, ..]. sinks: per head a score without a value, or None.
    Returns the outputs and what bounds their error: sum of weight * |value|, and the largest sum of |q k| scale of a row and head."""
    n, H, _ = q.shape
    g = H // k.shape[1]
    out, weight, reach = np.zeros((n, H, v.shape[2])), np.zeros((n, H, v.shape[2])), np.zeros((n, H, 1))
    for h in range(H):
        z = q[:, h] @ k[:, h // g].T * scale
        reach[:, h, 0] = (np.abs(q[:, h]) @ np.abs(k[:, h // g]).T * scale).max(1)
        for i, p in enumerate(pos):
            see = visible(p, len(k), window, keep, chunk)
            s = z[i, see] - (slopes[h] * (p - np.nonzero(see)[0]) if slopes is not None else 0.0)
            m = max(s.max(), sinks[h] if sinks is not None else -np.inf)
            e = np.exp(s - m)
            total = e.sum() + (np.exp(sinks[h] - m) if sinks is not None else 0.0)
            out[i, h] = e @ v[see, h // g] / total
            weight[i, h] = e @ np.abs(v[see, h // g]) / total
    return out, weight, reach


def bound(out, weight, reach, most):
    """How far a result in bf16 may be from `out`, whose largest cached value is `most`. Queries are rounded to fp16 (relative 2^-11), so a score is
    off by at most d = 2^-11 reach, and one part in 2^18 for fp32 sums and exponentials; a weight e^s / sum by the factor e^(2 d); weights are rounded to fp16 (2^-11);
    the result to bf16 (2^-8). Below 2^-24 of the largest weight there are no more bits."""
    d = reach * (2.0 ** -11 + 2.0 ** -18) + 2.0 ** -18
    return 2.0 ** -8 * np.abs(out) + (np.expm1(2 * d) + 2.0 ** -11 + 2.0 ** -16) * weight * (1 + 2.0 ** -8) + 2.0 ** -20 * most
