"""What the entry points of 8-bit products and drafted tokens refuse (every one of these calls returns before it reaches a device), and the arithmetic that their tests rest on."""
import ctypes as C

import numpy as np
import pytest

import drafts_oracle

P = 1 << 20                                            # a pointer that nothing follows


@pytest.mark.parametrize("args", [(None, 0, 10, 1, 10, P, 128, P), (P, 0, 10, 1, 10, None, 128, P), (P, 0, 10, 1, 10, P, 128, None), (P, 0, 10, 0, 10, P, 128, P), (P, 0, 10, -1, 10, P, 128, P),
                                  (P, 0, 9, 1, 10, P, 128, P), (P, 0, 10, 1, 0, P, 128, P), (P, 0, 1 << 20, 1, 131072, P, 131072, P), (P, 0, 10, 1, 10, P, 64, P), (P, 0, 200, 1, 200, P, 128, P),
                                  (P, 0, 10, 1, 10, P + 8, 128, P), (P, 0, 10, 1, 10, P, 128, P + 2), (P + 2, 0, 10, 1, 10, P, 128, P), (P + 1, 1, 10, 1, 10, P, 128, P), (P, 3, 10, 1, 10, P, 128, P),
                                  (P, -1, 10, 1, 10, P, 128, P)])
def test_quantize_rows(pkg, args):
    assert pkg.lib.cmlb200_quantize_rows(*args, None) == -1 and pkg.last_error()


def weight(pkg, **kw):
    return pkg.Dense8(**{**dict(rows=32, cols=100, ld=128, w=P, scale=P), **kw})


BAD = [dict(w=None), dict(scale=None), dict(rows=0), dict(cols=0), dict(cols=129), dict(cols=131072, ld=131072), dict(ld=100), dict(ld=192), dict(ld=0), dict(w=P + 8), dict(scale=P + 2), dict(bias=P + 1)]


@pytest.mark.parametrize("bad", BAD)
def test_weights(pkg, bad):
    w, L = weight(pkg, **bad), pkg.lib
    assert L.cmlb200_linear_dense8(w, P, 1, 200, 1, P, 200, P, None) == -1 and pkg.last_error()
    if "bias" not in bad:
        assert L.cmlb200_linear_dense8_glu(w, P, 1, 200, 1, 16, 0, P, 200, P, None) == -1 and pkg.last_error()


@pytest.mark.parametrize("args", [(None, 1, 100, 1, P, 32, P), (P, 1, 100, 1, None, 32, P), (P, 1, 100, 1, P, 32, None), (P, 1, 99, 1, P, 32, P), (P, 1, 100, 0, P, 32, P), (P, 1, 100, 1 << 21, P, 32, P),
                                  (P, 1, 100, 1, P, 31, P), (P, 3, 100, 1, P, 32, P), (P + 1, 1, 100, 1, P, 32, P), (P, 1, 100, 1, P + 2, 32, P), (P, 1, 100, 1, P, 32, P + 8)])
def test_products(pkg, args):
    assert pkg.lib.cmlb200_linear_dense8(weight(pkg), *args, None) == -1
    assert pkg.lib.cmlb200_linear_dense8(None, P, 1, 100, 1, P, 32, P, None) == -1


@pytest.mark.parametrize("args", [(P, 1, 100, 1, 0, 0, P, 16, P), (P, 1, 100, 1, 17, 0, P, 32, P), (P, 1, 100, 1, 16, 2, P, 16, P), (P, 1, 100, 1, 16, 4, P, 16, P), (P, 1, 100, 1, 16, -1, P, 16, P),
                                  (P, 1, 100, 1, 16, 0, P, 15, P), (P, 1, 100, 1, 16, 0, P + 1, 16, P), (P, 1, 100, 0, 16, 0, P, 16, P), (P, 1, 100, 1, 16, 0, None, 16, P)])
def test_gated_products(pkg, args):
    assert pkg.lib.cmlb200_linear_dense8_glu(weight(pkg), *args, None) == -1


def test_workspaces(pkg):
    L = pkg.lib
    assert L.cmlb200_dense8_work_bytes(0, 10, 10) == 0 and L.cmlb200_dense8_work_bytes(1, 0, 10) == 0 and L.cmlb200_dense8_work_bytes(1, 10, 0) == 0
    assert L.cmlb200_dense8_work_bytes(3, 10, 130) >= 3 * 256 + 12 and L.cmlb200_dense8_work_bytes(3, 10, 130) % 16 == 0
    assert L.cmlb200_verify_work_bytes(3, 4) == 0 and L.cmlb200_verify_work_bytes(3, 0) == 0 and L.cmlb200_verify_work_bytes(3, 3) > 0
    assert L.cmlb200_dense8_status(None, 0) == -1


def drafts(pkg, **kw):
    return pkg.Drafts(**{**dict(sequences=2, rows=5, first=P, tokens=P, logits=P, ld=50, temperature=P, random=P), **kw})


@pytest.mark.parametrize("bad", [dict(sequences=0), dict(sequences=-1), dict(rows=1), dict(rows=(1 << 20) + 1), dict(first=None), dict(tokens=None), dict(ld=49), dict(logits=P + 2), dict(random=P + 4),
                                 dict(temperature=None, random=None)])
def test_drafts(pkg, bad):
    assert pkg.lib.cmlb200_verify_drafts(drafts(pkg, **bad), P, 0, 50, 50, P, P, P, None) == -1 and pkg.last_error()


@pytest.mark.parametrize("args", [(None, 0, 50, 50, P, P, P), (P, 0, 49, 50, P, P, P), (P, 0, 50, 0, P, P, P), (P, 0, (1 << 28) + 1, (1 << 28) + 1, P, P, P), (P, 0, 50, 50, None, P, P), (P, 0, 50, 50, P, None, P), (P, 0, 50, 50, P, P, None),
                                  (P, 0, 50, 50, P, P, P + 8), (P + 2, 0, 50, 50, P, P, P), (P, 3, 50, 50, P, P, P), (P + 1, 1, 50, 50, P, P, P)])
def test_verify(pkg, args):
    assert pkg.lib.cmlb200_verify_drafts(drafts(pkg), *args, None) == -1
    assert pkg.lib.cmlb200_verify_drafts(None, P, 0, 50, 50, P, P, P, None) == -1


def test_random_words():
    """The known answers of the generator for counters and keys of zeros and of ones."""
    assert [int(x) for x in drafts_oracle.philox(0, [0], 0)[0]] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert len(set(drafts_oracle.philox(12345, np.arange(1000), 0).reshape(-1).tolist())) > 3990


def chi(counts, p):
    """Chi-square of counts against chances, by its mean and variance."""
    n, keep = counts.sum(), p > 0
    assert (counts[~keep] == 0).all()
    return ((counts[keep] - n * p[keep]) ** 2 / (n * p[keep])).sum(), keep.sum() - 1


@pytest.mark.parametrize("certain", [False, True])
def test_tokens_are_the_targets(certain):
    """Kept draft or drawn token: the first token that a sequence gets is distributed as the target's, whatever the drafter proposes."""
    rng = np.random.default_rng(5)
    vocab, trials = 7, 6000
    target, drafter = rng.normal(size=(2, vocab)) * 1.5, rng.normal(size=(1, vocab)) * 1.5
    p, q = drafts_oracle.chances(target[0], 0.8), drafts_oracle.chances(drafter[0], 0.8)
    counts = np.zeros(vocab)
    for _ in range(trials):
        draft = int(np.argmax(drafter[0])) if certain else int(rng.choice(vocab, p=q))
        kept, token, _ = drafts_oracle.verify(target, [draft], None if certain else drafter, 0.8, int(rng.integers(0, 2 ** 63)))
        counts[draft if kept else token] += 1
    c, freedom = chi(counts, p)
    assert c < freedom + 6 * np.sqrt(2 * freedom) + 6
