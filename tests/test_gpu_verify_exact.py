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
