"""Tokens drawn, drafts verified and sequences cut short through the models."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

import drafts_oracle
import lm_util
from lm_util import error
from test_gpu_lm_serving import feed, load, prompt  # noqa: F401 (load is a fixture)

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
PAGED = ["plain", "mixed", "odd", "latent", "latent_odd"]
STATES = ["streams", "loops_windows"]


def draws(rng, n):
    return rng.integers(0, 2 ** 64, n, dtype=np.uint64)


@pytest.mark.parametrize("name", PAGED + STATES)
@pytest.mark.parametrize("dtype", [6, 0])
def test_sampled(synth, tmp_path, load, name, dtype):  # noqa: F811
    """Every wanted row's token is the one that its logits and random number give, whatever portions the rows come in."""
    cfg, w, folder = lm_util.build(synth, tmp_path, name)
    rng = np.random.default_rng(2)
    m = load(folder, dtype)
    for sizes in ([40], [1] * 5, [3, 1, 20]):
        a, at, unsure = m.open(), 0, 0
        t = prompt(cfg, sum(sizes), 3)
        for k in sizes:
            b = m.fork(a)
            logits = m.step([(a, t[at:at + k], None)])[0]
            heat, key = rng.choice([0.0, 0.5, 1.0, 2.0], k).astype(np.float32), draws(rng, k)
            got = m.sampled([(b, t[at:at + k], None)], heat, key)
            for i in range(k):
                want = drafts_oracle.verify(logits[i][None], [], None, float(heat[i]), int(key[i]))
                unsure += want[2]
                assert want[2] or got[i] == want[1], (i, got[i], want)
            m.end(b)
            at += k
        m.end(a)
        assert unsure <= 2


@pytest.mark.parametrize("name", PAGED)
@pytest.mark.parametrize("cache", [0, 1])
def test_verified(pkg, synth, tmp_path, load, name, cache):  # noqa: F811
    """Kept drafts and next tokens as the logits of the same rows say; sequences then go on like ones that never had the others."""
    if cache and name.startswith("latent"):
        pytest.skip("latents have no 8-bit cache")
    cfg, w, folder = lm_util.build(synth, tmp_path, name)
    rng = np.random.default_rng(4)
    m = load(folder, cache=cache)
    seqs, lines = [m.open() for _ in range(3)], [list(prompt(cfg, n, n)) for n in (37, 16, 90)]
    for s, t in zip(seqs, lines):
        m.step([(s, t, [])])
    kept_all = []
    for r in range(6):
        copies = [m.fork(s) for s in seqs]
        entries = [[int(rng.integers(cfg["vocab"]))] for _ in seqs]
        for e, c in zip(entries, copies):                                 # drafts: what the model itself would say, mostly
            d = m.fork(c)
            for _ in range(int(rng.integers(0, 6))):
                e.append(int(m.step([(d, [e[-1]], None)], greedy=True)[0][0]) if rng.random() < 0.8 else int(rng.integers(cfg["vocab"])))
            m.end(d)
        logits = m.step([(c, e, None) for c, e in zip(copies, entries)])
        heat, key = np.array([0.0, 0.3, 1.0], np.float32), draws(rng, 3)
        kept, after = m.verified(list(zip(seqs, entries)), heat, key)
        for i in range(3):
            want = drafts_oracle.verify(logits[i], entries[i][1:], None, float(heat[i]), int(key[i]))
            assert want[2] or (kept[i], after[i]) == want[:2], (r, i, kept[i], after[i], want)
            lines[i] += entries[i][:1 + kept[i]]
            assert pkg.lib.cml_lm_sequence_length(m.h, seqs[i]) == len(lines[i])
            kept_all.append(int(kept[i]))
        for c in copies:
            m.end(c)
    assert max(kept_all) > 1 and min(kept_all) == 0
    for s, t in zip(seqs, lines):
        fresh = m.open()
        want = m.step([(fresh, t + [1, 2, 3], None)])[0][-3:]
        # (8-bit caches: dropped tokens may have left a group a larger scale)
        assert error(m.step([(s, [1, 2, 3], None)])[0], want) < (0.1 if cache else 2 * lm_util.TOL[6])
        m.end(fresh)


def test_truncate(pkg, synth, tmp_path, load):  # noqa: F811
    """Windows of 16 and 17 tokens: behind 100, the blocks in front of token 80 were let go of, so 96 tokens are the least that a sequence may keep (or none at all)."""
    cfg, w, folder = lm_util.build(synth, tmp_path, "plain")
    m = load(folder)
    t = list(prompt(cfg, 100))
    want = lm_util.reference(cfg, w, t)
    for length in (99, 97, 96):
        s = m.open()
        feed(m, s, t, [100])
        m.truncate(s, length)
        assert pkg.lib.cml_lm_sequence_length(m.h, s) == length
        assert error(feed(m, s, t[length:], [100]), want[length:]) < lm_util.TOL[6]
        for bad in (-1, 101, 95, 20, 1):
            with pytest.raises(pkg.CmlB200Error):
                m.truncate(s, bad)
        m.end(s)
    with pytest.raises(pkg.CmlB200Error):
        m.truncate(0, 0)
    free = pkg.lib.cml_lm_blocks_free(m.h)
    s = m.open()
    m.step([(s, t[:15], [])])
    m.truncate(s, 0)
    assert pkg.lib.cml_lm_blocks_free(m.h) == free and error(feed(m, s, t[:30], [30]), want[:30]) < lm_util.TOL[6]


def test_shared_blocks_are_not_cut_into(pkg, synth, tmp_path, load):  # noqa: F811
    cfg, w, folder = lm_util.build(synth, tmp_path, "mixed")
    m = load(folder)
    t = list(prompt(cfg, 40))
    a = m.open()
    m.step([(a, t, [])])
    b = m.fork(a)
    with pytest.raises(pkg.CmlB200Error):
        m.truncate(a, 31)
    m.truncate(a, 32)                                                     # the border of a shared block
    m.truncate(b, 35)
    want = lm_util.reference(cfg, w, t)
    assert error(feed(m, a, t[32:], [8]), want[32:]) < lm_util.TOL[6]
    assert error(feed(m, b, t[35:], [5]), want[35:]) < lm_util.TOL[6]


@pytest.mark.parametrize("name", STATES)
def test_models_with_states(pkg, synth, tmp_path, load, name):  # noqa: F811
    cfg, w, folder = lm_util.build(synth, tmp_path, name)
    m = load(folder)
    s = m.open()
    m.step([(s, prompt(cfg, 20), [])])
    with pytest.raises(pkg.CmlB200Error):
        m.truncate(s, 19)
    m.truncate(s, 20)
    with pytest.raises(pkg.CmlB200Error):
        m.verified([(s, [1, 2])], 0.0)
    assert pkg.lib.cml_lm_sequence_length(m.h, s) == 20
    kept, after = m.verified([(s, [1])], 0.0)
    assert kept[0] == 0 and 0 <= after[0] < cfg["vocab"] and pkg.lib.cml_lm_sequence_length(m.h, s) == 21
    with pytest.raises(pkg.CmlB200Error):
        m.generate_drafted(load(folder), 2, [1, 2], 4)


def test_what_is_refused(pkg, synth, tmp_path, load):  # noqa: F811
    cfg, w, folder = lm_util.build(synth, tmp_path, "plain")
    m = load(folder, max_sequences=2)
    s = m.open()
    m.step([(s, [1, 2, 3], [])])
    L = pkg.lib
    for bad in (lambda: m.sampled([(s, [1], None)]), lambda: m.sampled([(s, [1], None)], 1.0), lambda: m.sampled([(s, [1], None)], np.inf, [1]), lambda: m.sampled([(s, [99999], None)], 0.0),
                lambda: m.verified([(s, [1, 2])]), lambda: m.verified([(s, [])], 0.0), lambda: m.verified([(s, [1] * 257)], 0.0), lambda: m.verified([(s, [1]), (s, [2])], 0.0),
                lambda: m.verified([(s, [1, 99999])], 0.0), lambda: m.verified([(1, [1, 2])], 0.0), lambda: m.verified([(s, [1])] * 3, 0.0),
                lambda: m.generate_drafted(m, 2, [1, 2], 4), lambda: m.generate_drafted(load(folder), 0, [1, 2], 4), lambda: m.generate_drafted(load(folder), 33, [1, 2], 4)):
        with pytest.raises(pkg.CmlB200Error):
            bad()
        assert L.cml_lm_sequence_length(m.h, s) == 3
    other = load(lm_util.build(synth, tmp_path, "mixed")[2])
    with pytest.raises(pkg.CmlB200Error):
        m.generate_drafted(other, 2, [1, 2], 4)                           # another vocabulary
    assert L.cml_lm_step_sampled(None, None, 0, None, None, None) == -1 and L.cml_lm_step_verified(None, None, 0, None, None, None, None) == -1


@pytest.mark.parametrize("drafts", [1, 4, 9])
@pytest.mark.parametrize("name", PAGED)
def test_generation(synth, tmp_path, load, name, drafts):  # noqa: F811
    """Greedy: every token has (nearly) the largest logit behind those in front of it, with the model itself, its 8-bit form and another model of the vocabulary as drafters. Prompts longer than a step.
    The model itself is kept but for tokens that are so nearly the largest that a step of several rows and one of a single row see them differently: two of those at most, which cost a run of drafts each."""
    cfg, w, folder = lm_util.build(synth, tmp_path, name)
    other = lm_util.build(synth, tmp_path, name, seed=5)[2]
    m = load(folder, max_step_rows=40)
    t = list(prompt(cfg, 90))
    for drafter, itself in ((load(folder), True), (load(folder, weights=1, max_step_rows=24), False), (load(other), False)):
        got, (steps, drafted, accepted) = m.generate_drafted(drafter, drafts, t, 60)
        assert len(got) == 60 and steps <= 60 and 0 <= accepted <= drafted and (not itself or accepted >= drafted - 2 * drafts)
        logits = lm_util.reference(cfg, w, t + got)[len(t) - 1:-1]
        short = logits.max(1) - logits[np.arange(60), got]
        assert (short <= 6 * lm_util.TOL[6] * logits.std()).all(), short.max() / logits.std()
        assert pkg_free(m) and pkg_free(drafter)


def pkg_free(m):
    from __graft_entry__ import load_package
    L = load_package().lib
    return L.cml_lm_blocks_free(m.h) == L.cml_lm_blocks_total(m.h)


def test_generation_ends(synth, tmp_path, load):  # noqa: F811
    """At the end token, wherever among kept drafts it comes; and at the number asked for."""
    cfg, w, folder = lm_util.build(synth, tmp_path, "plain")
    m, d = load(folder), load(folder)
    t = list(prompt(cfg, 20))
    whole, _ = m.generate_drafted(d, 4, t, 40)
    for n in (1, 2, 3, 5, 6, 39):
        assert m.generate_drafted(d, 4, t, n)[0] == whole[:n]
    for eos in set(whole):
        assert m.generate_drafted(d, 4, t, 40, eos=eos)[0] == whole[:whole.index(eos) + 1]


def test_short_steps(synth, tmp_path, load):  # noqa: F811
    """Steps of a few tokens: as many drafts as go into one, a drafter that takes what it has not seen one by one, and no drafts where a step is a single token."""
    cfg, w, folder = lm_util.build(synth, tmp_path, "plain")
    t = list(prompt(cfg, 20))
    for rows, draft_rows in ((3, 1), (1, 1), (2, 2), (1, 40)):
        m, d = load(folder, max_step_rows=rows), load(folder, max_step_rows=draft_rows)
        got, (steps, drafted, accepted) = m.generate_drafted(d, 4, t, 30)
        assert len(got) == 30 and drafted <= steps * (rows - 1) and (drafted > 0) == (rows > 1)
        logits = lm_util.reference(cfg, w, t + got)[len(t) - 1:-1]
        assert (logits.max(1) - logits[np.arange(30), got] <= 6 * lm_util.TOL[6] * logits.std()).all()


def test_lengths_out_of_range(pkg, synth, tmp_path, load):  # noqa: F811
    cfg, w, folder = lm_util.build(synth, tmp_path, "plain")
    m, d = load(folder), load(folder)
    for n in (2 ** 31 - 1, 2 ** 31 - 40, 20000):        # (more than numbers, or the pool, hold: what was taken is given back)
        with pytest.raises(pkg.CmlB200Error):
            m.generate_drafted(d, 4, list(prompt(cfg, 30)), n)
        assert pkg_free(m) and pkg_free(d)


def test_sampled_generation(synth, tmp_path, load):  # noqa: F811
    """Drafted generation has the model's own distribution: third tokens of many runs, beside what the model's probabilities say of them, with a drafter that is another model."""
    cfg, w, folder = lm_util.build(synth, tmp_path, "plain")
    other = lm_util.build(synth, tmp_path, "plain", seed=7)[2]
    m, d = load(folder), load(other)
    t, runs, heat = list(prompt(cfg, 9)), 1500, 1.5
    first = drafts_oracle.chances(m.step([(m.open(), t, None)])[0][-1], heat)
    got = [tuple(m.generate_drafted(d, 2, t, 3, heat, seed)[0]) for seed in range(runs)]
    assert len(set(got)) > runs // 3
    # the distribution of the first two tokens by the model, summed over the first: what second tokens have
    top, seqs = np.arange(cfg["vocab"]), []
    second, third = np.zeros(cfg["vocab"]), 0
    s = m.open()
    m.step([(s, t, [])])
    for a in top:
        c = m.fork(s)
        second += first[a] * drafts_oracle.chances(m.step([(c, [a], None)])[0][0], heat)
        m.end(c)
    for place, p in ((0, first), (1, second)):
        count = np.bincount([g[place] for g in got], minlength=cfg["vocab"])
        big = p * runs >= 5
        seen, want = np.append(count[big], count[~big].sum()), np.append(p[big], p[~big].sum()) * runs
        freedom = len(want) - 1
        chi = ((seen - want) ** 2 / np.maximum(want, 1e-9)).sum()
        assert chi < freedom + 6 * np.sqrt(2 * freedom) + 6, (place, chi, freedom)


def test_program(synth, tmp_path):
    """cml_generate with 8-bit weights, and with drafts of the model's 8-bit form."""
    cfg, w, folder = lm_util.build(synth, tmp_path, "mixed")
    run = lambda *a: subprocess.run([str(ROOT / "bin" / "cml_generate"), "--model", str(folder), "--tokens", "5,6,7,8,9", "--tokens", "1,2", "--max-new", "12", *a], capture_output=True, text=True, timeout=300)
    for extra in ((), ("--weights", "int8"), ("--drafts", "3"), ("--drafts", "2", "--temperature", "0.9", "--seed", "4"), ("--drafts", "2", "--drafter", str(folder))):
        r = run(*extra)
        lines = [x.split("\t")[0].split() for x in r.stdout.splitlines()]
        assert r.returncode == 0 and [len(x) for x in lines] == [12, 12], (extra, r.stderr[-500:])
    assert run("--drafts", "2", "--temperature", "0.9", "--seed", "4").stdout == run("--drafts", "2", "--temperature", "0.9", "--seed", "4").stdout
    for bad in (("--weights", "int4"), ("--drafts", "0"), ("--drafts", "40"), ("--drafts", "x"), ("--drafter", str(folder)), ("--drafts", "2", "--top-k", "5", "--temperature", "1")):
        assert run(*bad).returncode == 2, bad
