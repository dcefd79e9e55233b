"""Language models with 8-bit caches, sequences that go on from others, pools made dense, and steps that score tokens: each by
itself against the plain restatements, and all of them in one run."""
import subprocess
from pathlib import Path

import numpy as np
import pytest

import lenedra_oracle
import llama_util
import lm_oracle
import lm_util
import zevilorn_oracle
from cache8_oracle import Sequence
from lm_util import TOL, cut, error

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
FORMS = {"i8": 1, "e4m3": 2}
GROUPED = ["mixed", "odd", "wide", "plain", "streams", "streams_odd", "streams_wide", "streams_full", "gated"]


@pytest.fixture
def load(pkg, torch_dev):
    made = []

    def f(folder, dtype=6, **kw):
        made.append(pkg.LanguageModel(folder, dtype, **kw))
        return made[-1]
    yield f
    for m in made:
        m.close()


def build(synth, tmp_path, name, monkeypatch):
    if name == "gated":                               # grouped heads with rotation beside recurrences, and nothing else
        G, S = synth.recurrent_layer, synth.sigmoid_mlp
        cfg = synth.looped_config(133, 96, [G((4, 2, 32, 24, 23), (8, 2000.0), 56, None, 2.5), G((3, 3, 24, 40, 90), (24, 900.0), 130, S(7, 7, 17)), G((12, 1, 64, 64, 400), (64, 1e4), 40, None)],
                                  (0, 2, 2), eps=1e-3)
        monkeypatch.setattr(lm_util, "variants", lambda synth: {"gated": cfg})
    made = lm_util.build(synth, tmp_path, name)
    monkeypatch.undo()
    return made


def held(x, form):
    s = Sequence(x.shape[1], x.shape[2], form)
    s.append(x)
    return s.held()


def with_cache(cfg, w, tokens, form, monkeypatch):
    """The restatement whose attention reads keys and values as 8-bit groups hold them."""
    plain, grouped, score, weigh = lm_oracle.attend, lenedra_oracle.grouped_attention, zevilorn_oracle.scores, zevilorn_oracle.weighted_values
    with monkeypatch.context() as m:
        m.setattr(lm_oracle, "attend", lambda q, k, v, *a: plain(q, held(k, form), held(v, form), *a))
        m.setattr(lenedra_oracle, "grouped_attention", lambda q, k, v, *a, **kw: grouped(q, held(k, form), held(v, form), *a, **kw))
        m.setattr(zevilorn_oracle, "scores", lambda q, k, *a: score(q, held(k, form), *a))
        m.setattr(zevilorn_oracle, "weighted_values", lambda p, v: weigh(p, held(v, form)))
        return lm_util.reference(cfg, w, tokens)


def prompt(cfg, n, seed=1):
    return np.random.default_rng(seed).integers(0, cfg["vocab"], n)


def feed(m, seq, tokens, sizes):
    return np.concatenate([m.step([(seq, tokens[a:b], None)])[0] for a, b in cut(len(tokens), sizes)])


@pytest.mark.parametrize("sizes", [[150], [1], [70, 2, 1, 1, 31], [16, 1, 64, 5]])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("name", GROUPED)
def test_8_bit_caches(synth, tmp_path, load, monkeypatch, name, form, sizes):
    """Against a cache of the same groups in 64 bits. The device's keys and values differ from the restatement's by bf16 products, which is what TOL allows for,
    and where that moves a value across the middle between two codes it ends a step away from the restatement's: an error like the codes' own, whose effect on the
    logits is the distance of the restatement with them from the one without."""
    cfg, w, folder = build(synth, tmp_path, name, monkeypatch)
    t = prompt(cfg, 150)
    plain, want = lm_util.reference(cfg, w, t), with_cache(cfg, w, t, form, monkeypatch)
    m = load(folder, cache=FORMS[form])
    assert error(feed(m, m.open(), t, sizes), want) < TOL[6] + error(want, plain)


@pytest.mark.parametrize("name", ["latent", "loops", "streams"])
def test_8_bit_caches_refused(synth, tmp_path, pkg, torch_dev, monkeypatch, name):
    cfg, w, folder = build(synth, tmp_path, name, monkeypatch)
    for cache in FORMS.values():
        o = pkg.LMOptions(0 if name == "streams" else 6, 256, 2, 0, cache)
        assert not pkg.lib.cml_lm_load(str(folder).encode(), o)


CONTINUED = [("mixed", 6, 0), ("mixed", 0, 0), ("mixed", 6, 1), ("mixed", 6, 2), ("odd", 6, 1), ("latent", 6, 0), ("latent", 0, 0), ("streams", 6, 0), ("streams", 0, 0), ("streams", 6, 2),
             ("streams_odd", 6, 1), ("loops", 6, 0), ("loops", 0, 0), ("loops_windows", 6, 0), ("loops_odd", 6, 0), ("gated", 6, 2)]


@pytest.mark.parametrize("tokens", [1, 16, 61, 128])
@pytest.mark.parametrize("name,dtype,cache", CONTINUED)
def test_forks_go_on_as_their_parents_would(synth, tmp_path, load, monkeypatch, name, dtype, cache, tokens):
    """Two sequences that were fed the same prompt apart, against one and its fork: the same steps give the same numbers, whichever blocks and slots they are in."""
    cfg, w, folder = build(synth, tmp_path, name, monkeypatch)
    t = prompt(cfg, 2 * tokens + 90, tokens)
    x, y = t[tokens:tokens + 40], t[tokens + 40:tokens + 80]
    steps = [(1, 1), (1, 7), (20, 1), (1, 1), (1, 1), (9, 25)]

    def go_on(m, a, b):
        out, i, j = [], 0, 0
        for p, q in steps:
            out += m.step([(a, x[i:i + p], None), (b, y[j:j + q], None)])
            i, j = i + p, j + q
        return out

    apart = load(folder, dtype, max_tokens=2048, max_sequences=4, cache=cache)
    s = [apart.open() for _ in range(2)]
    for k in s:
        feed(apart, k, t[:tokens], [50])
    want = go_on(apart, *s)
    m = load(folder, dtype, max_tokens=2048, max_sequences=4, cache=cache)
    gone = m.open()
    feed(m, gone, t[:33], [33])                        # blocks in front that are let go of later
    a = m.open()
    feed(m, a, t[:tokens], [50])
    b = m.fork(a)
    m.end(gone)
    assert m.compact() > 0
    got = go_on(m, a, b)
    for g, r in zip(got, want):
        assert np.array_equal(g, r)
    m.end(a)
    c = m.fork(b)                                       # and from a fork whose parent is gone
    m.compact()
    r1, r2 = m.step([(b, x[:3], None), (c, x[:3], None)])
    assert np.array_equal(r1, r2)


@pytest.mark.parametrize("name,dtype,cache", [("mixed", 6, 1), ("latent", 0, 0), ("streams", 6, 0), ("loops", 6, 0)])
def test_forks_of_what_has_just_begun(synth, tmp_path, load, monkeypatch, name, dtype, cache):
    """A fork of a sequence without tokens, in slots that others have left their states and tokens in, is another empty one."""
    cfg, w, folder = build(synth, tmp_path, name, monkeypatch)
    t = prompt(cfg, 60)
    m = load(folder, dtype, max_tokens=1024, max_sequences=2, cache=cache)
    old = [m.open(), m.open()]
    m.step([(old[0], t[:50], None), (old[1], t[10:], None)])
    for s in old:
        m.end(s)
    a = m.open()
    b = m.fork(a)
    got = [m.step([(a, t[:33], None), (b, t[:33], None)]), m.step([(a, t[33:34], None), (b, t[33:34], None)])]
    want = lm_util.reference(cfg, w, t[:34])
    for k in range(2):
        assert np.array_equal(got[0][0], got[0][1]) and np.array_equal(got[1][0], got[1][1])
        if not cache:
            assert error(np.concatenate([got[0][k], got[1][k]]), want) < TOL[dtype]


@pytest.mark.parametrize("name,cache", [("mixed", 1), ("streams", 2), ("gated", 1)])
def test_greedy_decoding_on_the_device(synth, tmp_path, load, monkeypatch, name, cache):
    """Captured steps over an 8-bit cache, of a sequence, its fork and another: every pick leads the logits of the same step by itself, up to what two ways to split the
    keys may differ by (each within TOL of the restatement's)."""
    cfg, w, folder = build(synth, tmp_path, name, monkeypatch)
    a, b = (load(folder, max_tokens=2048, max_sequences=4, cache=cache) for _ in range(2))
    t = prompt(cfg, 90)
    seqs = []
    for m in (a, b):
        x, y = m.open(), m.open()
        feed(m, x, t[:61], [61])
        feed(m, y, t[61:], [29])
        seqs.append([x, y, m.fork(x)])
    first = [int(v) for v in t[:3]]
    ids, _ = a.decode_greedy(seqs[0], first, 70)
    tokens = np.concatenate([np.array(first)[None], ids])
    for k in range(70):
        logits = b.step([(s, [int(tokens[k, i])], None) for i, s in enumerate(seqs[1])])
        for i, l in enumerate(logits):
            assert l[0][ids[k, i]] >= l[0].max() - 2 * TOL[6] * l.std() * np.sqrt(cfg["vocab"])


def soft(logits):
    z = np.asarray(logits, np.float64)
    z = z - z.max(-1, keepdims=True)
    return z - np.log(np.exp(z).sum(-1, keepdims=True))


def check_scores(logits, targets, top, lp, en, ids, best):
    """The operator's own error bound: a few roundings of the logits' spread and of the sum's logarithm."""
    p = soft(logits)
    tol = 2.0 ** -20 * (4 + np.abs(logits).max())
    at = np.arange(len(p))
    assert np.abs(lp - p[at, targets]).max() <= tol
    assert np.abs(en + (np.exp(p) * p).sum(-1)).max() <= tol * 8
    order = np.argsort(-np.asarray(logits), axis=-1, kind="stable")[:, :top]
    assert np.array_equal(ids, order)
    assert np.abs(best - np.take_along_axis(p, order, -1)).max(initial=0) <= tol


@pytest.mark.parametrize("name,dtype,cache", [("mixed", 6, 1), ("streams", 0, 0), ("loops", 6, 0), ("latent", 6, 0)])
def test_scored_steps(synth, tmp_path, load, monkeypatch, name, dtype, cache):
    """The scores of a step are those of the logits that the same step gives."""
    cfg, w, folder = build(synth, tmp_path, name, monkeypatch)
    t = prompt(cfg, 700)
    a, b = (load(folder, dtype, max_tokens=1024, max_sequences=3, cache=cache) for _ in range(2))
    s = [(m.open(), m.open()) for m in (a, b)]
    for top, parts in ((3, ((0, 300), (300, 330))), (0, ((330, 331), (331, 332))), (32, ((332, 600), (600, 609))), (1, ((609, 610), (610, 611)))):
        entries = [[(k, t[i:j], None) for k, (i, j) in zip(q, parts)] for q in s]
        logits = np.concatenate(a.step(entries[0]))
        targets = np.random.default_rng(top).integers(0, cfg["vocab"], len(logits)).astype(np.int32)
        check_scores(logits, targets, top, *b.scored(entries[1], targets, top))
    lp, en, ids, best = b.scored([(s[1][0], t[:2], [1])], None, 2)
    want = a.step([(s[0][0], t[:2], [1])])[0]
    assert lp is None and np.array_equal(ids, np.argsort(-want, -1, kind="stable")[:, :2]) and len(en) == 1


def test_scored_step_refusals(synth, tmp_path, load, pkg, monkeypatch):
    cfg, w, folder = build(synth, tmp_path, "plain", monkeypatch)
    m = load(folder, max_tokens=128, max_sequences=2)
    s = m.open()
    t, want, out = np.array([3], np.int32), np.array([0], np.int32), np.zeros(64, np.float32)
    e = pkg.LMEntry(s, t.ctypes.data, 1, want.ctypes.data, 1)
    call = lambda targets, top, lp, ids, best: pkg.lib.cml_lm_step_scored(m.h, e, 1, targets, top, lp, None, ids, best)
    P, T = pkg.np_ptr(out), pkg.np_ptr(t)
    for bad in ((None, 0, P, None, None), (T, 0, None, None, None), (None, -1, None, None, None), (None, 33, None, None, P), (None, 2, None, None, None), (None, 0, None, None, P)):
        assert call(*bad) == -1
    assert pkg.lib.cml_lm_sequence_length(m.h, s) == 0
    assert call(T, 1, P, None, pkg.np_ptr(out[8:])) == 0 and pkg.lib.cml_lm_sequence_length(m.h, s) == 1
    f = m.fork(s)
    assert pkg.lib.cml_lm_sequence_fork(m.h, s) == -1 and pkg.lib.cml_lm_sequence_fork(m.h, 7) == -1     # no slot, no sequence
    m.end(f)
    assert pkg.lib.cml_lm_sequence_fork(m.h, f) == -1


def test_llama_scored(pkg, tmp_path, load):
    import __graft_entry__ as entry
    cfg, path = llama_util.TINY, tmp_path / "tiny.gguf"
    meta = [(f"llama.{k}", 4, v) for k, v in (("block_count", cfg["layers"]), ("embedding_length", cfg["hidden"]), ("attention.head_count", cfg["heads"]),
                                              ("attention.head_count_kv", cfg["kv_heads"]), ("feed_forward_length", cfg["inter"]), ("context_length", cfg["max_seq"]))]
    llama_util.build(entry, np.random.default_rng(4), cfg, path, metadata=meta)
    t = np.random.default_rng(6).integers(0, cfg["vocab"], 20)
    a, b = (load(path, 0, max_tokens=96, max_sequences=3) for _ in range(2))
    s = [(m.open(), m.open()) for m in (a, b)]
    e = [[(q[0], t[:9], [8]), (q[1], t[:4], [3])] for q in s]
    check_scores(np.concatenate(a.step(e[0])), t[:2], 5, *b.scored(e[1], t[:2], 5))
    assert pkg.lib.cml_lm_sequence_fork(b.h, s[1][0]) == -1 and pkg.lib.cml_lm_compact(b.h) == -1
    assert not pkg.lib.cml_lm_load(str(path).encode(), pkg.LMOptions(6, 96, 2, 0, 1))


@pytest.mark.parametrize("name,cache", [("mixed", "i8"), ("streams", "e4m3"), ("gated", "i8")])
def test_a_run_of_all(synth, tmp_path, load, monkeypatch, name, cache):
    """Choosing the best of several continuations over an 8-bit cache: a prompt, three forks with their likeliest tokens, scores on the way, the worst given up, the
    pool made dense, two forks of the best; at each step the restatement's numbers."""
    cfg, w, folder = build(synth, tmp_path, name, monkeypatch)
    m = load(folder, max_tokens=640, max_sequences=6, cache=FORMS[cache])
    t = prompt(cfg, 75)
    root = m.open()
    lines = {root: list(t)}
    _, _, ids, _ = m.scored([(root, t, [74])], None, 4)
    kids = [m.fork(root) for _ in range(3)]
    for k in kids:
        lines[k] = list(t)
    total = dict.fromkeys(lines, 0.0)
    order = [root, *kids]
    feed_now = {k: int(i) for k, i in zip(order, ids[0])}
    for step in range(24):
        for k in order:
            lines[k].append(feed_now[k])
        nxt = [int(x) for x in prompt(cfg, len(order), 100 + step)]
        lp, en, ids, best = m.scored([(k, [feed_now[k]], None) for k in order], nxt, 2)
        if step % 6 == 5:
            for i, k in enumerate(order):
                want = with_cache(cfg, w, np.array(lines[k]), cache, monkeypatch)[-1:]
                plain = lm_util.reference(cfg, w, np.array(lines[k]))[-1:]
                p = soft(want)[0]
                # TOL and the codes' effect bound the deviation of a row's logits in units of their spread: a log probability is two of them away at most, were the
                # deviation shared evenly; a single place of V may take sqrt(V) of it
                allowed = 2 * (TOL[6] + error(want, plain)) * want.std() * np.sqrt(cfg["vocab"])
                assert abs(lp[i] - p[nxt[i]]) < allowed and abs(en[i] + (np.exp(p) * p).sum()) < allowed * (1 + np.abs(p).max())
        for i, k in enumerate(order):
            total[k] += float(lp[i])
            feed_now[k] = nxt[i]
        if step == 11:                                  # the worst of them makes room, the best goes on twice more
            order.sort(key=lambda k: -total[k])
            m.end(order.pop())
            m.compact()
            for _ in range(2):
                k = m.fork(order[0])
                lines[k], total[k], feed_now[k] = list(lines[order[0]]), total[order[0]], (feed_now[order[0]] + 1 + len(order)) % cfg["vocab"]
                order.append(k)
    for k in order:
        m.end(k)
    assert m.compact() == 0


def test_generate_program_with_an_8_bit_cache(pkg, synth, tmp_path, load, monkeypatch):
    cfg, w, folder = build(synth, tmp_path, "mixed", monkeypatch)
    t = prompt(cfg, 30).tolist()
    args = ["--model", str(folder), "--max-new", "12", "--tokens", ",".join(map(str, t))]
    for name, cache in (("int8", 1), ("e4m3", 2), ("default", 0)):
        r = subprocess.run([str(ROOT / "bin" / "cml_generate"), "--cache", name, *args], capture_output=True, text=True, timeout=600)
        assert r.returncode == 0, r.stderr
        got = [int(x) for x in r.stdout.split()]
        m = load(folder, max_tokens=8192, max_sequences=8, cache=cache)
        s, picked = m.open(), []
        nxt = int(m.step([(s, t, [len(t) - 1])], greedy=True)[0][0])
        for _ in range(12):
            picked.append(nxt)
            nxt = int(m.step([(s, [nxt], None)], greedy=True)[0][0])
        assert got[-12:] == picked
    r = subprocess.run([str(ROOT / "bin" / "cml_generate"), "--cache", "int4", *args], capture_output=True, text=True, timeout=600)
    assert r.returncode != 0
