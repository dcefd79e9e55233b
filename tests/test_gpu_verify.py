"""Drafted tokens kept and tokens drawn on the device, against 64 bits."""
import numpy as np
import pytest

import drafts_oracle

pytestmark = pytest.mark.gpu

FORMS = ["float32", "bfloat16", "float16"]


class Batch:
    """Sequences with `counts` drafts: logits of target and drafter as rows inside wider tensors."""

    def __init__(self, torch, dev, counts, vocab, seed, form="float32", drafter=True, temperatures=(1.0,), gap=0.7, spread=2.0, extra=0, lead=0):
        rng = np.random.default_rng(seed)
        self.torch, self.counts, self.vocab, self.form = torch, counts, vocab, form
        n, rows = sum(counts), sum(counts) + len(counts)
        self.first = np.concatenate([[0], np.cumsum(np.array(counts) + 1)]).astype(np.int32)
        kind = getattr(torch, form)

        def device_rows(a):
            t = torch.full((a.shape[0], lead + vocab + extra), float("nan"), dtype=kind)
            t[:, lead:lead + vocab] = torch.from_numpy(a).to(kind)
            return t.to(dev)[:, lead:lead + vocab]

        target = rng.normal(size=(rows, vocab)) * spread
        at = np.array([self.first[s] + i for s, c in enumerate(counts) for i in range(c)], int)
        self.target = device_rows(target)
        self.draft = device_rows(target[at] + rng.normal(size=(n, vocab)) * gap) if drafter and n else None
        self.t = np.array([temperatures[s % len(temperatures)] for s in range(len(counts))], np.float32)
        self.key = rng.integers(0, 2 ** 64, len(counts), dtype=np.uint64)
        # drafts as a drafter would draw them, some others among them
        source = (self.draft if self.draft is not None else self.target[torch.from_numpy(at).to(dev)]).double().cpu().numpy() if n else np.zeros((0, vocab))
        heat = np.repeat(self.t, counts)
        with np.errstate(invalid="ignore"):
            score = source + np.maximum(heat, 0)[:, None] * rng.gumbel(size=source.shape)
        self.tokens = np.argmax(score, 1).astype(np.int32) if n else np.zeros(0, np.int32)
        swap = rng.random(n) < 0.1
        self.tokens[swap] = rng.integers(0, vocab, swap.sum())
        self.dev = dev

    def call(self, pkg, stream=None, temperature=True, keep=None):
        torch, S = self.torch, len(self.counts)
        dt = {"float32": pkg.DT_F32, "bfloat16": pkg.DT_BF16, "float16": pkg.DT_F16}[self.form]
        up = lambda a: torch.from_numpy(a.copy()).to(self.dev)
        held = {"first": up(self.first), "tokens": up(np.append(self.tokens, 0).astype(np.int32)), "t": up(self.t), "key": up(self.key.view(np.int64))}
        out = torch.full((2, S + 1), -9, dtype=torch.int32, device=self.dev)
        rows = int(self.target.shape[0])
        work = torch.full((pkg.lib.cmlb200_verify_work_bytes(rows, S),), 171, dtype=torch.uint8, device=self.dev)
        d = pkg.Drafts(sequences=S, rows=rows, first=held["first"].data_ptr(), tokens=held["tokens"].data_ptr(), logits=self.draft.data_ptr() if self.draft is not None else None,
                       ld=self.draft.stride(0) if self.draft is not None else 0, temperature=held["t"].data_ptr() if temperature else None, random=held["key"].data_ptr())
        torch.cuda.synchronize()
        run = lambda st: pkg.check(pkg.lib.cmlb200_verify_drafts(d, self.target.data_ptr(), dt, self.target.stride(0), self.vocab, out[0].data_ptr(), out[1].data_ptr(), work.data_ptr(), st), "verify_drafts")
        if keep is not None:
            keep.update(held, out=out, work=work, d=d, run=run)
            return None
        run(stream)
        torch.cuda.synchronize()
        assert (out[:, S] == -9).all()
        return out[:, :S].cpu().numpy()

    def want(self):
        target = self.target.double().cpu().numpy()
        draft = self.draft.double().cpu().numpy() if self.draft is not None else None
        got = []
        for s, n in enumerate(self.counts):
            f = self.first[s]
            got.append(drafts_oracle.verify(target[f:f + n + 1], self.tokens[f - s:f - s + n].tolist(), draft[f - s:f - s + n] if draft is not None else None, float(self.t[s]), int(self.key[s])))
        return got

    def check(self, got, most_unsure=0.02):
        want = self.want()
        unsure = [w[2] for w in want]
        assert sum(unsure) <= 1 + most_unsure * len(unsure), "the inputs leave too much to rounding"
        for s, w in enumerate(want):
            if not w[2]:
                assert (got[0][s], got[1][s]) == w[:2], (s, self.counts[s], got[:, s], w)
        return want


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("counts,vocab", [([4], 32000), ([0], 1000), ([3, 0, 1, 7, 2, 0, 5], 517), ([1] * 40, 33), ([2, 5, 0, 3], 100003), ([12, 1, 4], 4097), ([600, 3], 40), ([0] * 90, 5), ([3, 2, 3, 1], 4),
                                          ([2, 0, 1], 3), ([1, 2], 2), ([2, 0, 1], 1), ([4] * 200, 700)])
def test_verify(pkg, torch_dev, form, drafter, counts, vocab):
    import torch
    b = Batch(torch, torch_dev, counts, vocab, len(counts) + vocab, form, drafter, (1.0, 0.7, 0.0, 1.6))
    want = b.check(b.call(pkg))
    if len(counts) > 50 and vocab > 100:                # every way that a sequence may end is met
        kept = np.array([w[0] for w in want])
        assert (kept == 4).any() and (kept == 0).any() and ((kept > 0) & (kept < 4)).any()


@pytest.mark.parametrize("extra,lead", [(1, 0), (3, 1), (8, 8), (5, 7)])
@pytest.mark.parametrize("form", FORMS)
def test_strides(pkg, torch_dev, form, extra, lead):
    import torch
    b = Batch(torch, torch_dev, [3, 0, 4, 1, 2], 1303, 11, form, True, (1.0, 0.0, 0.5), extra=extra, lead=lead)
    b.check(b.call(pkg))


def test_defaults(pkg, torch_dev):
    """No temperatures: all are 1. The same call gives the same tokens."""
    import torch
    b = Batch(torch, torch_dev, [2, 3, 0, 4] * 8, 5000, 3)
    got = b.call(pkg, temperature=False)
    b.check(got)
    assert (got == b.call(pkg)).all() and (got == b.call(pkg)).all()


@pytest.mark.parametrize("spread,temperature", [(0.0, 1.0), (0.01, 1.0), (30.0, 1.0), (300.0, 1.0), (2.0, 0.01), (2.0, 1e-4), (2.0, 100.0), (2.0, 9e-6), (2.0, -1.0)])
@pytest.mark.parametrize("drafter", [True, False])
def test_flat_and_steep(pkg, torch_dev, spread, temperature, drafter):
    import torch
    b = Batch(torch, torch_dev, [3, 0, 1, 2] * 5, 3001, 17, drafter=drafter, temperatures=(temperature,), spread=spread, gap=0.2 * spread)
    b.check(b.call(pkg), most_unsure=0.3)


def test_far_from_zero(pkg, torch_dev):
    """Logits that share a large offset lose no digits beyond their own."""
    import torch
    b = Batch(torch, torch_dev, [2, 0, 1] * 5, 2000, 71, gap=0.3)
    b.target += 4096.0
    b.draft += 1024.0
    b.check(b.call(pkg), most_unsure=0.2)


@pytest.mark.parametrize("vocab", [1, 2, 3, 4, 5, 6, 7, 9])
def test_few_tokens(pkg, torch_dev, vocab):
    """Waits of all lengths: with one token every one of them wins."""
    import torch
    b = Batch(torch, torch_dev, [0] * 3000, vocab, 73 + vocab, spread=0.3)
    b.check(b.call(pkg))


def test_close_calls(pkg, torch_dev):
    """Tokens whose weights over waits differ by less than 32 bits tell apart: the 64-bit comparison decides. Logits are waits' logarithms, so that all tokens come out nearly equal."""
    import torch
    b = Batch(torch, torch_dev, [0] * 64, 1500, 79)
    rng = np.random.default_rng(9)
    for s in range(64):
        z = np.log(drafts_oracle.waits(int(b.key[s]), 1500))
        keep = rng.permutation(1500)[:40]
        row = np.full(1500, -40.0)
        row[keep] = z[keep] + rng.normal(size=40) * 2e-5
        b.target[s] = torch.from_numpy(row).float()
    got = b.call(pkg)
    x = b.target.double().cpu().numpy()
    for s in range(64):
        z = x[s] - np.log(drafts_oracle.waits(int(b.key[s]), 1500))
        assert got[0][s] == 0 and got[1][s] == int(np.argmax(z)), (s, np.sort(z)[-3:], z[got[1][s]])


@pytest.mark.parametrize("vocab,at", [(2, (0, 1)), (4, (0, 3)), (4, (1, 2)), (50, (49, 48)), (5000, (2049, 2051)), (40000, (12, 2060)), (40000, (12, 4108))])
def test_close_neighbours(pkg, torch_dev, vocab, at):
    """The same where the two tokens are a thread's: of one group of four, or of groups that it looks at one after another."""
    import torch
    b = Batch(torch, torch_dev, [0] * 400, vocab, 80)
    rng, at = np.random.default_rng(vocab), list(at)
    x = np.full((400, vocab), -40.0)
    for s in range(400):
        x[s, at] = np.log(drafts_oracle.waits(int(b.key[s]), vocab))[at] + rng.normal(size=2) * 2e-6
    b.target[:] = torch.from_numpy(x).float()
    got, x = b.call(pkg), b.target.double().cpu().numpy()
    for s in range(400):
        z = x[s] - np.log(drafts_oracle.waits(int(b.key[s]), vocab))
        assert got[0][s] == 0 and got[1][s] == int(np.argmax(z)), (s, z[at] - z.max(), got[1][s])


def test_same_logits(pkg, torch_dev):
    """A drafter whose logits are the target's: everything is kept."""
    import torch
    b = Batch(torch, torch_dev, [5] * 20, 2000, 19, gap=0.0)
    b.tokens = np.array([drafts_oracle.verify(row[None], [], None, 1.0, int(k))[1] for row, k in zip(b.draft.double().cpu().numpy(), np.arange(100))], np.int32)
    got = b.call(pkg)
    assert (got[0] == 5).all()
    b.check(got)


@pytest.mark.parametrize("form", FORMS)
def test_without_end(pkg, torch_dev, form):
    """Infinite temperatures: any token that can come is as likely as any other, and those that cannot still do not. What is no temperature is greedy."""
    import torch
    b = Batch(torch, torch_dev, [4] * 30, 300, 8, form, True)
    b.target[:, ::3] = b.draft[:, ::3] = -float("inf")
    b.tokens = (b.tokens // 3 * 3 + 1).astype(np.int32)
    got = []
    for t in (np.inf, 1e38, 1e30, np.nan, 0.0):
        b.t[:] = t
        got.append(b.call(pkg))
    assert (got[0] == got[2]).all() and (got[1] == got[2]).all() and (got[3] == got[4]).all()
    assert (got[0][0] == 4).all()                      # p = q: u p < p
    assert (got[0][1] % 3 != 0).all() and len(set(got[0][1])) > 20


@pytest.mark.parametrize("form", FORMS)
def test_masked(pkg, torch_dev, form):
    """Tokens that cannot come: never drawn; a draft that the target rules out is turned down, one that the drafter ruled out is kept where the target allows it."""
    import torch
    b = Batch(torch, torch_dev, [2, 2, 2, 1, 0, 1, 1], 900, 23, form, True, (1.0,))
    inf = float("inf")
    b.target[:, ::3] = -inf
    b.draft[:, 1::3] = -inf
    b.tokens[:] = 2
    b.tokens[0], b.tokens[2], b.tokens[3] = 0, 1, 4
    b.target[4:6, :] = -inf                                               # sequence 1: one token is left, then none
    b.target[4, 77] = 1.0
    b.tokens[2:4] = 77
    b.target[9] = torch.finfo(getattr(torch, form)).min                   # sequence 3: nothing but the type's lowest number
    b.draft[6] = -inf                                                     # its drafter has nothing
    got = b.call(pkg)
    b.check(got, 0.3)
    assert got[1][1] == -1 and (got[1][[0, 2, 4, 5, 6]] % 3 != 0).all()


@pytest.mark.parametrize("drafter", [True, False])
def test_only_the_draft(pkg, torch_dev, drafter):
    """A target that allows one token, and a draft that is it or is not."""
    import torch
    b = Batch(torch, torch_dev, [1, 1, 1], 50, 29, "float32", drafter)
    b.target[:] = -float("inf")
    b.target[:, 9] = 3.0
    b.tokens[:] = (9, 8, 9)
    b.check(b.call(pkg))


def test_rows_that_are_not_numbers(pkg, torch_dev):
    import torch
    nan, inf = float("nan"), float("inf")
    for greedy in (0.0, 1.0):
        b = Batch(torch, torch_dev, [2] * 8, 700, 31, temperatures=(greedy,))
        b.target[0, 5] = nan
        b.target[4, 699] = nan
        b.target[8, 0] = inf
        b.target[9, 1] = nan
        b.target[9] = -inf
        b.draft[8, 3] = nan
        b.draft[10, 3] = inf
        b.draft[12] = -inf
        b.target[23, 0] = nan
        got = b.call(pkg)
        b.check(got)
        assert got[0][0] == 0 and got[1][0] == -1


def test_drafts_outside(pkg, torch_dev):
    import torch
    for drafter in (True, False):
        b = Batch(torch, torch_dev, [2, 3, 1, 2], 300, 37, drafter=drafter, temperatures=(1.0, 0.0))
        b.tokens[0], b.tokens[3], b.tokens[5], b.tokens[7] = 300, -1, 2 ** 31 - 1, -2 ** 31
        b.check(b.call(pkg))


@pytest.mark.parametrize("first", [[0, 3, 2, 6], [0, 7, 7, 7], [1, 2, 3, 9], [-4, 1, 3, 6], [0, 2, 9, 6], [0, 0, 1, 6], [0, 2 ** 31 - 1, -2 ** 31, 6], [0, 6, 6, 6]])
def test_rows_out_of_order(pkg, torch_dev, first):
    """Rows that are not a sequence's: no draft kept, no token; nothing is read that is not there, and sequences beside it keep theirs."""
    import torch
    b = Batch(torch, torch_dev, [1, 1, 1], 300, 41)
    b.first = np.array(first, np.int32)
    got = b.call(pkg)
    assert ((got[1] >= -1) & (got[1] < 300) & (got[0] >= 0) & (got[0] <= 5)).all()
    for s in range(3):
        if first[s + 1] <= first[s] or first[s] < s or first[s + 1] - s - 1 > 3:
            assert (got[:, s] == (0, -1)).all()


def test_far_rows(pkg, torch_dev):
    """Rows whose offsets pass 32 bits."""
    import torch
    V, ld = 1000, 1 << 28
    b = Batch(torch, torch_dev, [4, 5], V, 43, "float16")
    far = torch.empty(11 * ld, dtype=torch.float16, device=torch_dev)
    rows = far.as_strided((11, V), (ld, 1))
    rows.copy_(b.target)
    want = b.call(pkg)
    b.target = rows
    assert (b.call(pkg) == want).all()
    b.check(want)


def test_streams_and_graphs(pkg, torch_dev):
    import torch
    batches = [Batch(torch, torch_dev, [3, 1, 0, 4] * 4, 9000, 50 + i, gap=0.4) for i in range(2)]
    want = [b.call(pkg) for b in batches]
    kept = [{}, {}]
    for b, k in zip(batches, kept):
        b.call(pkg, keep=k)
    streams = [torch.cuda.Stream() for _ in batches]
    for _ in range(20):
        for k, st in zip(kept, streams):
            k["run"](st.cuda_stream)
    torch.cuda.synchronize()
    for k, w in zip(kept, want):
        assert (k["out"][:, :16].cpu().numpy() == w).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept[0]["run"](torch.cuda.current_stream().cuda_stream)
    b, other = batches
    b.target.copy_(other.target); b.draft.copy_(other.draft)
    for name in ("tokens", "key"):
        kept[0][name].copy_(kept[1][name])
    kept[0]["out"].fill_(-9)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert (kept[0]["out"][:, :16].cpu().numpy() == want[1]).all()


def test_draws_are_distributed(pkg, torch_dev):
    """20,000 sequences over the same logits: drawn tokens by the target's chances, and so are first tokens behind drafts from another distribution."""
    import torch
    rng = np.random.default_rng(3)
    S, V = 20000, 9
    p_row, q_row = rng.normal(size=V) * 1.3, rng.normal(size=V) * 1.3
    p, q = drafts_oracle.chances(p_row.astype(np.float32), 1.0), drafts_oracle.chances(q_row.astype(np.float32), 1.0)
    for n in (0, 1):
        b = Batch(torch, torch_dev, [n] * S, V, 60 + n)
        b.target.copy_(torch.from_numpy(np.tile(p_row, (len(b.target), 1))).float())
        if n:
            b.draft.copy_(torch.from_numpy(np.tile(q_row, (S, 1))).float())
            b.tokens = rng.choice(V, S, p=q).astype(np.int32)
        got = b.call(pkg)
        token = np.where(got[0] == 1, b.tokens if n else 0, got[1])
        count = np.bincount(token, minlength=V)
        chi = ((count - S * p) ** 2 / (S * p)).sum()
        assert chi < 8 + 6 * np.sqrt(16) + 6, (count / S, p)


CAPTURED_FIRST = """
import sys
sys.path.insert(0, {root!r})
sys.path.insert(0, {tests!r})
import torch
import __graft_entry__ as entry
from test_gpu_verify import Batch
pkg = entry.load_package()
b = Batch(torch, torch.device("cuda:0"), {counts}, 40000, 5)
k = {{}}
b.call(pkg, keep=k)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    k["run"](torch.cuda.current_stream().cuda_stream)
g.replay()
torch.cuda.synchronize()
b.check(k["out"][:, :len(b.counts)].cpu().numpy())
print("fine")
"""


@pytest.mark.parametrize("counts", [[3], [0, 2] * 20])
def test_captured_before_anything_else_ran(counts):
    import subprocess
    import sys
    from pathlib import Path
    tests = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST.format(root=str(tests.parent), tests=str(tests), counts=counts)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]
