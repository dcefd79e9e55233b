"""Attention over 8-bit paged caches: codes and scales have to be the definition's, outputs within what their roundings allow."""
import numpy as np
import pytest

import cache8_oracle as co

pytestmark = pytest.mark.gpu


def rms(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


class Layer:
    """A layer's descriptor over device pools filled with codes that nothing may read, and the same cache in the restatement."""

    def __init__(self, pkg, dev, form, heads, kv_heads, dim, vdim, page=16, slots=3, tokens=400, seed=0, window=0, keep=0, chunk=0, sink=None, slopes=False, norm=None,
                 temp=False, gate=None, rot=0, kav=False, scale=None, out_scale=0.0, spread=1.0):
        import torch
        self.t, self.pkg, self.dev, self.form = torch, pkg, dev, form
        self.H, self.G, self.D, self.V, self.page, self.slots = heads, kv_heads, dim, vdim, page, slots
        self.window, self.keep, self.chunk, self.norm, self.temp, self.gate, self.rot, self.kav, self.spread = window, keep, chunk, norm, temp, gate, rot, kav, spread
        r = self.rng = np.random.default_rng(seed)
        pad = lambda n: (n + 15) // 16 * 16
        up = lambda a, t=np.float32: torch.from_numpy(np.ascontiguousarray(a, t)).to(dev)
        per = -(-tokens // page)
        self.pages = per * slots + 2
        self.table = np.zeros((slots, per + 1), np.int32)
        self.table[:, :per] = r.permutation(self.pages)[:per * slots].reshape(slots, per)
        junk = 0x7F                                   # e4m3's NaN, int8's largest
        self.k = torch.full((self.pages, page, kv_heads, pad(dim)), junk, dtype=torch.int8, device=dev)
        self.v = torch.full((self.pages, page, kv_heads, pad(vdim)), junk, dtype=torch.int8, device=dev)
        self.ks, self.vs = (torch.full((self.pages, page // 16, kv_heads), float("nan"), device=dev) for _ in range(2))
        self.scale = scale or dim ** -0.5
        self.slopes = np.exp2(-8.0 * np.arange(1, heads + 1) / heads).astype(np.float32) if slopes else None
        self.sinks = None if sink is None else (np.zeros(heads) if sink == "zero" else r.standard_normal(heads).astype(np.float32))
        n = (heads * dim, kv_heads * dim) if norm == "whole" else (dim, dim)
        self.qn, self.kn = ((1 + 0.3 * r.standard_normal(m)).astype(np.float32) for m in n) if norm else (None, None)
        self.freq = (0.7 ** np.arange(rot // 2)).astype(np.float32) if rot else None
        self.eps, self.width = 1e-3, (heads + kv_heads) * dim + (0 if kav else kv_heads * vdim)
        self.out_scale = out_scale
        gates = 0 if gate is None else heads * vdim if gate == "wide" else heads
        self.ld = self.width + gates + 5
        self.held_on_device = [up(x) if x is not None else None for x in (self.slopes, self.sinks if sink == "own" else None, self.qn, self.kn, self.freq)]
        self.d_table = up(self.table, np.int32)
        ptr = lambda x: None if x is None else x.data_ptr()
        sl, si, qn, kn, fr = map(ptr, self.held_on_device)
        self.a = pkg.Attn(heads=heads, kv_heads=kv_heads, dim=dim, vdim=vdim, dim_ld=pad(dim), vdim_ld=pad(vdim), scale=self.scale, window=window, slopes=sl, sink=int(sink is not None),
                          sinks=si, q_norm=qn, k_norm=kn, eps=self.eps, temp_coef=0.3 if temp else 0.0, temp_every=7.0 if temp else 0.0, gate_col=self.width if gate else -1,
                          gate_wide=int(gate == "wide"), cache_dtype=pkg.DT_I8 if form == "i8" else pkg.DT_E4M3, k_pool=self.k.data_ptr(), v_pool=self.v.data_ptr(), k_scale=self.ks.data_ptr(),
                          v_scale=self.vs.data_ptr(), block_size=page, block_table=self.d_table.data_ptr(), table_ld=self.table.shape[1], keep=keep, chunk=chunk, head_norm=int(norm == "head"),
                          keys_as_values=int(kav), out_scale=out_scale, freq=fr, rot_dims=rot)
        self.seqs = [(co.Sequence(kv_heads, pad(dim), form), co.Sequence(kv_heads, pad(vdim), form)) for _ in range(slots)]
        self.worst = 0.0

    def fresh_rows(self, n):
        x = self.rng.standard_normal((n, self.ld)) * np.exp(self.rng.normal(0, self.spread, (n, 1)))      # tokens of different sizes: scales grow
        return x.astype(np.float32)

    def turn(self, x, pos):
        if not self.rot:
            return x
        y, ang = x.copy(), (pos[:, None].astype(np.float32) * self.freq).astype(np.float64)[:, None]
        a, b = x[..., 0:self.rot:2], x[..., 1:self.rot:2]
        y[..., 0:self.rot:2], y[..., 1:self.rot:2] = a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)
        return y

    def queries_and_keys(self, x, pos):
        n, H, G, D = len(x), self.H, self.G, self.D
        q, k = x[:, :H * D].astype(np.float64), x[:, H * D:(H + G) * D].astype(np.float64)
        if self.norm == "whole":
            q, k = rms(q, self.qn, self.eps), rms(k, self.kn, self.eps)
        q, k = q.reshape(n, H, D), k.reshape(n, G, D)
        if self.norm == "head":
            q, k = rms(q, self.qn, self.eps), rms(k, self.kn, self.eps)
        if self.temp:
            q = q * (1 + 0.3 * np.log(np.floor((pos + 1) / 7.0) + 1))[:, None, None]
        return self.turn(q, pos), self.turn(k, pos)

    def step(self, parts, rows=None, stream=None):
        """parts: (slot, tokens). Single tokens go through the decode kernel, portions through append and tiles; checks outputs."""
        parts = sorted(parts, key=lambda p: p[1] > 1)
        one = sum(n == 1 for _, n in parts)
        x = self.fresh_rows(sum(n for _, n in parts)) if rows is None else rows
        pos = np.concatenate([len(self.seqs[s][0].codes) + np.arange(n) for s, n in parts])
        slot = np.concatenate([np.full(n, s) for s, n in parts])
        had = {s: len(self.seqs[s][0].codes) for s, _ in parts}
        want, tol, at = [], [], 0
        for s, n in parts:
            part, p = x[at:at + n], pos[at:at + n]
            q, k = self.queries_and_keys(part, p)
            ks, vs = self.seqs[s]
            v = part[:, (self.H * self.D if self.kav else (self.H + self.G) * self.D):].astype(np.float64)[:, :self.G * self.V].reshape(n, self.G, self.V)
            widen = lambda a, w: np.concatenate([a, np.zeros(a.shape[:2] + (w - a.shape[2],))], 2)
            ks.append(widen(k, ks.codes.shape[2]))
            vs.append(widen(v, vs.codes.shape[2]))
            hk, hv = ks.held()[:, :, :self.D], vs.held()[:, :, :self.V]
            o, w, reach = co.attend(q, p, hk, hv, self.scale, self.slopes, self.sinks, self.window, self.keep, self.chunk)
            f = np.full((n, self.H, 1), self.out_scale or 1.0)
            if self.gate:
                g = part[:, self.width:self.width + (self.H * self.V if self.gate == "wide" else self.H)].astype(np.float64).reshape(n, self.H, -1)
                f = f / (1 + np.exp(-g))
            want.append((o * f).reshape(n, -1))
            tol.append(co.bound(o * f, w * np.abs(f), reach, np.abs(hv).max() * np.abs(f).max()).reshape(n, -1))
            at += n
        want, tol = np.concatenate(want), np.concatenate(tol)
        got = self.device(x, pos, slot, parts, one, had, stream)
        assert np.isfinite(got).all()
        off = np.abs(got - want) / tol
        self.worst = max(self.worst, float(off.max()))
        assert off.max() <= 1.0, (float(off.max()), np.unravel_index(off.argmax(), off.shape), got.flat[off.argmax()], want.flat[off.argmax()])
        return got

    def device(self, x, pos, slot, parts, one, had, stream=None):
        t, L, pkg = self.t, self.pkg.lib, self.pkg
        up = lambda a, k: t.from_numpy(np.ascontiguousarray(a, k)).to(self.dev)
        d, dp, ds = up(x, np.float32), up(pos, np.int32), up(slot, np.int32)
        ow, n = self.H * self.V, len(x)
        out = t.zeros((n, ow + 3), dtype=t.bfloat16, device=self.dev)
        tiles, at = [], one
        for s, m in parts[one:]:
            tiles += [[at + k, min(64, m - k), s, had[s] + k] for k in range(0, m, 64)]
            at += m
        st = None if stream is None else stream.cuda_stream
        t.cuda.synchronize()
        if n > one:
            dt = up(tiles, np.int32)
            if self.rot:
                pkg.check(L.cmlb200_rotate_append(self.a, d.data_ptr(), self.ld, dp.data_ptr(), ds.data_ptr(), one, n - one, one, None, st))
            else:
                pkg.check(L.cmlb200_qk_norm_append(self.a, d.data_ptr() + one * self.ld * 4, self.ld, dp.data_ptr() + one * 4, ds.data_ptr() + one * 4, n - one, st))
            pkg.check(L.cmlb200_attention_tiles(self.a, d.data_ptr(), self.ld, dt.data_ptr(), len(tiles), out.data_ptr(), ow + 3, st))
        if one:
            keys = max(had[s] for s, m in parts[:one])
            before = d[:one].clone()
            pkg.check(L.cmlb200_attention_one(self.a, d.data_ptr(), self.ld, dp.data_ptr(), ds.data_ptr(), one, keys, out.data_ptr(), ow + 3, st))
        t.cuda.synchronize()
        if one:
            assert t.equal(before, d[:one]), "decoded rows are read only"
        o = out.float().cpu().numpy()
        assert (o[:, ow:] == 0).all()
        return o[:, :ow].astype(np.float64)

    def check_cache(self, exact=True):
        """Codes and scales of every sequence; slots behind a sequence's end hold what they held."""
        raw = lambda p: (p.float() if self.form == "i8" else p.view(self.t.float8_e4m3fn).float()).cpu().numpy().astype(np.float64)
        used = np.zeros((self.pages, self.page), bool)
        for pool, scales, which in ((self.k, self.ks, 0), (self.v, self.vs, 1)):
            codes, sc = raw(pool), scales.cpu().numpy()
            for s in range(self.slots):
                seq = self.seqs[s][which]
                n = len(seq.codes)
                ids = self.table[s, :-(-n // self.page)]
                for j in range(n):
                    used[ids[j // self.page], j % self.page] = True
                if not n:
                    continue
                got = codes[ids].reshape(-1, self.G, codes.shape[3])[:n]
                gs = sc[ids].reshape(-1, self.G)[:-(-n // 16)]
                if exact:
                    assert np.array_equal(gs, seq.scales)
                    assert np.array_equal(got, seq.codes)
                else:                                 # normed or turned in fp32: a code may fall to the other side of a tie, a scale at its border
                    step = np.maximum(1.0, np.abs(seq.codes) / 8) if self.form == "e4m3" else 1.0
                    same = np.repeat(gs == seq.scales, 16, 0)[:n, :, None]
                    assert same.mean() > 0.99
                    assert (np.abs(got - seq.codes) <= step)[np.broadcast_to(same, got.shape)].all()
                    assert (got != seq.codes)[np.broadcast_to(same, got.shape)].mean() < 1e-2
            assert (pool.cpu().numpy()[~used] == 0x7F).all()


FORMS = ["i8", "e4m3"]
# heads, key/value heads, key and value sizes
SHAPES = [(32, 8, 128, 128), (4, 2, 64, 64), (3, 3, 13, 7), (8, 1, 80, 96), (20, 2, 72, 136), (16, 1, 128, 64), (6, 3, 256, 256), (12, 1, 192, 128), (34, 2, 64, 48), (5, 5, 16, 80)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("shape", SHAPES)
def test_portions_and_tokens(pkg, torch_dev, form, shape):
    L = Layer(pkg, torch_dev, form, *shape, page=16 if shape[0] % 4 else 64)
    L.step([(0, 70), (2, 17)])
    for i in range(20):                                # across the borders of groups, sequences alone and together
        L.step([(0, 1)] + ([(1, 1)] if i > 3 else []) + ([(2, 1)] if i % 3 else []))
    L.step([(0, 1), (1, 130), (2, 3)])
    L.step([(0, 65), (1, 1), (2, 2)])
    L.check_cache()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("mask", [dict(window=1), dict(window=16), dict(window=50), dict(window=33, keep=5), dict(window=20, keep=40), dict(chunk=48), dict(chunk=1, keep=1), dict(chunk=64, keep=17),
                                  dict(window=4000)])
def test_masks(pkg, torch_dev, form, mask):
    L = Layer(pkg, torch_dev, form, 8, 2, 64, 64, page=32, **mask)
    L.step([(0, 150), (1, 16)])
    for _ in range(18):
        L.step([(0, 1), (1, 1), (2, 1)])
    L.step([(0, 66), (1, 100), (2, 31)])
    L.check_cache()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("what", [dict(sink="zero"), dict(sink="own", slopes=True), dict(gate="head", out_scale=1.7), dict(temp=True), dict(kav=True), dict(scale=0.02), dict(slopes=True, window=40)])
def test_features(pkg, torch_dev, form, what):
    L = Layer(pkg, torch_dev, form, 12, 4, 64, 64, **what)
    L.step([(0, 80), (1, 33)])
    for _ in range(10):
        L.step([(0, 1), (2, 1), (1, 1)])
    L.step([(2, 64), (1, 1)])
    L.check_cache()


def test_wide_gate_of_portions(pkg, torch_dev):
    L = Layer(pkg, torch_dev, "i8", 4, 2, 64, 80, gate="wide")
    L.step([(0, 80), (1, 33)])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("what", [dict(norm="whole"), dict(norm="head"), dict(norm="whole", temp=True, slopes=True), dict(norm="head", kav=True)])
def test_norms(pkg, torch_dev, form, what):
    L = Layer(pkg, torch_dev, form, 8, 4, 96, 96, **what)
    L.step([(0, 80), (1, 33)])
    for _ in range(5):
        L.step([(0, 1), (2, 1)])
    L.check_cache(exact=False)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("rot", [2, 40, 64])
def test_rotation(pkg, torch_dev, form, rot):
    L = Layer(pkg, torch_dev, form, 6, 3, 64, 64, rot=rot)
    L.step([(0, 80), (1, 33)])
    for _ in range(5):
        L.step([(0, 1), (2, 1)])
    L.step([(0, 1), (1, 40)])
    L.check_cache(exact=False)


@pytest.mark.parametrize("form", FORMS)
def test_long_sequences(pkg, torch_dev, form):
    """Work of one row split over many CTAs; one key far back stands out."""
    L = Layer(pkg, torch_dev, form, 8, 2, 128, 128, page=16, slots=2, tokens=5100, spread=0.3)
    x = L.fresh_rows(5000)
    x[1234, L.H * L.D:(L.H + L.G) * L.D] *= 12
    # the restatement's attention of 5,000 rows takes long; the portion's outputs are not looked at
    attend, co.attend = co.attend, lambda q, p, k, v, *a: (np.zeros((len(q), L.H, L.V)), np.full((len(q), L.H, L.V), 1e30), np.zeros((len(q), L.H, 1)))
    try:
        L.step([(0, 5000)], rows=x)
    finally:
        co.attend = attend
    for _ in range(3):
        L.step([(0, 1), (1, 1)])
    L.step([(0, 7), (1, 5)])
    L.check_cache()


@pytest.mark.parametrize("form", FORMS)
def test_scales_far_apart(pkg, torch_dev, form):
    """Tokens from 1e-30 to 1e4, zeros, numbers beyond fp16, infinities and NaN."""
    L = Layer(pkg, torch_dev, form, 4, 2, 64, 64, scale=1e-6)
    x = L.fresh_rows(100) * np.exp(L.rng.uniform(-70, 9, (100, 1))).astype(np.float32)
    x[:, :L.H * L.D] = L.fresh_rows(100)[:, :L.H * L.D]
    x[10:30, L.H * L.D:] = 0
    x[5, L.H * L.D + 3], x[40, L.H * L.D + 130], x[41, L.H * L.D + 140], x[60, L.H * L.D] = 1e30, -np.inf, np.inf, np.nan
    L.step([(0, 37), (1, 63)], rows=x)
    for i in range(20):
        y = L.fresh_rows(2)
        y[:, L.H * L.D:] *= [1e-38, 1e-3, 0, 30][i % 4]
        L.step([(0, 1), (1, 1)], rows=y)
    L.check_cache()


@pytest.mark.parametrize("form", FORMS)
def test_values_at_the_edges_of_codes(pkg, torch_dev, form):
    """Ties between codes, the largest code exactly, and just beyond it."""
    L = Layer(pkg, torch_dev, form, 2, 1, 64, 64)
    full = co.FULL[form]
    x = L.fresh_rows(48)
    x[:, 2 * 64:] = (np.arange(48 * (L.ld - 128)).reshape(48, -1) % 509 - 254) / 2
    x[0, 128], x[16, 128], x[32, 128] = full, np.nextafter(np.float32(full), np.float32(1e9)), full / 2
    L.step([(0, 48)], rows=x)
    L.check_cache()


def test_a_page_taken_over_from_another_sequence(pkg, torch_dev):
    """A group that a new sequence begins takes no notice of the scale and codes that lie there."""
    L = Layer(pkg, torch_dev, "i8", 4, 2, 64, 64, spread=2.0)
    L.step([(0, 40)])
    L.table[1] = L.table[0]
    L.d_table.copy_(L.t.from_numpy(L.table))
    L.seqs[0] = (co.Sequence(2, 64, "i8"), co.Sequence(2, 64, "i8"))
    for _ in range(3):
        L.step([(1, 1)], rows=L.fresh_rows(1) * np.float32(1e-4))


def test_same_call_again_and_dropped_tokens(pkg, torch_dev):
    """A call that is repeated writes what it wrote; tokens after a rollback take the places of the dropped ones."""
    L = Layer(pkg, torch_dev, "e4m3", 4, 2, 64, 64)
    L.step([(0, 30)])
    x = L.fresh_rows(1)
    pos, slot = np.array([30]), np.array([0])
    a = L.device(x, pos, slot, [(0, 1)], 1, {0: 30})
    k, s = L.k.clone(), L.ks.clone()
    b = L.device(x, pos, slot, [(0, 1)], 1, {0: 30})
    assert np.array_equal(a, b) and L.t.equal(k, L.k) and L.t.equal(s.nan_to_num(), L.ks.nan_to_num())
    # position 30 again with another token: the group's scale stays where it was or grows
    y = L.fresh_rows(1) * np.float32(1e-3)
    grown = L.ks[L.table[0, 1], 0].cpu().numpy()
    L.device(y, pos, slot, [(0, 1)], 1, {0: 30})
    assert np.array_equal(L.ks[L.table[0, 1], 0].cpu().numpy(), grown)


def test_streams_and_graphs(pkg, torch_dev):
    """Another stream than the pools' own; a captured step, replayed with other rows in its buffers."""
    import torch
    L = Layer(pkg, torch_dev, "i8", 32, 8, 128, 128, slots=2)
    side = torch.cuda.Stream()
    L.step([(0, 40), (1, 20)], stream=side)
    L.step([(0, 1), (1, 1)], stream=side)
    x = L.fresh_rows(2)
    d = torch.from_numpy(x).to(torch_dev)
    pos, slot = (torch.tensor(v, dtype=torch.int32, device=torch_dev) for v in ([41, 21], [0, 1]))
    out = torch.zeros(2, L.H * L.V, dtype=torch.bfloat16, device=torch_dev)
    call = lambda st: pkg.check(pkg.lib.cmlb200_attention_one(L.a, d.data_ptr(), L.ld, pos.data_ptr(), slot.data_ptr(), 2, 128, out.data_ptr(), L.H * L.V, st))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        x = L.fresh_rows(2)
        d.copy_(torch.from_numpy(x))
        graph.replay()
        torch.cuda.synchronize()
        got = out.float().cpu().numpy()
        for s in range(2):
            q, k = L.queries_and_keys(x[s:s + 1], np.array([41 + i, 21 + i])[s:s + 1])
            L.seqs[s][0].append(k)
            L.seqs[s][1].append(x[s:s + 1, (L.H + L.G) * L.D:L.width].reshape(1, L.G, L.V))
            hk, hv = L.seqs[s][0].held(), L.seqs[s][1].held()
            o, w, reach = co.attend(q, np.array([len(hk) - 1]), hk, hv, L.scale)
            assert (np.abs(got[s] - o.reshape(-1)) <= co.bound(o, w, reach, np.abs(hv).max()).reshape(-1)).all()
        pos += 1
    L.check_cache()


@pytest.mark.parametrize("form,dim,what", [("i8", 128, {}), ("e4m3", 64, dict(slopes=True, sink="own", window=300)), ("i8", 64, dict(window=200, keep=150)), ("e4m3", 128, dict(chunk=256, gate="head"))])
def test_portions_of_many_tiles(pkg, torch_dev, form, dim, what):
    """Enough tiles for two blocks of rows a CTA."""
    L = Layer(pkg, torch_dev, form, 32, 8, dim, dim, slots=2, tokens=1500, **what)
    L.step([(0, 1290), (1, 77)])
    L.step([(0, 60), (1, 1210)])
    L.check_cache()


def test_bounded_waits_did_not_expire(pkg, torch_dev):
    import ctypes
    st = ctypes.c_int(-1)
    pkg.check(pkg.lib.cmlb200_attention8_status(ctypes.byref(st), 0))
    assert st.value == 0


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("heads,kv_heads", [(12, 1), (7, 1), (14, 2), (64, 2), (5, 5)])
def test_short_tiles_of_many_heads(pkg, torch_dev, form, heads, kv_heads):
    """Tiles whose rows and heads share blocks of 128 in every way: few rows of many heads, one less and one more than fill a block, the last tiles of longer portions."""
    L = Layer(pkg, torch_dev, form, heads, kv_heads, 40, 24, page=16, slopes=heads == 12, sink="own" if heads == 14 else None)
    L.ld += -L.ld % 4 if heads % 2 == 0 else 0         # rows that begin on 16 bytes, and that do not
    for parts in ([(0, 2), (1, 3), (2, 18)], [(0, 19), (1, 10), (2, 11)], [(0, 37), (1, 64), (2, 65)], [(0, 5), (1, 77), (2, 63)], [(0, 4), (1, 128), (2, 2)]):
        L.step(parts)
    L.check_cache()


def test_decode_far_into_the_pools(pkg, torch_dev):
    """Pages beyond the 32-bit offsets of a large pool, read and written through the table."""
    import torch
    pages, page, G, D = 70000, 64, 4, 128                                  # 2.3 GB a pool
    L = Layer(pkg, torch_dev, "i8", 8, G, D, D, page=page, slots=2, tokens=300)
    big = [torch.full((pages, page, G, D), 0x7F, dtype=torch.int8, device=torch_dev) for _ in range(2)]
    scales = [torch.full((pages, page // 16, G), float("nan"), device=torch_dev) for _ in range(2)]
    L.k, L.v, (L.ks, L.vs) = big[0], big[1], scales
    L.a.k_pool, L.a.v_pool, L.a.k_scale, L.a.v_scale = (x.data_ptr() for x in (*big, *scales))
    per = -(-300 // page)
    L.table[:, :per] = pages - 1 - np.arange(2 * per).reshape(2, per) * 3
    L.d_table.copy_(torch.from_numpy(L.table))
    for parts in ([(0, 70), (1, 200)], [(0, 1), (1, 1)], [(1, 1)], [(0, 65), (1, 1)]):
        L.step(parts)


CAPTURED_FIRST = """
import sys
sys.path[:0] = [{root!r}, {tests!r}]
import numpy as np, torch
import __graft_entry__ as entry
import test_gpu_cache8 as t
pkg = entry.load_package()
dev = torch.device("cuda:0")
L = t.Layer(pkg, dev, "i8", 8, 2, 64, 64, slots=2)
for s in range(2):
    for q in L.seqs[s]:
        q.append(np.zeros((0,) + q.codes.shape[1:]))
x, out = torch.randn(2, L.ld, device=dev), torch.zeros(2, 8 * 64, dtype=torch.bfloat16, device=dev)
pos, slot = torch.zeros(2, dtype=torch.int32, device=dev), torch.arange(2, dtype=torch.int32, device=dev)
tiles = torch.tensor([[0, 1, 0, 0], [1, 1, 1, 0]], dtype=torch.int32, device=dev)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    st = torch.cuda.current_stream().cuda_stream
    if {one}:
        pkg.check(pkg.lib.cmlb200_attention_one(L.a, x.data_ptr(), L.ld, pos.data_ptr(), slot.data_ptr(), 2, 0, out.data_ptr(), 512, st))
    else:
        pkg.check(pkg.lib.cmlb200_qk_norm_append(L.a, x.data_ptr(), L.ld, pos.data_ptr(), slot.data_ptr(), 2, st))
        pkg.check(pkg.lib.cmlb200_attention_tiles(L.a, x.data_ptr(), L.ld, tiles.data_ptr(), 2, out.data_ptr(), 512, st))
g.replay()
torch.cuda.synchronize()
v = x[:, L.width - 128:L.width].view(2, 2, 1, 64).expand(2, 2, 4, 64).reshape(2, 512)
assert (out.float() - v).abs().max() < v.abs().max() / 50, (out.float() - v).abs().max()
print("fine")
"""


@pytest.mark.parametrize("one", [True, False])
def test_captured_before_anything_else_ran(one):
    """The first call of a process is one that is being captured (a first token: attention returns its own value, an int8 rounding and bf16's away)."""
    import subprocess
    import sys
    from pathlib import Path
    tests = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST.format(root=str(tests.parent), tests=str(tests), one=one)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


def test_two_streams_at_once(pkg, torch_dev):
    """Decoding of two layers at a time, each over its own cache, gives what each gives alone."""
    import torch
    L = [Layer(pkg, torch_dev, f, 8, 2, 64, 64, slots=3, seed=k) for k, f in enumerate(("i8", "e4m3"))]
    for l in L:
        l.step([(0, 150), (1, 40), (2, 3)])
    streams = [torch.cuda.Stream(torch_dev) for _ in L]
    rows = [l.fresh_rows(3) for l in L]
    put = lambda a, k: torch.from_numpy(np.ascontiguousarray(a, k)).to(torch_dev)
    pos = [put([len(l.seqs[s][0].codes) for s in range(3)], np.int32) for l in L]
    slot, x = put([0, 1, 2], np.int32), [put(r, np.float32) for r in rows]
    out = [[torch.zeros(3, 512, dtype=torch.bfloat16, device=torch_dev) for _ in range(20)] for _ in L]
    torch.cuda.synchronize()
    for i in range(20):                                # (the same token again each time: it is the last of its group)
        for l, st, p, r, o in zip(L, streams, pos, x, out):
            pkg.check(pkg.lib.cmlb200_attention_one(l.a, r.data_ptr(), l.ld, p.data_ptr(), slot.data_ptr(), 3, 150, o[i].data_ptr(), 512, st.cuda_stream))
    torch.cuda.synchronize()
    for l, o, r in zip(L, out, rows):
        assert all(torch.equal(o[0], y) for y in o)
        got = l.step([(0, 1), (1, 1), (2, 1)], rows=r)
        assert np.array_equal(got, o[0].float().cpu().numpy().astype(np.float64))
