"""Which cache a model really keeps: its logits are nearest to the restatement with that cache, and its pools have that cache's bytes."""
import numpy as np
import pytest

import lm_oracle
import lm_util
from cache8_oracle import Sequence
from lm_util import cut, error
from test_gpu_lm_serving import FORMS, build, feed, load, prompt  # noqa: F401 (load is a fixture)

pytestmark = pytest.mark.gpu


def with_cache(cfg, w, tokens, form, sizes, monkeypatch):
    """The restatement over what an 8-bit cache holds while the prompt is fed in portions of those sizes: a group's scale grows with its tokens, and each portion sees what
    the cache then holds."""
    plain = lm_oracle.attend

    def attend(q, k, v, q_pos, k_pos, mixer):
        ks, vs, out = Sequence(*k.shape[1:], form), Sequence(*v.shape[1:], form), []
        for a, b in cut(len(q), sizes):
            ks.append(k[a:b])
            vs.append(v[a:b])
            out.append(plain(q[a:b], ks.held(), vs.held(), q_pos[a:b], k_pos[:b], mixer))
        return np.concatenate(out)
    with monkeypatch.context() as m:
        m.setattr(lm_oracle, "attend", attend)
        return lm_util.reference(cfg, w, tokens)


def with_large_channels(synth, cfg, w, folder, by=16):
    """The first channel of every value head, and of every key head by its norm, `by` times as large, with the weights that meet them as much smaller. The model computes what
    it did; groups' scales grow with their largest channel, so int8 has four bits less for the others, e4m3 as many as before."""
    for i, layer in enumerate(cfg["layers"]):
        x = layer["mixer"]
        for h in range(x["kv_heads"]):
            w[f"l{i}.mix.v"][h * x["vdim"]] *= by
            w[f"l{i}.mix.k.norm"][h * x["dim"]] *= by
        for h in range(x["heads"]):
            w[f"l{i}.mix.o"][:, h * x["vdim"]] /= by
            w[f"l{i}.mix.q.norm"][h * x["dim"]] /= by
    synth.write_layered(folder, cfg, w)


@pytest.mark.parametrize("sizes", [[150], [70, 2, 1, 1, 31], [1]])
def test_each_form_is_itself(synth, tmp_path, load, monkeypatch, sizes):  # noqa: F811
    """A model that kept another cache than it was asked for would be nearest to that one's restatement. (Channels are of different sizes because keys and values differ from
    the restatement's by bf16 products, 2^-9 of themselves: beside an int8 step of 2^-7 of the largest one that moves a fifth of the codes, as much of an error as the codes'
    own. With channel 0 sixteen times the others a step is as large as most values, and the restatements, fed keys and values 2^-9 off, are 0.12 to 0.15 (int8) and 0.06 (e4m3)
    from themselves, 0.30 to 0.43 and 0.10 to 0.43 from the others.)"""
    cfg, w, folder = build(synth, tmp_path, "plain", monkeypatch)
    with_large_channels(synth, cfg, w, folder)
    t = prompt(cfg, 150)
    want = {0: lm_util.reference(cfg, w, t), **{v: with_cache(cfg, w, t, form, sizes, monkeypatch) for form, v in FORMS.items()}}
    for cache in want:
        m = load(folder, cache=cache)
        got = feed(m, m.open(), t, sizes)
        off = {k: error(got, r) for k, r in want.items()}
        assert min(off, key=off.get) == cache, (cache, off)


def test_bytes_of_the_pools(synth, tmp_path, load, monkeypatch):  # noqa: F811
    """2^19 tokens of 2 layers with 1 and 2 heads of 32 and 32: 192 numbers a token, and 6 scales for 16 tokens."""
    import torch
    cfg, w, folder = build(synth, tmp_path, "plain", monkeypatch)
    tokens, room = 1 << 19, {}
    small = load(folder, max_tokens=1024, max_sequences=2, max_step_rows=64)       # (what a process's first model brings with it)
    for cache in (0, 1, 2):
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        m = load(folder, max_tokens=tokens, max_sequences=2, max_step_rows=64, cache=cache)
        room[cache] = before - torch.cuda.mem_get_info()[0]
        m.close()
    small.close()
    saved = tokens * 192 * (2 - 1) - tokens // 16 * 6 * 4
    for cache in (1, 2):                               # (each of up to 8 buffers is rounded to whole 2 MB)
        assert abs(room[0] - room[cache] - saved) < 16 << 20, room
