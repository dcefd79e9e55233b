"""What the entry points of 8-bit caches, pages and token scores refuse: every one of these calls returns before it reaches a device."""
import ctypes as C

import pytest

P = 1 << 20                                            # a pointer that nothing follows


def attn(pkg, **kw):
    base = dict(heads=4, kv_heads=2, dim=64, vdim=64, dim_ld=64, vdim_ld=64, scale=0.1, gate_col=-1, cache_dtype=pkg.DT_I8, k_pool=P, v_pool=P, block_size=16, block_table=P, table_ld=4, k_scale=P,
                v_scale=P)
    return pkg.Attn(**{**base, **kw})


BAD = [dict(k_scale=None), dict(v_scale=None), dict(scores=P, scores_ld=64), dict(talk=P), dict(taps=3, conv=P, ring=P), dict(cap=2.0), dict(dim=300, dim_ld=304), dict(vdim=300, vdim_ld=304),
       dict(cache_dtype=5), dict(cache_dtype=-1), dict(block_size=24), dict(block_size=8), dict(k_pool=P + 8), dict(dim_ld=72), dict(kv_heads=3), dict(k_pool=None), dict(block_table=None)]


@pytest.mark.parametrize("bad", BAD)
def test_8_bit_caches(pkg, bad):
    a, L = attn(pkg, **bad), pkg.lib
    assert L.cmlb200_attention_one(a, P, 512, P, P, 1, 10, P, 256, None) == -1
    assert L.cmlb200_attention_tiles(a, P, 512, P, 1, P, 256, None) == -1
    assert L.cmlb200_qk_norm_append(a, P, 512, P, P, 1, None) == -1
    assert L.cmlb200_rotate_append(a, P, 512, P, P, 0, 1, 0, None, None) == -1
    assert L.cmlb200_last_error()


def test_8_bit_caches_elsewhere(pkg):
    L = pkg.lib
    a = attn(pkg)
    assert L.cmlb200_attention_rows_f32(a, P, 512, P, P, 1, P, 256, None) == -1
    assert L.cmlb200_talk_scores_rows(a, P, P, P, 1, 64, P, 64, None) == -1
    assert L.cmlb200_talk_scores_tiles(a, P, P, 1, 64, P, 64, None) == -1
    assert L.cmlb200_attention_one(attn(pkg, gate_wide=1, gate_col=400), P, 700, P, P, 1, 10, P, 256, None) == -1
    assert L.cmlb200_rotate_append(attn(pkg, freq=P, rot_dims=64), P, 512, P, P, 0, 1, 0, P, None) == -1
    assert L.cmlb200_qk_norm_append(a, P, 511, P, P, 1, None) == -1
    assert L.cmlb200_attention_tiles(a, P, 512, P + 4, 1, P, 256, None) == -1
    assert L.cmlb200_attention_one(a, P, 512, P, P, 0, 10, P, 256, None) == -1
    assert L.cmlb200_attention_one(a, P, 512, P, P, 1, -1, P, 256, None) == -1


@pytest.mark.parametrize("args", [(None, 0, 10, 1, 10, P, 0, P, P, None, None), (P, 0, 9, 1, 10, P, 0, P, P, None, None), (P, 0, 10, 0, 10, P, 0, P, P, None, None),
                                  (P, 0, 10, 1, 0, P, 0, P, P, None, None), (P, 0, 10, 1, 10, P, 11, P, P, P, P), (P, 0, 100, 1, 100, P, 33, P, P, P, P), (P, 0, 10, 1, 10, P, -1, P, P, P, P),
                                  (P, 0, 10, 1, 10, P, 3, P, P, None, None), (P, 0, 10, 1, 10, None, 0, P, P, None, None), (P, 0, 10, 1, 10, P, 0, None, P, None, None),
                                  (P, 0, 10, 1, 10, None, 0, None, None, None, None), (P, 3, 10, 1, 10, P, 0, P, P, None, None), (P + 2, 0, 10, 1, 10, P, 0, P, P, None, None),
                                  (P + 1, 1, 10, 1, 10, P, 0, P, P, None, None)])
def test_token_scores(pkg, args):
    assert pkg.lib.cmlb200_token_scores(*args, None) == -1


def test_pages(pkg):
    L = pkg.lib
    ok = dict(pools=2, pool=P, most=64, pages=10, table=P, slots=2, table_ld=4)
    for bad in (dict(pool=None), dict(pools=-1), dict(pools=65535), dict(pages=0), dict(slots=0), dict(table_ld=0), dict(most=1 << 40), dict(pools=0, pool=None, table=None)):
        assert L.cmlb200_pages_copy(pkg.Pages(**{**ok, **bad}), P, 1, None) == -1
    for bad in (dict(pool=None), dict(table=None), dict(slots=0)):
        assert L.cmlb200_pages_fork(pkg.Pages(**{**ok, **bad}), P, 1, None) == -1
    p = pkg.Pages(**ok)
    assert L.cmlb200_pages_copy(None, P, 1, None) == -1 and L.cmlb200_pages_copy(p, None, 1, None) == -1 and L.cmlb200_pages_copy(p, P, 0, None) == -1
    assert L.cmlb200_pages_copy(p, P + 4, 1, None) == -1 and L.cmlb200_pages_fork(p, P + 8, 1, None) == -1 and L.cmlb200_pages_fork(p, P, -1, None) == -1
