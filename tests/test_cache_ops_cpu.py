"""CPU tests of the cache operators' argument checks and rotary plans (no device needed: every
refusal here happens before the library touches one)."""
import ctypes as C
import math

import numpy as np
import pytest

import cache_ref as ref

INVALID, SHAPE, SMALL = 1, 2, 6
P = 0x1000        # an aligned address that no refused call reads


def append(ckl, **kw):
    f = dict(q=P, k=0x100000, v=0x200000, q_stride=1024, k_stride=256, v_stride=256, q_out=0x300000,
             k_cache=0x1000000, v_cache=0x2000000, kv_indptr=P, kv_indices=P, kv_last_page_len=P,
             q_indptr=P, positions=None, B=2, N=3, Hq=8, Hkv=2, num_pages=4)
    f.update(kw)
    return ckl.AppendParams(*[f[n] for n, _ in ckl.AppendParams._fields_])


@pytest.mark.parametrize("kw,status", [
    (dict(N=-1), INVALID), (dict(Hkv=0), INVALID), (dict(k=None), INVALID), (dict(q_out=None), INVALID),
    (dict(v_cache=None), INVALID), (dict(kv_indices=None), INVALID), (dict(q_indptr=None), INVALID),
    (dict(num_pages=0), INVALID), (dict(k=P + 2), INVALID), (dict(q_stride=1020), INVALID),
    (dict(k_stride=128), INVALID), (dict(v_stride=252), INVALID), (dict(q_out=P + 1024), INVALID),
    (dict(k_cache=0x100000), INVALID), (dict(v_cache=0x1000000), INVALID), (dict(Hkv=70000), SHAPE),
])
def test_append_refuses(ckl, kw, status):
    r = ckl.rope_plan(64)
    assert ckl.lib().ckl_rope_append(C.byref(append(ckl, **kw)), C.byref(r), None) == status
    assert ckl.lib().ckl_last_error_string()


def test_append_refuses_a_rope_that_is_no_plan_and_null(ckl):
    r = ckl.Rope()
    assert ckl.lib().ckl_rope_append(C.byref(append(ckl)), C.byref(r), None) == INVALID
    assert ckl.lib().ckl_rope_append(None, None, None) == INVALID
    # an empty batch is nothing to do
    assert ckl.lib().ckl_rope_append(C.byref(append(ckl, N=0)), None, None) == 0


def tree(ckl, **kw):
    f = dict(q=P, k_cache=P, v_cache=P, kv_indptr=P, kv_indices=P, kv_last_page_len=P, q_indptr=P,
             tree_mask=None, positions=None, slopes=None, B=2, N=5, Hq=8, Hkv=2, max_q=4, mask_words=0,
             num_chunks=1, chunk_tokens=32, window=0, num_pages=4, sm_scale=0.1, softcap=0.0)
    f.update(kw)
    return ckl.TreeParams(*[f[n] for n, _ in ckl.TreeParams._fields_])


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), INVALID), (dict(Hq=7), INVALID), (dict(Hq=258, Hkv=2), SHAPE), (dict(q=None), INVALID),
    (dict(q=P + 8), INVALID), (dict(kv_last_page_len=None), INVALID), (dict(num_pages=0), INVALID),
    (dict(max_q=0), INVALID), (dict(q_indptr=None), INVALID), (dict(tree_mask=P), INVALID),
    (dict(tree_mask=P, mask_words=1, max_q=33), INVALID), (dict(window=-1), INVALID),
    (dict(softcap=-1.0), INVALID), (dict(softcap=math.nan), INVALID), (dict(sm_scale=0.0), INVALID),
    (dict(sm_scale=math.inf), INVALID), (dict(B=70000), SHAPE),
])
def test_tree_and_weights_refuse(ckl, kw, status):
    p = tree(ckl, **kw)
    assert ckl.lib().ckl_tree_attention(C.byref(p), P, P, None, 0, None) == status
    assert ckl.lib().ckl_cache_weights(C.byref(p), P, P, 64, 1.0, None) == status


def test_tree_attention_refuses_split_outputs_and_workspace(ckl):
    L = ckl.lib()
    for kw in (dict(num_chunks=0), dict(chunk_tokens=24), dict(num_chunks=70000)):
        assert L.ckl_tree_attention(C.byref(tree(ckl, **kw)), P, P, P, 1 << 40, None) == INVALID
    assert L.ckl_tree_attention(C.byref(tree(ckl)), None, P, None, 0, None) == INVALID
    assert L.ckl_tree_attention(C.byref(tree(ckl)), P + 2, P, None, 0, None) == INVALID
    p = tree(ckl, num_chunks=3)
    need = L.ckl_tree_workspace_size(C.byref(p))
    assert need == 5 * 8 * 3 * 128 * 4 + 512
    assert L.ckl_tree_attention(C.byref(p), P, P, P, need - 1, None) == SMALL
    assert L.ckl_tree_attention(C.byref(p), P, P, None, need, None) == SMALL
    assert L.ckl_tree_attention(C.byref(p), P, P, P + 16, need, None) == INVALID
    assert L.ckl_tree_workspace_size(C.byref(tree(ckl))) == 0
    assert L.ckl_tree_attention(C.byref(tree(ckl, N=0)), P, P, None, 0, None) == 0


def test_weights_refuse(ckl):
    L, p = ckl.lib(), tree(ckl)
    assert L.ckl_cache_weights(C.byref(p), P, P, 0, 1.0, None) == INVALID
    assert L.ckl_cache_weights(C.byref(p), None, P, 64, 1.0, None) == INVALID
    for d in (-0.5, 1.5, math.nan):
        assert L.ckl_cache_weights(C.byref(p), P, P, 64, d, None) == INVALID
    assert L.ckl_cache_weights(C.byref(tree(ckl, B=0)), P, P, 64, 1.0, None) == 0


def test_tree_plan_covers_every_key(ckl):
    for G, B, Hkv, T, L, w, force in [(4, 2, 8, 6, 1000, 0, 3), (1, 1, 1, 1, 1, 0, 1), (8, 3, 2, 64, 70000, 0, 9),
                                      (4, 2, 8, 6, 100000, 500, 4), (4, 2, 8, 6, 0, 0, 2), (4, 1, 1, 1, 40, 0, 1000)]:
        nc, ct = C.c_int(), C.c_int()
        assert ckl.lib().ckl_tree_plan(G, B, Hkv, T, L, w, force, C.byref(nc), C.byref(ct)) == 0
        assert ct.value % 16 == 0 and 1 <= nc.value <= force
        assert nc.value * ct.value >= (min(L, w + T + 16) if w else L)
        assert (nc.value - 1) * ct.value < max(L, 1)                 # no chunk is empty for the longest
    for bad in [(0, 1, 1, 1, 1, 0, 1), (1, 0, 1, 1, 1, 0, 1), (1, 1, 1, 0, 1, 0, 1), (1, 1, 1, 1, -1, 0, 1)]:
        assert ckl.lib().ckl_tree_plan(*bad, C.byref(nc), C.byref(ct)) == INVALID
    assert ckl.lib().ckl_tree_plan(129, 1, 1, 1, 1, 0, 1, C.byref(nc), C.byref(ct)) == SHAPE


def test_select_and_compact_and_mask_refuse(ckl):
    L = ckl.lib()
    sel = lambda *a: L.ckl_cache_select(*a)
    assert sel(P, 64, P, P, 2, 8, 5, 4, P, P, None) == INVALID        # sink + recent > keep
    assert sel(P, 64, P, P, 2, 0, 0, 0, P, P, None) == INVALID
    assert sel(P, 0, P, P, 2, 8, 0, 0, P, P, None) == INVALID
    assert sel(None, 64, P, P, 2, 8, 0, 0, P, P, None) == INVALID
    assert sel(P, 64, P, P, 0, 8, 0, 0, P, P, None) == 0
    com = lambda k, v, B=2, Hkv=2, pages=4, idx=P, ks=8, cnt=P, acc=None, st=0: L.ckl_cache_compact(
        k, v, P, P, P, B, Hkv, pages, idx, ks, cnt, None, acc, st, None, None)
    assert com(P, 0x100000, idx=None) == INVALID
    assert com(P + 2, 0x100000) == INVALID
    assert com(P, P) == INVALID
    assert com(P, 0x100000, ks=0) == INVALID
    assert com(P, 0x100000, acc=P, st=0) == INVALID
    assert com(P, 0x100000, Hkv=0) == INVALID
    assert com(P, 0x100000, B=70000) == SHAPE
    assert com(P, 0x100000, B=0) == 0
    assert L.ckl_tree_mask(P, P, P, P, 2, 4, 0, P, None, None) == INVALID
    assert L.ckl_tree_mask(None, P, P, P, 2, 4, 1, P, None, None) == INVALID
    assert L.ckl_tree_mask(P, P, P, P, 70000, 4, 1, P, None, None) == SHAPE
    assert L.ckl_tree_mask(P, P, P, P, 2, 0, 1, P, None, None) == 0


@pytest.mark.parametrize("rot", [2, 20, 64, 128])
@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "by_parts"])
def test_rope_plan_turns(ckl, rot, scaling):
    """turns[i] is f_i / 2 pi as a binary fraction of 2^64 (f_i comes from pow in 64 bits: 2^-50
    of it is allowed)."""
    f, scale = ref.rope_angles(rot, scaling=scaling, factor=8.0)
    r = ckl.rope_plan(rot, scaling=scaling, factor=8.0, original_len=4096)
    assert r.rot_dim == rot and r.interleaved == 0 and abs(r.scale - scale) <= 2.0 ** -23 * scale
    for i in range(rot // 2):
        want = f[i] / (2 * np.longdouble(np.pi)) * np.longdouble(2) ** 64
        assert abs(float(np.longdouble(r.turns[i]) - want)) <= float(want) * 2.0 ** -50 + 2
    own = ckl.rope_plan(rot, inv_freq=[float(x) for x in f], scale=scale, interleaved=True)
    assert own.interleaved == 1
    assert all(abs(own.turns[i] - r.turns[i]) <= 2.0 ** -50 * r.turns[i] + 4 for i in range(rot // 2))


@pytest.mark.parametrize("kw", [dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=130), dict(base=1.0),
                                dict(base=math.inf), dict(scaling="linear", factor=0.5),
                                dict(scaling="by_parts", factor=2.0), dict(scaling="other"),
                                dict(scaling="by_parts", factor=2.0, original_len=4096, beta_fast=1.0),
                                dict(rot_dim=4, inv_freq=[1.0, -1.0]), dict(rot_dim=4, inv_freq=[1.0]),
                                dict(rot_dim=4, inv_freq=[1.0, math.nan]), dict(rot_dim=2, inv_freq=[4.0])])
def test_rope_plan_refuses(ckl, kw):
    with pytest.raises(ckl.CklError) as e:
        ckl.rope_plan(**kw)
    assert e.value.status == INVALID


def test_compact_refuses_outputs_that_overlap(ckl):
    """What one part of the call writes, other parts still read."""
    L = ckl.lib()
    # caches of 4 pages x 16 x 2 heads x 256 bytes = 32 KB; five sequences
    com = lambda k, v, cnt=P, start=None, new=None: L.ckl_cache_compact(
        k, v, P + 0x400, P, P + 0x800, 5, 2, 4, P, 8, cnt, start, None, 0, new, None)
    assert com(0x100000, 0x100000 + 32768 - 16) == INVALID
    assert com(0x100000 + 16, 0x100000) == INVALID
    for new in (P - 16, P, P + 16):
        assert com(0x100000, 0x200000, new=new) == INVALID                 # keep_count
    assert com(0x100000, 0x200000, start=P + 0x100, new=P + 0x100) == INVALID
    assert com(0x100000, 0x200000, new=P + 0x414) == INVALID               # the end of kv_indptr
    assert com(0x100000, 0x200000, new=P + 0x800) == INVALID               # kv_last_page_len
