"""GPU tests of the operators that write, verify and trim the paged cache, against their
64-bit restatements (tests/cache_ref.py, where the tolerances are derived)."""
import numpy as np
import pytest

import cache_ref as ref

pytestmark = pytest.mark.gpu


def up(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def table(bt, dev):
    return dict(kv_indptr=up(bt.indptr, dev), kv_indices=up(bt.indices, dev),
                kv_last_page_len=up(bt.last, dev))


def finish(ckl):
    import torch
    torch.cuda.synchronize()
    ckl.check_device_error()


# ------------------------------------------------------------------ rotary append
ROPES = [(128, False, "none"), (128, True, "by_parts"), (64, False, "ntk"), (64, True, "linear"),
         (48, False, "none"), (40, True, "none"), (20, False, "by_parts"), (18, True, "none"),
         (2, False, "ntk"), (126, True, "linear")]


@pytest.mark.parametrize("rot,inter,scaling", ROPES)
@pytest.mark.parametrize("toks,Hq,Hkv", [([1, 1, 1], 8, 2), ([5, 0, 33, 1], 6, 3), ([70], 4, 4)])
def test_rope_append(ckl, dev, rot, inter, scaling, toks, Hq, Hkv):
    import torch
    lens = [t + c for t, c in zip(toks, (40, 0, 7, 300))]
    bt = ref.Batch(lens, toks, Hq, Hkv, 3, extra_rows=2)
    r = np.random.default_rng(5)
    N = bt.N
    qkv = up(r.standard_normal((N, (Hq + 2 * Hkv) * 128)).astype(np.float16), dev)
    pos = r.integers(-50, 2 ** 31 - 1, N).astype(np.int32)
    pos[:1] = 2 ** 31 - 1
    q, k, v = qkv.split([Hq * 128, Hkv * 128, Hkv * 128], 1)
    kc, vc = up(bt.k, dev), up(bt.v, dev)
    q_out = torch.full((N, Hq, 128), 7.0, dtype=torch.float16, device=dev)
    plan = ckl.rope_plan(rot, interleaved=inter, scaling=scaling, factor=4.0, original_len=4096)
    p = ckl.make_append_params(q.unflatten(1, (Hq, 128)), k.unflatten(1, (Hkv, 128)),
                               v.unflatten(1, (Hkv, 128)), kc, vc, **table(bt, dev), q_out=q_out,
                               q_indptr=up(bt.q_indptr, dev), positions=up(pos, dev))
    ckl.rope_append(p, plan)
    finish(ckl)
    f, scale = ref.rope_angles(rot, scaling=scaling, factor=4.0)
    x = qkv.cpu().numpy().reshape(N, Hq + 2 * Hkv, 128)
    y, tol = ref.rotate(x[:, :Hq + Hkv], pos, rot, inter, f, scale)
    n = bt.T_total
    got = q_out.float().cpu().numpy()
    assert np.all(np.abs(got[:n] - y[:n, :Hq]) <= tol[:n, :Hq])
    assert np.all(got[n:] == 7.0)                             # rows behind the last sequence
    wk, wv = bt.k.copy().reshape(-1, Hkv, 128), bt.v.copy().reshape(-1, Hkv, 128)
    gk, gv = kc.cpu().numpy().reshape(-1, Hkv, 128), vc.cpu().numpy().reshape(-1, Hkv, 128)
    touched = np.zeros(len(wk), bool)
    for b in range(bt.B):
        s = bt.slots(b)[bt.lens[b] - bt.toks[b]:]
        touched[s] = True
        rows = slice(bt.q_indptr[b], bt.q_indptr[b + 1])
        assert np.all(np.abs(gk[s].astype(np.float64) - y[rows, Hq:]) <= tol[rows, Hq:])
        assert np.array_equal(gv[s], x[rows, Hq + Hkv:])
    assert np.array_equal(gk[~touched], wk[~touched], equal_nan=True)
    assert np.array_equal(gv[~touched], wv[~touched], equal_nan=True)


def test_rope_append_one_token_each_places_and_copies(ckl, dev):
    """q_indptr None, positions None (the cache places), rope None (a copy), q None."""
    import torch
    bt = ref.Batch([1, 16, 17, 500], [1] * 4, 4, 2, 8)
    r = np.random.default_rng(1)
    q, k, v = (up(r.standard_normal((4, h, 128)).astype(np.float16), dev) for h in (4, 2, 2))
    kc, vc = up(bt.k, dev), up(bt.v, dev)
    p = ckl.make_append_params(q, k, v, kc, vc, **table(bt, dev))
    out = ckl.rope_append(p, ckl.rope_plan(128))
    finish(ckl)
    f, scale = ref.rope_angles(128)
    place = np.array(bt.lens) - 1
    y, tol = ref.rotate(q.cpu().numpy(), place, 128, False, f, scale)
    assert np.all(np.abs(out.float().cpu().numpy() - y) <= tol)
    p = ckl.make_append_params(None, k, v, kc, vc, **table(bt, dev))
    assert ckl.rope_append(p) is None
    finish(ckl)
    s = [bt.slots(b)[-1] for b in range(4)]
    assert torch.equal(kc.view(-1, 2, 128)[s], k) and torch.equal(vc.view(-1, 2, 128)[s], v)


def test_rope_append_without_a_place(ckl, dev):
    """Tokens that the page table has no place for, and pages outside the cache, are not
    written; their q is."""
    import torch
    bt = ref.Batch([3, 20], [5, 4], 2, 1, 8)                  # 5 new tokens, 3 places
    kc, vc = up(bt.k, dev), up(bt.v, dev)
    t = table(bt, dev)
    ids = bt.indices.copy()
    ids[-1] = bt.num_pages + 5                                # the second sequence's last page
    t["kv_indices"] = up(ids, dev)
    r = np.random.default_rng(1)
    q, k, v = (up(r.standard_normal((9, h, 128)).astype(np.float16), dev) for h in (2, 1, 1))
    p = ckl.make_append_params(q, k, v, kc, vc, **t, q_indptr=up(bt.q_indptr, dev))
    out = ckl.rope_append(p)
    finish(ckl)
    want = bt.k.copy().reshape(-1, 1, 128)
    want[bt.slots(0)] = k.cpu().numpy()[2:5]
    assert np.array_equal(kc.cpu().numpy().reshape(-1, 1, 128), want, equal_nan=True)
    assert torch.equal(out, q)


# ------------------------------------------------------------------ tree attention
def run_tree(ckl, dev, bt, max_len=None, force=0, max_q=None, q_indptr=True, **opt):
    kw = {}
    if opt.get("mask") is not None:
        kw["tree_mask"] = up(opt["mask"], dev)
    if opt.get("positions") is not None:
        kw["positions"] = up(opt["positions"], dev)
    if opt.get("slopes") is not None:
        kw["slopes"] = up(opt["slopes"].astype(np.float32), dev)
    p = ckl.make_tree_params(up(bt.q, dev), up(bt.k, dev), up(bt.v, dev), **table(bt, dev),
                             max_len=max_len or max(bt.lens), q_indptr=up(bt.q_indptr, dev) if q_indptr else None,
                             max_q=max_q or max(max(bt.toks), 1), softcap=opt.get("softcap", 0.0),
                             window=opt.get("window", 0), force_chunks=force, **kw)
    return p


def check_tree(ckl, dev, bt, force=0, max_len=None, **opt):
    import torch
    p = run_tree(ckl, dev, bt, force=force, max_len=max_len, **opt)
    out = torch.full((bt.N, bt.Hq, 128), 9.0, dtype=torch.float16, device=dev)
    lse = torch.full((bt.N, bt.Hq), 9.0, dtype=torch.float32, device=dev)
    ckl.tree_attention(p, out=out, lse=lse)
    finish(ckl)
    want, wl, tol, ltol = ref.attention(bt, **opt)
    o, l, n = out.float().cpu().numpy(), lse.cpu().numpy(), bt.T_total
    assert np.all(o[n:] == 9.0) and np.all(l[n:] == 9.0)      # rows behind the last sequence
    assert np.isfinite(o[:n]).all()
    err = np.abs(o[:n] - want) - tol
    assert np.all(err <= 0), f"out off by {err.max():.3e} more than its bound"
    dead = np.isneginf(wl)
    assert np.array_equal(dead, np.isneginf(l[:n])) and np.all(o[:n][dead] == 0)
    lerr = np.abs(l[:n][~dead] - wl[~dead]) - ltol[~dead]
    assert np.all(lerr <= 0), f"lse off by {lerr.max():.3e} more than its bound"
    return o, l


SHAPES = [([1], [1], 1, 1), ([40, 16, 17], [3, 16, 1], 8, 2), ([300, 1000], [7, 6], 32, 8),
          ([130, 64, 5, 700], [33, 64, 5, 2], 8, 2), ([90, 33], [17, 9], 5, 1), ([260], [140], 2, 1),
          ([50, 49], [3, 2], 128, 1), ([2000, 31], [1, 1], 14, 2)]


@pytest.mark.parametrize("lens,toks,Hq,Hkv", SHAPES)
@pytest.mark.parametrize("force", [1, 0, 5])
def test_tree_chain(ckl, dev, lens, toks, Hq, Hkv, force):
    check_tree(ckl, dev, ref.Batch(lens, toks, Hq, Hkv, 11, extra_rows=1), force=force)


OPTS = [dict(), dict(softcap=5.0), dict(window=20), dict(bias=True), dict(softcap=30.0, bias=True, window=100)]


@pytest.mark.parametrize("lens,toks,Hq,Hkv", SHAPES[1:])
@pytest.mark.parametrize("opt", OPTS, ids=str)
def test_tree_masks_and_scores(ckl, dev, lens, toks, Hq, Hkv, opt):
    bt = ref.Batch(lens, toks, Hq, Hkv, 12, qscale=2.0)
    _, mask, pos = bt.random_tree(4)
    o = dict(opt)
    if o.pop("bias", False):
        o["slopes"] = np.float32(2.0) ** (-8.0 * (np.arange(Hq, dtype=np.float32) + 1) / Hq)
    check_tree(ckl, dev, bt, force=3, mask=mask, positions=pos, **o)


@pytest.mark.parametrize("toks,Hq", [([6, 5, 20], 4), ([6, 5, 40], 8)])
def test_tree_rows_that_see_nothing(ckl, dev, toks, Hq):
    """Empty mask rows without context, sequences without tokens or keys, more tokens than
    cached places, and a window that ends before the first key."""
    bt = ref.Batch([6, 0, 20, 37, 3], [toks[0], 0, toks[2] - 1 if toks[2] <= 20 else 20, 0, 5], Hq, 2, 5)
    mask = np.zeros((bt.N, 2), np.int32)
    mask[1, 0] = 1
    mask[bt.q_indptr[2] + 3, 0] = -1
    mask[bt.q_indptr[4]:, 0] = 0b11101
    for force in (1, 2):
        check_tree(ckl, dev, bt, force=force, mask=mask)
        check_tree(ckl, dev, bt, force=force)
        far = np.full(bt.N, 2 ** 31 - 1, np.int32)
        check_tree(ckl, dev, bt, force=force, positions=far, window=7)


@pytest.mark.parametrize("toks,Hq", [([4, 3], 4), ([30, 40], 8)])
@pytest.mark.parametrize("force", [1, 3])
def test_tree_unseen_keys_do_not_leak(ckl, dev, toks, Hq, force):
    """Infinities and NaN in keys that a token does not see (other branches, out of its window)
    leave it as it is; NaN behind the sequence never matters."""
    bt = ref.Batch([70, 55], toks, Hq, 2, 6)
    _, mask, pos = bt.random_tree(9)
    clean = check_tree(ckl, dev, bt, force=force, mask=mask, positions=pos)
    m = mask.view(np.uint32)
    for b in range(2):
        q0, T = bt.q_indptr[b], bt.toks[b]
        j = T - 1                                             # the last drafted token: a leaf
        s = bt.slots(b)[bt.lens[b] - 1]
        bt.k.reshape(-1, 2, 128)[s, :, 5] = np.nan
        bt.v.reshape(-1, 2, 128)[s, 0, ::7] = np.inf
        bt.v.reshape(-1, 2, 128)[s, 1, 3::5] = np.nan
        bt.v.reshape(-1, 2, 128)[s, 1, 2::5] = -np.inf
    p = run_tree(ckl, dev, bt, force=force, mask=mask, positions=pos)
    out, lse = ckl.tree_attention(p)
    finish(ckl)
    o, l = out.float().cpu().numpy(), lse.cpu().numpy()
    for b in range(2):
        q0, T = bt.q_indptr[b], bt.toks[b]
        for i in range(T):
            if (m[q0 + i, (T - 1) // 32] >> np.uint32((T - 1) % 32)) & 1:
                assert np.isnan(o[q0 + i]).any()              # the one that sees it does not hide it
            else:
                want, _, tol, _ = clean_ref(bt, b, i, mask, pos)
                assert np.all(np.abs(o[q0 + i] - want) <= tol)
                assert np.array_equal(l[q0 + i], clean[1][q0 + i])
    # an infinite value that its token sees reaches it as infinity, where the scores are finite
    bt = ref.Batch([40, 33], toks, Hq, 2, 6) if max(toks) < 33 else ref.Batch([80, 73], toks, Hq, 2, 6)
    for b in range(2):
        bt.v.reshape(-1, 2, 128)[bt.slots(b)[-1], :, 9] = np.inf
    o = ckl.tree_attention(run_tree(ckl, dev, bt, force=force))[0].float().cpu().numpy()
    finish(ckl)
    for b in range(2):
        q0, T = bt.q_indptr[b], bt.toks[b]
        assert np.all(np.isposinf(o[q0 + T - 1, :, 9]))
        assert np.isfinite(np.delete(o[q0 + T - 1], 9, axis=1)).all() and np.isfinite(o[q0:q0 + T - 1]).all()


def clean_ref(bt, b, i, mask, pos):
    """The result of token i of sequence b, the other tokens' bad keys unseen."""
    q0 = bt.q_indptr[b]
    s, big = ref.scores(bt, b, mask=mask, positions=pos)
    v = bt.v.reshape(-1, bt.Hkv, 128)[bt.slots(b)].astype(np.float64)
    out, tol = np.zeros((bt.Hq, 128)), np.zeros((bt.Hq, 128))
    for h in range(bt.Hq):
        x = s[h, i]
        see = x > -np.inf
        p = np.exp(x[see] - x[see].max())
        vv = v[see, h // bt.G]
        out[h] = (p[:, None] * vv).sum(0) / p.sum()
        mag = (p[:, None] * np.abs(vv)).sum(0) / p.sum()
        ds = 2.0 ** -24 * (128 * 40.0 + 8 * 40.0)             # |q.k| scale: below 40 here
        tol[h] = mag * (2.0 ** -10 + 2 * ds + 2.0 ** -18) + 2.0 ** -25 * (1 + len(p) * np.abs(vv).max() / p.sum())
    return out, None, tol, None


def test_tree_window_reads_the_right_keys(ckl, dev):
    """Windows around page and chunk borders, sequences longer than planned for."""
    bt = ref.Batch([333, 1200, 15], [3, 5, 2], 8, 2, 21)
    for w in (1, 2, 15, 16, 17, 64, 1199, 5000):
        check_tree(ckl, dev, bt, force=3, window=w)
    check_tree(ckl, dev, bt, force=4, max_len=100)
    check_tree(ckl, dev, bt, force=4, max_len=100, window=800)


def test_tree_one_token_equals_decode(ckl, dev):
    """One token per sequence without options: decode_attention's results (each is within the
    bound of the 64-bit result; the two differ by at most both bounds)."""
    bt = ref.Batch([5, 300, 2049, 1], [1] * 4, 32, 8, 7)
    p = run_tree(ckl, dev, bt, q_indptr=False)
    o, l = ckl.tree_attention(p)
    od, ld = ckl.decode_attention(up(bt.q, dev), up(np.nan_to_num(bt.k), dev), up(np.nan_to_num(bt.v), dev),
                                  **table(bt, dev))
    finish(ckl)
    _, _, tol, ltol = ref.attention(bt)
    assert np.all(np.abs(o.float().cpu().numpy() - od.float().cpu().numpy()) <= 2 * tol)
    assert np.all(np.abs(l.cpu().numpy() - ld.cpu().numpy()) <= 2 * ltol)


def test_tree_more_tokens_than_max_q(ckl, dev):
    import torch
    bt = ref.Batch([50, 60], [9, 2], 4, 2, 3)
    p = run_tree(ckl, dev, bt, max_q=4)
    out = torch.full((bt.N, 4, 128), 9.0, dtype=torch.float16, device=dev)
    ckl.tree_attention(p, out=out)
    torch.cuda.synchronize()
    with pytest.raises(ckl.CklError) as e:
        ckl.check_device_error()
    assert e.value.status == 1
    want, _, tol, _ = ref.attention(bt)
    o = out.float().cpu().numpy()
    assert np.all(o[4:9] == 9.0)
    rows = [0, 1, 2, 3, 9, 10]
    assert np.all(np.abs(o[rows] - want[rows]) <= tol[rows])


@pytest.mark.parametrize("toks,Hq", [([3, 5], 8), ([40, 37], 8)])
def test_tree_repeats_streams_and_graphs(ckl, dev, toks, Hq):
    """Same bits again, on another stream, two calls at once with a workspace each, and
    captured and replayed after the inputs changed."""
    import torch
    bt, bt2 = (ref.Batch([900, 1100], toks, Hq, 2, s) for s in (31, 32))
    _, mask, pos = bt.random_tree(1)
    p = run_tree(ckl, dev, bt, force=4, mask=mask, positions=pos)
    q = run_tree(ckl, dev, bt2, force=4)
    a, al = ckl.tree_attention(p)
    c, _ = ckl.tree_attention(q)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(3):
        outs.append((ckl.tree_attention(p, stream=s1)[0], ckl.tree_attention(q, stream=s2)[0]))
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(x, a) and torch.equal(y, c)
    out, lse = torch.empty_like(a), torch.empty_like(al)
    ws = torch.empty(ckl.tree_workspace_size(p), dtype=torch.uint8, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ckl.tree_attention(p, out=out, lse=lse, workspace=ws)
    for _ in range(2):
        out.fill_(3.0)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, a) and torch.equal(lse, al)
    p._keep[0].copy_(-p._keep[0])
    g.replay()
    want = ckl.tree_attention(p)[0]
    finish(ckl)
    assert torch.equal(out, want) and not torch.equal(out, a)


@pytest.mark.parametrize("toks,Hq", [(9, 8), (33, 16), (3, 8)])
def test_tree_many_calls_in_a_row(ckl, dev, toks, Hq):
    """Hundreds of calls without a wait between them: the same bits, and no barrier that gave up
    (one that a fast warp could pass twice shows as a time-out here)."""
    import torch
    bt = ref.Batch([1800 + 130 * i for i in range(8)], [toks] * 8, Hq, 2, 41)
    p = run_tree(ckl, dev, bt)
    ws = torch.empty(max(ckl.tree_workspace_size(p), 256), dtype=torch.uint8, device=dev)
    want, wl = ckl.tree_attention(p)
    out, lse = torch.empty_like(want), torch.empty_like(wl)
    acc = torch.zeros((8, 3000), device=dev)
    one = ckl.cache_weights(p, wl, acc.clone())
    for _ in range(300):
        ckl.tree_attention(p, out=out, lse=lse, workspace=ws)
        ckl.cache_weights(p, wl, acc, decay=0.0)
    finish(ckl)
    assert torch.equal(out, want) and torch.equal(lse, wl) and torch.equal(acc, one)


def test_tree_mask_of_parents(ckl, dev):
    bt = ref.Batch([30, 90, 4, 50], [5, 70, 0, 33], 2, 1, 3, extra_rows=2)
    parents, mask, pos = bt.random_tree(8)
    m, p = ckl.tree_mask(up(parents, dev), up(bt.q_indptr, dev), up(bt.indptr, dev), up(bt.last, dev), 70)
    finish(ckl)
    n = bt.T_total
    assert np.array_equal(m.cpu().numpy()[:n], mask[:n]) and np.array_equal(p.cpu().numpy()[:n], pos[:n])
    # a parent that is not lower than its child is a root; tokens behind the words have no bit
    bad = np.array([0, 5, 0, 7], np.int32)
    m, p = ckl.tree_mask(up(bad, dev), up(np.array([0, 4], np.int32), dev), up(np.array([0, 1], np.int32), dev),
                         up(np.array([10], np.int32), dev), 4)
    finish(ckl)
    assert m.cpu().numpy()[:, 0].tolist() == [1, 2, 5, 8] and p.cpu().numpy().tolist() == [6, 6, 7, 6]


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("lens,toks,Hq,Hkv", SHAPES + [([100, 600], [1, 3], 48, 12), ([400], [64], 16, 1)])
@pytest.mark.parametrize("opt", OPTS[:1] + OPTS[-1:], ids=str)
def test_cache_weights(ckl, dev, lens, toks, Hq, Hkv, opt):
    import torch
    bt = ref.Batch(lens, toks, Hq, Hkv, 15)
    _, mask, pos = bt.random_tree(4)
    o = dict(opt)
    if o.pop("bias", False):
        o.update(slopes=np.float32(2.0) ** (-8.0 * (np.arange(Hq, dtype=np.float32) + 1) / Hq),
                 mask=mask, positions=pos)
    _, lse, _, _ = ref.attention(bt, **o)
    lse = lse.astype(np.float32)
    p = run_tree(ckl, dev, bt, **o)
    r = np.random.default_rng(2)
    for decay, stride in ((1.0, max(lens)), (0.25, max(lens) + 5), (0.0, max(1, max(lens) - 9))):
        acc = r.random((len(lens), stride)).astype(np.float32)
        buf = up(acc, dev)
        if decay == 0.0:
            buf.fill_(float("nan"))                           # not read
        ckl.cache_weights(p, up(lse, dev), buf, decay=decay)
        finish(ckl)
        want, tol = ref.weights(bt, acc, lse, decay, **o)
        got = buf.cpu().numpy()
        for b, L in enumerate(lens):
            n = min(L, stride)
            assert np.all(np.abs(got[b, :n] - want[b, :n]) <= tol[b, :n] + 2.0 ** -23 * np.abs(want[b, :n]))
            assert np.array_equal(got[b, n:], buf.cpu().numpy()[b, n:], equal_nan=True)
            if decay:
                assert np.array_equal(got[b, n:], acc[b, n:])


def test_cache_weights_sum_and_repeat(ckl, dev):
    """Every row gives away a weight of 1 in all; the same bits every time."""
    import torch
    bt = ref.Batch([3000, 17], [4, 1], 16, 4, 3)
    p = run_tree(ckl, dev, bt)
    _, lse = ckl.tree_attention(p)
    got = [ckl.cache_weights(p, lse, torch.zeros((2, 3000), device=dev)) for _ in range(3)]
    finish(ckl)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    s = got[0].double().sum(1).cpu().numpy()
    # lse and weights are within 2^-14 here (tests above): so are the sums
    assert np.all(np.abs(s - np.array([64.0, 16.0])) <= np.array([64.0, 16.0]) * 2.0 ** -13)


# ------------------------------------------------------------------ select
def run_select(ckl, dev, acc, lens, keep, sink=0, recent=0):
    np_ = [(l + 15) // 16 for l in lens]
    indptr = np.concatenate([[0], np.cumsum(np_)]).astype(np.int32)
    last = np.array([l - (n - 1) * 16 if n else 0 for l, n in zip(lens, np_)], np.int32)
    i, c = ckl.cache_select(up(acc, dev), up(indptr, dev), up(last, dev), keep, sink=sink, recent=recent)
    finish(ckl)
    wi, wc = ref.select(acc, lens, keep, sink, recent)
    assert np.array_equal(c.cpu().numpy(), wc)
    assert np.array_equal(i.cpu().numpy(), wi)


@pytest.mark.parametrize("L,keep,sink,recent", [(1, 1, 0, 0), (5, 8, 2, 2), (100, 100, 4, 4), (101, 100, 4, 4),
                                                (1000, 1, 0, 0), (1000, 10, 6, 4), (1025, 300, 0, 17),
                                                (5000, 4999, 1, 1), (40000, 9000, 16, 1000), (140000, 333, 0, 0)])
@pytest.mark.parametrize("kind", ["smooth", "ties", "same"])
def test_cache_select(ckl, dev, L, keep, sink, recent, kind):
    r = np.random.default_rng(L)
    lens = [L, max(1, L // 2), max(1, L - 3)]
    acc = r.random((3, L)).astype(np.float32) ** 4
    if kind == "ties":
        acc = np.round(acc * 8).astype(np.float32) / 8
    if kind == "same":
        acc[:] = 0.5
    run_select(ckl, dev, acc, lens, keep, sink, recent)


def test_cache_select_odd_values(ckl, dev):
    """NaN ranks last, then -inf; -0 and 0 tie; denormals count; places behind acc rank as NaN."""
    r = np.random.default_rng(3)
    pool = np.array([np.nan, -np.inf, -1.0, -0.0, 0.0, 1e-45, -1e-45, 1.0, np.inf, 3e38], np.float32)
    acc = pool[r.integers(0, len(pool), (4, 300))]
    for keep in (1, 30, 150, 299):
        run_select(ckl, dev, acc, [300, 290, 17, 0], keep)
    run_select(ckl, dev, acc[:, :100].copy(), [300, 290, 17, 0], 150, 3, 9)


# ------------------------------------------------------------------ compact
def lists(bt, how, n, seed):
    r = np.random.default_rng(seed)
    rows, start = [], []
    for L, T in zip(bt.lens, bt.toks):
        s = L - T if how == "path" else 0
        k = min(n, L - s)
        rows.append(np.sort(r.choice(np.arange(s, L), k, replace=False)))
        start.append(s)
    idx = np.full((bt.B, n), 12345678, np.int32)
    for b, x in enumerate(rows):
        idx[b, :len(x)] = x
    return idx, np.array([len(x) for x in rows], np.int32), np.array(start, np.int32)


def want_compact(bt, idx, count, start, acc):
    k, v, a = bt.k.copy().reshape(-1, bt.Hkv, 128), bt.v.copy().reshape(-1, bt.Hkv, 128), None if acc is None else acc.copy()
    for b in range(bt.B):
        s, n, L = bt.slots(b), count[b], bt.lens[b]
        src, dst = idx[b, :n], np.arange(start[b], start[b] + n)
        k[s[dst]], v[s[dst]] = k[s[src]].copy(), v[s[src]].copy()
        if a is not None:
            m = a.shape[1]
            row = np.concatenate([a[b], np.zeros(max(0, L - m), np.float32)])
            new = row.copy()
            new[dst] = row[src]
            new[start[b] + n:L] = 0
            a[b] = new[:m]
    return k, v, a


@pytest.mark.parametrize("lens,toks,Hkv", [([40, 17, 1], [6, 17, 1], 2), ([5000, 900], [64, 3], 8), ([20000], [30], 1),
                                           ([300] * 40, [20] * 40, 3)])
@pytest.mark.parametrize("how,frac", [("path", 0.0), ("evict", 0.02), ("evict", 0.5), ("evict", 1.0)])
def test_cache_compact(ckl, dev, lens, toks, Hkv, how, frac):
    bt = ref.Batch(lens, toks, Hkv, Hkv, 9)
    n = 5 if how == "path" else max(1, int(max(lens) * frac))
    idx, count, start = lists(bt, how, n, 2)
    for cols in (None, max(lens) + 3, max(1, max(lens) // 2)):
        acc = None if cols is None else np.random.default_rng(1).random((bt.B, cols)).astype(np.float32)
        k, v = up(bt.k, dev), up(bt.v, dev)
        a = None if acc is None else up(acc, dev)
        new = ckl.cache_compact(k, v, **table(bt, dev), keep_idx=up(idx, dev), keep_count=up(count, dev),
                                dst_start=up(start, dev) if how == "path" else None, acc=a)
        finish(ckl)
        wk, wv, wa = want_compact(bt, idx, count, start, acc)
        assert np.array_equal(k.cpu().numpy().reshape(wk.shape), wk, equal_nan=True)
        assert np.array_equal(v.cpu().numpy().reshape(wv.shape), wv, equal_nan=True)
        assert np.array_equal(new.cpu().numpy(), start + count)
        if acc is not None:
            assert np.array_equal(a.cpu().numpy(), wa)


def test_cache_compact_refuses_lists(ckl, dev):
    """A list that falls, repeats, starts before its place or leaves the sequence moves nothing
    of its sequence; the others are moved."""
    import torch
    bt = ref.Batch([50] * 8, [4] * 8, 2, 2, 9)
    good = np.array([3, 9, 10, 30], np.int32)
    idx = np.stack([good, [3, 9, 8, 30], [3, 9, 9, 30], [-1, 9, 10, 30], [3, 9, 10, 50], good, good, good])
    count = np.array([4, 4, 4, 4, 4, 4, 0, 99], np.int32)
    start = np.array([0, 0, 0, 0, 0, 4, 51, 2], np.int32)
    k, v = up(bt.k, dev), up(bt.v, dev)
    acc = up(np.ones((8, 50), np.float32), dev)
    new = ckl.cache_compact(k, v, **table(bt, dev), keep_idx=up(idx.astype(np.int32), dev), keep_count=up(count, dev),
                            dst_start=up(start, dev), acc=acc)
    torch.cuda.synchronize()
    with pytest.raises(ckl.CklError) as e:
        ckl.check_device_error()
    assert e.value.status == 1
    ckl.check_device_error()
    moved = [0, 7]
    assert new.cpu().tolist() == [4] + [50] * 6 + [6]
    wk = bt.k.copy().reshape(-1, 2, 128)
    for b in moved:
        s = bt.slots(b)
        wk[s[np.arange(4) + start[b]]] = bt.k.reshape(-1, 2, 128)[s[good]]
    assert np.array_equal(k.cpu().numpy().reshape(wk.shape), wk, equal_nan=True)
    a = acc.cpu().numpy()
    assert np.all(a[1:7] == 1) and np.all(a[0, :4] == 1) and np.all(a[0, 4:] == 0) and np.all(a[7, 6:] == 0)


# ------------------------------------------------------------------ together
def trimmed(bt, new_len):
    """The page table after the lengths shrank (the pages behind them are free)."""
    np_ = [(int(l) + 15) // 16 for l in new_len]
    indptr = np.concatenate([[0], np.cumsum(np_)]).astype(np.int32)
    ids = np.concatenate([bt.indices[bt.indptr[b]:bt.indptr[b] + n] for b, n in enumerate(np_)])
    last = np.array([int(l) - (n - 1) * 16 for l, n in zip(new_len, np_)], np.int32)
    return indptr, ids.astype(np.int32), last


def test_draft_verify_and_evict_together(ckl, dev):
    """Drafts are appended, verified against the cache and the accepted path kept; the cache is
    then trimmed by the weights of a decode step and decoded from again. All on one stream, the
    host reads only the lengths; every stage is checked against the 64-bit restatement on the
    bytes the stage before it left."""
    import torch
    Hq, Hkv = 8, 2
    bt = ref.Batch([200, 61, 333], [12, 20, 7], Hq, Hkv, 77)
    parents, mask, pos = bt.random_tree(5)
    r = np.random.default_rng(6)
    q, k, v = (up(r.standard_normal((bt.N, h, 128)).astype(np.float16), dev) for h in (Hq, Hkv, Hkv))
    kc, vc, t, qi = up(bt.k, dev), up(bt.v, dev), table(bt, dev), up(bt.q_indptr, dev)
    m, ps = ckl.tree_mask(up(parents, dev), qi, t["kv_indptr"], t["kv_last_page_len"], 20)
    ap = ckl.make_append_params(q, k, v, kc, vc, **t, q_indptr=qi, positions=ps)
    qr = ckl.rope_append(ap, ckl.rope_plan(128))
    tp = ckl.make_tree_params(qr, kc, vc, **t, max_len=333, q_indptr=qi, max_q=20, tree_mask=m, positions=ps)
    out, lse = ckl.tree_attention(tp)
    finish(ckl)
    f, scale = ref.rope_angles(128)
    y, tol = ref.rotate(q.cpu().numpy(), pos, 128, False, f, scale)
    assert np.all(np.abs(qr.float().cpu().numpy() - y) <= tol)
    bt.q, bt.k, bt.v = qr.cpu().numpy(), kc.cpu().numpy(), vc.cpu().numpy()
    want, wl, otol, ltol = ref.attention(bt, mask=mask, positions=pos)
    assert np.all(np.abs(out.float().cpu().numpy() - want) <= otol)
    # accept the path to each sequence's deepest token
    paths = []
    for b in range(3):
        q0, T, c = bt.q_indptr[b], bt.toks[b], bt.lens[b] - bt.toks[b]
        i = int(np.argmax(pos[q0:q0 + T]))
        path = []
        while i >= 0:
            path.append(c + i)
            i = int(parents[q0 + i])
        paths.append(path[::-1])
    n = max(map(len, paths))
    idx = np.array([p + [0] * (n - len(p)) for p in paths], np.int32)
    cnt, start = np.array([len(p) for p in paths], np.int32), np.array(bt.lens, np.int32) - np.array(bt.toks, np.int32)
    new = ckl.cache_compact(kc, vc, **t, keep_idx=up(idx, dev), keep_count=up(cnt, dev), dst_start=up(start, dev))
    wk, wv, _ = want_compact(bt, idx, cnt, start, None)
    indptr, ids, last = trimmed(bt, new.cpu().numpy())
    finish(ckl)
    assert np.array_equal(kc.cpu().numpy().reshape(wk.shape), wk, equal_nan=True)
    # the accepted tokens' cache: weights of one more decode step, then the cache is halved
    b2 = ref.Batch([int(x) for x in new.cpu()], [1] * 3, Hq, Hkv, 78)
    b2.indptr, b2.indices, b2.last, b2.num_pages = indptr, ids, last, bt.num_pages
    b2.k, b2.v = kc.cpu().numpy(), vc.cpu().numpy()
    t2 = table(b2, dev)
    # pages past the new lengths hold the drafts' leftovers and NaN: neither may show
    dp = ckl.make_tree_params(up(b2.q, dev), kc, vc, **t2, max_len=max(b2.lens))
    o2, l2 = ckl.tree_attention(dp)
    acc = ckl.cache_weights(dp, l2, torch.zeros((3, 400), device=dev))
    ki, kn = ckl.cache_select(acc, t2["kv_indptr"], t2["kv_last_page_len"], 60, sink=4, recent=16)
    finish(ckl)
    want, wl, otol, ltol = ref.attention(b2)
    assert np.all(np.abs(o2.float().cpu().numpy() - want) <= otol)
    wacc, atol = ref.weights(b2, np.zeros((3, 400), np.float32), l2.cpu().numpy(), 1.0)
    a = acc.cpu().numpy()
    assert np.all(np.abs(a - wacc) <= atol + 1e-30)
    wi, wc = ref.select(a, b2.lens, 60, 4, 16)
    assert np.array_equal(ki.cpu().numpy(), wi) and np.array_equal(kn.cpu().numpy(), wc)
    new = ckl.cache_compact(kc, vc, **t2, keep_idx=ki, keep_count=kn, acc=acc)
    wk, wv, wa = want_compact(b2, wi, wc, np.zeros(3, np.int32), a)
    indptr, ids, last = trimmed(b2, new.cpu().numpy())
    finish(ckl)
    assert np.array_equal(vc.cpu().numpy().reshape(wv.shape), wv, equal_nan=True)
    assert np.array_equal(acc.cpu().numpy(), wa)
    b3 = ref.Batch([int(x) for x in new.cpu()], [1] * 3, Hq, Hkv, 79)
    b3.indptr, b3.indices, b3.last, b3.num_pages = indptr, ids, last, bt.num_pages
    b3.k, b3.v = kc.cpu().numpy(), vc.cpu().numpy()
    o3, _ = ckl.decode_attention(up(b3.q, dev), torch.nan_to_num(kc), torch.nan_to_num(vc), **table(b3, dev))
    finish(ckl)
    want, _, otol, _ = ref.attention(b3)
    assert np.all(np.abs(o3.float().cpu().numpy() - want) <= otol)


def test_python_refusals(ckl, dev):
    import torch
    bt = ref.Batch([20, 30], [2, 3], 4, 2, 1)
    t = table(bt, dev)
    q, k, v = up(bt.q, dev), up(bt.k, dev), up(bt.v, dev)
    mk = lambda **kw: ckl.make_tree_params(**{**dict(q=q, k_cache=k, v_cache=v, max_len=30, max_q=3,
                                                     q_indptr=up(bt.q_indptr, dev)), **t, **kw})
    for kw in (dict(q=q.float()), dict(q=q[:, :3]), dict(k_cache=k[:, :8]), dict(q_indptr=up(bt.q_indptr[:2], dev)),
               dict(positions=t["kv_indptr"][:2]), dict(tree_mask=t["kv_indptr"]), dict(slopes=torch.ones(3, device=dev)),
               dict(kv_last_page_len=t["kv_last_page_len"][:1]), dict(kv_indices=bt.indices)):
        with pytest.raises(ckl.CklError):
            mk(**kw)
    p = mk()
    for kw in (dict(out=torch.empty(3, device=dev)), dict(lse=torch.empty((5, 4), device=dev, dtype=torch.float64))):
        with pytest.raises(ckl.CklError):
            ckl.tree_attention(p, **kw)
    qkv = torch.zeros((5, 8 * 128), dtype=torch.float16, device=dev)
    with pytest.raises(ckl.CklError):
        ckl.make_append_params(q, q[:, :2].transpose(0, 1), q[:, :2], k, v, **t)
    with pytest.raises(ckl.CklError):                          # the output in place of the input
        ckl.rope_append(ckl.make_append_params(q, q[:, :2], q[:, 2:], k, v, **t, q_out=q,
                                               q_indptr=up(bt.q_indptr, dev)), ckl.rope_plan(128))
    with pytest.raises(ckl.CklError):
        ckl.cache_weights(p, torch.empty((5, 4), device=dev), torch.empty((1, 30), device=dev))


def test_python_refuses_what_is_no_tensor(ckl, dev):
    import torch
    bt = ref.Batch([20, 30], [2, 3], 4, 2, 1)
    t = table(bt, dev)
    q, k, v = up(bt.q, dev), up(bt.k, dev), up(bt.v, dev)
    for bad in (None, bt.k, 3):
        with pytest.raises(ckl.CklError):
            ckl.make_tree_params(q, bad, v, **t, max_len=30)
        with pytest.raises(ckl.CklError):
            ckl.make_append_params(q, bad, q[:, 2:], k, v, **t)
        with pytest.raises(ckl.CklError):
            ckl.make_append_params(q, q[:, :2], q[:, 2:], k, bad, **t)
        with pytest.raises(ckl.CklError):
            ckl.cache_select(bad, t["kv_indptr"], t["kv_last_page_len"], 4)
    idx = torch.zeros((2, 4), dtype=torch.int32, device=dev)
    cnt = torch.zeros(2, dtype=torch.int32, device=dev)
    with pytest.raises(ckl.CklError):                          # the lengths over the counts
        ckl.cache_compact(k, v, **t, keep_idx=idx, keep_count=cnt, new_len=cnt)


def test_tree_and_weights_calls_longer_than_the_wait_limit(ckl, dev):
    """The limit on a wait bounds a wait, not a call: 6144 units of 64 key blocks (about 42 a CTA,
    over 2 ms) with a limit of 1 ms give what they give without one."""
    import torch
    T, G, Hkv, B, L = 6144, 1, 32, 8, 8192
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.randn((B * T, Hkv * G, 128), device=dev, dtype=torch.float16, generator=g)
    k = torch.randn((64, 16, Hkv, 128), device=dev, dtype=torch.float16, generator=g)
    v = torch.randn((64, 16, Hkv, 128), device=dev, dtype=torch.float16, generator=g)
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device=dev)
    pages = L // 16
    indptr = i32([b * pages for b in range(B + 1)])
    indices = torch.randint(0, 64, (B * pages,), device=dev, dtype=torch.int32, generator=g)
    p = ckl.make_tree_params(q, k, v, indptr, indices, i32([16] * B), max_len=L, max_q=T,
                             q_indptr=i32([b * T for b in range(B + 1)]))
    out, lse = ckl.tree_attention(p)
    acc = ckl.cache_weights(p, lse, torch.zeros((B, L), device=dev))
    finish(ckl)
    ckl.lib().ckl_set_spin_timeout_ns(1000000)
    try:
        o2, l2 = ckl.tree_attention(p)
        a2 = ckl.cache_weights(p, lse, torch.zeros((B, L), device=dev))
        finish(ckl)
    finally:
        ckl.lib().ckl_set_spin_timeout_ns(1000000000)
    assert torch.equal(out, o2) and torch.equal(lse, l2) and torch.equal(acc, a2)


@pytest.mark.parametrize("toks,Hq", [(16, 16), (32, 16), (5, 16)])
def test_tree_short_sequences_many_times(ckl, dev, toks, Hq):
    """Two to four key blocks a sequence: the softmax ends the last block while the product of the
    one before it may still wait for its V. The output must hold both, in every call."""
    bt = ref.Batch([129 + 17 * i for i in range(20)], [toks] * 20, Hq, 2, 43)
    o, l = check_tree(ckl, dev, bt, force=1)
    p = run_tree(ckl, dev, bt, force=1)
    for _ in range(100):
        out, lse = ckl.tree_attention(p)
        assert np.array_equal(out.float().cpu().numpy(), o) and np.array_equal(lse.cpu().numpy(), l)
    finish(ckl)
