"""GPU tests of the cache operators at the edges of what their header allows."""
import numpy as np
import pytest

import cache_ref as ref
from test_cache_ops_gpu import check_tree, finish, run_tree, table, up

pytestmark = pytest.mark.gpu


def score_error(bt, b, s, big, softcap=0.0, **_):
    """Bound of a score's error in nats: 128 fp32 additions of exact products and a handful of
    roundings, and of a cap 2^-21 of the score up to 0.45 of the cap, 2^-21 of the cap beyond (where
    the score is above 0.42 of it): at most 2^-21 of 2.4 of the greatest score, or of the cap."""
    fin = s[np.isfinite(s)]
    top = float(np.abs(fin).max()) if fin.size else 0.0
    return 2.0 ** -24 * (128 * min(big, 1e30) + 8 * top) + 2.0 ** -21 * min(softcap, 2.4 * top)


def attend(bt, **opt):
    """out, lse and their bounds, as in cache_ref.attention but for the error of a cap (score_error)
    and for weights far below the greatest: P is kept 2^7 above fp16's own range, so that at
    most 2^-32 of the greatest weight is lost of each."""
    out = np.zeros((bt.T_total, bt.Hq, 128))
    lse = np.full((bt.T_total, bt.Hq), -np.inf)
    tol, ltol = np.zeros_like(out), np.zeros_like(lse)
    for b in range(bt.B):
        L, T, q0 = bt.lens[b], bt.toks[b], bt.q_indptr[b]
        if T == 0 or L == 0:
            continue
        s, big = ref.scores(bt, b, **opt)
        ds = score_error(bt, b, s, big, **opt)
        v = bt.v.reshape(-1, bt.Hkv, 128)[bt.slots(b)].astype(np.float64)
        for h in range(bt.Hq):
            vh = np.where(np.isfinite(s[h]).any(0)[:, None], v[:, h // bt.G], 0.0)
            for i in range(T):
                m = s[h, i].max()
                p = np.exp(s[h, i] - m)
                z = p.sum()
                o, mag = p @ vh / z, p @ np.abs(vh) / z
                out[q0 + i, h], lse[q0 + i, h] = o, m + np.log(z)
                tol[q0 + i, h] = (mag * (2.0 ** -11 + 2 * ds + 2.0 ** -18) + np.abs(o) * 2.0 ** -11
                                  + 2.0 ** -32 * L * np.abs(vh).max() / z + 2.0 ** -25)
                ltol[q0 + i, h] = 2 * ds + 2.0 ** -20 * (1 + abs(lse[q0 + i, h]))
    return out, lse, tol, ltol


def check(ckl, bt, p, **opt):
    out, lse = ckl.tree_attention(p)
    finish(ckl)
    want, wl, tol, ltol = attend(bt, **opt)
    o, l, n = out.float().cpu().numpy(), lse.cpu().numpy(), bt.T_total
    assert np.isfinite(o[:n]).all() and np.isfinite(l[:n]).all()
    err, lerr = np.abs(o[:n] - want) - tol, np.abs(l[:n] - wl) - ltol
    assert np.all(err <= 0) and np.all(lerr <= 0), f"out {err.max():.3e}, lse {lerr.max():.3e} beyond their bounds"


def slopes_of(Hq):
    return np.float32(2.0) ** (-8.0 * (np.arange(Hq, dtype=np.float32) + 1) / Hq)


# rows of a kv head: 12 (registers), 28 and 120 (one tile), 160 (two)
CAPPED = [([300, 290], [3, 2], 8, 2), ([400, 333], [7, 5], 8, 2), ([400, 333], [15, 9], 8, 1), ([600, 280], [40, 33], 4, 1)]


# ------------------------------------------------------------------ caps
@pytest.mark.parametrize("lens,toks,Hq,Hkv", CAPPED)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cap", [1e-12, 0.5, 30.0, 1e4, 1e8, 1e30])
def test_caps_of_every_size(ckl, dev, lens, toks, Hq, Hkv, bias, cap):
    """From a cap that levels every score to one that leaves them as they are; at 30 every key part
    that all rows see whole is below 0.45 of the cap."""
    bt = ref.Batch(lens, toks, Hq, Hkv, 51)
    _, mask, pos = bt.random_tree(4)
    opt = dict(mask=mask, positions=pos, softcap=cap)
    if bias:
        opt["slopes"] = slopes_of(Hq)
    check(ckl, bt, run_tree(ckl, dev, bt, force=2, **opt), **opt)


@pytest.mark.parametrize("lens,toks,Hq,Hkv", CAPPED)
def test_cap_below_some_scores(ckl, dev, lens, toks, Hq, Hkv):
    """One head in four far beyond the cap, the others far below it, in the same warps."""
    bt = ref.Batch(lens, toks, Hq, Hkv, 52)
    bt.q[:, ::4] *= 20
    opt = dict(softcap=30.0)
    check(ckl, bt, run_tree(ckl, dev, bt, force=2, **opt), **opt)


@pytest.mark.parametrize("lens,toks,Hq,Hkv", CAPPED)
@pytest.mark.parametrize("cap", [1e-30, 1e-12, 1.0, 1e30])
def test_caps_of_scores_of_zero(ckl, dev, lens, toks, Hq, Hkv, cap):
    bt = ref.Batch(lens, toks, Hq, Hkv, 53, qscale=0.0)
    check(ckl, bt, run_tree(ckl, dev, bt, force=1, softcap=cap), softcap=cap)


@pytest.mark.parametrize("lens,toks,Hq,Hkv", CAPPED)
@pytest.mark.parametrize("cap", [1e-12, 0.5, 30.0, 1e4, 1e8, 1e30])
def test_cache_weights_caps(ckl, dev, lens, toks, Hq, Hkv, cap):
    import torch
    bt = ref.Batch(lens, toks, Hq, Hkv, 54)
    _, mask, pos = bt.random_tree(4)
    opt = dict(mask=mask, positions=pos, softcap=cap)
    _, lse, _, _ = attend(bt, **opt)
    lse = lse.astype(np.float32)
    acc = ckl.cache_weights(run_tree(ckl, dev, bt, **opt), up(lse, dev), torch.zeros((2, max(lens)), device=dev))
    finish(ckl)
    for b in range(2):
        s, big = ref.scores(bt, b, **opt)
        l = lse[bt.q_indptr[b]:bt.q_indptr[b + 1]].astype(np.float64).T[:, :, None]
        want = np.exp(s - l).sum((0, 1))
        ds = score_error(bt, b, s, big, **opt)
        # 2^-24 of lse from its own rounding, 2^-23 of each of the score and lse in the exponent
        ds += 2.0 ** -22 * float(np.abs(lse).max())
        tol = want * (2 * ds + 2.0 ** -20 + Hq * toks[b] * 2.0 ** -24) + 1e-30
        assert np.all(np.abs(acc.cpu().numpy()[b, :lens[b]] - want) <= tol)


# ------------------------------------------------------------------ small weights
@pytest.mark.parametrize("toks,Hq", [(1, 4), (6, 4), (40, 4)])
def test_many_small_weights(ckl, dev, toks, Hq):
    """Four keys far above 60,000 others, each of which weighs 2^-25.7 of the greatest: together they
    are all of the result."""
    L = 60000
    bt = ref.Batch([L], [toks], Hq, 1, 61)
    s = bt.slots(0)
    bt.q[:] = 0
    bt.q[:, :, 0] = 14.2
    k, v = bt.k.reshape(-1, 128), bt.v.reshape(-1, 128)
    k[s], v[s] = 0, 512
    k[s, 0] = -14.2
    # one for each of the four warps that take pages in turn
    k[s[[0, 16, 32, 48]], 0] = 0
    v[s[[0, 16, 32, 48]]] = 0
    check(ckl, bt, run_tree(ckl, dev, bt, force=1))


# ------------------------------------------------------------------ neighbours
@pytest.mark.parametrize("softcap", [0.0, 30.0])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("toks,Hq", [([5, 9], 8), ([37, 20], 8), ([3, 30], 8)])
def test_neighbours_leave_the_same_bits(ckl, dev, toks, Hq, softcap, bias):
    """What the other sequences of a batch hold -- their q lie in the same tiles, their keys where a
    last block's are missing -- changes no bit of a sequence's results."""
    import torch
    lens = [525, 700]                                        # 33 pages: the last block of 128 keys has one
    opt = dict(softcap=softcap)
    if bias:
        opt["slopes"] = slopes_of(Hq)
    got = []
    for scale in (1.0, 60.0):
        bt = ref.Batch(lens, toks, Hq, 2, 71)
        bt.q[bt.q_indptr[1]:] *= scale
        bt.k.reshape(-1, 2, 128)[bt.slots(1)] *= scale
        p = run_tree(ckl, dev, bt, force=1, **opt)
        out, lse = ckl.tree_attention(p)
        acc = ckl.cache_weights(p, lse, torch.zeros((2, 700), device=dev))
        finish(ckl)
        got.append([x[:toks[0]].cpu() for x in (out, lse)] + [acc[0].cpu()])
    for x, y in zip(*got):
        assert torch.equal(x, y)


# ------------------------------------------------------------------ rows of weights
def test_cache_weights_leaves_the_rest(ckl, dev):
    """Places from the length on are left for every decay, 0 too."""
    import torch
    lens, toks = [40, 300, 1], [3, 5, 1]
    bt = ref.Batch(lens, toks, 8, 2, 72)
    p = run_tree(ckl, dev, bt)
    _, lse = ckl.tree_attention(p)
    for decay in (0.0, 0.5, 1.0):
        acc = torch.rand((3, 333), device=dev)
        was = acc.clone()
        ckl.cache_weights(p, lse, acc, decay=decay)
        finish(ckl)
        for b, L in enumerate(lens):
            assert torch.equal(acc[b, L:], was[b, L:]) and not torch.equal(acc[b, :L], was[b, :L])


def test_weights_that_are_columns_of_something_wider(ckl, dev):
    """acc as columns of a wider tensor, sequences longer than its rows: what a contiguous acc of
    those rows gives, and the columns beside it are neither read nor written."""
    import torch
    lens, toks = [300, 70, 390], [3, 5, 1]
    bt = ref.Batch(lens, toks, 8, 2, 72)
    p = run_tree(ckl, dev, bt)
    _, lse = ckl.tree_attention(p)
    t = table(bt, dev)
    big = torch.full((3, 500), 1e9, device=dev)
    view = big[:, 100:250]
    view.copy_(torch.rand((3, 150), device=dev))

    def both(call):
        plain = view.clone()
        a, b = call(view), call(plain)
        finish(ckl)
        assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(view, plain)
        assert torch.all(big[:, :100] == 1e9) and torch.all(big[:, 250:] == 1e9)

    for decay in (1.0, 0.5, 0.0):
        both(lambda acc: [ckl.cache_weights(p, lse, acc, decay=decay)])
    idx = up(np.array([[0, 5, 149, 160, 299], [1, 2, 3, 4, 69], [7, 150, 200, 251, 389]], np.int32), dev)
    cnt = up(np.full(3, 5, np.int32), dev)

    def compact(acc):
        k, v = up(bt.k, dev), up(bt.v, dev)
        return [ckl.cache_compact(k, v, **t, keep_idx=idx, keep_count=cnt, acc=acc), acc]

    both(lambda acc: ckl.cache_select(acc, t["kv_indptr"], t["kv_last_page_len"], 60, sink=2, recent=20))
    both(compact)


def test_compact_refuses_lengths_over_the_page_table(ckl, dev):
    import torch
    bt = ref.Batch([90, 70], [3, 5], 2, 2, 73)
    t = table(bt, dev)
    k, v = up(bt.k, dev), up(bt.v, dev)
    n = t["kv_indices"].numel()
    idx, cnt = up(np.zeros((2, 1), np.int32), dev), up(np.ones(2, np.int32), dev)
    for at in (0, n // 2, n - 2):
        with pytest.raises(ckl.CklError) as e:
            ckl.cache_compact(k, v, **t, keep_idx=idx, keep_count=cnt, new_len=t["kv_indices"][at:at + 2])
        assert e.value.status == 1
    assert torch.equal(t["kv_indices"], up(bt.indices, dev))


# ------------------------------------------------------------------ limits on waits
def long_context(ckl, dev, T, G, L, B=1):
    """B sequences of L tokens over 64 pages that repeat, one kv head."""
    import torch
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.randn((B * T, G, 128), device=dev, dtype=torch.float16, generator=g)
    k, v = (torch.randn((64, 16, 1, 128), device=dev, dtype=torch.float16, generator=g) for _ in range(2))
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32, device=dev)
    ids = torch.randint(0, 64, (B * L // 16,), device=dev, dtype=torch.int32, generator=g)
    return ckl.make_tree_params(q, k, v, i32([b * L // 16 for b in range(B + 1)]), ids, i32([16] * B), max_len=L, max_q=T,
                                q_indptr=i32([b * T for b in range(B + 1)]), force_chunks=1)


@pytest.fixture
def wait_limit(ckl):
    yield ckl.lib().ckl_set_spin_timeout_ns
    ckl.lib().ckl_set_spin_timeout_ns(1000000000)


@pytest.mark.parametrize("T,G", [(1, 4), (6, 4), (64, 4)])
def test_one_run_of_keys_longer_than_the_wait_limit(ckl, dev, wait_limit, T, G):
    """The limit is one wait's: a CTA that walks 400,000 keys (several ms) under a limit of 1 ms."""
    import torch
    p = long_context(ckl, dev, T, G, 400000)
    out, lse = ckl.tree_attention(p)
    finish(ckl)
    wait_limit(1000000)
    o2, l2 = ckl.tree_attention(p)
    finish(ckl)
    assert torch.equal(out, o2) and torch.equal(lse, l2)


@pytest.mark.parametrize("T,G", [(1, 4), (6, 4), (6, 5), (64, 4), (70, 5)])
def test_waits_that_may_give_up(ckl, dev, wait_limit, T, G):
    """A limit below what some waits take: the calls return, one that gave up is recorded as
    CKL_TIMEOUT, and the next calls give what they gave before. (A wait that ends within the
    hardware's own suspension never looks at the limit, so a call may also be right.)"""
    import torch
    p = long_context(ckl, dev, T, G, 4000, B=3)
    out, lse = ckl.tree_attention(p)
    acc = ckl.cache_weights(p, lse, torch.zeros((3, 4000), device=dev))
    finish(ckl)

    def attend():
        o, l = ckl.tree_attention(p)
        return torch.equal(o, out) and torch.equal(l, lse)

    def weigh():
        return torch.equal(ckl.cache_weights(p, lse, torch.zeros((3, 4000), device=dev)), acc)

    for call in [attend, weigh] * 5:
        wait_limit(1)
        right = call()
        torch.cuda.synchronize()
        if not right:
            with pytest.raises(ckl.CklError) as e:
                ckl.check_device_error()
            assert e.value.status == 5                         # CKL_TIMEOUT
        else:
            try:
                ckl.check_device_error()
            except ckl.CklError as e:
                assert e.status == 5
        wait_limit(1000000000)
        assert attend() and weigh()
        finish(ckl)


# ------------------------------------------------------------------ nothing there
def test_a_batch_without_a_page(ckl, dev):
    """Every sequence empty, so that there is no page id: tokens see nothing and have no place,
    lists of nothing move nothing."""
    import torch
    bt = ref.Batch([0, 0, 0], [1, 2, 0], 8, 2, 81)
    t = table(bt, dev)
    assert t["kv_indices"].numel() == 0
    k, v = up(bt.k, dev), up(bt.v, dev)
    q = up(bt.q, dev)
    p = ckl.make_append_params(q, q[:, :2], q[:, 2:4], k, v, **t, q_indptr=up(bt.q_indptr, dev))
    assert torch.equal(ckl.rope_append(p), q)
    tp = ckl.make_tree_params(q, k, v, **t, max_len=0, max_q=2, q_indptr=up(bt.q_indptr, dev))
    out, lse = ckl.tree_attention(tp)
    acc = ckl.cache_weights(tp, lse, torch.ones((3, 4), device=dev), decay=0.5)
    idx, cnt = ckl.cache_select(acc, t["kv_indptr"], t["kv_last_page_len"], 5)
    new = ckl.cache_compact(k, v, **t, keep_idx=idx, keep_count=cnt, acc=acc)
    finish(ckl)
    assert torch.all(out == 0) and torch.all(torch.isneginf(lse)) and torch.all(acc == 1)
    assert torch.all(idx == -1) and torch.all(cnt == 0) and torch.all(new == 0)
    assert np.array_equal(k.cpu().numpy(), bt.k, equal_nan=True)


# ------------------------------------------------------------------ many sequences, graphs
@pytest.mark.parametrize("toks,Hq,opt", [(1, 4, dict()), (3, 4, dict(window=21)), (9, 4, dict(softcap=20.0)),
                                         (33, 8, dict(window=40, bias=True))], ids=str)
def test_many_sequences(ckl, dev, toks, Hq, opt):
    """More sequences than a warp has lanes, a third of them without tokens or without keys."""
    r = np.random.default_rng(91)
    lens = [int(r.choice([0, 1, 40, 300])) for _ in range(75)]
    bt = ref.Batch(lens, [0 if b % 3 == 1 else min(toks, L) for b, L in enumerate(lens)], Hq, 2, 92, extra_rows=2)
    _, mask, pos = bt.random_tree(3)
    opt = dict(opt, mask=mask, positions=pos)
    if opt.pop("bias", False):
        opt["slopes"] = slopes_of(Hq)
    check_tree(ckl, dev, bt, force=1, **opt)
    p = run_tree(ckl, dev, bt, **opt)
    import torch
    _, lse = ckl.tree_attention(p)
    lse[bt.T_total:] = 0
    acc = np.random.default_rng(1).random((75, 300)).astype(np.float32)
    got = ckl.cache_weights(p, lse, up(acc, dev), decay=0.5)
    finish(ckl)
    want, tol = ref.weights(bt, acc, lse.cpu().numpy(), 0.5, **opt)
    assert np.all(np.abs(got.cpu().numpy() - want) <= tol + 2.0 ** -23 * np.abs(want))


def test_a_step_captured_on_a_stream_and_replayed(ckl, dev):
    """Append, masks, attention, weights, selection and compaction in one graph on a stream of its
    own; each replay does to fresh caches what the calls do one by one."""
    import torch
    bt = ref.Batch([200, 61, 333], [12, 20, 7], 8, 2, 77)
    parents, _, _ = bt.random_tree(5)
    r = np.random.default_rng(6)
    q, k, v = (up(r.standard_normal((bt.N, h, 128)).astype(np.float16), dev) for h in (8, 2, 2))
    t, qi, par = table(bt, dev), up(bt.q_indptr, dev), up(parents, dev)
    plan = ckl.rope_plan(128)
    clean = [up(np.nan_to_num(bt.k), dev), up(np.nan_to_num(bt.v), dev)]
    kc, vc = (x.clone() for x in clean)
    acc = torch.zeros((3, 400), device=dev)

    def step(stream=None):
        m, ps = ckl.tree_mask(par, qi, t["kv_indptr"], t["kv_last_page_len"], 20, stream=stream)
        qr = ckl.rope_append(ckl.make_append_params(q, k, v, kc, vc, **t, q_indptr=qi, positions=ps), plan, stream=stream)
        tp = ckl.make_tree_params(qr, kc, vc, **t, max_len=333, q_indptr=qi, max_q=20, tree_mask=m, positions=ps)
        out, lse = ckl.tree_attention(tp, stream=stream)
        ckl.cache_weights(tp, lse, acc, decay=0.5, stream=stream)
        ki, kn = ckl.cache_select(acc, t["kv_indptr"], t["kv_last_page_len"], 60, sink=4, recent=16, stream=stream)
        new = ckl.cache_compact(kc, vc, **t, keep_idx=ki, keep_count=kn, acc=acc, stream=stream)
        return m, qr, out, lse, ki, kn, new

    def fresh():
        kc.copy_(clean[0])
        vc.copy_(clean[1])
        acc.zero_()

    fresh()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        got = step(side)
    for scale in (1.0, -0.5):
        q.mul_(scale)
        fresh()
        want = [x.clone() for x in step()] + [kc.clone(), vc.clone(), acc.clone()]
        fresh()
        g.replay()
        finish(ckl)
        for x, y in zip(list(got) + [kc, vc, acc], want):
            assert torch.equal(x, y)


def test_a_workspace_that_is_no_tensor_is_refused(ckl, dev):
    import torch
    p = run_tree(ckl, dev, ref.Batch([300], [9], 8, 2, 82))
    for bad in (3, np.empty(1 << 20, np.uint8), torch.empty(1 << 20, dtype=torch.uint8)):
        with pytest.raises(ckl.CklError):
            ckl.tree_attention(p, workspace=bad)
