"""Plain 64-bit restatements of the cache operators (rotary append, draft-tree attention, cache
weights, selection, compaction) and the batches their tests run on."""
import math

import numpy as np

D, PAGE = 128, 16


class Batch:
    """Paged sequences with their new tokens: pages of the pool in random order, NaN in spare
    pages and behind every sequence."""

    def __init__(self, lens, toks, Hq, Hkv, seed, extra_rows=0, qscale=1.0):
        r = np.random.default_rng(seed)
        self.lens, self.toks, self.Hq, self.Hkv, self.G = list(lens), list(toks), Hq, Hkv, Hq // Hkv
        self.B = len(lens)
        np_ = [(l + PAGE - 1) // PAGE for l in lens]
        self.indptr = np.concatenate([[0], np.cumsum(np_)]).astype(np.int32)
        total = int(self.indptr[-1])
        self.num_pages = total + 3
        self.indices = r.permutation(self.num_pages)[:total].astype(np.int32)
        self.last = np.array([l - (n - 1) * PAGE if n else 0 for l, n in zip(lens, np_)], np.int32)
        self.q_indptr = np.concatenate([[0], np.cumsum(toks)]).astype(np.int32)
        self.T_total = int(self.q_indptr[-1])
        self.N = self.T_total + extra_rows
        self.q = (r.standard_normal((self.N, Hq, D)) * qscale).astype(np.float16)
        self.k = np.full((self.num_pages, PAGE, Hkv, D), np.nan, np.float16)
        self.v = np.full((self.num_pages, PAGE, Hkv, D), np.nan, np.float16)
        for b in range(self.B):
            s = self.slots(b)
            self.k.reshape(-1, Hkv, D)[s] = r.standard_normal((len(s), Hkv, D)).astype(np.float16)
            self.v.reshape(-1, Hkv, D)[s] = r.standard_normal((len(s), Hkv, D)).astype(np.float16)

    def slots(self, b):
        pages = self.indices[self.indptr[b]:self.indptr[b + 1]].astype(np.int64)
        return (pages[:, None] * PAGE + np.arange(PAGE)).reshape(-1)[:self.lens[b]]

    def random_tree(self, seed, words=None):
        """(parents, mask words int32 [N, W], positions) of random trees."""
        r = np.random.default_rng(seed)
        W = words or max(1, (max(self.toks) + 31) // 32)
        parents = np.full(self.N, -1, np.int32)
        mask = np.zeros((self.N, W), np.uint32)
        pos = np.zeros(self.N, np.int32)
        for b in range(self.B):
            q0 = self.q_indptr[b]
            for i in range(self.toks[b]):
                p = int(r.integers(max(-1, i - 6), i)) if i else -1
                parents[q0 + i] = p
                pos[q0 + i] = pos[q0 + p] + 1 if p >= 0 else self.lens[b] - self.toks[b]
                if p >= 0:
                    mask[q0 + i] = mask[q0 + p]
                mask[q0 + i, i // 32] |= np.uint32(1 << (i % 32))
        return parents, mask.view(np.int32), pos


def seen(bt, b, mask=None, positions=None, window=0):
    """[T, L] who sees what, and the positions of the tokens and keys of sequence b."""
    L, T, q0 = bt.lens[b], bt.toks[b], bt.q_indptr[b]
    ctx = L - T
    kpos = np.arange(L, dtype=np.int64)
    qpos = np.arange(T, dtype=np.int64) + ctx
    if positions is not None:
        qpos = positions[q0:q0 + T].astype(np.int64)
        for p in range(max(ctx, 0), L):
            kpos[p] = qpos[p - ctx]
    vis = np.ones((T, L), bool)
    for i in range(T):
        for p in range(max(ctx, 0), L):
            j = p - ctx
            if mask is None:
                vis[i, p] = j <= i
            else:
                m = mask.view(np.uint32)
                vis[i, p] = j // 32 < m.shape[1] and bool((m[q0 + i, j // 32] >> np.uint32(j % 32)) & 1)
    if window:
        vis &= (qpos[:, None] - kpos[None]) < window
    return vis, qpos, kpos


def scores(bt, b, mask=None, positions=None, slopes=None, softcap=0.0, window=0, scale=None):
    """[Hq, T, L] scores, -inf where unseen; and the largest sum |q_d k_d| * scale of a seen key."""
    L, T, q0, G = bt.lens[b], bt.toks[b], bt.q_indptr[b], bt.G
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    vis, qpos, kpos = seen(bt, b, mask, positions, window)
    q = bt.q[q0:q0 + T].astype(np.float64)
    k = bt.k.reshape(-1, bt.Hkv, D)[bt.slots(b)].astype(np.float64)
    s = np.full((bt.Hq, T, L), -np.inf)
    big = 0.0
    for h in range(bt.Hq):
        with np.errstate(invalid="ignore"):
            x = q[:, h] @ k[:, h // G].T * scale
            a = np.abs(q[:, h]) @ np.abs(k[:, h // G]).T * scale
        if softcap:
            x = softcap * np.tanh(x / softcap)
        if slopes is not None:
            x = x + float(slopes[h]) * (kpos[None] - qpos[:, None])
        s[h] = np.where(vis, x, -np.inf)
        if vis.any():
            big = max(big, float(np.max(a[vis])))
    return s, big


def attention(bt, **opt):
    """out [T_total, Hq, D], lse, and per-row tolerances of both.

    The tolerances follow the arithmetic: ds bounds a score's error (128 fp32 additions of exact
    products, 2^-24 each of the largest sum of magnitudes, and a handful more roundings of the
    score itself, of a cap's tanh -- 2^-21 of the cap -- and of a bias); a weight is then off by
    2 ds, by 2^-11 of itself when it is rounded to fp16 and by at most 2^-25 of the largest weight
    where fp16 is subnormal; the result is rounded to fp16 once (2^-11, or 2^-25 when subnormal)."""
    out = np.zeros((bt.T_total, bt.Hq, D))
    lse = np.full((bt.T_total, bt.Hq), -np.inf)
    tol = np.zeros_like(out)
    ltol = np.zeros_like(lse)
    for b in range(bt.B):
        L, T, q0, G = bt.lens[b], bt.toks[b], bt.q_indptr[b], bt.G
        if T == 0 or L == 0:
            continue
        s, big = scores(bt, b, **opt)
        fin = s[np.isfinite(s)]
        top = float(np.abs(fin).max()) if fin.size else 0.0
        ds = 2.0 ** -24 * (128 * big + 8 * top) + 2.0 ** -21 * opt.get("softcap", 0.0)
        v = bt.v.reshape(-1, bt.Hkv, D)[bt.slots(b)].astype(np.float64)
        for h in range(bt.Hq):
            for i in range(T):
                x = s[h, i]
                see = x > -np.inf
                if not see.any():
                    continue
                m = x[see].max()
                p = np.exp(x[see] - m)
                vv = v[see, h // G]
                o = (p[:, None] * vv).sum(0) / p.sum()
                mag = (p[:, None] * np.abs(vv)).sum(0) / p.sum()
                out[q0 + i, h] = o
                lse[q0 + i, h] = m + np.log(p.sum())
                tol[q0 + i, h] = (mag * (2.0 ** -11 + 2 * ds + 2.0 ** -18) + np.abs(o) * 2.0 ** -11
                                  + 2.0 ** -25 * len(p) * np.abs(vv).max() / p.sum() + 2.0 ** -25)
                ltol[q0 + i, h] = 2 * ds + 2.0 ** -20 * (1 + abs(lse[q0 + i, h]))
    return out, lse, tol, ltol


def weights(bt, acc, lse, decay, **opt):
    """acc after a call, and its tolerance."""
    ref, tol = acc.astype(np.float64).copy(), np.zeros(acc.shape)
    for b in range(bt.B):
        L, q0, T = bt.lens[b], bt.q_indptr[b], bt.toks[b]
        n = min(L, acc.shape[1])
        ref[b, :n] *= decay
        tol[b, :n] = np.abs(ref[b, :n]) * 2.0 ** -23
        if T == 0 or L == 0:
            continue
        s, big = scores(bt, b, **opt)
        fin = s[np.isfinite(s)]
        top = float(np.abs(fin).max()) if fin.size else 0.0
        ds = 2.0 ** -24 * (128 * big + 16 * top) + 2.0 ** -21 * opt.get("softcap", 0.0)
        l = lse[q0:q0 + T].astype(np.float64).T[:, :, None]
        with np.errstate(invalid="ignore"):
            add = np.where(np.isneginf(l), 0.0, np.exp(s - l)).sum((0, 1))
        ref[b, :n] += add[:n]
        tol[b, :n] += add[:n] * (2 * ds + 2.0 ** -20 + bt.Hq * T * 2.0 ** -24) + 1e-30
    return ref, tol


def select(acc, lens, keep, sink, recent):
    idx = np.full((len(lens), keep), -1, np.int32)
    count = np.zeros(len(lens), np.int32)
    for b, L in enumerate(lens):
        if L <= keep:
            got = list(range(L))
        else:
            val = [acc[b, p] if p < acc.shape[1] and not np.isnan(acc[b, p]) else None for p in range(L)]
            rest = sorted(range(sink, L - recent),
                          key=lambda p: ((0, -val[p]) if val[p] is not None else (1, 0.0), p))
            got = sorted(list(range(sink)) + list(range(L - recent, L)) + rest[:keep - sink - recent])
        idx[b, :len(got)] = got
        count[b] = len(got)
    return idx, count


def rope_angles(rot, base=10000.0, scaling="none", factor=1.0, original_len=4096, fast=32.0, slow=1.0):
    """(angle per position of each pair, scale)."""
    if scaling == "ntk" and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)], np.longdouble)
    scale = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "by_parts":
        at = lambda t: rot * math.log(original_len / (t * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - low) / max(high - low, 0.001), 0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1.0
    return f, scale


def rotate(x, pos, rot, interleaved, f, scale):
    """x [N, H, D] turned at positions pos, in 64 bits, and the error bound of an fp32 rotation
    rounded once to fp16: 2^-11 of the result (2^-25 when subnormal), and 2^-20 of the pair's
    magnitudes for the angle (2^-24 of half a turn from its fp32 conversion), sine and products."""
    x = x.astype(np.float64)
    y, mag = x.copy(), np.zeros_like(x)
    turn = np.asarray(pos, np.longdouble)[:, None] * (f / (2 * np.longdouble(np.pi)))
    ang = ((turn - np.floor(turn)) * 2 * np.longdouble(np.pi)).astype(np.float64)
    c, s = np.cos(ang)[:, None] * scale, np.sin(ang)[:, None] * scale
    i = np.arange(rot // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    a, b = x[:, :, ia], x[:, :, ib]
    y[:, :, ia], y[:, :, ib] = a * c - b * s, a * s + b * c
    mag[:, :, ia] = mag[:, :, ib] = (np.abs(a) + np.abs(b)) * scale
    return y, 2.0 ** -11 * np.abs(y) + 2.0 ** -20 * mag + 2.0 ** -25
