"""Measured cases of the operators that write, read, weigh and trim the paged K/V cache.

rope     rotary positions on q and k, and the append of k and v to the paged cache
tree     attention of drafted tokens (a tree, a chain, or one token) over the cache, with capped
         scores, a distance bias and a sliding window as options
weights  the attention weight every cached token received, accumulated
select   the tokens to keep of each sequence, by accumulated weight
compact  the kept rows moved to the front, in place

Where `own` is false, run() computes them with elementary torch operations in 32 bits.
"""
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
D = 128          # head size
PAGE = 16        # tokens per page


def _ckl():
    p = os.path.join(ROOT, "cuda-kernel-lab_b200")
    if p not in sys.path:
        sys.path.insert(0, p)
    import ckl
    return ckl


# ---------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a small serving batch: latency
        dict(name="rope_decode_8", op="rope", B=8, T=1, L=2048, Hq=32, Hkv=8, rot=128,
             interleaved=False, scaling="none", factor=1.0, far=0),
        # prompts of uneven lengths, part of the head rotated in the interleaved layout, a
        # context stretched 8 times, far positions
        dict(name="rope_prefill_ragged", op="rope", B=5, T=2500, L=2500, Hq=32, Hkv=8, rot=64,
             interleaved=True, scaling="by_parts", factor=8.0, far=40000),
        # one request, a chain of 6 drafted tokens: latency
        dict(name="tree_chain_1x1000", op="tree", B=1, T=6, L=1000, Hq=32, Hkv=8, tree=False,
             softcap=0.0, bias=False, window=0, ragged=False),
        # a ragged batch, 24-token trees, capped scores, 8 query heads per kv head
        dict(name="tree_16x24_capped", op="tree", B=16, T=24, L=6000, Hq=64, Hkv=8, tree=True,
             softcap=30.0, bias=False, window=0, ragged=True),
        # wide trees over long contexts
        dict(name="tree_8x64_long", op="tree", B=8, T=64, L=16384, Hq=32, Hkv=8, tree=True,
             softcap=0.0, bias=False, window=0, ragged=False),
        # single-token decode with a distance bias and a sliding window
        dict(name="decode_bias_window", op="tree", B=64, T=1, L=4096, Hq=32, Hkv=8, tree=False,
             softcap=0.0, bias=True, window=2000, ragged=True),
        # weights of one decode step
        dict(name="weights_decode_8x8192", op="weights", B=8, T=1, L=8192, Hq=32, Hkv=8, decay=1.0,
             ragged=False),
        # weights of a prompt's last 32 tokens
        dict(name="weights_observe_3x32", op="weights", B=3, T=32, L=7001, Hq=32, Hkv=4, decay=0.5,
             ragged=True),
        # a batch trimmed to a budget
        dict(name="select_64x4096", op="select", B=64, L=4096, keep=1024, sink=4, recent=128),
        # one very long sequence
        dict(name="select_1x131072", op="select", B=1, L=131072, keep=16384, sink=16, recent=1024),
        # the accepted path of a draft tree moved up
        dict(name="compact_accept_32", op="compact", B=32, L=2000, T=24, n=5, Hkv=8, acc=False),
        # half of a long cache evicted, the accumulated weights moved along
        dict(name="compact_evict_8x8192", op="compact", B=8, L=8192, T=0, n=4096, Hkv=8, acc=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "tree", "tree", "tree", "weights", "select", "compact"])
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 4, 8])
    if op == "rope":
        B = _log(rng, 1, 64)
        T = _log(rng, 1, max(1, 8000 // B))
        return dict(op=op, B=B, T=T, L=T + _log(rng, 1, 2000), Hq=Hkv * G, Hkv=Hkv,
                    rot=2 * rng.randint(1, 64), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "ntk", "by_parts"]),
                    factor=rng.choice([2.0, 4.0, 8.0]), far=rng.choice([0, 0, 100000, 1000000]))
    if op == "tree":
        B = _log(rng, 1, 48)
        T = _log(rng, 1, 64)
        return dict(op=op, B=B, T=T, L=T + _log(rng, 1, max(64, min(30000, 60000 // B))),
                    Hq=Hkv * G, Hkv=Hkv, tree=rng.random() < 0.6,
                    softcap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.3,
                    window=rng.choice([0, 0, 0, 100, 1500]), ragged=rng.random() < 0.6)
    if op == "weights":
        B = _log(rng, 1, 16)
        T = rng.choice([1, 1, 5, 16, 32])
        return dict(op=op, B=B, T=T, L=T + _log(rng, 1, 64000 // B), Hq=Hkv * G, Hkv=Hkv,
                    decay=rng.choice([1.0, 0.75]), ragged=rng.random() < 0.6)
    if op == "select":
        B = _log(rng, 1, 64)
        L = _log(rng, 16, 131072 // B)
        keep = max(1, int(L * rng.uniform(0.05, 1.1)))
        return dict(op=op, B=B, L=L, keep=keep, sink=min(rng.choice([0, 4, 16]), keep // 4),
                    recent=rng.randint(0, keep // 2))
    B = _log(rng, 1, 32)
    if rng.random() < 0.5:
        T = rng.randint(2, 64)
        return dict(op=op, B=B, L=T + _log(rng, 1, 36000 // B), T=T, n=rng.randint(1, min(T, 12)),
                    Hkv=Hkv, acc=rng.random() < 0.5)
    L = _log(rng, 32, 36000 // B)
    return dict(op=op, B=B, L=L, T=0, n=max(1, int(L * rng.uniform(0.1, 0.9))), Hkv=Hkv,
                acc=rng.random() < 0.7)


# ---------------------------------------------------------------------------- sizes
def _lens(case):
    """Cached tokens of every sequence, drafted ones included: from the case alone."""
    B, L = case["B"], case["L"]
    low = max(case.get("T", 0), 1)
    if not case.get("ragged", False) or B == 1:
        return [L] * B
    return [max(low, L - (((b * 7) % B) * 3 * L) // (4 * (B - 1))) for b in range(B)]


def _tokens(case):
    """New (drafted) tokens of every sequence."""
    B, T = case["B"], case["T"]
    if case["op"] == "rope" and T > 64:                  # prompts of uneven lengths
        return [max(1, T - ((b * 5) % B) * T // (2 * B)) for b in range(B)]
    if case["op"] == "tree" and case["ragged"] and T > 2:
        return [max(1, T - (b % 3)) for b in range(B)]
    return [T] * B


def work(case):
    op, B = case["op"], case["B"]
    if op == "rope":
        N = sum(_tokens(case))
        heads = case["Hq"] + 2 * case["Hkv"]
        return dict(bytes=4 * N * heads * D, flops=3 * N * (case["Hq"] + case["Hkv"]) * case["rot"])
    if op in ("tree", "weights"):
        lens, toks = _lens(case), _tokens(case)
        w = case.get("window", 0)
        row = case["Hkv"] * D * 2
        keys = sum(min(l, w + t) if w else l for l, t in zip(lens, toks))
        pairs = sum(t * (min(l, w) if w else l) for l, t in zip(lens, toks))
        N = sum(toks)
        if op == "tree":
            return dict(bytes=2 * keys * row + 4 * N * case["Hq"] * D + 4 * N * case["Hq"],
                        flops=4 * D * case["Hq"] * pairs)
        return dict(bytes=keys * row + 2 * N * case["Hq"] * D + 4 * N * case["Hq"] + 8 * keys,
                    flops=2 * D * case["Hq"] * pairs)
    if op == "select":
        return dict(bytes=4 * B * case["L"] + 4 * B * min(case["keep"], case["L"]), flops=B * case["L"])
    n = case["n"]
    if case["T"]:
        moved = max(n - 1, 1)                            # the root stays in its place
    else:
        moved = max(n - min(4, n), 1)                    # the first tokens stay in theirs
    rows = B * moved
    return dict(bytes=rows * 4 * case["Hkv"] * D * 2 + 4 * B * n + (8 * rows if case["acc"] else 0), flops=0)


# ---------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _pages(lens, g):
    """A page table with the pages of the pool in random order."""
    np_ = [(l + PAGE - 1) // PAGE for l in lens]
    total = sum(np_)
    indptr = [0]
    for n in np_:
        indptr.append(indptr[-1] + n)
    i32 = dict(dtype=torch.int32, device="cuda")
    ids = torch.randperm(total + 3, generator=g, device="cuda")[:total].to(torch.int32)
    last = [l - (n - 1) * PAGE if n else 0 for l, n in zip(lens, np_)]
    return torch.tensor(indptr, **i32), ids.contiguous(), torch.tensor(last, **i32), total + 3


def _half(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).half()


def _slots(s, b):
    """Rows (page * 16 + place) of the cached tokens of sequence b, in order."""
    L = s["lens"][b]
    p0 = s["h_indptr"][b]
    n = (L + PAGE - 1) // PAGE
    ids = s["indices"][p0:p0 + n].long()
    return (ids[:, None] * PAGE + torch.arange(PAGE, device="cuda")).reshape(-1)[:L]


def _tree(T, g):
    """Parents (-1: the root) of a random draft tree in topological order."""
    par = [-1]
    r = torch.rand(max(T, 1), generator=g, device="cuda").tolist()
    for i in range(1, T):
        lo = max(0, i - 8)
        par.append(lo + int(r[i] * (i - lo)))
    return par


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case=case)
    i32 = dict(dtype=torch.int32, device="cuda")
    if op == "select":
        B, L = case["B"], case["L"]
        lens = [max(1, L - (b * 37) % max(1, L // 8)) for b in range(B)]
        s["indptr"], _, s["last"], _ = _pages(lens, g)
        s["lens"] = lens
        # heavy-tailed weights; coarse, so that values tie
        a = torch.rand(B, L, generator=g, device="cuda").pow(6.0) * 64.0
        s["acc"] = torch.where(a < 1.0, (a * 256).round() / 256, a)
        s["n"] = [min(case["keep"], l) for l in lens]
        if own:
            s["idx"] = torch.empty(B, case["keep"], **i32)
            s["count"] = torch.empty(B, **i32)
        return s
    Hkv = case["Hkv"]
    lens = _lens(case)
    s["lens"] = lens
    s["indptr"], s["indices"], s["last"], P = _pages(lens, g)
    s["h_indptr"] = [0]
    for l in lens:
        s["h_indptr"].append(s["h_indptr"][-1] + (l + PAGE - 1) // PAGE)
    s["k_cache"] = _half(g, P, PAGE, Hkv, D)
    s["v_cache"] = _half(g, P, PAGE, Hkv, D)
    if op == "compact":
        B, n = case["B"], case["n"]
        rows, start = [], []
        for b in range(B):
            if case["T"]:                        # a path through the drafted tokens, root first
                c = lens[b] - case["T"]
                r = torch.randperm(case["T"] - 1, generator=g, device="cuda")[:n - 1] + 1
                rows.append(c + torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), r.sort().values]))
                start.append(c)
            else:                                # the first tokens and any others
                k = min(4, n)
                r = torch.randperm(lens[b] - k, generator=g, device="cuda")[:n - k] + k
                rows.append(torch.cat([torch.arange(k, device="cuda"), r.sort().values]))
                start.append(0)
        s["idx"] = torch.stack(rows).to(torch.int32)
        s["count"] = torch.full((B,), n, **i32)
        s["start"] = torch.tensor(start, **i32)
        s["h_start"] = start
        s["acc"] = torch.rand(B, case["L"], generator=g, device="cuda") if case["acc"] else None
        if own:
            s["new_len"] = torch.empty(B, **i32)
        return s
    toks = _tokens(case)
    s["toks"] = toks
    Hq, N = case["Hq"], sum(toks)
    h_q = [0]
    for t in toks:
        h_q.append(h_q[-1] + t)
    s["h_q"] = h_q
    s["q_indptr"] = torch.tensor(h_q, **i32)
    if op == "rope":
        s["qkv"] = _half(g, N, (Hq + 2 * Hkv) * D)       # the output of one fused projection
        pos = torch.cat([torch.arange(l - t, l) for l, t in zip(lens, toks)]) + case["far"]
        s["positions"] = pos.to(**i32)
        if own:
            ckl = _ckl()
            q, k, v = s["qkv"].split([Hq * D, Hkv * D, Hkv * D], 1)
            s["rope"] = ckl.rope_plan(case["rot"], interleaved=case["interleaved"],
                                      scaling=case["scaling"], factor=case["factor"],
                                      original_len=4096)
            s["q_out"] = torch.empty(N, Hq, D, dtype=torch.float16, device="cuda")
            s["p"] = ckl.make_append_params(
                q.unflatten(1, (Hq, D)), k.unflatten(1, (Hkv, D)), v.unflatten(1, (Hkv, D)),
                s["k_cache"], s["v_cache"], s["indptr"], s["indices"], s["last"], q_out=s["q_out"],
                q_indptr=s["q_indptr"], positions=s["positions"])
        return s
    s["q"] = _half(g, N, Hq, D, scale=1.5)
    s["mask"] = s["positions"] = s["slopes"] = None
    if case.get("tree", False):
        W = (max(toks) + 31) // 32
        m, pos = torch.zeros(N, W, dtype=torch.int64), []
        for b, t in enumerate(toks):
            bits, depth = [], []
            for i, par in enumerate(_tree(t, g)):
                bits.append((bits[par] if par >= 0 else 0) | (1 << i))
                depth.append(depth[par] + 1 if par >= 0 else 0)
                for w in range(W):
                    m[h_q[b] + i, w] = (bits[i] >> (32 * w)) & 0xffffffff
                pos.append(lens[b] - t + depth[i])
        s["mask"] = torch.where(m >= 1 << 31, m - (1 << 32), m).to(**i32)
        s["positions"] = torch.tensor(pos, **i32)
    if case.get("bias", False):
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) for h in range(Hq)],
                                   dtype=torch.float32, device="cuda")
    if op == "weights":
        s["acc"] = torch.rand(case["B"], case["L"], generator=g, device="cuda") * 4
        s["lse"] = torch.empty(N, Hq, dtype=torch.float32, device="cuda")
        for b in range(case["B"]):
            sc = _scores(s, b, torch.float64)
            rows = slice(h_q[b], h_q[b + 1])
            s["lse"][rows] = torch.logsumexp(sc, 2).permute(1, 0).float()
    if own:
        ckl = _ckl()
        s["p"] = ckl.make_tree_params(
            s["q"], s["k_cache"], s["v_cache"], s["indptr"], s["indices"], s["last"],
            q_indptr=s["q_indptr"], max_q=max(toks), max_len=max(lens), tree_mask=s["mask"],
            positions=s["positions"], slopes=s["slopes"], softcap=case.get("softcap", 0.0),
            window=case.get("window", 0))
        if op == "tree":
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(N, Hq, dtype=torch.float32, device="cuda")
            s["ws"] = torch.empty(max(ckl.tree_workspace_size(s["p"]), 256), dtype=torch.uint8,
                                  device="cuda")
    return s


# ---------------------------------------------------------------------------- plain forms
def _scores(s, b, dtype):
    """Scores [Hq, T, L] of the drafted tokens of sequence b, -inf where a key is not seen."""
    c = s["case"]
    L, T, Hq, Hkv = s["lens"][b], s["toks"][b], c["Hq"], c["Hkv"]
    rows = slice(s["h_q"][b], s["h_q"][b + 1])
    k = s["k_cache"].view(-1, Hkv, D)[_slots(s, b)].to(dtype)
    q = s["q"][rows].to(dtype).view(T, Hkv, Hq // Hkv, D)
    sc = torch.matmul(q.permute(1, 2, 0, 3).reshape(Hkv, -1, D), k.permute(1, 2, 0))
    sc = sc.view(Hq, T, L) * (1.0 / math.sqrt(D))
    if c.get("softcap", 0.0):
        sc = torch.tanh(sc / c["softcap"]) * c["softcap"]
    kpos = torch.arange(L, device="cuda")
    qpos = kpos[L - T:]
    if s["positions"] is not None:
        qpos = s["positions"][rows].long()
        kpos = torch.cat([kpos[:L - T], qpos])
    dist = qpos[:, None] - kpos[None, :]
    if s["slopes"] is not None:
        sc = sc - s["slopes"].to(dtype)[:, None, None] * dist
    seen = torch.ones(T, L, dtype=torch.bool, device="cuda")
    j = torch.arange(T, device="cuda")
    if s["mask"] is not None:
        m = s["mask"][rows]
        seen[:, L - T:] = ((m[:, j // 32] >> (j % 32)) & 1) != 0
    else:
        seen[:, L - T:] = j[None, :] <= j[:, None]
    if c.get("window", 0):
        seen &= dist < c["window"]
    return sc.masked_fill(~seen, float("-inf"))


def _inv_freq(case, dtype):
    """Angle per position of every rotated pair, and the factor on cosine and sine."""
    r, base, f = case["rot"], 10000.0, case["factor"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    if case["scaling"] == "ntk" and r > 2:
        base *= f ** (r / (r - 2))
    inv = base ** (-2.0 * i / r)
    scale = 1.0
    if case["scaling"] == "linear":
        inv = inv / f
    if case["scaling"] == "by_parts":
        at = [r * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), r - 1)
        ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv / f * ramp + inv * (1 - ramp)
        scale = 0.1 * math.log(f) + 1.0
    return inv.to(dtype), scale


def _rope_plain(s):
    c = s["case"]
    Hq, Hkv, r = c["Hq"], c["Hkv"], c["rot"]
    inv, scale = _inv_freq(c, torch.float64)             # far positions need the angle in 64 bits
    ang = s["positions"].double()[:, None] * inv
    cos, sin = (ang.cos() * scale).float()[:, None], (ang.sin() * scale).float()[:, None]
    x = s["qkv"].float().view(-1, Hq + 2 * Hkv, D)
    y = x[:, :Hq + Hkv].clone()
    if c["interleaved"]:
        a, b = x[:, :Hq + Hkv, 0:r:2], x[:, :Hq + Hkv, 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[:, :Hq + Hkv, :r // 2], x[:, :Hq + Hkv, r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = a * cos - b * sin, a * sin + b * cos
    y = y.half()
    at = torch.cat([_slots(s, b)[l - t:] for b, (l, t) in enumerate(zip(s["lens"], s["toks"]))])
    s["k_cache"].view(-1, Hkv, D)[at] = y[:, Hq:]
    s["v_cache"].view(-1, Hkv, D)[at] = x[:, Hq + Hkv:].half()
    return dict(q=y[:, :Hq].contiguous(), k_cache=s["k_cache"], v_cache=s["v_cache"])


def _tree_plain(s):
    c = s["case"]
    Hq, Hkv = c["Hq"], c["Hkv"]
    outs, lses = [], []
    for b in range(c["B"]):
        sc = _scores(s, b, torch.float32)
        m = sc.amax(2, keepdim=True)
        p = torch.exp(sc - m)
        l = p.sum(2, keepdim=True)
        v = s["v_cache"].view(-1, Hkv, D)[_slots(s, b)].float().permute(1, 0, 2)
        o = torch.matmul(p.view(Hkv, -1, p.shape[2]), v).view(Hq, -1, D) / l
        outs.append(o.permute(1, 0, 2).half())
        lses.append((m + torch.log(l)).squeeze(2).t())
    return dict(out=torch.cat(outs), lse=torch.cat(lses))


def _weights_plain(s):
    c = s["case"]
    s["acc"].copy_(torch.stack([
        torch.cat([s["acc"][b, :s["lens"][b]] * c["decay"] + torch.exp(
            _scores(s, b, torch.float32) - s["lse"][s["h_q"][b]:s["h_q"][b + 1]].t()[:, :, None]).sum((0, 1)),
            s["acc"][b, s["lens"][b]:]]) for b in range(c["B"])]))
    return dict(acc=s["acc"])


def _select_plain(s):
    c = s["case"]
    B, keep = c["B"], c["keep"]
    idx = torch.full((B, keep), -1, dtype=torch.int32, device="cuda")
    for b, (L, n) in enumerate(zip(s["lens"], s["n"])):
        if L <= keep:
            idx[b, :L] = torch.arange(L, dtype=torch.int32, device="cuda")
            continue
        a = s["acc"][b, :L].clone()
        a[:c["sink"]] = float("inf")
        a[L - c["recent"]:] = float("inf")
        top = torch.sort(a, descending=True, stable=True).indices[:keep]
        idx[b] = top.sort().values.to(torch.int32)
    return dict(idx=idx, count=torch.tensor(s["n"], dtype=torch.int32, device="cuda"))


def _compact_plain(s):
    c = s["case"]
    n, Hkv = c["n"], c["Hkv"]
    for b in range(c["B"]):
        at = _slots(s, b)
        src, dst = at[s["idx"][b].long()], at[s["h_start"][b]:s["h_start"][b] + n]
        for name in ("k_cache", "v_cache"):
            rows = s[name].view(-1, Hkv, D)
            rows[dst] = rows[src]
        if s["acc"] is not None:
            a, end = s["acc"][b], s["h_start"][b] + n
            a[s["h_start"][b]:end] = a[s["idx"][b].long()]
            a[end:s["lens"][b]] = 0
    out = dict(k_cache=s["k_cache"], v_cache=s["v_cache"], new_len=s["start"] + s["count"])
    if s["acc"] is not None:
        out["acc"] = s["acc"]
    return out


def run(s):
    c = s["case"]
    op = c["op"]
    if not own:
        return {"rope": _rope_plain, "tree": _tree_plain, "weights": _weights_plain,
                "select": _select_plain, "compact": _compact_plain}[op](s)
    ckl = _ckl()
    if op == "rope":
        ckl.rope_append(s["p"], s["rope"])
        return dict(q=s["q_out"], k_cache=s["k_cache"], v_cache=s["v_cache"])
    if op == "tree":
        ckl.tree_attention(s["p"], out=s["out"], lse=s["lse"], workspace=s["ws"])
        return dict(out=s["out"], lse=s["lse"])
    if op == "weights":
        ckl.cache_weights(s["p"], s["lse"], s["acc"], decay=c["decay"])
        return dict(acc=s["acc"])
    if op == "select":
        ckl.cache_select(s["acc"], s["indptr"], s["last"], c["keep"], sink=c["sink"],
                         recent=c["recent"], keep_idx=s["idx"], keep_count=s["count"])
        return dict(idx=s["idx"], count=s["count"])
    ckl.cache_compact(s["k_cache"], s["v_cache"], s["indptr"], s["indices"], s["last"], s["idx"],
                      s["count"], dst_start=s["start"], acc=s["acc"], new_len=s["new_len"])
    out = dict(k_cache=s["k_cache"], v_cache=s["v_cache"], new_len=s["new_len"])
    if s["acc"] is not None:
        out["acc"] = s["acc"]
    return out


# ---------------------------------------------------------------------------- 64 bits
def _row_of(s, b, p):
    """Cache row of token p of sequence b, through the page table."""
    return s["indices"][s["h_indptr"][b] + p // PAGE].long() * PAGE + p % PAGE


def _attend64(s, b, i):
    """Scores [Hq, L] of drafted token i of sequence b in 64 bits, and the cache rows."""
    c = s["case"]
    L, T, Hq, Hkv = s["lens"][b], s["toks"][b], c["Hq"], c["Hkv"]
    n = s["h_q"][b] + i
    p = torch.arange(L, device="cuda")
    at = _row_of(s, b, p)
    k = s["k_cache"].view(-1, Hkv, D)[at].double()
    q = s["q"][n].double().view(Hkv, Hq // Hkv, D)
    x = torch.einsum("hgd,phd->hgp", q, k).reshape(Hq, L) / D ** 0.5
    cap = c.get("softcap", 0.0)
    if cap:
        x = cap * torch.tanh(x / cap)
    first = L - T
    pos = p.clone()
    if s["positions"] is not None:
        pos[first:] = s["positions"][s["h_q"][b]:s["h_q"][b] + T].long()
    if s["slopes"] is not None:
        x = x + s["slopes"].double()[:, None] * (pos - pos[first + i])[None]
    hide = torch.zeros(L, dtype=torch.bool, device="cuda")
    for w in range((T + 31) // 32):
        for j in range(32 * w, min(T, 32 * w + 32)):
            if s["mask"] is None:
                if j > i:
                    hide[first + j:] = True
                    break
    if s["mask"] is not None:
        bits = [int(v) & 0xffffffff for v in s["mask"][n].tolist()]
        hide[first:] = torch.tensor([not (bits[j // 32] >> (j % 32)) & 1 for j in range(T)], device="cuda")
    if c.get("window", 0):
        hide |= (pos[first + i] - pos) >= c["window"]
    x[:, hide] = float("-inf")
    return x, at


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    op = case["op"]
    if op == "select":
        rows, count = [], []
        for b, L in enumerate(s["lens"]):
            a = s["acc"][b].tolist()[:L]
            pin = set(range(min(case["sink"], L))) | set(range(max(0, L - case["recent"]), L))
            rest = sorted((i for i in range(L) if i not in pin), key=lambda i: (-a[i], i))
            got = list(range(L)) if L <= case["keep"] else sorted(list(pin) + rest[:case["keep"] - len(pin)])
            count.append(len(got))
            rows.append(got + [-1] * (case["keep"] - len(got)))
        return dict(idx=torch.tensor(rows), count=torch.tensor(count))
    if op == "compact":
        k, v = s["k_cache"].clone(), s["v_cache"].clone()
        for b in range(case["B"]):
            src = s["idx"][b].long()
            dst = torch.arange(case["n"], device="cuda") + s["h_start"][b]
            for old, new in ((s["k_cache"], k), (s["v_cache"], v)):
                new.view(-1, case["Hkv"], D)[_row_of(s, b, dst)] = old.view(-1, case["Hkv"], D)[_row_of(s, b, src)]
        out = dict(k_cache=k, v_cache=v, new_len=torch.tensor(s["h_start"]) + case["n"])
        if s["acc"] is not None:
            a = s["acc"].double()
            for b in range(case["B"]):
                st, n = s["h_start"][b], case["n"]
                row = a[b].clone()
                a[b, st:st + n] = row[s["idx"][b].long()]
                a[b, st + n:s["lens"][b]] = 0.0
            out["acc"] = a
        return out
    if op == "rope":
        Hq, Hkv, r = case["Hq"], case["Hkv"], case["rot"]
        inv, scale = _inv_freq(case, torch.float64)
        k, v = s["k_cache"].double(), s["v_cache"].double()
        qs = []
        for b in range(case["B"]):
            lo, hi, L, T = s["h_q"][b], s["h_q"][b + 1], s["lens"][b], s["toks"][b]
            x = s["qkv"][lo:hi].double().view(T, Hq + 2 * Hkv, D)
            pairs = torch.arange(r, device="cuda").view(r // 2, 2) if case["interleaved"] else \
                torch.arange(r, device="cuda").view(2, r // 2).t()
            turn = torch.polar(torch.full((T, r // 2), scale, dtype=torch.float64, device="cuda"),
                               s["positions"][lo:hi].double()[:, None] * inv[None])
            z = torch.complex(x[:, :Hq + Hkv, pairs[:, 0]], x[:, :Hq + Hkv, pairs[:, 1]]) * turn[:, None]
            y = x[:, :Hq + Hkv].clone()
            y[:, :, pairs[:, 0]], y[:, :, pairs[:, 1]] = z.real, z.imag
            qs.append(y[:, :Hq])
            at = _row_of(s, b, torch.arange(L - T, L, device="cuda"))
            k.view(-1, Hkv, D)[at] = y[:, Hq:]
            v.view(-1, Hkv, D)[at] = x[:, Hq + Hkv:]
        return dict(q=torch.cat(qs), k_cache=k, v_cache=v)
    N, Hq, Hkv = sum(s["toks"]), case["Hq"], case["Hkv"]
    G = Hq // Hkv
    if op == "weights":
        acc = s["acc"].double()
        for b in range(case["B"]):
            acc[b, :s["lens"][b]] *= case["decay"]
            for i in range(s["toks"][b]):
                x, _ = _attend64(s, b, i)
                acc[b, :s["lens"][b]] += (x - s["lse"][s["h_q"][b] + i].double()[:, None]).exp().sum(0)
        return dict(acc=acc)
    if sum(l * t for l, t in zip(s["lens"], s["toks"])) * Hq > 1 << 31:
        return None
    out = torch.zeros(N, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.zeros(N, Hq, dtype=torch.float64, device="cuda")
    for b in range(case["B"]):
        for i in range(s["toks"][b]):
            x, at = _attend64(s, b, i)
            top = x.max(1, keepdim=True).values
            e = (x - top).exp()
            n = s["h_q"][b] + i
            v = s["v_cache"].view(-1, Hkv, D)[at].double()
            out[n] = torch.einsum("hgp,phd->hgd", (e / e.sum(1, keepdim=True)).view(Hkv, G, -1), v).reshape(Hq, D)
            lse[n] = top[:, 0] + e.sum(1).log()
    return dict(out=out, lse=lse)
