"""Cases of the speculative-decoding and bounded-cache operators over the paged multi-turn cache:

* ``tree``    dvattn_tree_sdpa: attention of a tree of drafted tokens over the paged cache and the tree's own
              keys (a token sees the cache and its ancestors in the tree);
* ``commit``  dvattn_tree_append: the accepted tokens of the tree, keys rotated, written into the pages;
* ``mass``    dvattn_paged_mass: the attention weight that every cached key received, added to a running sum;
* ``evict``   dvattn_paged_evict: the keys of least accumulated weight leave the cache, the survivors behind the
              kept length fill the holes.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end),
or, where ``own`` is true, calls dvattn_b200.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one fp32 sequence of the plumbing configuration (16/1 heads, 1024 keys), four drafted tokens: latency
        {"name": "tree-one-f32", "op": "tree", "dtype": "f32", "W": 1, "Hq": 16, "Hkv": 1, "E": 128, "R": 64, "BS": 16,
         "F": 1, "lo": 1024, "hi": 1024, "S": 4, "fan": 2, "layout": 1},
        # the batched bf16 decode configuration (32 sequences, 64/4 heads, two turns) verifying 8 drafted tokens
        {"name": "tree-batch-bf16", "op": "tree", "dtype": "bf16", "W": 32, "Hq": 64, "Hkv": 4, "E": 128, "R": 64, "BS": 16,
         "F": 2, "lo": 512, "hi": 8192, "S": 8, "fan": 2, "layout": 2},
        # the long-context fp16 configuration (128/8 heads, full rotary, pages of 64), ragged lengths up to 128k
        {"name": "tree-long-f16", "op": "tree", "dtype": "f16", "W": 4, "Hq": 128, "Hkv": 8, "E": 128, "R": 128, "BS": 64,
         "F": 1, "lo": 65001, "hi": 131072, "S": 16, "fan": 3, "layout": 3},
        # the serving mix (head dim 256, 1-4 turns), a short odd tree
        {"name": "tree-serve-e256-f16", "op": "tree", "dtype": "f16", "W": 48, "Hq": 32, "Hkv": 2, "E": 256, "R": 64, "BS": 64,
         "F": 4, "lo": 16, "hi": 6000, "S": 5, "fan": 2, "layout": 4},
        # a wide tree of 61 tokens for 8 sequences of the prefill configuration's heads: bound by the products
        {"name": "tree-wide-bf16", "op": "tree", "dtype": "bf16", "W": 8, "Hq": 32, "Hkv": 2, "E": 128, "R": 32, "BS": 16,
         "F": 1, "lo": 2001, "hi": 16384, "S": 61, "fan": 4, "layout": 5},
        # the accepted tokens of one verification step of the batched decode
        {"name": "commit-step-bf16", "op": "commit", "dtype": "bf16", "W": 32, "Hq": 64, "Hkv": 4, "E": 128, "R": 64, "BS": 16,
         "lo": 512, "hi": 1024, "S": 8, "A": 4, "layout": 6},
        # a large batch with wide trees and long accepted runs
        {"name": "commit-wide-f16", "op": "commit", "dtype": "f16", "W": 256, "Hq": 32, "Hkv": 8, "E": 128, "R": 128, "BS": 64,
         "lo": 100, "hi": 700, "S": 64, "A": 37, "layout": 7},
        # one fp32 sequence of the plumbing configuration
        {"name": "mass-one-f32", "op": "mass", "dtype": "f32", "W": 1, "Hq": 16, "Hkv": 1, "E": 128, "R": 64, "BS": 16,
         "F": 1, "lo": 1024, "hi": 1024, "S": 1, "layout": 8},
        # one decode step of the batched bf16 configuration
        {"name": "mass-step-bf16", "op": "mass", "dtype": "bf16", "W": 32, "Hq": 64, "Hkv": 4, "E": 128, "R": 64, "BS": 16,
         "F": 2, "lo": 512, "hi": 8192, "S": 1, "layout": 9},
        # the last 31 queries of long prompts score their keys before the prompt is thinned out
        {"name": "mass-window-f16", "op": "mass", "dtype": "f16", "W": 4, "Hq": 128, "Hkv": 8, "E": 128, "R": 128, "BS": 64,
         "F": 1, "lo": 20001, "hi": 32768, "S": 31, "layout": 10},
        # every step of a decode at its budget: a few tokens over 4096 leave
        {"name": "evict-step-bf16", "op": "evict", "dtype": "bf16", "W": 32, "Hq": 64, "Hkv": 4, "E": 128, "BS": 16,
         "lo": 4100, "hi": 4128, "keep": 4096, "sink": 4, "recent": 64, "layout": 11},
        # prompts of up to 30000 tokens thinned out to about 4000
        {"name": "evict-prompt-f16", "op": "evict", "dtype": "f16", "W": 8, "Hq": 128, "Hkv": 8, "E": 128, "BS": 64,
         "lo": 9001, "hi": 30000, "keep": 4001, "sink": 4, "recent": 257, "layout": 12},
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "commit", "mass", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    E = rng.choice([64, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    Hq = Hkv * rng.choice([1, 2, 4, 5, 8, 16])
    W = _logint(rng, 1, 48)
    BS = rng.choice([1, 8, 16, 16, 32, 64, 96])
    R = rng.choice([0, 32, E // 2, E])
    layout = rng.randrange(1 << 20)
    c = {"op": op, "dtype": dtype, "W": W, "Hq": Hq, "Hkv": Hkv, "E": E, "BS": BS, "layout": layout}
    # the cached keys of the whole batch stay under 0.5 GiB a tensor, the scores under 1 GiB
    most = (1 << 29) // (W * Hkv * E * 4)
    if op == "commit":
        S = _logint(rng, 1, 64)
        c.update(R=R, lo=1, hi=max(1, min(1024, most - S)), S=S, A=rng.randint(1, S))
    elif op == "evict":
        hi = max(2, min(_logint(rng, 2, 40000), most))
        keep = rng.randint(1, hi)
        c.update(lo=rng.randint(1, hi), hi=hi, keep=keep, sink=rng.randint(0, 5), recent=rng.randint(0, 1 + keep // 8))
    else:
        S = _logint(rng, 1, 64)
        F = rng.choice([1, 1, 2, 3])
        hi = max(1, min(_logint(rng, 1, 40000), most // F, (1 << 28) // (F * W * Hq * S)))
        c.update(R=R, F=F, lo=rng.randint(1, hi), hi=hi, S=S)
        if op == "tree":
            c["fan"] = rng.randint(1, 4)
    return c


def _turns(c):
    """Keys of turn f cached for sequence w [W, F], and the turns' padded lengths [F]."""
    rs = np.random.RandomState(c["layout"])
    n = rs.randint(c["lo"], c["hi"] + 1, size=c["W"])
    n[0] = c["hi"]
    cuts = np.sort(rs.randint(0, n[:, None] + 1, size=(c["W"], c["F"] - 1)), axis=1)
    edges = np.concatenate([np.zeros((c["W"], 1), int), cuts, n[:, None]], axis=1)
    tl = np.diff(edges, axis=1)
    return rs, tl, tl.max(axis=0)


def _tree(c, rs):
    """Parents [W, S] (-1: a child of the context, -2: no token, at the end of shorter trees) and depths."""
    W, S = c["W"], c["S"]
    par, dep = np.full((W, S), -2, int), np.zeros((W, S), int)
    for w in range(W):
        n = S if w == 0 else rs.randint(max(1, S // 2), S + 1)
        for j in range(n):
            p = (j - 1) // c["fan"] if rs.rand() < 0.8 else rs.randint(-1, j)
            p = -1 if j == 0 else p
            par[w, j], dep[w, j] = p, 0 if p < 0 else dep[w, p] + 1
    return par, dep


def _pages(c, rs, positions):
    """A table of distinct pages, in no order, for `positions` logical positions of every sequence."""
    maxb = max(1, -(-int(positions) // c["BS"]))
    return rs.permutation(c["W"] * maxb).reshape(c["W"], maxb)


# ------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------
def _rotary(pos, R):
    i = torch.arange(R // 2, dtype=torch.float64, device=DEV)
    a = torch.as_tensor(pos, device=DEV).double()[..., None] * 10000.0 ** (-2.0 * i / max(R, 1))
    return [torch.cat([t, t], -1).float().contiguous() for t in (a.cos(), a.sin())]


def prepare(case, seed):
    c = case
    T, W, Hq, Hkv, E, BS = TYPES[c["dtype"]], c["W"], c["Hq"], c["Hkv"], c["E"], c["BS"]
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=T)

    def ints(a):
        return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device=DEV)

    s = {"op": c["op"], "scale": 1.0 / math.sqrt(E)}
    if c["op"] in ("tree", "mass"):
        rs, tl, L = _turns(c)
        F, S = c["F"], c["S"]
        bt = _pages(c, rs, L.sum())
        par, dep = _tree(c, rs) if c["op"] == "tree" else (None, np.arange(S)[None].repeat(W, 0) - S)
        left = tl[:, ::-1].cumsum(axis=1)[:, ::-1]  # keys of turn f and the turns after it
        s["cos"], s["sin"] = _rotary(left.T[:, :, None] + dep[None], c["R"])
        loc = np.repeat(tl.T[:, :, None] - 1, S, axis=2)
        if c["op"] == "mass":  # the queries are the sequence's last tokens: causal within the last turn
            loc[-1] -= np.minimum(np.arange(S)[::-1][None], tl[:, -1:])
        s.update(loc=ints(loc), L=ints(L), bt=ints(bt), q=normal(W, Hq, S, E), kc=normal(bt.size, BS, Hkv, E))
        if c["op"] == "tree":
            s.update(parents=ints(par), vc=normal(bt.size, BS, Hkv, E), dk=normal(W, Hkv, S, E), dv=normal(W, Hkv, S, E))
        else:
            sc = _scores(s).permute(1, 2, 3, 0, 4).flatten(3)
            s["lse"] = sc.logsumexp(-1).view(W, Hq, S).contiguous()  # what the attention of this step gave
            s["mass"] = torch.rand((W, Hkv, bt.shape[1] * BS), generator=g, device=DEV) * 4
        return s
    rs = np.random.RandomState(c["layout"])
    n = rs.randint(c["lo"], c["hi"] + 1, size=W)
    n[0] = c["hi"]
    bt = _pages(c, rs, c["hi"] + c.get("S", 0))
    s.update(bt=ints(bt), kc=normal(bt.size, BS, Hkv, E), vc=normal(bt.size, BS, Hkv, E))
    if c["op"] == "commit":
        S, A = c["S"], c["A"]
        acc = np.sort(np.stack([rs.permutation(S)[:A] for _ in range(W)]), axis=1)
        s["cos"], s["sin"] = _rotary(n[:, None] + np.arange(S)[None] // 2, c["R"])
        s.update(dk=normal(W, Hkv, S, E), dv=normal(W, Hkv, S, E), positions=ints(n), accepted=ints(acc),
                 counts=ints(rs.randint(0, A + 1, size=W)))
    else:
        # accumulated weights are heavy-tailed; some keys were never seen
        m = torch.randn((W, Hkv, bt.shape[1] * BS), generator=g, device=DEV).mul_(2).exp_()
        m[torch.rand(m.shape, generator=g, device=DEV) < 0.05] = 0
        s.update(mass=m, starts=ints(np.zeros(W)), lengths=ints(n), keep=ints(np.full(W, c["keep"])), sink=c["sink"],
                 recent=c["recent"], mass_out=torch.empty_like(m), source=torch.empty(m.shape, dtype=torch.int32, device=DEV))
    return s


# ------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------
def run(state):
    return _kernels(state) if own else _plain(state)


def _kernels(s):
    import dvattn_b200 as dv
    if s["op"] == "tree":
        lse = torch.empty(s["q"].shape[:3], dtype=torch.float32, device=s["q"].device)
        out = dv.dvattn_tree_sdpa(s["q"], s["parents"], s["loc"], s["cos"], s["sin"], s["L"], s["kc"], s["vc"], s["bt"],
                                  s["dk"], s["dv"], s["scale"], lse=lse)
        return out, lse
    if s["op"] == "commit":
        dv.dvattn_tree_append(s["kc"], s["vc"], s["dk"], s["dv"], s["cos"], s["sin"], s["bt"], s["positions"], s["accepted"],
                              s["counts"])
        return s["kc"], s["vc"]
    if s["op"] == "mass":
        return dv.dvattn_paged_mass(s["mass"], s["q"], s["lse"], s["loc"], s["cos"], s["sin"], s["L"], s["kc"], s["bt"], s["scale"])
    dv.dvattn_paged_evict(s["kc"], s["vc"], s["mass"], s["bt"], s["starts"], s["lengths"], s["keep"], sink=s["sink"],
                          recent=s["recent"], mass_out=s["mass_out"], source=s["source"])
    return s["kc"], s["vc"], s["mass_out"], s["source"]


def _rotate(x, cos, sin):
    """The first R dims turned pairwise (e, e + R/2), in 32 bits, rounded to x's type; the others as they are."""
    R = cos.shape[-1]
    a, b, rest = x[..., :R // 2].float(), x[..., R // 2:R].float(), x[..., R:]
    c, s = cos[..., :R // 2], sin[..., :R // 2]
    lo, hi = (a * c + -b * s).to(x.dtype), (b * c + a * s).to(x.dtype)
    return torch.cat([lo, hi, rest.expand(lo.shape[:-1] + rest.shape[-1:])], -1)


def _queries(s):
    """Per turn rotated queries, the query heads of a key head side by side: [F, W, Hkv, G * S, E] in 32 bits."""
    W, Hq, S, E = s["q"].shape
    q = _rotate(s["q"][None], s["cos"][:, :, None], s["sin"][:, :, None])
    return q.float().view(-1, W, s["kc"].shape[2], Hq // s["kc"].shape[2] * S, E)


def _gather(cache, bt, pos):
    """Rows [..., Hkv, E] of the logical positions pos [..., W, n] of every sequence, in 32 bits."""
    W, BS = bt.shape[0], cache.shape[1]
    w = torch.arange(W, device=bt.device)[:, None]
    page = bt[w, (pos // BS).clamp(max=bt.shape[1] - 1)].long()
    return cache[page, pos % BS].float()


def _positions(s):
    """Logical positions [F, W, n] of the keys of every turn, n the longest turn's length."""
    L = s["L"].long()
    n = torch.arange(s["bt"].shape[1] * s["kc"].shape[1], device=L.device)[:int(s["L"].max())]
    return ((L.cumsum(0) - L)[:, None, None] + n).expand(-1, s["bt"].shape[0], -1)


def _scores(s):
    """Scaled scores of every turn's keys, -inf where a query does not see the key: [F, W, Hkv, G * S, n]."""
    W, Hq, S, E = s["q"].shape
    Hkv = s["kc"].shape[2]
    k = _gather(s["kc"], s["bt"], _positions(s))
    sc = _queries(s) @ k.permute(0, 1, 3, 4, 2) * s["scale"]
    l = torch.arange(sc.shape[-1], device=sc.device)
    sees = (l <= s["loc"][..., None]) & (l < s["L"][:, None, None, None])
    sees = sees[:, :, None, None].expand(-1, -1, Hkv, Hq // Hkv, -1, -1).flatten(3, 4)
    return sc.masked_fill_(~sees, -math.inf)


def _plain(s):
    if s["op"] == "tree":
        return _plain_tree(s)
    if s["op"] == "commit":
        W, Hkv, S, E = s["dk"].shape
        BS, A = s["kc"].shape[1], s["accepted"].shape[1]
        i = torch.arange(A, device=s["kc"].device)
        on = i < s["counts"][:, None]
        w = torch.arange(W, device=i.device)[:, None].expand(W, A)[on]
        node = s["accepted"].long()[on]
        pos = (s["positions"][:, None] + i)[on].long()
        page = s["bt"].long()[w, pos // BS]
        k = _rotate(s["dk"], s["cos"][:, None], s["sin"][:, None])
        s["kc"][page, pos % BS] = k[w, :, node]
        s["vc"][page, pos % BS] = s["dv"][w, :, node]
        return s["kc"], s["vc"]
    if s["op"] == "mass":
        W, Hq, S, E = s["q"].shape
        Hkv, n = s["kc"].shape[2], int(s["L"].max())
        lse = s["lse"].view(1, W, Hkv, -1, 1)
        lse = lse.masked_fill(lse == -math.inf, math.inf)  # a query that saw nothing gives no weight
        p = (_scores(s) - lse).exp_().sum(3)  # [F, W, Hkv, n]
        pos = _positions(s)[:, :, None].expand_as(p).clamp(max=s["mass"].shape[2] - 1)
        s["mass"].scatter_add_(2, pos.permute(1, 2, 0, 3).flatten(2), p.permute(1, 2, 0, 3).flatten(2))
        return s["mass"]
    return _plain_evict(s)


def _plain_tree(s):
    W, Hq, S, E = s["q"].shape
    Hkv = s["kc"].shape[2]
    par = s["parents"].long()
    eye = torch.eye(S, device=par.device)
    up = (par[:, :, None] == torch.arange(S, device=par.device)).float()
    anc = torch.linalg.matrix_power(eye + up, S) > 0  # a token's ancestors and itself
    there = (anc & (par == -1)[:, None]).any(-1)
    anc = (anc & there[:, :, None])[:, None, None].expand(-1, Hkv, Hq // Hkv, -1, -1).flatten(2, 3)
    there = there[:, None, None].expand(-1, Hkv, Hq // Hkv, -1).flatten(2)
    q = _queries(s)[-1]
    dk = _rotate(s["dk"], s["cos"][-1][:, None], s["sin"][-1][:, None]).float()
    draft = (q @ dk.mT * s["scale"]).masked_fill_(~anc, -math.inf)
    sc = torch.cat([_scores(s).permute(1, 2, 3, 0, 4).flatten(3), draft], -1)
    sc.masked_fill_(~there[..., None], -math.inf)
    v = _gather(s["vc"], s["bt"], _positions(s)).permute(1, 3, 0, 2, 4).flatten(2, 3)
    v = torch.cat([v, s["dv"].float()], 2)
    top = sc.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
    p = sc.sub_(top).exp_()
    l = p.sum(-1, keepdim=True)
    out = (p @ v / l).masked_fill_(~there[..., None], 0.0)
    return out.view(W, Hq, S, E).to(s["q"].dtype), (top + l.log()).view(W, Hq, S)


def _plain_evict(s):
    W, Hkv, N = s["mass"].shape
    i = torch.arange(N, device=s["mass"].device)
    first, n, keep = (s[k].long()[:, None, None] for k in ("starts", "lengths", "keep"))
    at = i - first
    inside = (at >= 0) & (at < n)
    order = torch.where((at < s["sink"]) | (at >= n - s["recent"]), math.inf, s["mass"])
    order = torch.where(inside, order, -math.inf)
    rank = order.argsort(dim=-1, descending=True, stable=True).argsort(dim=-1)
    stays = inside & (rank < keep)
    hole, mover = inside & ~stays & (at < keep), stays & (at >= keep)
    from_ = (~mover).to(torch.uint8).argsort(dim=-1, stable=True)  # the movers first, in their order
    source = torch.where(hole, from_.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), i.expand_as(hole))
    gone = inside & (at >= torch.minimum(n, keep))
    s["mass_out"].copy_(s["mass"].gather(-1, source).masked_fill_(gone, 0.0))
    s["source"].copy_(source.masked_fill(gone, -1))
    bt, BS = s["bt"].long(), s["kc"].shape[1]
    w, h = torch.arange(W, device=i.device)[:, None, None], torch.arange(Hkv, device=i.device)[None, :, None]
    src, dst = (bt[w, source // BS], source % BS, h), (bt[w, i // BS].expand_as(source), (i % BS).expand_as(source), h)
    s["kc"][dst] = s["kc"][src]
    s["vc"][dst] = s["vc"][src]
    return s["kc"], s["vc"], s["mass_out"], s["source"]


# ------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------
def work(case):
    c, es = case, SIZE[case["dtype"]]
    W, Hq, Hkv, E = c["W"], c["Hq"], c["Hkv"], c["E"]
    row = Hkv * E * es  # one token's keys (or values)
    if c["op"] in ("tree", "mass"):
        rs, tl, L = _turns(c)
        F, S, R = c["F"], c["S"], c["R"]
        keys = int(tl.sum())
        tables = sum(-(-int(t) // c["BS"]) for t in tl.sum(axis=1)) * 4 + F * W * S * 4 + F * W * S * R * 4
        if c["op"] == "mass":
            return {"bytes": keys * (row + 8 * Hkv) + W * Hq * S * (E * es + 4) + tables, "flops": 2 * Hq * S * E * keys}
        rs2, _, _ = _turns(c)
        _pages(c, rs2, L.sum())
        par, dep = _tree(c, rs2)
        live = (par > -2).sum(axis=1)
        pairs = int((live * tl.sum(axis=1)).sum()) + int((dep[par > -2] + 1).sum())
        n = int(live.sum())
        return {"bytes": (keys + n) * 2 * row + W * S * Hq * (2 * E * es + 4) + tables + W * S * 4, "flops": 4 * Hq * E * pairs}
    rs = np.random.RandomState(c["layout"])
    n = rs.randint(c["lo"], c["hi"] + 1, size=W)
    n[0] = c["hi"]
    _pages(c, rs, c["hi"] + c.get("S", 0))
    if c["op"] == "commit":
        for _ in range(W):
            rs.permutation(c["S"])
        got = int(rs.randint(0, c["A"] + 1, size=W).sum())
        return {"bytes": got * (4 * row + 2 * c["R"] * 4 + 8) + W * 8, "flops": 3 * got * Hkv * c["R"]}
    # of the evicted tokens a share keep / n lies in front of the kept length: those holes are filled
    cut = np.maximum(0, n - c["keep"])
    moves = float((cut * np.minimum(1, c["keep"] / n)).sum())
    return {"bytes": moves * 4 * row + float(n.sum()) * Hkv * 12, "flops": float(n.sum()) * Hkv}


# ------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------------------
def _turned(x, cos, sin):
    """x [..., E] with each pair (x[e], x[e + R/2]) turned by its angle, rounded to x's type, in 64 bits."""
    h = cos.shape[-1] // 2
    y = x.double().clone()
    lo, hi = y[..., :h].clone(), y[..., h:2 * h].clone()
    y[..., :h] = lo * cos[..., :h].double() - hi * sin[..., :h].double()
    y[..., h:2 * h] = hi * cos[..., :h].double() + lo * sin[..., :h].double()
    return y.to(x.dtype).double()


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "commit":
        # copies and one rotation of single rows: token by token
        bt, pos, acc, cnt = (s[k].cpu().numpy() for k in ("bt", "positions", "accepted", "counts"))
        k, v = s["kc"].double(), s["vc"].double()
        if int(cnt.sum()) > 20000:
            return None
        BS = s["kc"].shape[1]
        for w in range(len(pos)):
            turned = _turned(s["dk"][w], s["cos"][w], s["sin"][w])
            for i in range(cnt[w]):
                p = int(pos[w]) + i
                page = int(bt[w, p // BS])
                k[page, p % BS] = turned[:, acc[w, i]]
                v[page, p % BS] = s["dv"][w, :, acc[w, i]].double()
        return k, v
    if s["op"] == "evict":
        mass = s["mass"].cpu().numpy()
        W, Hkv, N = mass.shape
        if mass.size > 4_000_000:
            return None
        bt, n, keep = (s[k].cpu().numpy() for k in ("bt", "lengths", "keep"))
        source = np.tile(np.arange(N, dtype=np.int32), (W, Hkv, 1))
        out = mass.astype(np.float64)
        k, v = s["kc"].double().cpu().numpy(), s["vc"].double().cpu().numpy()
        BS = k.shape[1]
        for w in range(W):
            for h in range(Hkv):
                m, kept = mass[w, h, :n[w]].astype(np.float64).copy(), min(int(n[w]), int(keep[w]))
                m[:s["sink"]] = np.inf
                if s["recent"]:
                    m[max(0, n[w] - s["recent"]):] = np.inf
                stay = np.sort(np.lexsort((np.arange(n[w]), -m))[:kept])
                holes, movers = np.setdiff1d(np.arange(kept), stay), stay[stay >= kept]
                source[w, h, holes], source[w, h, kept:n[w]] = movers, -1
                out[w, h, holes], out[w, h, kept:n[w]] = mass[w, h, movers], 0
                a, b = (bt[w, holes // BS], holes % BS, h), (bt[w, movers // BS], movers % BS, h)
                k[a], v[a] = k[b], v[b]
        return [torch.from_numpy(x) for x in (k, v, out, source)]
    W, Hq, S, E = s["q"].shape
    Hkv, BS = s["kc"].shape[2], s["kc"].shape[1]
    G, L = Hq // Hkv, s["L"].tolist()
    loc, bt = s["loc"].cpu(), s["bt"].long()
    if s["op"] == "tree":
        out = torch.zeros((W, Hq, S, E), dtype=torch.float64, device=DEV)
        lse = torch.full((W, Hq, S), -math.inf, dtype=torch.float64, device=DEV)
        parents = s["parents"].tolist()
    else:
        mass = s["mass"].double()
    for w in range(W):
        rows = lambda cache, p: cache[bt[w, p // BS], p % BS].double()  # noqa: E731
        spans, first = [], 0
        for f, length in enumerate(L):
            spans.append(torch.arange(first, first + min(length, int(loc[f, w].max()) + 1), device=DEV))
            first += length
        if s["op"] == "tree":
            line = []  # each token's line of ancestors, itself at the end
            for j, p in enumerate(parents[w]):
                line.append([j] if p == -1 else line[p] + [j] if 0 <= p < j and line[p] else [])
            sees = torch.zeros((S, S), dtype=torch.bool)
            for j in range(S):
                sees[j, line[j]] = True
            sees = sees.to(DEV)
            there = sees.any(1)
        for h in range(Hkv):
            z = []
            for f, p in enumerate(spans):
                q = _turned(s["q"][w, h * G:(h + 1) * G], s["cos"][f, w], s["sin"][f, w])  # [G, S, E]
                x = s["scale"] * (q @ rows(s["kc"], p)[:, h].T) if len(p) else q.new_zeros((G, S, 0))
                z.append(x.masked_fill(torch.arange(len(p), device=DEV) > s["loc"][f, w][:, None], -math.inf))
            if s["op"] == "mass":
                got = torch.cat(z, -1) - s["lse"][w, h * G:(h + 1) * G].double()[..., None]
                mass[w, h].index_add_(0, torch.cat(spans), got.exp().nan_to_num(nan=0.0).sum((0, 1)))
                continue
            keys = _turned(s["dk"][w, h], s["cos"][-1, w], s["sin"][-1, w])
            z.append((s["scale"] * (q @ keys.T)).masked_fill(~sees, -math.inf))
            z = torch.cat(z, -1)[:, there]
            v = torch.cat([rows(s["vc"], p)[:, h] for p in spans] + [s["dv"][w, h].double()])
            out[w][h * G:(h + 1) * G, there] = z.softmax(-1) @ v
            lse[w][h * G:(h + 1) * G, there] = z.logsumexp(-1)
    return (out, lse) if s["op"] == "tree" else mass
