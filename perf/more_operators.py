"""Cases of the operators of a paged multi-turn cache held in 8 bits (e4m3, one scale per page and KV head), and of
the pages behind it:

* ``attend``   dvattn_paged_sdpa_q8: the paged decode attention over such a cache;
* ``prefill``  dvattn_varlen_paged_sdpa_q8: the packed chunked prefill over it;
* ``append``   dvattn_paged_append_q8: new tokens, keys rotated, rounded to 8 bits and written into the pages, whose
               scales grow where the new tokens need it;
* ``pages``    dvattn_assign_pages and dvattn_release_pages: block tables and slot maps from request lengths, pages
               taken from a free list and given back.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once at the end), or,
where ``own`` is true, calls dvattn_b200.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
F8 = torch.float8_e4m3fn
TOP = 448.0  # the largest e4m3 value
LEAST = 2.0 ** -60  # the smallest scale that the append sets


# ------------------------------------------------------------------------------------------------------------
# cases
# ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one fp32 sequence of the plumbing configuration (16/1 heads, 1024 keys), one token: latency
        {"name": "attend-one-f32", "op": "attend", "dtype": "f32", "W": 1, "Hq": 16, "Hkv": 1, "E": 128, "R": 64, "BS": 16,
         "F": 1, "lo": 1024, "hi": 1024, "S": 1, "layout": 1},
        # a decode step of the batched bf16 configuration (32 sequences, 64/4 heads, two turns)
        {"name": "attend-batch-bf16", "op": "attend", "dtype": "bf16", "W": 32, "Hq": 64, "Hkv": 4, "E": 128, "R": 64, "BS": 16,
         "F": 2, "lo": 512, "hi": 8192, "S": 1, "layout": 2},
        # the long-context fp16 configuration (128/8 heads, full rotary, pages of 64), ragged lengths up to 128k
        {"name": "attend-long-f16", "op": "attend", "dtype": "f16", "W": 4, "Hq": 128, "Hkv": 8, "E": 128, "R": 128, "BS": 64,
         "F": 1, "lo": 65001, "hi": 131072, "S": 1, "layout": 3},
        # the serving mix (head dim 256, 1-4 turns)
        {"name": "attend-serve-e256-f16", "op": "attend", "dtype": "f16", "W": 96, "Hq": 32, "Hkv": 2, "E": 256, "R": 64, "BS": 64,
         "F": 4, "lo": 16, "hi": 6000, "S": 1, "layout": 4},
        # the last five tokens of each of 24 sequences at once (a short chunk), small heads, few query heads to a KV head
        {"name": "attend-chunk-bf16", "op": "attend", "dtype": "bf16", "W": 24, "Hq": 32, "Hkv": 8, "E": 64, "R": 32, "BS": 32,
         "F": 2, "lo": 101, "hi": 9001, "S": 5, "layout": 5},
        # chunks of prompts behind their contexts, packed (the prefill configuration's heads)
        {"name": "prefill-chunks-bf16", "op": "prefill", "dtype": "bf16", "W": 8, "Hq": 32, "Hkv": 2, "E": 128, "R": 32, "BS": 16,
         "F": 1, "lo": 1, "hi": 8192, "n": 777, "layout": 6},
        # one new token for each sequence of the batched decode
        {"name": "append-step-bf16", "op": "append", "dtype": "bf16", "W": 32, "Hq": 64, "Hkv": 4, "E": 128, "R": 64, "BS": 16,
         "lo": 512, "hi": 1024, "n": 1, "layout": 7},
        # prompts of up to 2048 tokens for 16 sequences
        {"name": "append-prompts-bf16", "op": "append", "dtype": "bf16", "W": 16, "Hq": 32, "Hkv": 2, "E": 128, "R": 32, "BS": 16,
         "lo": 0, "hi": 1000, "n": 2048, "layout": 8},
        # wide chunks in long pages, full rotary
        {"name": "append-chunks-f16", "op": "append", "dtype": "f16", "W": 32, "Hq": 128, "Hkv": 8, "E": 128, "R": 128, "BS": 64,
         "lo": 0, "hi": 300, "n": 501, "layout": 9},
        # a decode step of 256 sequences: one in 16 begins a page
        {"name": "pages-step", "op": "pages", "W": 256, "BS": 16, "lo": 16, "hi": 32000, "n": 1, "spare": 100, "layout": 10},
        # prompts of up to 32k tokens
        {"name": "pages-prompts", "op": "pages", "W": 48, "BS": 16, "lo": 0, "hi": 600, "n": 32000, "spare": 1000, "layout": 11},
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "prefill", "append", "append", "pages"])
    layout = rng.randrange(1 << 20)
    if op == "pages":
        W = _logint(rng, 1, 1024)
        n = _logint(rng, 1, max(1, 1500000 // W) if W > 48 else 32000)
        BS = rng.choice([1, 8, 16, 16, 32, 64, 96])
        return {"op": op, "W": W, "BS": BS, "lo": 0, "hi": _logint(rng, 1, min(32000, 2000000 * BS // W)), "n": n,
                "spare": rng.choice([0, 10, 1000, -5, -500]), "layout": layout}
    dtype = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    E = rng.choice([64, 128, 128, 128, 256])
    Hkv = rng.choice([1, 2, 3, 4, 5, 8])
    Hq = Hkv * rng.choice([1, 2, 4, 5, 8, 16])
    W = _logint(rng, 1, 48)
    BS = rng.choice([1, 6, 8, 16, 16, 32, 64, 96])
    R = rng.choice([0, 32, E // 2, E])
    c = {"op": op, "dtype": dtype, "W": W, "Hq": Hq, "Hkv": Hkv, "E": E, "R": R, "BS": BS, "layout": layout}
    # the cached keys of the whole batch stay under 0.5 GiB a tensor in 32 bits, the scores under 1 GiB
    most = (1 << 29) // (W * Hkv * E * 4)
    if op == "append":
        n = min(_logint(rng, 1, 2048), max(1, most // 2))
        c.update(lo=0, hi=_logint(rng, 1, max(1, min(1024, most - n))), n=n)
    elif op == "attend":
        S = rng.choice([1, 1, 1, _logint(rng, 1, 16)])
        F = rng.choice([1, 1, 2, 3])
        hi = max(1, min(_logint(rng, 1, 60000), most // F, (1 << 28) // (F * W * Hq * S)))
        c.update(F=F, lo=rng.randint(1, hi), hi=hi, S=S)
    else:
        F = rng.choice([1, 1, 2])
        n = min(_logint(rng, 1, 1024), most // (2 * F))
        hi = max(1, min(_logint(rng, 1, 16000), most // F - n, (1 << 27) // (F * W * Hq * n) - n))
        c.update(F=F, lo=rng.randint(1, hi), hi=hi, n=n)
    return c


def _turns(c, extra=0):
    """Keys of turn f cached for sequence w [W, F] (`extra` more in the last turn) and the turns' padded lengths [F]."""
    rs = np.random.RandomState(c["layout"])
    n = rs.randint(c["lo"], c["hi"] + 1, size=c["W"])
    n[0] = c["hi"]
    new = np.zeros(c["W"], int)
    if extra:
        new = rs.randint(1, extra + 1, size=c["W"])
        new[-1] = extra
    cuts = np.sort(rs.randint(0, n[:, None] + 1, size=(c["W"], c["F"] - 1)), axis=1)
    edges = np.concatenate([np.zeros((c["W"], 1), int), cuts, n[:, None]], axis=1)
    tl = np.diff(edges, axis=1)
    tl[:, -1] += new
    return rs, tl, new, tl.max(axis=0)


def _pages(c, rs, positions):
    """A table of distinct pages, in no order, for `positions` logical positions of every sequence."""
    maxb = max(1, -(-int(positions) // c["BS"]))
    return rs.permutation(c["W"] * maxb).reshape(c["W"], maxb)


def _requests(c):
    """Cached and new tokens of every sequence, the table's width and the pages that the new ones need."""
    rs = np.random.RandomState(c["layout"])
    n = rs.randint(c["lo"], c["hi"] + 1, size=c["W"])
    new = rs.randint(1, c["n"] + 1, size=c["W"])
    have, end = -(-n // c["BS"]), -(-(n + new) // c["BS"])
    return rs, n, new, have, end - have, -(-(c["hi"] + c["n"]) // c["BS"])


# ------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------
def _rotary(pos, R):
    i = torch.arange(R // 2, dtype=torch.float64, device=DEV)
    a = torch.as_tensor(pos, device=DEV).double()[..., None] * 10000.0 ** (-2.0 * i / max(R, 1))
    return [torch.cat([t, t], -1).float().contiguous() for t in (a.cos(), a.sin())]


def prepare(case, seed):
    c = case
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def ints(a):
        return torch.as_tensor(np.ascontiguousarray(a), dtype=torch.int32, device=DEV)

    s = {"op": c["op"], "BS": c["BS"]}
    if c["op"] == "pages":
        rs, n, new, have, need, maxb = _requests(c)
        # other inputs from another seed: the pages' order
        order = torch.randperm(int(have.sum() + need.sum() + max(0, c["spare"])), generator=g, device=DEV).int()
        bt = torch.full((c["W"], maxb), -1, dtype=torch.int32, device=DEV)
        there = torch.arange(maxb, device=DEV) < ints(have)[:, None]
        bt[there] = order[:int(have.sum())]
        left = order[int(have.sum()):]
        count = max(0, int(need.sum()) + c["spare"])  # fewer than needed where spare is negative
        s.update(bt=bt, free=left.contiguous(), count=torch.tensor([count], dtype=torch.int32, device=DEV), starts=ints(n), counts=ints(new),
                 granted=torch.empty(c["W"], dtype=torch.int32, device=DEV), slots=torch.empty((c["W"], c["n"]), dtype=torch.int64, device=DEV))
        return s

    T, W, Hq, Hkv, E, BS = TYPES[c["dtype"]], c["W"], c["Hq"], c["Hkv"], c["E"], c["BS"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=T)

    def pool(pages):
        """A cache in 8 bits [pages, BS, Hkv, E] whose scales are as the append sets them."""
        q = torch.randn((pages, BS, Hkv, E), generator=g, device=DEV, dtype=torch.float16).mul_(100).clamp_(-TOP, TOP).to(F8)
        return q, torch.randint(-8, -5, (pages, Hkv), generator=g, device=DEV).float().exp2()

    s["scale"] = 1.0 / math.sqrt(E)
    if c["op"] == "append":
        rs = np.random.RandomState(c["layout"])
        n = rs.randint(c["lo"], c["hi"] + 1, size=W)
        counts = rs.randint(1, c["n"] + 1, size=W)
        counts[0] = c["n"]
        bt = _pages(c, rs, c["hi"] + c["n"])
        s["kc"], s["ks"] = pool(bt.size)
        s["vc"], s["vs"] = pool(bt.size)
        pad = c["n"] - counts  # left padding
        s["cos"], s["sin"] = _rotary(np.maximum(0, n[:, None] + np.arange(c["n"])[None] - pad[:, None]), c["R"])
        s.update(bt=ints(bt), k=normal(W, Hkv, c["n"], E), v=normal(W, Hkv, c["n"], E), positions=ints(n), counts=ints(counts))
        return s
    rs, tl, new, L = _turns(c, c.get("n", 0))
    F, S = c["F"], c.get("S", c.get("n"))
    bt = _pages(c, rs, L.sum())
    s["kc"], s["ks"] = pool(bt.size)
    s["vc"], s["vs"] = pool(bt.size)
    left = tl[:, ::-1].cumsum(axis=1)[:, ::-1]  # keys of turn f and the turns after it
    # query j of the sequence's last S tokens: the last key of each turn that it sees, its place from the turn's start
    back = np.arange(S)[::-1][None]
    loc = np.repeat(tl.T[:, :, None] - 1, S, axis=2)
    loc[-1] -= np.minimum(back, tl[:, -1:]) if not c.get("n") else back
    place = left.T[:, :, None] - 1 - back[None]
    s.update(L=ints(L), bt=ints(bt))
    if c["op"] == "attend":
        s["cos"], s["sin"] = _rotary(place, c["R"])
        s.update(loc=ints(loc), q=normal(W, Hq, S, E))
        return s
    # packed: the last new[w] of the S columns are sequence w's tokens
    live = back[0][None] < new[:, None]  # [W, S]
    cos, sin = _rotary(place[:, live], c["R"])
    s.update(cos=cos[..., :c["R"] // 2].contiguous(), sin=sin[..., :c["R"] // 2].contiguous(), loc=ints(loc[:, live]),
             q=normal(int(new.sum()), Hq, E), cu=ints(np.concatenate([[0], new.cumsum()])), longest=S)
    return s


# ------------------------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------------------------
def run(state):
    return _kernels(state) if own else _plain(state)


def _kernels(s):
    import dvattn_b200 as dv
    if s["op"] == "attend":
        lse = torch.empty(s["q"].shape[:3], dtype=torch.float32, device=s["q"].device)
        out = dv.dvattn_paged_sdpa_q8(s["q"], s["loc"], s["cos"], s["sin"], s["L"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"],
                                      s["scale"], lse=lse)
        return out, lse
    if s["op"] == "prefill":
        lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=s["q"].device)
        out = dv.dvattn_varlen_paged_sdpa_q8(s["q"], s["loc"], s["cos"], s["sin"], s["L"], s["kc"], s["vc"], s["ks"], s["vs"], s["bt"],
                                             s["cu"], None, s["scale"], lse=lse)
        return out, lse
    if s["op"] == "append":
        dv.dvattn_paged_append_q8(s["kc"], s["vc"], s["ks"], s["vs"], s["k"], s["v"], s["cos"], s["sin"], s["bt"], s["positions"],
                                  s["counts"])
        return s["kc"], s["ks"], s["vc"], s["vs"]
    granted = dv.dvattn_assign_pages(s["bt"], s["free"], s["count"], s["starts"], s["counts"], s["BS"], granted=s["granted"],
                                     slots=s["slots"])
    dv.dvattn_release_pages(s["bt"], s["free"], s["count"], s["starts"], s["BS"])
    return granted, s["slots"], s["bt"], s["free"], s["count"]


def _rotate(x, cos, sin):
    """The first R dims turned pairwise (e, e + R/2), in 32 bits, rounded to x's type; the others as they are."""
    R = 2 * cos.shape[-1]
    a, b, rest = x[..., :R // 2].float(), x[..., R // 2:R].float(), x[..., R:]
    lo, hi = (a * cos + -b * sin).to(x.dtype), (b * cos + a * sin).to(x.dtype)
    return torch.cat([lo, hi, rest.expand(lo.shape[:-1] + rest.shape[-1:])], -1)


def _half(t):
    return t[..., :t.shape[-1] // 2]


def _gather(cache, scales, bt, pos):
    """Rows [..., Hkv, E] of the logical positions pos [..., W, n] of every sequence, the values that they stand for."""
    W, BS = bt.shape[0], cache.shape[1]
    w = torch.arange(W, device=bt.device)[:, None]
    page = bt[w, (pos // BS).clamp(max=bt.shape[1] - 1)].long()
    return cache.view(torch.uint8)[page, pos % BS].view(F8).float().mul_(scales[page][..., None])


def _attend(s, q, loc, cos, sin):
    """q [W, Hq, S, E], loc [F, W, S], cos/sin [F, W, S, R / 2] -> out [W, Hq, S, E] and lse [W, Hq, S] in 32 bits."""
    W, Hq, S, E = q.shape
    Hkv, L, bt = s["kc"].shape[2], s["L"].long(), s["bt"]
    q = _rotate(q[None], cos[:, :, None], sin[:, :, None]).float().view(-1, W, Hkv, Hq // Hkv * S, E)
    n = torch.arange(bt.shape[1] * s["BS"], device=L.device)[:int(L.max())]
    pos = ((L.cumsum(0) - L)[:, None, None] + n).expand(-1, W, -1)
    k = _gather(s["kc"], s["ks"], bt, pos)
    sc = (q @ k.permute(0, 1, 3, 4, 2)).mul_(s["scale"])  # [F, W, Hkv, G * S, n]
    del k
    sees = (n <= loc[..., None]) & (n < L[:, None, None, None])
    sees = sees[:, :, None, None].expand(-1, -1, Hkv, Hq // Hkv, -1, -1).flatten(3, 4)
    sc = sc.masked_fill_(~sees, -math.inf).permute(1, 2, 3, 0, 4).flatten(3)
    top = sc.amax(-1, keepdim=True).nan_to_num(neginf=0.0)
    p = sc.sub_(top).exp_()
    l = p.sum(-1, keepdim=True)
    v = _gather(s["vc"], s["vs"], bt, pos).permute(1, 3, 0, 2, 4).flatten(2, 3)
    out = (p @ v / l).masked_fill_(l == 0, 0.0)
    return out.view(W, Hq, S, E), (top + l.log()).view(W, Hq, S)


def _plain(s):
    if s["op"] == "attend":
        out, lse = _attend(s, s["q"], s["loc"], _half(s["cos"]), _half(s["sin"]))
        return out.to(s["q"].dtype), lse
    if s["op"] == "prefill":
        # unpacked: sequence w's tokens in front of S columns
        cu = s["cu"].long()
        j = torch.arange(s["longest"], device=cu.device)
        live = j < (cu[1:] - cu[:-1])[:, None]
        t = (cu[:-1, None] + j).clamp(max=cu[-1] - 1)
        out, lse = _attend(s, s["q"][t].transpose(1, 2), s["loc"][:, t].masked_fill(~live, -1), s["cos"][:, t], s["sin"][:, t])
        return out.transpose(1, 2)[live].to(s["q"].dtype), lse.transpose(1, 2)[live]
    return _plain_append(s) if s["op"] == "append" else _plain_pages(s)


def _plain_append(s):
    W, Hkv, n, E = s["k"].shape
    NB, BS, i = s["kc"].shape[0], s["BS"], torch.arange(n, device=s["k"].device)
    first = n - s["counts"].long()
    live = i >= first[:, None]
    w = torch.arange(W, device=i.device)[:, None].expand(W, n)[live]
    pos = (s["positions"].long()[:, None] + i - first[:, None])[live]
    page, off = s["bt"].long()[w, pos // BS], pos % BS
    # tokens that were in a page before: those in front of the first new one
    began = torch.full((NB,), BS, device=i.device).scatter_reduce_(0, page, off, "amin")
    held = torch.arange(BS, device=i.device) < began[:, None]
    touched = torch.zeros(NB, dtype=torch.bool, device=i.device).index_fill_(0, page, True)
    old = (held & touched[:, None])[..., None, None]

    def write(cache, scales, x):
        x = x.transpose(1, 2)[live].float()  # [tokens, Hkv, E]
        amax = torch.zeros((NB, Hkv), device=x.device).scatter_reduce_(0, page[:, None].expand(-1, Hkv), x.abs().amax(-1), "amax")
        m, e = torch.frexp(amax)  # amax = m 2^e, 0.5 <= m < 1; 448 = 0.875 2^9
        e = torch.where(amax == 0, -60, e - 9 + (m > 0.875)).clamp(min=-60)
        need = ((e + 127).int() << 23).view(torch.float32)  # 2^e, LEAST or more
        new = torch.where((began == 0)[:, None], need, torch.maximum(scales, need))
        new = torch.where(touched[:, None], new, scales)
        again = (cache.float() * scales[:, None, :, None] / new[:, None, :, None]).to(F8)
        bits = torch.where(old, again.view(torch.uint8), cache.view(torch.uint8))
        bits[page, off] = (x / new[page][..., None]).to(F8).view(torch.uint8)
        cache.copy_(bits.view(F8))
        scales.copy_(new)

    write(s["kc"], s["ks"], _rotate(s["k"], _half(s["cos"])[:, None], _half(s["sin"])[:, None]))
    write(s["vc"], s["vs"], s["v"])
    return s["kc"], s["ks"], s["vc"], s["vs"]


def _plain_pages(s):
    bt, free, BS, slots = s["bt"], s["free"], s["BS"], s["slots"]
    W, maxb = bt.shape
    j = torch.arange(maxb, device=bt.device)
    starts, counts, have = s["starts"].long(), s["counts"].long(), s["count"].long()
    ok = starts + counts <= maxb * BS
    need = (j >= (starts // BS)[:, None]) & (j * BS < (starts + counts)[:, None]) & ok[:, None] & (bt < 0)
    per = need.sum(1)
    upto = per.cumsum(0)
    given = ok & ((per == 0) | (upto <= have))
    used = torch.where(upto <= have, upto, 0).amax()
    at = (have - used + need.flatten().cumsum(0).view(W, maxb) - 1).clamp(0, max(0, free.numel() - 1))
    take = need & given[:, None]
    if free.numel():
        bt.copy_(torch.where(take, free[at], bt))
    s["count"].copy_(have - used)
    granted = torch.where(given, s["counts"], 0)
    i = torch.arange(slots.shape[1], device=bt.device)
    p = starts[:, None] + i
    slot = bt.long().gather(1, (p // BS).clamp(max=maxb - 1)) * BS + p % BS
    slots.copy_(torch.where(i < granted[:, None], slot, -1))
    # given back: the pages behind each sequence's start
    back = (j * BS >= starts[:, None]) & (bt >= 0)
    to = (s["count"] + back.flatten().cumsum(0) - 1)[back.flatten()]
    free[to] = bt[back]
    s["count"].add_(back.sum())
    bt.masked_fill_(back, -1)
    return granted, slots, bt, free, s["count"]


# ------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------------------------
def work(case):
    c = case
    W, BS = c["W"], c["BS"]
    if c["op"] == "pages":
        rs, n, new, have, need, maxb = _requests(c)
        # taken and given back: an entry and a free page read, then both written, twice; a slot per token
        return {"bytes": float(16 * need.sum() + 8 * new.sum() + 12 * W), "flops": float(new.sum())}
    es, Hq, Hkv, E, R = SIZE[c["dtype"]], c["Hq"], c["Hkv"], c["E"], c["R"]
    row = Hkv * E  # one token's keys (or values) in 8 bits
    if c["op"] == "append":
        rs = np.random.RandomState(c["layout"])
        rs.randint(c["lo"], c["hi"] + 1, size=W)
        counts = rs.randint(1, c["n"] + 1, size=W)
        counts[0] = c["n"]
        got = int(counts.sum())
        pages = sum(-(-int(x) // BS) for x in counts)
        return {"bytes": got * (2 * row * (es + 1) + 2 * R * 4) + pages * (4 + 16 * Hkv) + 8 * W, "flops": got * Hkv * (3 * R + 2 * E)}
    rs, tl, new, L = _turns(c, c.get("n", 0))
    F, keys = c["F"], int(tl.sum())
    if c["op"] == "attend":
        tokens, pairs = W * c["S"], c["S"] * keys
    else:
        tokens, pairs = int(new.sum()), int((new * tl.sum(axis=1)).sum() - (new * (new - 1) // 2).sum())
    pages = sum(-(-int(t) // BS) for t in tl.sum(axis=1))
    half = R if c["op"] == "attend" else R // 2
    return {"bytes": keys * 2 * row + pages * (4 + 8 * Hkv) + tokens * (Hq * (2 * E * es + 4) + F * (4 + 8 * half)),
            "flops": 4 * Hq * E * pairs}


# ------------------------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------------------
def _turned(x, cos, sin, h):
    """x [..., E] with each pair (x[e], x[e + h]) turned by its angle, rounded to x's type, in 64 bits."""
    y = x.double().clone()
    lo, hi = y[..., :h].clone(), y[..., h:2 * h].clone()
    y[..., :h] = lo * cos[..., :h].double() - hi * sin[..., :h].double()
    y[..., h:2 * h] = hi * cos[..., :h].double() + lo * sin[..., :h].double()
    return y.to(x.dtype).double()


def _exact_append(s):
    bt, pos, cnt = (s[k].cpu().numpy() for k in ("bt", "positions", "counts"))
    W, Hkv, n, E = s["k"].shape
    BS, h = s["BS"], s["cos"].shape[-1] // 2
    got = []
    for x, cache, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
        values, steps = cache.double(), scales.double()
        for w in range(W):
            rows = (_turned(x[w], s["cos"][w], s["sin"][w], h) if x is s["k"] else x[w].double())[:, n - int(cnt[w]):].transpose(0, 1)
            i = 0
            while i < cnt[w]:  # page by page
                p = int(pos[w]) + i
                page, a = int(bt[w, p // BS]), p % BS
                m = min(BS - a, int(cnt[w]) - i)
                top = rows[i:i + m].abs().amax((0, 2)).clamp(min=1e-300)
                step = torch.exp2((top / TOP).log2().ceil()).clamp(min=LEAST)
                if a:
                    step = torch.maximum(step, steps[page])
                    values[page, :a] = (values[page, :a] * (steps[page] / step)[:, None]).float().to(F8).double()
                values[page, a:a + m] = (rows[i:i + m] / step[:, None]).float().to(F8).double()
                steps[page] = step
                i += m
        got += [values, steps]
    return got


def exact(case, seed):
    if case["op"] == "pages":
        return None
    s = prepare(case, seed)
    if s["op"] == "append":
        return _exact_append(s) if int(s["counts"].sum()) < 10000 * s["BS"] else None
    packed = s["op"] == "prefill"
    q = s["q"]
    Hq, E, Hkv, BS = q.shape[1], q.shape[-1], s["kc"].shape[2], s["BS"]
    G, L, bt = Hq // Hkv, s["L"].tolist(), s["bt"].long()
    h = s["cos"].shape[-1] // (1 if packed else 2)
    out = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    lse = torch.full(q.shape[:-1], -math.inf, dtype=torch.float64, device=DEV)
    cu = s["cu"].tolist() if packed else None
    for w in range(bt.shape[0]):
        t = slice(cu[w], cu[w + 1]) if packed else w
        loc = s["loc"][:, t]  # [F, tokens]
        qw = q[t].transpose(0, 1) if packed else q[w]  # [Hq, tokens, E]
        at, first = [], 0
        for f, length in enumerate(L):
            at.append(torch.arange(first, first + max(0, min(length, int(loc[f].max()) + 1)), device=DEV))
            first += length
        for kv in range(Hkv):
            z, vals = [], []
            for f, p in enumerate(at):
                page = bt[w, p // BS]
                k = s["kc"][page, p % BS, kv].double() * s["ks"][page, kv].double()[:, None]
                vals.append(s["vc"][page, p % BS, kv].double() * s["vs"][page, kv].double()[:, None])
                x = s["scale"] * (_turned(qw[kv * G:(kv + 1) * G], s["cos"][f, t], s["sin"][f, t], h) @ k.T)
                z.append(x.masked_fill(torch.arange(len(p), device=DEV) > loc[f][:, None], -math.inf))
            z = torch.cat(z, -1)
            o = (z.softmax(-1) @ torch.cat(vals)).nan_to_num(nan=0.0)  # a token that sees nothing: zeros
            if packed:
                out[t, kv * G:(kv + 1) * G], lse[t, kv * G:(kv + 1) * G] = o.transpose(0, 1), z.logsumexp(-1).T
            else:
                out[w, kv * G:(kv + 1) * G], lse[w, kv * G:(kv + 1) * G] = o, z.logsumexp(-1)
    return out, lse
