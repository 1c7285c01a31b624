"""The draft-tree attention, the accumulated attention weight and the eviction in 64 bits, written
from their definitions key by key and turn by turn, and the error bounds their kernels are
held to."""
import math

import numpy as np
import torch

# unit roundoff of the types: half the distance from 1 to the next number above
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
U32 = 2.0 ** -23  # a 32-bit operation (a tensor core's sum may cut instead of round: twice the unit roundoff)


def rotate(x, cos, sin):
    """x [..., E] T with pairs (e, e + R/2) turned by cos/sin [..., R] (first half), rounded to T, in 64 bits."""
    h = cos.shape[-1] // 2
    y = x.double().clone()
    a, b = x[..., :h].double(), x[..., h:2 * h].double()
    y[..., :h] = a * cos[..., :h].double() - b * sin[..., :h].double()
    y[..., h:2 * h] = b * cos[..., :h].double() + a * sin[..., :h].double()
    return y.to(x.dtype).double()


def ancestors(parents):
    """Sees [S, S] of one tree: token s's ancestors and itself; a token that is not there sees nothing."""
    S = len(parents)
    sees = torch.zeros((S, S), dtype=torch.bool)
    for s in range(S):
        line, c = [], s
        while c >= 0 and -1 <= parents[c] < c:
            line.append(c)
            c = parents[c]
        if c == -1:
            sees[s, line] = True
    return sees


def turns(L, cap):
    """(first position, readable keys) of every turn."""
    out, off = [], 0
    for n in L:
        out.append((off, max(0, min(int(n), cap - off))))
        off += int(n)
    return out


def key_rows(cache, table, first, n, h):
    """Rows [n, E] of KV head h at logical positions first.., pages outside the pool as zeros, in 64 bits."""
    BS = cache.size(1)
    pos = torch.arange(first, first + n)
    page = table[pos // BS].long()
    ok = (page >= 0) & (page < cache.size(0))
    rows = cache[page.clamp(0, max(cache.size(0) - 1, 0)), pos % BS, h].double()
    return torch.where(ok[:, None], rows, torch.zeros((), dtype=torch.float64))


def scores(c, w, h):
    """Per turn (first, [G, S, n] scaled scores with -inf where not seen) of one sequence and KV head."""
    Hkv = c["kc"].size(2)
    G = c["q"].size(1) // Hkv
    cap = c["bt"].size(1) * c["kc"].size(1)
    out = []
    for f, (first, n) in enumerate(turns(c["L"].tolist(), cap)):
        q = rotate(c["q"][w, h * G:(h + 1) * G], c["cos"][f, w], c["sin"][f, w])
        s = c["scale"] * q @ key_rows(c["kc"], c["bt"][w], first, n, h).T
        out.append((first, s.masked_fill(torch.arange(n) > c["loc"][f, w][:, None], -math.inf)))
    return out


def tree(c):
    """(out, lse, weight): out [W,Hq,S,E], lse [W,Hq,S], and per output the softmax-weighted sum of |v|."""
    W, Hq, S, E = c["q"].shape
    Hkv = c["kc"].size(2)
    G = Hq // Hkv
    cap = c["bt"].size(1) * c["kc"].size(1)
    out = torch.zeros((W, Hq, S, E), dtype=torch.float64)
    mag, lse = torch.zeros_like(out), torch.full((W, Hq, S), -math.inf, dtype=torch.float64)
    for w in range(W):
        sees = ancestors(c["parents"][w].tolist())
        there = sees.any(1)
        for h in range(Hkv):
            hs = slice(h * G, (h + 1) * G)
            parts = [s for _, s in scores(c, w, h)]
            q = rotate(c["q"][w, hs], c["cos"][-1, w], c["sin"][-1, w])
            k = rotate(c["dk"][w, h], c["cos"][-1, w], c["sin"][-1, w])
            parts.append((c["scale"] * q @ k.T).masked_fill(~sees, -math.inf))
            z = torch.cat(parts, -1)[:, there]
            v = [key_rows(c["vc"], c["bt"][w], first, n, h) for first, n in turns(c["L"].tolist(), cap)]
            v = torch.cat(v + [c["dv"][w, h].double()])
            p = z.softmax(-1)
            # 0 * NaN: a key that nobody of the sequence sees does not count, whatever lies there
            v = torch.where((p > 0).flatten(0, 1).any(0)[:, None], v, torch.zeros((), dtype=torch.float64))
            out[w, hs, there.nonzero()[:, 0]] = p @ v
            mag[w, hs, there.nonzero()[:, 0]] = p @ v.abs()
            lse[w, hs, there.nonzero()[:, 0]] = z.logsumexp(-1)
    return out, lse, mag


def mass(c):
    """(new mass, the weight added) [W, Hkv, N]."""
    W, Hq, S, E = c["q"].shape
    Hkv = c["kc"].size(2)
    G, N = Hq // Hkv, c["mass"].size(2)
    add = torch.zeros((W, Hkv, N + 1), dtype=torch.float64)
    for w in range(W):
        for h in range(Hkv):
            lse = c["lse"][w, h * G:(h + 1) * G].double()[..., None]
            for first, s in scores(c, w, h):
                p = torch.where(lse == -math.inf, torch.zeros_like(s), (s - lse).exp())
                p = torch.where(s == -math.inf, torch.zeros_like(s), p).sum((0, 1))
                n = min(p.numel(), max(N - first, 0))
                add[w, h, first:first + n] += p[:n]
    return c["mass"].double() + add[..., :N], add[..., :N]


def evict(kc, vc, mass, bt, starts, lengths, keep, sink, recent):
    """(kc, vc, mass_out, source) after the eviction, by sorting."""
    kc, vc, out = kc.clone(), vc.clone(), mass.clone()
    W, Hkv, N = mass.shape
    BS, NB = kc.size(1), kc.size(0)
    source = torch.arange(N, dtype=torch.int32).expand(W, Hkv, N).clone()
    lim = min(N, bt.size(1) * BS)
    for w in range(W):
        st, n, kp = int(starts[w]), int(lengths[w]), max(0, int(keep[w]))
        n = 0 if st < 0 else max(0, min(n, lim - st))
        kept = min(n, kp)
        for h in range(Hkv):
            m = mass[w, h, st:st + n].double().numpy()
            tier = np.where(np.isnan(m), 2, 1)
            i = np.arange(n)
            tier[(i < sink) | (i >= n - recent)] = 0
            value = np.where(tier == 1, -np.nan_to_num(m, nan=0.0, posinf=np.inf, neginf=-np.inf), 0.0)
            stay = np.sort(np.lexsort((i, value, tier))[:kept])
            holes, movers = np.setdiff1d(np.arange(kept), stay), stay[stay >= kept]
            for d, s in zip(holes + st, movers + st):
                out[w, h, d], source[w, h, d] = mass[w, h, s], int(s)
                pd, ps = int(bt[w, d // BS]), int(bt[w, s // BS])
                if 0 <= pd < NB and 0 <= ps < NB:
                    kc[pd, d % BS, h] = kc[ps, s % BS, h]
                    vc[pd, d % BS, h] = vc[ps, s % BS, h]
            out[w, h, st + kept:st + n], source[w, h, st + kept:st + n] = 0, -1
    return kc, vc, out, source


# ---- bounds, from the operations (probabilistic rounding analysis: a sum of n rounded terms is off by a
# small multiple, here 8, of sqrt(n) unit roundoffs of the sum of magnitudes) ----
def score_error(c):
    """Of a scaled score in 32 bits: the dot product of E terms, at most |q| |k| scale in magnitude."""
    E = c["q"].size(-1)
    keys = [c["kc"]] + ([c["dk"]] if "dk" in c else [])
    top = max(float(torch.nan_to_num(k.float(), nan=0.0, posinf=0.0, neginf=0.0).norm(dim=-1).max()) for k in keys if k.numel())
    b = abs(c["scale"]) * float(torch.nan_to_num(c["q"].float()).norm(dim=-1).max()) * top
    return U32 * (8 * math.sqrt(E) + 4) * b


def out_bound(c, out, mag, keys):
    """Rounding of the result and of the weights to T, of the scores and of the sums over the keys in 32 bits."""
    u = UNIT[c["q"].dtype]
    rel = 2 * score_error(c) + U32 * (16 * math.sqrt(keys) + 32)
    pu = 0.0 if c["q"].dtype == torch.float32 else u
    return u * out.abs() + (pu + rel) * mag + 1e-30


def lse_bound(c, lse, keys):
    return score_error(c) + U32 * (8 * math.sqrt(keys) + 16) + 2 * U32 * lse.abs()


def mass_bound(c, new, add):
    rows = c["q"].size(1) // c["kc"].size(2) * c["q"].size(2)
    return (score_error(c) + U32 * (8 * math.sqrt(rows) + 32 + 2 * float(c["lse"][c["lse"].abs() < math.inf].abs().max()))) * add + U32 * new.abs()
