"""The attention over an 8-bit paged cache, the append into one and the page assignment, written from their
definitions in 64 bits (whole numbers: as loops), with the error bounds that the kernels are held to."""
import math

import torch

import plain64

F8 = torch.float8_e4m3fn
LEAST = 2.0 ** -60


def rotate32(x, cos, sin):
    """x [..., E] T with pairs (e, e + h) turned by cos/sin [..., h] as the operators define it: products and sum each
    rounded to 32 bits, the result to T."""
    h = cos.shape[-1]
    y = x.clone()
    a, b = x[..., :h].float(), x[..., h:2 * h].float()
    y[..., :h] = (a * cos + -b * sin).to(x.dtype)
    y[..., h:2 * h] = (b * cos + a * sin).to(x.dtype)
    return y


def quantise(x, pow2=True):
    """x [NB, BS, Hkv, E] in 8 bits with a scale per page and head that its largest finite element just fits (or, pow2, the
    power of two above)."""
    top = torch.nan_to_num(x.float(), nan=0.0, posinf=0.0, neginf=0.0).abs().amax((1, 3)).clamp(min=1e-12)
    s = (top.double() / 448).float()
    if pow2:
        s = torch.exp2(torch.log2(s.double()).ceil()).float()
    return (x.float() / s[:, None, :, None]).clamp(-448, 448).to(F8), s


def values(cache, scales):
    """What a cache in 8 bits stands for, in 64 bits."""
    return cache.double() * scales.double()[:, None, :, None]


def attend(q, loc, cos, sin, L, kc, vc, table, scale):
    """One sequence: q [Hq, S, E], loc [F, S], cos/sin [F, S, h], kc/vc values in 64 bits, table [maxb] ->
    out [Hq, S, E], lse [Hq, S], softmax-weighted sum of |v|, largest |v| seen."""
    Hq, S, E = q.shape
    Hkv = kc.size(2)
    G, cap = Hq // Hkv, table.numel() * kc.size(1)
    out, lse = torch.zeros((Hq, S, E), dtype=torch.float64), torch.full((Hq, S), -math.inf, dtype=torch.float64)
    mag, top = torch.zeros_like(out), 0.0
    for h in range(Hkv):
        hs, z, v = slice(h * G, (h + 1) * G), [], []
        for f, (first, n) in enumerate(plain64.turns([max(0, x) for x in L.tolist()], cap)):
            qr = rotate32(q[hs], cos[f], sin[f]).double()
            s = scale * qr @ plain64.key_rows(kc, table, first, n, h).T
            z.append(s.masked_fill(torch.arange(n) > loc[f][:, None], -math.inf))
            v.append(plain64.key_rows(vc, table, first, n, h))
        if not z:
            continue
        z, v = torch.cat(z, -1), torch.cat(v)
        seen = z > -math.inf
        p = torch.where(seen.any(-1, keepdim=True), z, torch.zeros(())).softmax(-1) * seen
        # 0 * NaN: a key that a query does not see does not count for it, whatever lies there
        weight = torch.where(p[..., None] > 0, p[..., None] * v, torch.zeros((), dtype=torch.float64)) if torch.isnan(v).any() else None
        out[hs] = p @ v if weight is None else weight.sum(2)
        mag[hs] = out[hs].abs() if weight is not None else p @ v.abs()
        lse[hs] = z.logsumexp(-1) if z.size(-1) else lse[hs]
        top = max(top, float(torch.nan_to_num(v).abs().max()) if v.numel() else 0.0)
    return out, lse, mag, top


def paged(c):
    """(out, lse, mag, top) of a call with c["kc"], c["vc"] in 8 bits."""
    k, v, h = values(c["kc"], c["ks"]), values(c["vc"], c["vs"]), c["cos"].shape[-1] // 2
    got = [attend(c["q"][w], c["loc"][:, w], c["cos"][:, w, :, :h], c["sin"][:, w, :, :h], c["L"], k, v, c["bt"][w], c["scale"])
           for w in range(c["q"].size(0))]
    return tuple(torch.stack([g[i] for g in got]) for i in range(3)) + (max(g[3] for g in got),)


def varlen(c):
    """(out [T, Hq, E], lse [T, Hq], mag, top) of a packed call; token t belongs to the first w with t < cu[w + 1], else 0."""
    k, v, cu = values(c["kc"], c["ks"]), values(c["vc"], c["vs"]), c["cu"].tolist()
    T = c["q"].size(0)
    out, mag = torch.zeros(c["q"].shape, dtype=torch.float64), torch.zeros(c["q"].shape, dtype=torch.float64)
    lse, top = torch.zeros(c["q"].shape[:2], dtype=torch.float64), 0.0
    owner = [next((w for w in range(len(cu) - 1) if t < cu[w + 1]), 0) for t in range(T)]
    for w in set(owner):
        t = [i for i in range(T) if owner[i] == w]
        o, l, m, x = attend(c["q"][t].transpose(0, 1), c["loc"][:, t], c["cos"][:, t], c["sin"][:, t], c["L"], k, v, c["bt"][w], c["scale"])
        out[t], lse[t], mag[t], top = o.transpose(0, 1), l.T, m.transpose(0, 1), max(top, x)
    return out, lse, mag, top


def score_error(c):
    """Of a scaled score: the dot product of E terms in 32 bits, at most |q| |k| scale in magnitude; q's elements under 2^-27 of the
    row's largest keep 2^-39 of it, less than the sum's own rounding."""
    k = values(c["kc"], c["ks"])
    top = float(torch.nan_to_num(k).norm(dim=-1).max()) if k.numel() else 0.0
    b = abs(c["scale"]) * float(torch.nan_to_num(c["q"].float()).norm(dim=-1).max()) * top
    return plain64.U32 * (8 * math.sqrt(c["q"].size(-1)) + 4) * b


def out_bound(c, out, mag, top, keys, wide=False):
    """The result's rounding to T; the weights' to f16 (32-bit queries: to a pair, 2^-22) and to nothing under 2^-32 of the largest;
    scores and sums over the keys in 32 bits.  wide: the packed prefill, whose weights and widened values are rounded to T."""
    T = c["q"].dtype
    rel = 2 * score_error(c) + plain64.U32 * (16 * math.sqrt(keys) + 32)
    pu = 2.0 ** -22 if T == torch.float32 else 2 * plain64.UNIT[T] + 2.0 ** -11 if wide else 2.0 ** -11
    return plain64.UNIT[T] * out.abs() + (pu + rel) * mag + keys * 2.0 ** (-24 if wide and T == torch.float16 else -32) * top + 1e-30


def lse_bound(c, lse, keys):
    return score_error(c) + plain64.U32 * (8 * math.sqrt(keys) + 16) + 2 * plain64.U32 * lse.abs()


def append(kc, vc, ks, vs, k, v, cos, sin, bt, positions, counts):
    """The caches and scales after the append, page by page; all that is rounded is rounded as the operator says."""
    W, Hkv, n, E = k.shape
    NB, BS, h = kc.size(0), kc.size(1), cos.shape[-1] // 2
    got = []
    for x, cache, scales, key in ((k, kc, ks, True), (v, vc, vs, False)):
        bits, scales = cache.clone().view(torch.uint8), scales.clone()
        for w in range(W):
            cnt = max(0, min(n, int(counts[w]) if counts is not None else n))
            rows = rotate32(x[w], cos[w, :, :h], sin[w, :, :h]) if key else x[w]
            tokens = {}
            for i in range(cnt):
                p = int(positions[w]) + i
                if 0 <= p < bt.size(1) * BS:
                    tokens.setdefault(p // BS, []).append((p % BS, rows[:, n - cnt + i].float()))
            for j, new in tokens.items():
                page, a = int(bt[w, j]), new[0][0]
                if not 0 <= page < NB:
                    continue
                fresh = torch.stack([r for _, r in new], 1)  # [Hkv, tokens, E]
                top = torch.where(torch.isfinite(fresh), fresh.abs(), torch.zeros(())).amax((1, 2)).double()
                need = torch.exp2(torch.log2(top.clamp(min=1e-300) / 448).ceil()).clamp(min=LEAST).float()
                s = torch.maximum(scales[page], need) if a else need
                if a:
                    grown = s > scales[page]
                    again = (bits[page, :a].view(F8).float() * scales[page][:, None] / s[:, None]).to(F8).view(torch.uint8)
                    bits[page, :a] = torch.where(grown[:, None], again, bits[page, :a])
                q = torch.where(torch.isfinite(fresh), fresh / s[:, None, None], torch.full((), math.nan))
                bits[page, a:a + len(new)] = q.to(F8).view(torch.uint8).transpose(0, 1)
                scales[page] = s
        got += [bits, scales]
    return got


def assign(bt, free, count, starts, counts, BS, n=None):
    """(bt, count, granted, slots) by a loop over the sequences."""
    bt, W, maxb = bt.clone(), bt.size(0), bt.size(1)
    need, bad = [], []
    for w in range(W):
        s, c = int(starts[w]), max(0, int(counts[w]))
        bad.append(s < 0 or s + c > maxb * BS)
        need.append([] if bad[w] or c == 0 else [j for j in range(s // BS, (s + c - 1) // BS + 1) if bt[w, j] < 0])
    have = max(0, min(int(count), free.numel()))
    upto, used, served = 0, 0, []
    for w in range(W):
        upto += len(need[w])
        served.append(not bad[w] and (not need[w] or upto <= have))
        if upto <= have:
            used = upto
    i = 0
    for w in range(W):
        if served[w]:
            for j in need[w]:
                bt[w, j] = free[have - used + i]
                i += 1
    granted = torch.tensor([max(0, int(counts[w])) if served[w] else 0 for w in range(W)], dtype=torch.int32)
    slots = None
    if n is not None:
        slots = torch.full((W, n), -1, dtype=torch.int64)
        for w in range(W):
            for i in range(min(n, int(granted[w]))):
                p = int(starts[w]) + i
                if bt[w, p // BS] >= 0:
                    slots[w, i] = int(bt[w, p // BS]) * BS + p % BS
    return bt, have - used, granted, slots


def release(bt, free, count, keep, BS):
    bt, free, have = bt.clone(), free.clone(), max(0, min(int(count), free.numel()))
    for w in range(bt.size(0)):
        for j in range(max(0, -(-int(keep[w]) // BS)), bt.size(1)):
            if bt[w, j] >= 0 and have < free.numel():
                free[have] = bt[w, j]
                have += 1
                bt[w, j] = -1
    return bt, free, have
