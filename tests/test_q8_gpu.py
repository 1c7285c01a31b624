"""GPU tests of the attention over an 8-bit paged cache, the append into one and the page assignment against
their definitions in 64 bits (plain_q8.py), with bounds derived there from the operations."""
import math

import numpy as np
import pytest
import torch

import dvattn_b200
import plain_q8
from dvattn_b200 import capi
from dvattn_b200 import workloads as wl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
F8 = torch.float8_e4m3fn
TYPES = [F32, F16, BF16]


def make(turn_lens, S, Hq, Hkv, E, R, BS, dtype, seed=0, pow2=True, spread=True, extra_pages=0):
    """Inputs of one call (CPU): the cache of workloads.make_paged in 8 bits, pages of different magnitudes."""
    c = wl.make_paged(turn_lens, Hq, Hkv, E, R, BS, dtype, seed=seed, S=S, extra_pages=extra_pages)
    g = torch.Generator().manual_seed(seed + 1)
    kc, vc = c.k_cache.float(), c.v_cache.float()
    if spread:
        vc = vc * torch.exp2(torch.randint(-6, 7, vc.shape[:1] + (1,) + vc.shape[2:3] + (1,), generator=g).float())
        kc = kc * torch.exp2(torch.randint(-3, 1, kc.shape[:1] + (1,) + kc.shape[2:3] + (1,), generator=g).float())
    (k8, ks), (v8, vs) = plain_q8.quantise(kc, pow2), plain_q8.quantise(vc, pow2)
    return dict(q=c.queries, loc=c.locations, cos=c.cosines, sin=c.sines, L=c.fragment_lengths, kc=k8, vc=v8, ks=ks, vs=vs,
                bt=c.block_tables, scale=c.scale)


def on_gpu(c):
    return {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}


def call(c, out=None, **kw):
    lse = torch.full(c["q"].shape[:3], float("nan"), device=DEV)
    if out is None:
        out = torch.full_like(c["q"], float("nan"))
    dvattn_b200.dvattn_paged_sdpa_q8(c["q"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"],
                                     c["scale"], out=out, lse=lse, **kw)
    return out, lse


def close(c, out, lse, ref, ref_lse, mag, top, what="", wide=False):
    keys = int(c["L"].clamp(min=0).sum())
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(lse == -math.inf, ref_lse == -math.inf), what
    fin = ref_lse > -math.inf
    err, bound = (lse[fin] - ref_lse[fin]).abs(), plain_q8.lse_bound(c, ref_lse[fin], keys)
    assert bool((err <= bound).all()), (what, "lse", float((err / bound).max()))
    err, bound = (out - ref).abs(), plain_q8.out_bound(c, ref, mag, top, keys, wide)
    # a result past the type's largest number is an infinity in that type
    past = (ref.abs() + bound > torch.finfo(c["q"].dtype).max) & (out == torch.where(ref > 0, math.inf, -math.inf))
    assert bool(((err <= bound) | past).all()), (what, "out", float((err / bound)[~past].max()))


def check(c, what=""):
    out, lse = call(on_gpu(c))
    torch.cuda.synchronize()
    close(c, out, lse, *plain_q8.paged(c), what)
    return out, lse


# ---- attention -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_one_sequence(dtype):
    check(make([[100]], 1, 16, 1, 128, 64, 16, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,S", [(16, 1, 1), (8, 8, 1), (15, 3, 7), (32, 2, 3)])
def test_heads_types_dims(dtype, E, Hq, Hkv, S):
    check(make([[70, 33], [1, 260], [0, 5]], S, Hq, Hkv, E, 32, 16, dtype, seed=E + S))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Hkv", [1, 2, 3, 4, 5, 6, 8, 12, 16])
def test_kv_heads(dtype, Hkv):
    check(make([[131, 57]], 1, 4 * Hkv, Hkv, 64 if Hkv > 8 else 128, 32, 16, dtype, seed=Hkv))


@pytest.mark.parametrize("dtype,E", [(F32, 128), (BF16, 64), (F16, 128), (BF16, 256)])
@pytest.mark.parametrize("BS", [1, 3, 8, 24, 48, 64, 96, 128, 256])
def test_page_sizes(dtype, E, BS):
    """Pages that end inside a window, are larger than one, hold a single token, or are no whole boxes."""
    check(make([[131, 200, 17], [300, 1, 0]], 2, 8, 2, E, 64, BS, dtype, seed=BS))


@pytest.mark.parametrize("R", [0, 2, 24, 32, 128])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_rotary_dims(dtype, R):
    check(make([[90, 65]], 2, 8, 2, 128, R, 16, dtype, seed=R))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,G", [(1, 1), (2, 16), (3, 16), (17, 16), (16, 1), (17, 1), (13, 5), (130, 4), (300, 2)])
def test_tokens_by_group(dtype, S, G):
    """Row counts around the tiles (16 and 32 rows), many tiles, tokens that see nothing (S longer than the cache)."""
    check(make([[150], [40]], S, 2 * G, 2, 128, 64, 16, dtype, seed=S + G))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [0, 1, 7, 8, 31, 32, 33, 127, 128, 129, 257, 5000])
def test_context_lengths(dtype, n):
    """Empty caches and lengths around the windows; 5000 keys are split over many blocks."""
    check(make([[n]], 1, 4, 1, 128, 64, 16, dtype, seed=n))
    check(make([[n]], 1, 16, 4, 64, 64, 16, dtype, seed=n))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_sequences(dtype):
    """More sequences than CTAs, ragged, empty ones among them, three turns."""
    rs = np.random.RandomState(5)
    tl = rs.randint(0, 90, size=(700, 3))
    tl[rs.rand(700, 3) < 0.4] = 0
    check(make(tl, 1, 4, 2, 64, 32, 16, dtype))


def test_more_sequences_than_a_launch_takes():
    tl = np.random.RandomState(6).randint(0, 20, size=(4200, 1))
    check(make(tl, 1, 2, 1, 64, 0, 8, BF16))


def test_no_turns_and_no_pages():
    c = on_gpu(make([[20], [30]], 1, 8, 2, 128, 64, 16, BF16))
    e = dict(c, L=c["L"][:0], loc=c["loc"][:0], cos=c["cos"][:0], sin=c["sin"][:0])
    out, lse = call(e)
    assert not out.any() and bool((lse == -math.inf).all())
    e = dict(c, kc=c["kc"][:0], vc=c["vc"][:0], ks=c["ks"][:0], vs=c["vs"][:0])
    out, lse = call(e)
    assert not out.any() and bool((lse == -math.inf).all())
    e = dict(c, bt=c["bt"][:, :0].contiguous())
    out, lse = call(e)
    assert not out.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_any_scales(dtype):
    """Scales that are no powers of two, from 2^-60 to 2^40, keys of different pages deciding the softmax."""
    c = make([[260, 40], [90, 300]], 3, 8, 2, 128, 64, 16, dtype, pow2=False)
    check(c)
    g = torch.Generator().manual_seed(3)
    c["vs"] = c["vs"] * torch.exp2(torch.randint(-50, 40, c["vs"].shape, generator=g).float())
    check(c)


@pytest.mark.parametrize("dtype", TYPES)
def test_zero_values_and_smallest_scales(dtype):
    c = make([[300]], 1, 8, 2, 128, 64, 16, dtype)
    c["vc"] = torch.zeros_like(c["vc"].view(torch.uint8)).view(F8)
    c["vs"][:] = plain_q8.LEAST
    out, lse = check(c)
    assert not out.any()
    c = make([[300]], 1, 8, 2, 128, 64, 16, dtype)
    c["vs"][:] = 0.0  # an empty scale: values of zero
    out, lse = check(c)


@pytest.mark.parametrize("dtype", TYPES)
def test_query_magnitudes(dtype):
    """Rows of very small and large queries: the row's power of two."""
    c = make([[200]], 2, 16, 2, 128, 64, 16, dtype)
    top = {F32: 60, F16: 10, BF16: 60}[dtype]
    e = torch.linspace(-top, top, 16).round()
    c["q"] = (c["q"].float() * torch.exp2(e)[None, :, None, None]).to(dtype)
    c["scale"] = 2.0 ** -top
    check(c)


@pytest.mark.parametrize("dtype", TYPES)
def test_locations(dtype):
    """Locations of any order and sign, beyond the turn, and a query that sees nothing."""
    c = make([[100, 60, 80]], 5, 8, 2, 128, 64, 16, dtype)
    c["loc"][:, 0] = torch.tensor([[-1, 3, 500, 99, -7], [59, -1, 0, 2147483647, -1], [-1, -5, 40, 79, -2147483648]], dtype=torch.int32)
    out, lse = check(c)
    assert not out[0, :, 4].any() and bool((lse[0, :, 4] == -math.inf).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_tables_that_end_early(dtype):
    """Positions behind the table are not seen; pages outside the pool are zeros; fragment lengths below zero are empty."""
    c = make([[100, 60]], 2, 8, 2, 128, 64, 16, dtype)
    check(dict(c, bt=c["bt"][:, :5].contiguous()))
    bt = c["bt"].clone()
    bt[0, 1], bt[0, 3] = -1, c["kc"].size(0) + 3
    check(dict(c, bt=bt))
    c["L"][0] = -4
    check(c)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("BS", [16, 6])
def test_nan_reaches_who_sees_it(dtype, BS):
    """NaN in unseen positions, behind the last key and in keys and values that some tokens see."""
    S = 4
    c = make([[75]], S, 8, 2, 128, 64, BS, dtype, extra_pages=2)
    k, v = c["kc"].view(torch.uint8), c["vc"].view(torch.uint8)
    for t in (k, v):  # behind the last key
        for p in range(75, c["bt"].size(1) * BS):
            t[int(c["bt"][0, p // BS]), p % BS] = 0x7F
    check(c)
    # the last token's own key, which the tokens before it do not see
    page = int(c["bt"][0, 74 // BS])
    v[page, 74 % BS, :, 5] = 0xFF
    ref, _, _, _ = plain_q8.paged(c)
    out, lse = call(on_gpu(c))
    assert torch.equal(torch.isnan(out).cpu(), torch.isnan(ref))
    assert torch.isnan(ref[:, :, -1, 5]).all() and not torch.isnan(ref[:, :, :-1]).any() and not torch.isnan(lse).any()
    k[page, 74 % BS, 0, 7] = 0x7F
    out, lse = call(on_gpu(c))
    assert torch.isnan(out[:, :4, -1]).all() and torch.isnan(lse[:, :4, -1]).all()
    assert not torch.isnan(out[:, :, :-1]).any() and not torch.isnan(lse[:, :, :-1]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_scales_of_unseen_pages_do_not_matter(dtype):
    c = make([[70, 5], [20, 90]], 3, 8, 2, 128, 64, 16, dtype, extra_pages=3)
    used = torch.zeros(c["kc"].size(0), dtype=torch.bool)
    used[c["bt"].flatten().long()] = True
    for s in (c["ks"], c["vs"]):
        s[~used] = float("nan")
    # pages that only hold padding of a turn are in the table, too
    check(c)


def test_optional_outputs_and_repeat():
    c = on_gpu(make([[500, 31], [77, 900], [0, 3]], 2, 32, 4, 128, 64, 16, BF16))
    o32 = torch.full(c["q"].shape, float("nan"), device=DEV)
    out, lse = call(c, out_f32=o32)
    assert torch.equal(out, o32.to(BF16))
    for _ in range(3):  # the order of all sums is fixed
        again, lse2 = call(c)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    only = dvattn_b200.dvattn_paged_sdpa_q8(c["q"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"], c["scale"])
    assert torch.equal(only, out)


def test_unaligned_angles():
    c = on_gpu(make([[150], [40]], 2, 8, 2, 128, 64, 16, BF16))
    ref, _ = call(c)
    for k in ("cos", "sin"):
        buf = torch.empty(c[k].numel() + 1, device=DEV)
        buf[1:] = c[k].flatten()
        c[k] = buf[1:].view(c[k].shape)
    assert torch.equal(call(c)[0], ref)


def test_stream_graph_and_shared_workspace():
    """On another stream; captured twice with one workspace and replayed in order on new queries."""
    c = on_gpu(make([[300, 40], [77, 200]], 1, 32, 4, 128, 64, 16, F16))
    ref, ref_lse = call(c)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        out, _ = call(c)
    s.synchronize()
    assert torch.equal(out, ref)
    d = dict(c, q=c["q"].flip(1).contiguous())
    want, _ = call(d)
    outs = [torch.zeros_like(ref), torch.zeros_like(ref)]
    lse = torch.zeros_like(ref_lse)
    ws = capi.paged_sdpa_q8(outs[0], c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"], lse=lse)
    graphs = []
    for x, o in zip((c, d), outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            capi.paged_sdpa_q8(o, x["scale"], x["loc"], x["q"], x["cos"], x["sin"], x["L"], x["kc"], x["vc"], x["ks"], x["vs"], x["bt"], workspace=ws)
        graphs.append(g)
    for _ in range(3):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref) and torch.equal(outs[1], want)
    assert capi.workspace_status(ws) == 0


# ---- packed prefill ------------------------------------------------------------------------------------------
def make_varlen(ctx, new, Hq, Hkv, E, R, BS, dtype, seed=0, extra_pages=0):
    """Sequence w: ctx[w] = keys of every turn, new[w] tokens that are the last ones of the last turn."""
    ctx, new = np.asarray(ctx), np.asarray(new)
    tl = ctx.copy()
    tl[:, -1] += new
    c = make(tl, 1, Hq, Hkv, E, R, BS, dtype, seed=seed, extra_pages=extra_pages)
    F, T = tl.shape[1], int(new.sum())
    loc = np.zeros((F, T), np.int32)
    pos = np.zeros((F, T), np.int64)
    t = 0
    for w in range(len(new)):
        for j in range(new[w]):
            back = new[w] - 1 - j
            loc[:, t] = tl[w] - 1
            loc[-1, t] -= back
            pos[:, t] = tl[w, ::-1].cumsum()[::-1] - 1 - back
            t += 1
    cos, sin = wl.rope_angles(torch.from_numpy(pos), R)
    g = torch.Generator().manual_seed(seed + 7)
    return dict(c, q=torch.randn((T, Hq, E), generator=g).to(dtype), loc=torch.from_numpy(loc), cos=cos[..., :R // 2].contiguous(),
                sin=sin[..., :R // 2].contiguous(), cu=torch.tensor([0] + new.cumsum().tolist(), dtype=torch.int32))


def call_varlen(c):
    lse = torch.full(c["q"].shape[:2], float("nan"), device=DEV)
    out = torch.full_like(c["q"], float("nan"))
    dvattn_b200.dvattn_varlen_paged_sdpa_q8(c["q"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"],
                                            c["cu"], None, c["scale"], out=out, lse=lse)
    return out, lse


def check_varlen(c):
    out, lse = call_varlen(on_gpu(c))
    torch.cuda.synchronize()
    close(c, out, lse, *plain_q8.varlen(c), wide=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,BS", [(64, 16), (128, 16), (128, 6), (256, 64)])
def test_varlen(dtype, E, BS):
    check_varlen(make_varlen([[50, 9], [0, 0], [120, 40]], [3, 1, 20], 8, 2, E, 32, BS, dtype, seed=E))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_varlen_on_the_tensor_core_prefill(dtype):
    """Enough tokens for the 16-bit prefill kernel (148 work items of 16 tokens)."""
    check_varlen(make_varlen([[60], [0], [130]], [700, 300, 260], 32, 2, 128, 32, 16, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_varlen_tables(dtype):
    """A pool larger than the batch's tables (the widened pages have a table of their own), pages outside the pool, a token behind
    the last sequence (the first one's, as in the 16-bit call) and an empty sequence."""
    c = make_varlen([[50, 9], [30, 11], [120, 40]], [3, 2, 9], 8, 2, 128, 32, 16, dtype, extra_pages=70)
    check_varlen(c)
    c["bt"][2, 1], c["bt"][0, 0] = -1, c["kc"].size(0)
    check_varlen(c)
    c["cu"] = torch.tensor([0, 3, 3, 13], dtype=torch.int32)
    check_varlen(c)


def test_varlen_stale_workspace_and_graph():
    """The workspace's content from other calls does not matter; a captured call follows new cache contents."""
    c = on_gpu(make_varlen([[50], [30]], [8, 5], 8, 2, 128, 32, 16, BF16))
    ref, _ = call_varlen(c)
    a = capi.varlen_args(ref, c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"], c["cu"])
    n = capi.lib().dvattn_varlen_paged_sdpa_q8_workspace_size(a)
    ws = torch.full((n,), 0x7F, dtype=torch.uint8, device=DEV)
    out = torch.zeros_like(ref)

    def go():
        capi.varlen_paged_sdpa_q8(out, c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"], c["cu"],
                                  workspace=ws)
    go()
    assert torch.equal(out, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
    c["vs"].mul_(2.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call_varlen(c)[0]) and not torch.equal(out, ref)


# ---- append --------------------------------------------------------------------------------------------------
def make_append(W, Hkv, n, E, R, BS, dtype, positions, maxb, seed=0, magnitude=0.0):
    g = torch.Generator().manual_seed(seed)
    NB = W * maxb + 2
    mag = torch.exp2(magnitude * torch.randn((W, Hkv, n, 1), generator=g))
    k, v = (torch.randn((W, Hkv, n, E), generator=g) * mag).to(dtype), (torch.randn((W, Hkv, n, E), generator=g) * mag).to(dtype)
    pos = torch.tensor(positions, dtype=torch.int32)
    cos, sin = wl.rope_angles(pos.long()[:, None] + torch.arange(n)[None], R)
    old = [torch.randint(0, 256, (NB, BS, Hkv, E), generator=g, dtype=torch.uint8) for _ in range(2)]
    for o in old:
        o[(o & 0x7F) == 0x7F] = 0
    scales = [torch.exp2(torch.randint(-9, -4, (NB, Hkv), generator=g).float()) for _ in range(2)]
    bt = torch.randperm(NB, generator=g)[:W * maxb].view(W, maxb).int()
    return dict(kc=old[0].view(F8), vc=old[1].view(F8), ks=scales[0], vs=scales[1], k=k, v=v, cos=cos, sin=sin, bt=bt, positions=pos)


def run_append(c, counts=None):
    d = on_gpu(c)
    dvattn_b200.dvattn_paged_append_q8(d["kc"], d["vc"], d["ks"], d["vs"], d["k"], d["v"], d["cos"], d["sin"], d["bt"], d["positions"],
                                       None if counts is None else counts.to(DEV))
    torch.cuda.synchronize()
    return d["kc"].view(torch.uint8).cpu(), d["ks"].cpu(), d["vc"].view(torch.uint8).cpu(), d["vs"].cpu()


def same_bytes(a, b):
    """Equal; zeros of either sign and NaN of either sign are one value."""
    a, b = [torch.where((x & 0x7F) == 0, 0, torch.where((x & 0x7F) == 0x7F, 0x7F, x.int())) for x in (a, b)]
    return torch.equal(a, b)


def check_append(c, counts=None):
    got = run_append(c, counts)
    ref = plain_q8.append(c["kc"], c["vc"], c["ks"], c["vs"], c["k"], c["v"], c["cos"], c["sin"], c["bt"], c["positions"], counts)
    for i, name in enumerate(("k", "k scales", "v", "v scales")):
        ok = torch.equal(got[i], ref[i]) if i & 1 else same_bytes(got[i], ref[i])
        assert ok, (name, int((got[i] != ref[i]).sum()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,BS", [(1, 16), (5, 16), (40, 16), (40, 1), (40, 3), (130, 64), (300, 128)])
@pytest.mark.parametrize("E,R", [(64, 32), (128, 128), (256, 24)])
def test_append(dtype, n, BS, E, R):
    maxb = -(-(n + 40) // BS)
    check_append(make_append(3, 2, n, E, R, BS, dtype, [0, 7, 33], maxb, seed=n + E, magnitude=2.0))


@pytest.mark.parametrize("dtype", TYPES)
def test_append_counts_and_bad_pages(dtype):
    """Left padding, counts of none, of more than there are and below zero, positions before the first and behind the table, pages
    outside the pool."""
    c = make_append(7, 3, 9, 64, 16, 16, dtype, [0, 12, 30, -3, 2147483640, 5, 44], 3, magnitude=3.0)
    c["bt"][5, 0] = -2
    c["bt"][6, 2] = c["kc"].size(0)
    check_append(c, torch.tensor([9, 4, 20, 8, 9, 9, 9], dtype=torch.int32))
    check_append(c, torch.tensor([0, -1, 1, 9, 0, 9, 2], dtype=torch.int32))
    check_append(c)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_special_values(dtype):
    """NaN and infinities of a page leave the other elements alone; zeros; the largest and smallest numbers; ties."""
    c = make_append(2, 2, 20, 64, 0, 16, dtype, [0, 5], 3)
    c["k"][0, 0, 3, 7], c["k"][1, 1, 2, 9], c["v"][0, 1, 17, 0] = float("nan"), float("inf"), -float("inf")
    c["v"][1, 0] = 0.0
    c["v"][0, 0, :16] = torch.finfo(dtype).max
    c["v"][1, 1, :, ::2] = torch.finfo(dtype).tiny
    c["k"][1, 0, :, :] = torch.linspace(-448, 448, 64)[None].to(dtype)  # borders between values
    check_append(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_append_scale_borders(dtype):
    """The largest element exactly 448 times a power of two, and the next above."""
    c = make_append(4, 1, 1, 64, 0, 16, dtype, [0, 0, 0, 0], 1)
    up = {F32: 448 * (1 + 2.0 ** -22), BF16: 450.0}[dtype]
    for w, x in enumerate((448.0, up, 448.0 * 2.0 ** -9, 3.5)):
        c["v"][w] = c["v"][w].clamp(-x, x)
        c["v"][w, 0, 0, 11] = x
    check_append(c)
    got = run_append(c)
    assert [float(got[3][int(c["bt"][w, 0]), 0]) for w in range(4)] == [1.0, 2.0, 2.0 ** -9, 2.0 ** -7]


@pytest.mark.parametrize("dtype", [F32, F16])
def test_append_scales_of_others(dtype):
    """Pages begun with scales that are no powers of two, are larger than needed, or are zero."""
    c = make_append(3, 2, 6, 64, 32, 16, dtype, [4, 9, 15], 2)
    c["ks"] *= 1.37
    c["vs"] *= 0.61
    c["vs"][int(c["bt"][0, 0])] = 0.0
    c["ks"][int(c["bt"][1, 0])] = 77.7
    check_append(c)


def test_append_step_by_step_equals_the_values():
    """Tokens appended one by one: every stored value is within e4m3's half step (2^-4 of it, or half the smallest step) of the key, each
    growth of the scale adding nothing but the smallest step's."""
    g = torch.Generator().manual_seed(1)
    Hkv, E, BS, n = 2, 128, 16, 50
    k = torch.randn((1, Hkv, n, E), generator=g) * torch.exp2(torch.arange(n).float() / 8)[None, None, :, None]
    kc = torch.zeros((4, BS, Hkv, E), device=DEV).to(F8)
    vc, ks, vs = kc.clone(), torch.zeros((4, Hkv), device=DEV), torch.zeros((4, Hkv), device=DEV)
    bt = torch.tensor([[2, 0, 3, 1]], dtype=torch.int32, device=DEV)
    none = torch.zeros((1, 1, 0), device=DEV)
    for i in range(n):
        x = k[:, :, i:i + 1].contiguous().to(DEV)
        dvattn_b200.dvattn_paged_append_q8(kc, vc, ks, vs, x, x, none, none, bt, torch.tensor([i], dtype=torch.int32, device=DEV))
    got = plain_q8.values(kc.cpu(), ks.cpu())
    for i in range(n):
        page = int(bt[0, i // BS])
        x, s = k[0, :, i].double(), ks[page].double().cpu()[:, None]
        # rounding to a normal value, and to a multiple of the final and of each smaller scale's smallest step 2^-9
        assert bool(((got[page, i % BS] - x).abs() <= 2.0 ** -4 * x.abs() + 2 * 2.0 ** -10 * s).all())


# ---- pages ---------------------------------------------------------------------------------------------------
def run_pages(bt, free, count, starts, counts, BS, n, size=None):
    dev = [t.to(DEV) for t in (bt, free, torch.tensor([count], dtype=torch.int32), starts, counts)]
    slots = None if n is None else torch.full((bt.size(0), n), -9, dtype=torch.int64, device=DEV)
    granted = dvattn_b200.dvattn_assign_pages(*dev, BS, slots=slots)
    torch.cuda.synchronize()
    return dev[0].cpu(), int(dev[2]), granted.cpu(), None if slots is None else slots.cpu(), dev


@pytest.mark.parametrize("W,BS,maxb,longest", [(1, 16, 8, 100), (3, 1, 50, 40), (40, 16, 30, 300), (300, 8, 12, 60), (1000, 16, 6, 1), (5, 96, 40, 3500)])
@pytest.mark.parametrize("spare", [5, 0, -1, -40])
def test_pages(W, BS, maxb, longest, spare):
    """Requests of every length, tables with pages in the middle, too few pages, ones that pass the table; then back again."""
    rs = np.random.RandomState(W + BS)
    starts = rs.randint(0, maxb * BS, size=W)
    counts = rs.randint(0, longest + 1, size=W)
    starts[0], counts[0] = 0, min(longest, maxb * BS)
    if W > 2:
        starts[2], counts[1] = -3, -2
    bt = torch.full((W, maxb), -1, dtype=torch.int32)
    ids = iter(rs.permutation(100000).tolist())
    for w in range(W):
        for j in range(maxb):
            if j * BS < starts[w] or rs.rand() < 0.1:
                bt[w, j] = next(ids)
    starts, counts = torch.tensor(starts, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)
    needed = plain_q8.assign(bt, torch.zeros(10 ** 6, dtype=torch.int32), 10 ** 6, starts, counts, BS)[1]
    count = max(0, 10 ** 6 - needed + spare)
    free = torch.tensor([next(ids) for _ in range(min(count + 3, 60000))], dtype=torch.int32)
    count = min(count, free.numel())
    n = longest + 2 if W < 500 else None
    got = run_pages(bt, free, count, starts, counts, BS, n)
    ref = plain_q8.assign(bt, free, count, starts, counts, BS, n)
    assert torch.equal(got[0], ref[0]) and got[1] == ref[1] and torch.equal(got[2], ref[2])
    assert n is None or torch.equal(got[3], ref[3])
    keep = torch.tensor(rs.randint(-2, maxb * BS + 9, size=W), dtype=torch.int32)
    dbt, dfree, dcount = got[4][0], got[4][1], got[4][2]
    dvattn_b200.dvattn_release_pages(dbt, dfree, dcount, keep.to(DEV), BS)
    back = plain_q8.release(ref[0], free, ref[1], keep, BS)
    assert torch.equal(dbt.cpu(), back[0]) and torch.equal(dfree.cpu(), back[1]) and int(dcount) == back[2]


def test_pages_long_slot_map():
    """A slot map that a launch of its own writes."""
    W, BS, maxb = 20, 16, 300
    starts, counts = torch.arange(W, dtype=torch.int32) * 7, torch.full((W,), 4000, dtype=torch.int32)
    bt = torch.full((W, maxb), -1, dtype=torch.int32)
    bt[:, 0] = torch.arange(W, dtype=torch.int32)
    free = torch.arange(100, 100 + 250 * 18, dtype=torch.int32)  # not enough for the last ones
    got = run_pages(bt, free, free.numel(), starts, counts, BS, 4001)
    ref = plain_q8.assign(bt, free, free.numel(), starts, counts, BS, 4001)
    assert torch.equal(got[0], ref[0]) and got[1] == ref[1] and torch.equal(got[2], ref[2]) and torch.equal(got[3], ref[3])
    assert 0 < int((got[2] == 0).sum()) < W


def test_pages_in_a_graph():
    """Captured once: replays take the next pages of the stack, as requests grow."""
    W, BS = 4, 16
    bt = torch.full((W, 10), -1, dtype=torch.int32, device=DEV)
    free, count = torch.arange(39, -1, -1, dtype=torch.int32, device=DEV), torch.tensor([40], dtype=torch.int32, device=DEV)
    lens, one = torch.zeros(W, dtype=torch.int32, device=DEV), torch.ones(W, dtype=torch.int32, device=DEV)
    granted, slots = torch.empty_like(lens), torch.empty((W, 1), dtype=torch.int64, device=DEV)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        dvattn_b200.dvattn_assign_pages(bt, free, count, lens, one, BS, granted=granted, slots=slots)
        lens += granted
    for step in range(40):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(granted, one)
        page = bt.cpu()[:, step // BS].long()
        assert torch.equal(slots.cpu()[:, 0], page * BS + step % BS)
    assert int(count) == 40 - W * 3 and sorted(bt[bt >= 0].tolist()) == list(range(12))


# ---- together ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_serving_loop(dtype):
    """Pages assigned, prompts appended and prefilled, tokens appended and attended to, pages given back: the attention over the 8-bit
    cache follows the attention over the unrounded keys within e4m3's rounding, and exactly that over the values kept."""
    W, Hq, Hkv, E, R, BS, maxb = 3, 8, 2, 128, 64, 16, 8
    g = torch.Generator().manual_seed(2)
    NB = W * maxb
    i32 = dict(dtype=torch.int32, device=DEV)
    bt, free, count = torch.full((W, maxb), -1, **i32), torch.randperm(NB, generator=g).int().to(DEV), torch.tensor([NB], **i32)
    kc = torch.zeros((NB, BS, Hkv, E), device=DEV).to(F8)
    vc, ks, vs = kc.clone(), torch.zeros((NB, Hkv), device=DEV), torch.zeros((NB, Hkv), device=DEV)
    lens = torch.zeros(W, **i32)
    scale = 1 / math.sqrt(E)
    n = [37, 5, 60]

    def angles(pos):
        return [t.to(DEV) for t in wl.rope_angles(pos, R)]

    # prompts, left-padded
    N = max(n)
    k, v = [torch.randn((W, Hkv, N, E), generator=g).to(dtype).to(DEV) for _ in range(2)]
    counts = torch.tensor(n, **i32)
    granted = dvattn_b200.dvattn_assign_pages(bt, free, count, lens, counts, BS)
    assert granted.tolist() == n
    pos = torch.arange(N)[None] - (N - torch.tensor(n))[:, None]
    dvattn_b200.dvattn_paged_append_q8(kc, vc, ks, vs, k, v, *angles(pos.clamp(min=0)), bt, lens, granted)
    lens += granted
    live = pos >= 0
    q = torch.randn((sum(n), Hq, E), generator=g).to(dtype)
    cos, sin = [t[None].contiguous() for t in angles(pos[live])]
    c = dict(q=q, loc=pos[live][None].int(), cos=cos.cpu()[..., :R // 2].contiguous(), sin=sin.cpu()[..., :R // 2].contiguous(),
             L=torch.tensor([N], dtype=torch.int32), kc=kc.cpu(), vc=vc.cpu(), ks=ks.cpu(), vs=vs.cpu(), bt=bt.cpu(), scale=scale,
             cu=torch.tensor([0] + np.cumsum(n).tolist(), dtype=torch.int32))
    check_varlen(c)
    # ten tokens each
    for step in range(10):
        granted = dvattn_b200.dvattn_assign_pages(bt, free, count, lens, torch.ones(W, **i32), BS)
        assert granted.tolist() == [1] * W
        k, v = [torch.randn((W, Hkv, 1, E), generator=g).to(dtype).to(DEV) for _ in range(2)]
        cos, sin = angles(lens.cpu().long()[:, None])
        dvattn_b200.dvattn_paged_append_q8(kc, vc, ks, vs, k, v, cos, sin, bt, lens, granted)
        lens += granted
        c = dict(q=torch.randn((W, Hq, 1, E), generator=g).to(dtype), loc=(lens - 1).cpu().view(1, W, 1), cos=cos[None].cpu(), sin=sin[None].cpu(),
                 L=lens.max().view(1).cpu(), kc=kc.cpu(), vc=vc.cpu(), ks=ks.cpu(), vs=vs.cpu(), bt=bt.cpu(), scale=scale)
        check(c)
    used = sum(-(-(x + 10) // BS) for x in n)
    assert int(count) == NB - used
    dvattn_b200.dvattn_release_pages(bt, free, count, torch.tensor([0, 15, 33], **i32), BS)
    kept = 0 + 1 + 3
    assert int(count) == NB - kept and int((bt >= 0).sum()) == kept
    assert sorted(free[:NB - kept].tolist() + bt[bt >= 0].tolist()) == list(range(NB))
