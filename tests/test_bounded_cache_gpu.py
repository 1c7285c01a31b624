"""GPU tests of the accumulated attention weight (dvattn_paged_mass) and the eviction by it
(dvattn_paged_evict) against their definitions in 64 bits (plain64.py)."""
import math

import numpy as np
import pytest
import torch

import dvattn_b200
import plain64
from dvattn_b200 import capi
from dvattn_b200 import workloads as wl

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


# ---- accumulated weight -----------------------------------------------------------------------------------
def make(turn_lens, S, Hq, Hkv, E, R, BS, dtype, seed=0, N=None):
    c = wl.make_paged(turn_lens, Hq, Hkv, E, R, BS, dtype, seed=seed, S=S)
    W = len(turn_lens)
    g = torch.Generator().manual_seed(seed)
    c = dict(q=c.queries, loc=c.locations, cos=c.cosines, sin=c.sines, L=c.fragment_lengths, kc=c.k_cache, bt=c.block_tables, scale=c.scale)
    c["mass"] = torch.rand((W, Hkv, c["bt"].size(1) * BS if N is None else N), generator=g)
    lse = []
    for w in range(W):
        for h in range(Hkv):
            lse.append(torch.cat([s for _, s in plain64.scores(c, w, h)], -1).logsumexp(-1))
    c["lse"] = torch.stack(lse).reshape(W, Hq, S).float()
    return c


def add_mass(c, mass=None):
    mass = c["mass"].to(DEV) if mass is None else mass
    g = [c[k].to(DEV) for k in ("q", "lse", "loc", "cos", "sin", "L", "kc", "bt")]
    got = dvattn_b200.dvattn_paged_mass(mass, *g, c["scale"])
    assert got.data_ptr() == mass.data_ptr()
    return mass


def check(c, what=""):
    got = add_mass(c).double().cpu()
    ref, add = plain64.mass(c)
    untouched = add == 0
    assert torch.equal(got[untouched], c["mass"].double()[untouched]), what
    err, bound = (got - ref).abs(), plain64.mass_bound(c, ref, add)
    assert bool((err <= bound).all()), (what, float((err / bound.clamp(min=1e-300)).max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,S", [(16, 1, 1), (8, 8, 1), (15, 3, 7), (32, 2, 33)])
def test_mass_heads_types_dims(dtype, E, Hq, Hkv, S):
    check(make([[70, 133], [1, 260], [10, 55]], S, Hq, Hkv, E, 32, 16, dtype, seed=E + S))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("BS", [1, 3, 48, 64, 96, 256])
def test_mass_page_sizes(dtype, BS):
    check(make([[131, 200, 17], [300, 1, 40]], 2, 8, 2, 128, 64, BS, dtype, seed=BS))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,G", [(1, 1), (8, 16), (9, 16), (31, 16), (33, 16), (70, 16), (257, 2), (600, 1)])
def test_mass_rows(dtype, S, G):
    """Row counts around the tiles; several turns' worth of queries."""
    check(make([[700], [601]], S, 2 * G, 2, 128, 64, 16, dtype, seed=S))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 31, 32, 33, 127, 128, 129, 4099])
def test_mass_lengths(dtype, n):
    check(make([[n]], 1, 4, 1, 128, 64, 16, dtype, seed=n))


@pytest.mark.parametrize("dtype", TYPES)
def test_mass_masks(dtype):
    """Queries that saw nothing, were taken out (lse -inf, with NaN in their rows), locations by query,
    NaN in keys that nobody sees, pages outside the pool, fewer mass positions than cached ones."""
    c = make([[200, 40], [77, 64]], 6, 8, 2, 128, 64, 16, dtype, seed=3)
    c["loc"][:, 0, 1] = -1
    c["lse"][0, :, 1] = -math.inf
    c["lse"][1, :, 2] = -math.inf
    c["q"][1, :, 2] = float("nan")
    c["loc"][0, 0, 3] = 2 ** 31 - 1
    c["loc"][0, 0, 4] = 100
    check(c)
    # positions 80..95 of turn 0, which sequence 1 does not reach, in a page of their own
    c["loc"][0, 1] = 76
    c["kc"] = torch.cat([c["kc"], torch.full_like(c["kc"][:1], float("nan"))])
    c["bt"][1, 5] = c["kc"].size(0) - 1
    c["bt"][0, 1] = -1
    c["bt"][0, 2] = c["kc"].size(0)
    check(c, "pages")
    c["mass"] = c["mass"][:, :, :37].contiguous()
    check(c, "few positions")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [64, 256])
@pytest.mark.parametrize("S,G", [(3, 5), (40, 16)])
def test_mass_of_keys_that_are_not_finite(dtype, E, S, G):
    """Next to queries that give no weight (taken out, or the padding of a row tile): a key with -inf where every
    counted query is positive weighs nothing, a key with NaN gets NaN, and no other key does."""
    c = make([[700]], S, G, 1, E, 0, 16, dtype, seed=E + S)
    c["q"][..., 1] = 0.5 + c["q"][..., 1].abs().clamp(max=2)
    rows = c["bt"][0].long()
    for p in (5, 300, 640):
        c["kc"][rows[p // 16], p % 16, 0, 1] = -math.inf
    finite = torch.ones(c["mass"].shape, dtype=torch.bool)
    lse = torch.cat([s for _, s in plain64.scores(c, 0, 0)], -1).logsumexp(-1)
    c["lse"] = lse.reshape(1, G, S).float()
    c["lse"][:, :, 1] = -math.inf
    check(c)
    c["kc"][rows[20], 3, 0, 2] = math.nan
    finite[:, :, 20 * 16 + 3] = False
    got = add_mass(c).double().cpu()
    assert torch.equal(torch.isfinite(got), finite) and bool(torch.isnan(got[~finite]).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("BS", [65536, 65537])
def test_mass_of_as_many_positions_as_there_are(dtype, BS):
    """A turn of 2^31 - 1 keys, one page under all of them; the mass holds the first ones."""
    n, E, N = 2 ** 31 - 1, 64, 70000
    g = torch.Generator().manual_seed(17)
    kc = torch.randn((1, BS, 1, E), generator=g).to(dtype)
    q = torch.randn((1, 2, 1, E), generator=g).to(dtype)
    none = torch.zeros((1, 1, 1, 0))
    c = dict(q=q, loc=torch.full((1, 1, 1), n, dtype=torch.int32), cos=none, sin=none, L=torch.tensor([n], dtype=torch.int32), kc=kc,
             bt=torch.zeros((1, 32769), dtype=torch.int32), scale=0.125, mass=torch.rand((1, 1, N), generator=g), lse=torch.full((1, 2, 1), 3.0))
    got = add_mass(c).double().cpu()
    add = (0.125 * q[0, :, 0].double() @ kc[0, :, 0].double().T - 3.0).exp().sum(0)
    add = torch.cat([add, add])[:N][None, None]
    ref = c["mass"].double() + add
    assert bool(((got - ref).abs() <= plain64.mass_bound(c, ref, add)).all())


def test_mass_repeats_streams_and_c_abi():
    c = make([[3000, 20], [40, 700]], 9, 8, 2, 128, 64, 16, BF16, seed=9)
    a, b = add_mass(c), add_mass(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        d = add_mass(c)
    side.synchronize()
    m = c["mass"].to(DEV)
    g = {k: c[k].to(DEV) for k in ("q", "lse", "loc", "cos", "sin", "L", "kc", "bt")}
    ws = capi.paged_mass(m, c["scale"], g["loc"], g["q"], g["lse"], g["cos"], g["sin"], g["L"], g["kc"], g["bt"])
    assert capi.workspace_status(ws) == 0
    assert torch.equal(a, b) and torch.equal(a, d) and torch.equal(a, m)


@pytest.mark.parametrize("E", [64, 128, 256])
@pytest.mark.parametrize("S", [5, 8, 9, 17, 33, 35, 67])
def test_mass_repeats_with_row_passes(E, S):
    """Rows of one and several passes, with an odd number of row tiles: a key's sum has one order."""
    c = make([[2500, 1100], [40, 1700]], S, 16, 1, E, 64, 16, F16, seed=S)
    a = add_mass(c)
    assert all(torch.equal(a, add_mass(c)) for _ in range(3))
    check(c)


def test_mass_of_a_decode_sums_to_the_queries():
    """With the lse of the attention call itself, the weights of every query add up to one."""
    c = wl.make_paged([[500, 77], [64, 300]], 32, 2, 128, 64, 16, BF16, seed=4, device=DEV)
    lse = torch.empty((2, 32, 1), device=DEV)
    dvattn_b200.dvattn_paged_sdpa(c.queries, c.locations, c.cosines, c.sines, c.fragment_lengths, c.k_cache, c.v_cache,
                                  c.block_tables, c.scale, lse=lse)
    m = torch.zeros((2, 2, c.block_tables.size(1) * 16), device=DEV)
    dvattn_b200.dvattn_paged_mass(m, c.queries, lse, c.locations, c.cosines, c.sines, c.fragment_lengths, c.k_cache,
                                  c.block_tables, c.scale)
    # 16 queries per key head; both calls' scores and sums are within 1e-4 of exact (the lse tolerance)
    assert bool(((m.sum(-1) - 16).abs() <= 16 * 2e-4).all())


# ---- eviction ---------------------------------------------------------------------------------------------
def pool(W, positions, Hkv, E, BS, dtype, seed=0):
    rs = np.random.RandomState(seed)
    maxb = -(-positions // BS)
    g = torch.Generator().manual_seed(seed)
    kc, vc = (torch.randn((W * maxb, BS, Hkv, E), generator=g).to(dtype) for _ in range(2))
    return kc, vc, torch.from_numpy(rs.permutation(W * maxb).reshape(W, maxb).astype(np.int32)), g


def evict_both(kc, vc, mass, bt, starts, lengths, keep, sink=0, recent=0, in_place=False):
    i32 = lambda x: torch.as_tensor(x, dtype=torch.int32)  # noqa: E731
    starts, lengths, keep = i32(starts), i32(lengths), i32(keep)
    ref = plain64.evict(kc, vc, mass, bt, starts, lengths, keep, sink, recent)
    k, v, m = kc.to(DEV), vc.to(DEV), mass.to(DEV)
    src = torch.full(mass.shape, 77, dtype=torch.int32, device=DEV)
    mout = m if in_place else torch.full_like(m, 5)
    out = dvattn_b200.dvattn_paged_evict(k, v, m, bt.to(DEV), starts.to(DEV), lengths.to(DEV), keep.to(DEV), sink, recent,
                                         mass_out=None if in_place else mout, source=src)
    assert out.data_ptr() == mout.data_ptr()
    assert torch.equal(src.cpu(), ref[3])
    assert torch.equal(torch.nan_to_num(out.cpu(), nan=-7.0), torch.nan_to_num(ref[2], nan=-7.0))
    assert torch.equal(k.cpu(), ref[0]) and torch.equal(v.cpu(), ref[1])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,E,BS", [(BF16, 128, 16), (F16, 256, 64), (F32, 64, 1), (F32, 128, 96)])
def test_evict_types(dtype, E, BS, in_place):
    kc, vc, bt, g = pool(4, 300, 3, E, BS, dtype, seed=E)
    mass = torch.rand((4, 3, bt.size(1) * BS), generator=g)
    evict_both(kc, vc, mass, bt, [0, 5, 100, 0], [300, 250, 77, 64], [64, 249, 10, 64], sink=2, recent=7, in_place=in_place)


@pytest.mark.parametrize("n,keep", [(0, 3), (1, 0), (1, 1), (2, 1), (32, 31), (33, 1), (1000, 0), (1000, 999), (1000, 1000), (1000, 5000),
                                    (5000, 2500), (9001, 17), (40000, 39000), (70001, 4000)])
def test_evict_lengths(n, keep):
    kc, vc, bt, g = pool(1, max(n, 1), 2, 16, 16, BF16, seed=n)
    mass = torch.randn((1, 2, bt.size(1) * 16), generator=g).mul_(2).exp_()
    evict_both(kc, vc, mass, bt, [0], [n], [keep], sink=1, recent=min(5, n))


def test_evict_rows_longer_than_shared_memory():
    """800000 positions: the survivors' bitmaps lie in the workspace."""
    n = 800_000
    kc, vc, bt, g = pool(1, n, 1, 8, 64, BF16, seed=5)
    mass = torch.randint(0, 50, (1, 1, bt.size(1) * 64), generator=g).float()
    i32 = lambda x: torch.tensor([x], dtype=torch.int32, device=DEV)  # noqa: E731
    k, v = kc.to(DEV), vc.to(DEV)
    src = torch.empty(mass.shape, dtype=torch.int32, device=DEV)
    out = dvattn_b200.dvattn_paged_evict(k, v, mass.to(DEV), bt.to(DEV), i32(0), i32(n), i32(500_000), source=src)
    m = mass[0, 0, :n].numpy()
    stay = np.sort(np.lexsort((np.arange(n), -m))[:500_000])
    want = np.arange(n)
    want[np.setdiff1d(np.arange(500_000), stay)] = stay[stay >= 500_000]
    want[500_000:] = -1
    assert np.array_equal(src[0, 0, :n].cpu().numpy(), want)
    assert np.array_equal(out[0, 0, :500_000].cpu().numpy(), m[want[:500_000]])
    assert torch.equal(k.cpu()[bt[0].long()].reshape(-1, 8)[:500_000], kc[bt[0].long()].reshape(-1, 8)[torch.from_numpy(want[:500_000])])


def test_evict_ties_and_special_values():
    """Equal masses (all of them, zeros of both signs), infinities, NaN, denormals, negatives: larger first,
    NaN last, equal ones by position."""
    kc, vc, bt, g = pool(5, 640, 2, 16, 16, F16, seed=6)
    mass = torch.zeros((5, 2, 640))
    mass[1] = torch.randint(0, 3, (2, 640), generator=g).float()
    mass[2] = torch.where(torch.rand((2, 640), generator=g) < 0.5, 0.0, -0.0)
    special = torch.tensor([math.inf, -math.inf, math.nan, -math.nan, 1e-42, -1e-42, 0.0, -0.0, 1.0, -1.0, 3e38])
    mass[3] = special[torch.randint(0, len(special), (2, 640), generator=g)]
    mass[4] = math.nan
    for keep in (1, 63, 320, 600):
        evict_both(kc, vc, mass, bt, [0] * 5, [640, 639, 640, 640, 500], [keep] * 5, sink=3, recent=9)


def test_evict_protected_beyond_the_budget_and_odd_ranges():
    """More protected tokens than are kept; ranges outside the mass or the table; negative sizes; pages
    outside the pool (their rows do not move)."""
    kc, vc, bt, g = pool(8, 200, 2, 32, 16, F32, seed=7)
    mass = torch.rand((8, 2, 150), generator=g)
    bt[7, 2] = -1
    bt[7, 8] = kc.size(0)
    evict_both(kc, vc, mass, bt, [0, 10, -1, 149, 150, 2 ** 31 - 1, 140, 0], [200, -4, 50, 5, 5, 2 ** 31 - 1, 2 ** 31 - 1, 150],
               [20, 5, 5, 1, 1, 1, -3, 60], sink=15, recent=20)
    evict_both(kc, vc, torch.rand((8, 2, 1000), generator=g), bt, [0] * 8, [2 ** 31 - 1] * 8, [100] * 8, sink=2 ** 31 - 1, recent=2 ** 31 - 1)


def test_evict_then_attend():
    """Attention over the kept positions equals attention over the survivors where they were."""
    W, Hkv, n, keep, E = 2, 2, 256, 100, 128
    kc, vc, bt, g = pool(W, n, Hkv, E, 16, F32, seed=8)
    mass = torch.rand((W, Hkv, n), generator=g)
    q = torch.randn((W, 8, 1, E), generator=g)
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    k, v, src = kc.to(DEV), vc.to(DEV), torch.empty((W, Hkv, n), dtype=torch.int32, device=DEV)
    dvattn_b200.dvattn_paged_evict(k, v, mass.to(DEV), bt.to(DEV), ints(0, 0), ints(n, n), ints(keep, keep), sink=4, recent=16, source=src)
    none = torch.zeros((1, W, 1, 0), device=DEV)
    loc = torch.full((1, W, 1), keep - 1, dtype=torch.int32, device=DEV)
    out = dvattn_b200.dvattn_paged_sdpa(q.to(DEV), loc, none, none, ints(n), k, v, bt.to(DEV), E ** -0.5)
    for w in range(W):
        for h in range(Hkv):
            at = src[w, h, :keep].long().cpu()
            kk, vv = (plain64.key_rows(t, bt[w], 0, n, h)[at] for t in (kc, vc))
            p = (q[w, 4 * h:4 * h + 4, 0].double() @ kk.T * E ** -0.5).softmax(-1)
            # the sums of 100 terms and the scores of 128 in 32 bits (plain64's analysis): below 1e-4 of the weights
            assert bool(((out[w, 4 * h:4 * h + 4, 0].cpu().double() - p @ vv).abs() <= 1e-4 * (p @ vv.abs())).all())


def test_evict_repeats_and_c_abi():
    kc, vc, bt, g = pool(3, 2000, 2, 64, 16, BF16, seed=9)
    mass = torch.rand((3, 2, 2000), generator=g)
    i = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 1, 2], [2000, 1500, 30], [700, 100, 30])]
    runs = []
    for via in (dvattn_b200.dvattn_paged_evict, capi.paged_evict, dvattn_b200.dvattn_paged_evict):
        k, v, m, out = kc.to(DEV), vc.to(DEV), mass.to(DEV), torch.empty((3, 2, 2000), device=DEV)
        for _ in range(2):  # the same call again moves the same rows
            via(k, v, m, bt.to(DEV), *i, sink=1, recent=2, mass_out=out)
        runs.append([k, v, out])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_append_mass_and_eviction_replayed_from_a_graph():
    """Captured once, replayed over changed inputs: what the calls themselves give."""
    W, Hkv, S, E, BS, n = 3, 2, 4, 64, 16, 300
    kc, vc, bt, g = pool(W, n + 20, Hkv, E, BS, BF16, seed=10)
    N = bt.size(1) * BS
    kc, vc, bt = (t.to(DEV) for t in (kc, vc, bt))
    dk, dv = (torch.randn((W, Hkv, S, E), generator=g).to(BF16).to(DEV) for _ in range(2))
    q = torch.randn((W, 4 * Hkv, S, E), generator=g).to(BF16).to(DEV)
    angles = torch.rand((1, W, S, 32), generator=g).to(DEV)
    lse = torch.full((W, 4 * Hkv, S), 6.0, device=DEV)
    mass = torch.rand((W, Hkv, N), generator=g).to(DEV)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    pos, acc, cnt, L = ints([n, n - 9, 17]), ints([[0, 1, 3]] * W), ints([3, 2, 1]), ints([N])
    zero, source = ints([0] * W), torch.zeros((W, Hkv, N), dtype=torch.int32, device=DEV)
    state = [kc, vc, mass, source]
    start = [t.clone() for t in state]

    def step():
        dvattn_b200.dvattn_tree_append(kc, vc, dk, dv, angles[0], angles[0], bt, pos, acc, cnt)
        seen = (pos + cnt)[None, :, None].expand(1, W, S).contiguous() - 1
        dvattn_b200.dvattn_paged_mass(mass, q, lse, seen, angles, angles, L, kc, bt, 0.125)
        dvattn_b200.dvattn_paged_evict(kc, vc, mass, bt, zero, pos + cnt, (pos + cnt).clamp(max=256), sink=2, recent=8, source=source)

    def run(call, positions):
        for t, x in zip(state, start):
            t.copy_(x)
        pos.copy_(positions)
        call()
        torch.cuda.synchronize()
        return [t.clone() for t in state]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for positions in ([n, n - 9, 17], [280, 3, 255], [n, n, n]):
        want = run(step, ints(positions))
        for _ in range(2):
            assert all(torch.equal(a, b) for a, b in zip(run(graph.replay, ints(positions)), want))


# ---- refusals ---------------------------------------------------------------------------------------------
def test_refusals():
    c = make([[10, 4], [3, 3]], 3, 4, 2, 64, 32, 16, F16, seed=14)
    g = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}
    for name, bad, word in [("mass", g["mass"].double(), "float32"), ("mass", g["mass"][:1].contiguous(), "mass must be"),
                            ("lse", g["lse"][:, :2].contiguous(), "lse must be"), ("q", g["q"].float(), "dtype"),
                            ("loc", g["loc"].long(), "int32"), ("kc", g["kc"][:, ::2], "contiguous"), ("lse", g["lse"].cpu(), "CUDA"),
                            ("bt", g["bt"][:1].contiguous(), "block_tables"), ("cos", g["cos"][:1].contiguous(), "cosines/sines")]:
        a = {**g, name: bad}
        with pytest.raises(RuntimeError, match=word):
            dvattn_b200.dvattn_paged_mass(a["mass"], *(a[k] for k in ("q", "lse", "loc", "cos", "sin", "L", "kc", "bt")), 0.1)
    kc, vc, bt, gen = pool(2, 64, 2, 64, 16, F16)
    t = dict(k_cache=kc, v_cache=vc, mass=torch.zeros((2, 2, 64)), block_tables=bt, starts=torch.zeros(2, dtype=torch.int32),
             lengths=torch.zeros(2, dtype=torch.int32), keep=torch.zeros(2, dtype=torch.int32))
    t = {k: v.to(DEV) for k, v in t.items()}
    flat = torch.zeros(2 * 2 * 64 + 8, device=DEV)
    for name, bad, word in [("mass", t["mass"][:, :1].contiguous(), "mass"), ("keep", t["keep"].long(), "int32"), ("sink", -1, "sink"),
                            ("starts", t["starts"][:1], "starts"), ("v_cache", t["v_cache"].float(), "dtype"),
                            ("mass_out", torch.zeros((2, 2, 63), device=DEV), "mass_out"),
                            ("source", torch.zeros((2, 2, 64), device=DEV), "int32")]:
        with pytest.raises(RuntimeError, match=word):
            dvattn_b200.dvattn_paged_evict(**{**t, name: bad})
    with pytest.raises(RuntimeError, match="invalid argument"):  # overlaps the mass without being it
        dvattn_b200.dvattn_paged_evict(**{**t, "mass": flat[:256].view(2, 2, 64), "mass_out": flat[8:].view(2, 2, 64)})
