"""GPU tests of the draft-tree attention (dvattn_tree_sdpa) and the append of accepted tokens
(dvattn_tree_append) against their definitions in 64 bits (plain64.py), with bounds derived
there from the operations."""
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


def random_tree(rs, S, fan=3):
    return [-1] + [int(rs.randint(max(-1, (j - 1) // fan - 1), j)) for j in range(1, S)]


def make(turn_lens, S, Hq, Hkv, E, R, BS, dtype, seed=0, parents=None):
    """Inputs of one call (CPU): the cache of workloads.make_paged, a random tree per sequence."""
    rs = np.random.RandomState(seed)
    tl = np.asarray(turn_lens)
    W, F = tl.shape
    if parents is None:
        parents = [random_tree(rs, S) for _ in range(W)]
    depth = np.zeros((W, S), int)
    for w in range(W):
        for j, p in enumerate(parents[w]):
            depth[w, j] = depth[w, p] + 1 if 0 <= p < j else 0
    left = tl[:, ::-1].cumsum(axis=1)[:, ::-1].T[:, :, None] + depth[None]
    loc = np.repeat(tl.T[:, :, None] - 1, S, axis=2)
    c = wl.make_paged(turn_lens, Hq, Hkv, E, R, BS, dtype, seed=seed, S=S, loc_override=loc, rot_offsets=left)
    g = torch.Generator().manual_seed(seed + 1)
    return dict(q=c.queries, parents=torch.tensor(parents, dtype=torch.int32), loc=c.locations, cos=c.cosines, sin=c.sines,
                L=c.fragment_lengths, kc=c.k_cache, vc=c.v_cache, bt=c.block_tables, scale=c.scale,
                dk=torch.randn((W, Hkv, S, E), generator=g).to(dtype), dv=torch.randn((W, Hkv, S, E), generator=g).to(dtype))


def on_gpu(c):
    return {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in c.items()}


def call(c, out=None):
    lse = torch.full(c["q"].shape[:3], float("nan"), device=DEV)
    if out is None:
        out = torch.full_like(c["q"], float("nan"))
    dvattn_b200.dvattn_tree_sdpa(c["q"], c["parents"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"],
                                 c["dk"], c["dv"], c["scale"], out=out, lse=lse)
    return out, lse


def check(c, what=""):
    out, lse = call(on_gpu(c))
    torch.cuda.synchronize()
    ref, ref_lse, mag = plain64.tree(c)
    keys = int(c["L"].sum()) + c["q"].size(2)
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(lse == -math.inf, ref_lse == -math.inf), what
    fin = ref_lse > -math.inf
    err, bound = (lse[fin] - ref_lse[fin]).abs(), plain64.lse_bound(c, ref_lse[fin], keys)
    assert bool((err <= bound).all()), (what, "lse", float((err / bound).max()))
    err, bound = (out - ref).abs(), plain64.out_bound(c, ref, mag, keys)
    assert bool((err <= bound).all()), (what, "out", float((err / bound).max()))
    return out, lse


TYPES = [F32, F16, BF16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E", [64, 128, 256])
@pytest.mark.parametrize("Hq,Hkv,S", [(16, 1, 4), (8, 8, 1), (15, 3, 7), (32, 2, 33)])
def test_heads_types_dims(dtype, E, Hq, Hkv, S):
    check(make([[70, 33], [1, 260], [0, 5]], S, Hq, Hkv, E, 32, 16, dtype, seed=E + S))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("BS", [1, 3, 8, 48, 64, 96, 128, 256])
def test_page_sizes(dtype, BS):
    """Pages that end inside a window, are larger than one, or hold a single token."""
    check(make([[131, 200, 17], [300, 1, 0]], 5, 8, 2, 128, 64, BS, dtype, seed=BS))


@pytest.mark.parametrize("R", [0, 2, 24, 32, 128])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_rotary_dims(dtype, R):
    check(make([[90, 65]], 6, 8, 2, 128, R, 16, dtype, seed=R))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,G", [(1, 1), (1, 16), (8, 16), (9, 16), (17, 16), (64, 5), (129, 1), (130, 4), (257, 2), (1024, 1)])
def test_tokens_by_group(dtype, S, G):
    """Row counts around the tiles (32, 128, 256 rows) and trees longer than a key window."""
    check(make([[150], [40]], S, 2 * G, 2, 128, 64, 16, dtype, seed=S + G))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 127, 128, 129, 255, 256, 257, 5000])
def test_context_lengths(dtype, n):
    """Empty caches and lengths around the windows; 5000 keys are split over many blocks."""
    check(make([[n]], 3, 4, 1, 128, 64, 16, dtype, seed=n))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_sequences(dtype):
    """More sequences than blocks, lengths from nothing to a few pages."""
    rs = np.random.RandomState(1)
    check(make([[int(rs.randint(0, 60)), int(rs.randint(0, 9))] for _ in range(333)], 2, 2, 1, 64, 32, 8, dtype, seed=2))


@pytest.mark.parametrize("dtype", TYPES)
def test_shapes_of_trees(dtype):
    """A chain, a star, a forest of roots, a comb."""
    S = 40
    chain, star = list(range(-1, S - 1)), [-1] + [0] * (S - 1)
    roots, comb = [-1] * S, [-1] + [j - 1 if j % 2 else j - 2 for j in range(1, S)]
    check(make([[77]] * 4, S, 4, 2, 128, 64, 16, dtype, seed=3, parents=[chain, star, roots, [max(p, -1) for p in comb]]))


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_that_are_not_there(dtype):
    """Padding (-2), a parent that comes after its child, an own parent, indices far outside, and the
    descendants of all these: zeros and -inf; what lies in their keys, values and queries does not matter."""
    parents = [[-1, 0, 1, -2, -2, -2], [-1, 5, 1, 2, 0, -2], [0, 0, -1, 3, 2, 2 ** 31 - 1], [-2] * 6, [-2 ** 31, -1, 1, 0, 1, 4]]
    c = make([[50], [3], [0], [20], [9]], 6, 8, 2, 128, 64, 16, dtype, seed=4, parents=parents)
    gone = [(w, j) for w in range(5) for j in range(6) if not bool(plain64.ancestors(parents[w])[j, j])]
    for w, j in gone:
        c["dk"][w, :, j] = float("nan")
        c["dv"][w, :, j] = float("inf")
        c["q"][w, :, j] = float("nan")
        c["loc"][:, w, j] = 2 ** 31 - 1
    out, lse = check(c)
    for w, j in gone:
        assert not bool(out[w, :, j].any()) and bool((lse[w, :, j] == -math.inf).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_places_do_not_matter(dtype):
    """Keys that no token sees hold NaN and infinities: past the locations, in a skipped turn, in pages
    that only padding uses; pages outside the pool read as zeros."""
    c = make([[200, 130], [90, 40]], 5, 8, 2, 128, 64, 16, dtype, seed=5)
    c["loc"][0, 0] = 99
    c["loc"][1, 1] = -1
    c["loc"][1, 0, 2] = -2 ** 31
    bt, BS = c["bt"], 16
    off = int(c["L"][0])
    for w, (a, b) in enumerate([(100, 130), (90, 0)]):
        for p in list(range(a, off)) + list(range(off + b, bt.size(1) * BS)):
            page = int(bt[w, p // BS])
            live = any(int(bt[x, y // BS]) == page and y % BS == p % BS for x, m in ((0, [(0, 100), (off, off + 130)]), (1, [(0, 90)]))
                       for lo, hi in m for y in range(lo, hi) if y % BS == p % BS)
            if not live:
                c["kc"][page, p % BS] = float("nan")
                c["vc"][page, p % BS] = float("inf")
    check(c)
    c["bt"][0, 2] = -5
    c["bt"][0, 3] = c["kc"].size(0)
    c["bt"][1, 0] = 2 ** 31 - 1
    check(c, "pages outside the pool")


@pytest.mark.parametrize("dtype", TYPES)
def test_locations_by_token(dtype):
    """Locations that differ from token to token, past the turn's end and past the block table."""
    c = make([[300, 64]], 12, 8, 2, 64, 32, 16, dtype, seed=6)
    rs = np.random.RandomState(6)
    c["loc"] = torch.from_numpy(rs.randint(-3, 400, size=(2, 1, 12)).astype(np.int32))
    check(c)
    c["L"] = torch.tensor([300, 5000], dtype=torch.int32)  # longer than the table
    c["loc"][1] = 4999
    check(c, "past the table")


@pytest.mark.parametrize("dtype", [F32, F16])
def test_large_scores(dtype):
    """Scores in the hundreds: the running maximum carries the sums."""
    c = make([[400]], 7, 8, 2, 128, 64, 16, dtype, seed=7)
    c["kc"], c["dk"] = c["kc"] * 8, c["dk"] * 8
    c["q"] = c["q"] * 8
    check(c)
    c["scale"] = -c["scale"]
    check(c, "negative scale")


@pytest.mark.parametrize("nats", [15.0, 16.0, 17.0, 18.03])
@pytest.mark.parametrize("E,S,G", [(64, 1, 4), (128, 1, 4), (256, 1, 4), (64, 33, 4), (128, 33, 4)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_one_key_far_above_many(dtype, E, S, G, nats):
    """A key whose value is zero, and thousands of keys that far below it whose values have one sign: their
    weights are small for the type, their sum is the result.  Many sequences share the pages, so that a
    sequence's keys are one block's work."""
    W, n, BS = 300, 20000, 64
    pages = -(-n // BS)
    g = torch.Generator().manual_seed(E + S)
    kc = torch.zeros((pages, BS, 1, E), dtype=dtype)
    vc = (0.5 + torch.rand((pages, BS, 1, E), generator=g)).to(dtype)
    dv = (0.5 + torch.rand((1, 1, S, E), generator=g)).to(dtype)
    kc[0, 0, 0, 0], vc[0, 0] = nats, 0
    q = torch.zeros((W, G, S, E), dtype=dtype)
    q[..., 0] = 1
    none = torch.zeros((1, W, S, 0))
    c = dict(q=q, parents=torch.full((W, S), -1, dtype=torch.int32), loc=torch.full((1, W, S), n - 1, dtype=torch.int32), cos=none, sin=none,
             L=torch.tensor([n], dtype=torch.int32), kc=kc, vc=vc, bt=torch.arange(pages, dtype=torch.int32).repeat(W, 1), scale=1.0,
             dk=torch.zeros((W, 1, S, E), dtype=dtype), dv=dv.repeat(W, 1, 1, 1))
    out, lse = call(on_gpu(c))
    top = math.exp(float(kc[0, 0, 0, 0]))
    total = top + n  # the dominant key, n - 1 others and the token itself
    ref = (vc.reshape(-1, E)[:n].double().sum(0) + dv[0, 0].double()) / total  # [S, E]
    bound = plain64.out_bound(c, ref, ref, n + 1)
    if dtype == F16:  # a weight's rounding is at most 2^-32 of the largest weight where fp16 is subnormal
        bound = bound + n * 2.0 ** -32 * 1.5
    assert bool(((out.double().cpu() - ref).abs() <= bound).all())
    assert bool(((lse.double().cpu() - math.log(total)).abs() <= plain64.lse_bound(c, torch.tensor(math.log(total)).double(), n + 1)).all())


def test_equal_to_a_causal_decode_of_the_appended_chain():
    """A chain of drafts gives what the paged decode gives once the chain is in the cache."""
    S = 5
    c = make([[100], [37]], S, 32, 2, 128, 64, 16, BF16, seed=8, parents=[list(range(-1, S - 1))] * 2)
    g = on_gpu(c)
    out, lse = call(g)
    pages = 10
    kc, vc = (torch.zeros((2 * pages, 16, 2, 128), dtype=BF16, device=DEV) for _ in range(2))
    bt = torch.arange(2 * pages, dtype=torch.int32, device=DEV).reshape(2, pages)
    for w, n in enumerate((100, 37)):
        pos = torch.arange(n, device=DEV)
        old = g["bt"][w].long()[pos // 16]
        kc[bt[w].long()[pos // 16], pos % 16], vc[bt[w].long()[pos // 16], pos % 16] = g["kc"][old, pos % 16], g["vc"][old, pos % 16]
    n = torch.tensor([100, 37], dtype=torch.int32, device=DEV)
    chain = torch.arange(S, dtype=torch.int32, device=DEV).expand(2, S).contiguous()
    dvattn_b200.dvattn_tree_append(kc, vc, g["dk"], g["dv"], g["cos"][0], g["sin"][0], bt, n, chain)
    loc = (n[:, None] + chain)[None].contiguous()
    L = torch.tensor([160], dtype=torch.int32, device=DEV)
    lse2 = torch.empty_like(lse)
    ref = dvattn_b200.dvattn_paged_sdpa(g["q"], loc, g["cos"], g["sin"], L, kc, vc, bt, c["scale"], lse=lse2)
    torch.cuda.synchronize()
    # both are within the bound of the same exact value
    exact, exact_lse, mag = plain64.tree(c)
    assert bool(((out - ref).double().abs().cpu() <= 2 * plain64.out_bound(c, exact, mag, 105)).all())
    assert bool(((lse - lse2).double().abs().cpu() <= 2 * plain64.lse_bound(c, exact_lse, 105)).all())


def visible(c):
    """[W, S, keys] which cached key of each turn, then which drafted key, a token sees."""
    W, S = c["parents"].shape
    cap = c["bt"].size(1) * c["kc"].size(1)
    anc = torch.stack([plain64.ancestors(p) for p in c["parents"].tolist()])
    there = anc.any(-1)
    parts = [(torch.arange(n) <= c["loc"][f][..., None]) & there[..., None] for f, (_, n) in enumerate(plain64.turns(c["L"].tolist(), cap))]
    return torch.cat(parts + [anc], -1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,S,G,BS", [(64, 7, 2, 16), (64, 70, 4, 16), (128, 7, 2, 16), (128, 1, 16, 16), (128, 7, 2, 6), (128, 70, 4, 16),
                                      (128, 70, 4, 6), (128, 300, 1, 16), (256, 7, 2, 16), (256, 40, 4, 5)])
def test_values_that_are_not_finite_reach_who_sees_them(dtype, E, S, G, BS):
    """Infinities and NaN in values of drafted tokens and of cached keys that some tokens see: an element of
    who sees one is not finite, everything else has the bits of the same call with zeros in these places."""
    c = make([[500, 130], [90, 61]], S, 2 * G, 2, E, 32, BS, dtype, seed=E + S, parents=None if S > 1 else [[-1], [-1]])
    rs = np.random.RandomState(E + S + BS)
    if S > 1:
        c["parents"][1, S - 1] = -2
        # locations by token: past the end, inside a window, in front of the turn
        c["loc"][0, 0] = torch.from_numpy(rs.choice([499, 77, 430, -1], size=S).astype(np.int32))
        c["loc"][1, 1] = torch.from_numpy(rs.choice([60, 40], size=S).astype(np.int32))
        c["loc"][1, 0] = torch.from_numpy(rs.choice([129, 128], size=S).astype(np.int32))
    # pages of every sequence's own
    pages = c["bt"].size(1)
    g = torch.Generator().manual_seed(18)
    c["kc"], c["vc"] = (torch.randn((2 * pages, BS, 2, E), generator=g).to(dtype) for _ in range(2))
    c["bt"] = torch.from_numpy(rs.permutation(2 * pages).reshape(2, pages).astype(np.int32))
    spans = plain64.turns(c["L"].tolist(), pages * BS)
    where = torch.cat([torch.arange(first, first + n) for first, n in spans])
    cached = where.numel()
    clean = {**c, "vc": c["vc"].clone(), "dv": c["dv"].clone()}
    bad = torch.zeros((2, 2, cached + S, E))  # what lies there, 0: a finite value
    special = [math.inf, -math.inf, math.nan]
    spots = [(0, 70), (0, 80), (0, 429), (0, 431), (0, 499), (1, 499 + 41), (1, 499 + 62), (0, 500 + 129)]
    spots += [(int(w), cached + int(j)) for w, j in zip(rs.randint(0, 2, 8), rs.randint(0, S, 8))]
    for x, (w, key) in enumerate(spots):
        if key >= bad.size(2):
            continue
        bad[w, x % 2, key, rs.randint(0, E, 3)] = special[x % 3]
    for w in range(2):
        for h in range(2):
            for key in bad[w, h].ne(0).any(-1).nonzero()[:, 0].tolist():
                b = bad[w, h, key]
                row = lambda t: t["vc"][int(t["bt"][w, where[key] // BS]), where[key] % BS, h] if key < cached else t["dv"][w, h, key - cached]  # noqa: E731
                row(clean)[:] = torch.where(b != 0, torch.zeros((), dtype=dtype), row(clean))
                row(c)[:] = torch.where(b != 0, b.to(dtype), row(c))
    want, want_lse = call(on_gpu(clean))
    out, lse = call(on_gpu(c))
    assert bool(torch.isfinite(want).all())
    sees = visible(c).float()  # [W, S, keys]
    hit = bad != 0
    # per output: how many of each it sees
    n = {v: torch.einsum("wsk,whke->whse", sees, (bad.isnan() if v != v else bad == v).float()) for v in special}
    nan = (n[special[2]] > 0) | ((n[math.inf] > 0) & (n[-math.inf] > 0))
    expect = want.cpu().view(2, 2, G, S, E).float()
    for v in (math.inf, -math.inf):
        expect = torch.where((n[v] > 0)[:, :, None], torch.tensor(v), expect)
    expect = torch.where(nan[:, :, None], torch.tensor(math.nan), expect)
    got = out.cpu().view(2, 2, G, S, E).float()
    assert bool(hit.any()) and not bool(torch.isfinite(got).all())
    assert torch.equal(got.isnan(), expect.isnan())
    assert torch.equal(got.nan_to_num(nan=0.0), expect.nan_to_num(nan=0.0))
    assert torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("BS", [65536, 65537])
def test_as_many_positions_as_there_are(dtype, BS):
    """A block table of more than 2^31 positions, one page under all of them: the first 2^31 - 256 are read."""
    n, E, most = 2 ** 31 - 1, 64, 2 ** 31 - 256
    g = torch.Generator().manual_seed(16)
    kc, vc = (torch.randn((1, BS, 1, E), generator=g).to(dtype) for _ in range(2))
    q, dk, dv = (torch.randn((1, h, 1, E), generator=g).to(dtype) for h in (2, 1, 1))
    none = torch.zeros((1, 1, 1, 0))
    c = dict(q=q, parents=torch.tensor([[-1]], dtype=torch.int32), loc=torch.full((1, 1, 1), n, dtype=torch.int32), cos=none, sin=none,
             L=torch.tensor([n], dtype=torch.int32), kc=kc, vc=vc, bt=torch.zeros((1, 32769), dtype=torch.int32), scale=0.125, dk=dk, dv=dv)
    out, lse = call(on_gpu(c))
    times = torch.tensor([(most - p + BS - 1) // BS for p in range(BS)] + [1], dtype=torch.float64)
    z = 0.125 * q[0, :, 0].double() @ torch.cat([kc[0, :, 0], dk[0, 0]]).double().T
    w = z.exp() * times
    v = torch.cat([vc[0, :, 0], dv[0, 0]]).double()
    ref, mag = (w @ v / w.sum(1, keepdim=True))[None, :, None], (w @ v.abs() / w.sum(1, keepdim=True))[None, :, None]
    assert bool(((out.double().cpu() - ref).abs() <= plain64.out_bound(c, ref, mag, most)).all())
    want = w.sum(1).log()
    assert bool(((lse.double().cpu()[0, :, 0] - want).abs() <= plain64.lse_bound(c, want, most)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R", [24, 64])
def test_drafted_keys_are_those_that_the_append_writes(dtype, R):
    """cos/sin rows whose halves differ: a drafted key is turned by both, like the key that goes into the cache."""
    S = 6
    c = make([[90], [31]], S, 8, 2, 128, R, 16, dtype, seed=15, parents=[[-1, 0, 0, 1, 1, 2]] * 2)
    g = torch.Generator().manual_seed(15)
    c["cos"][..., R // 2:], c["sin"][..., R // 2:] = torch.rand((2,) + c["cos"][..., R // 2:].shape, generator=g)
    out, lse = call(on_gpu(c))
    cos, sin = c["cos"][0][:, None], c["sin"][0][:, None]
    k, h = c["dk"].double(), R // 2
    turned = k.clone()
    turned[..., :h] = k[..., :h] * cos[..., :h].double() - k[..., h:R] * sin[..., :h].double()
    turned[..., h:R] = k[..., h:R] * cos[..., h:].double() + k[..., :h] * sin[..., h:].double()
    turned = turned.to(dtype).double()
    sees = plain64.ancestors(c["parents"][0].tolist())
    for w, n in enumerate((90, 31)):
        for kv in range(2):
            q = plain64.rotate(c["q"][w, 4 * kv:4 * kv + 4], c["cos"][0, w], c["sin"][0, w])
            cached = plain64.scores(c, w, kv)[0][1]
            z = torch.cat([cached, (c["scale"] * q @ turned[w, kv].T).masked_fill(~sees, -math.inf)], -1)
            v = torch.cat([plain64.key_rows(c["vc"], c["bt"][w], 0, cached.size(-1), kv), c["dv"][w, kv].double()])
            p = z.softmax(-1)
            v = torch.where((p > 0).flatten(0, 1).any(0)[:, None], v, torch.zeros((), dtype=torch.float64))
            got, got_lse = (t[w, 4 * kv:4 * kv + 4].double().cpu() for t in (out, lse))
            # the rotated keys' own rounding: in 64 bits here, of 32-bit products there: an ulp of T of the
            # rare element that lies between two, on a row of E elements
            s = plain64.UNIT[dtype] * 2 * abs(c["scale"]) * float(q.norm(dim=-1).max()) * float(turned.abs().max())
            assert bool(((got - p @ v).abs() <= plain64.out_bound(c, p @ v, p @ v.abs(), 96) + 2 * s * (p @ v.abs())).all())
            assert bool(((got_lse - z.logsumexp(-1)).abs() <= plain64.lse_bound(c, z.logsumexp(-1), 96) + s).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_repeats_and_streams(dtype):
    """The same bits again, on another stream too, with a workspace full of another call's data."""
    a = on_gpu(make([[3000, 20], [40, 700]], 9, 8, 2, 128, 64, 16, dtype, seed=9))
    b = on_gpu(make([[10]], 2, 4, 2, 64, 32, 16, dtype, seed=10))
    first = call(a)
    call(b)
    again = call(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = call(a)
    side.synchronize()
    torch.cuda.synchronize()
    for x, y, z in zip(first, again, third):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_c_abi_and_status():
    c = on_gpu(make([[600], [31]], 6, 16, 2, 128, 64, 16, F16, seed=11))
    out, lse = call(c)
    got, got_lse = torch.empty_like(out), torch.empty_like(lse)
    ws = torch.full((64 << 20,), 0xff, dtype=torch.uint8, device=DEV)
    capi.tree_sdpa(got, c["scale"], c["parents"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"],
                   c["dk"], c["dv"], lse=got_lse, workspace=ws)
    assert capi.workspace_status(ws) == 0
    assert torch.equal(got, out) and torch.equal(got_lse, lse)


def test_replayed_from_a_graph():
    c = on_gpu(make([[900], [250]], 6, 16, 2, 128, 64, 16, BF16, seed=12))
    out, lse = call(c)
    got = torch.zeros_like(out)
    call(c, got)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dvattn_b200.dvattn_tree_sdpa(c["q"], c["parents"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"],
                                     c["dk"], c["dv"], c["scale"], out=got)
    got.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, out)


def test_nothing_to_do():
    c = on_gpu(make([[10]], 2, 4, 2, 64, 32, 16, F16, seed=13))
    empty = {k: (v[:0] if k in ("q", "parents", "bt", "dk", "dv") else v[:, :0] if k in ("loc", "cos", "sin") else v) for k, v in c.items()}
    assert call(empty)[0].shape == (0, 4, 2, 64)


# ---- the append of accepted tokens ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,E,R,BS", [(BF16, 128, 64, 16), (F16, 256, 128, 64), (F32, 64, 0, 8), (BF16, 128, 24, 1), (F32, 128, 12, 96)])
@pytest.mark.parametrize("via", ["op", "capi"])
def test_append_accepted(dtype, E, R, BS, via):
    rs = np.random.RandomState(E + R)
    W, Hkv, S, A = 6, 3, 21, 9
    maxb = -(-120 // BS)
    NB = W * maxb
    g = torch.Generator().manual_seed(3)
    kc, vc = (torch.randn((NB, BS, Hkv, E), generator=g).to(dtype) for _ in range(2))
    dk, dv = (torch.randn((W, Hkv, S, E), generator=g).to(dtype) for _ in range(2))
    cos, sin = wl.rope_angles(torch.from_numpy(rs.randint(0, 9000, (W, S))), R)
    bt = torch.from_numpy(rs.permutation(NB).reshape(W, maxb).astype(np.int32))
    pos = torch.from_numpy(rs.randint(0, 100, size=W).astype(np.int32))
    pos[1], pos[2] = maxb * BS - 3, -2  # runs past the table; begins before it
    bt[3, int(pos[3]) // BS] = NB       # a page outside the pool
    acc = torch.from_numpy(np.sort(np.stack([rs.permutation(S)[:A] for _ in range(W)]), axis=1).astype(np.int32))
    acc[4, 1], acc[4, 3] = -1, S        # no such tokens
    cnt = torch.tensor([A, A, A, 5, 7, 0], dtype=torch.int32)
    ek, ev = kc.clone(), vc.clone()
    # apply_rotary_pos_emb in the type's own rounding: 32-bit products and sum, rounded once
    rk = dvattn_b200.apply_rotary_pos_emb(dk.float(), cos, sin).to(dtype) if R else dk
    for w in range(W):
        for i in range(int(cnt[w])):
            p, node = int(pos[w]) + i, int(acc[w, i])
            if 0 <= p < maxb * BS and 0 <= node < S and 0 <= int(bt[w, p // BS]) < NB:
                ek[int(bt[w, p // BS]), p % BS], ev[int(bt[w, p // BS]), p % BS] = rk[w, :, node], dv[w, :, node]
    got_k, got_v = kc.to(DEV), vc.to(DEV)
    fn = dvattn_b200.dvattn_tree_append if via == "op" else capi.tree_append
    fn(got_k, got_v, *(t.to(DEV) for t in (dk, dv, cos, sin, bt, pos, acc, cnt)))
    torch.cuda.synchronize()
    assert torch.equal(got_k.cpu(), ek) and torch.equal(got_v.cpu(), ev)


# ---- refusals ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("change,word", [
    (lambda c: c.update(q=c["q"].transpose(1, 2)), "contiguous|output must be"),
    (lambda c: c.update(kc=c["kc"].float()), "dtype"),
    (lambda c: c.update(parents=c["parents"].long()), "int32"),
    (lambda c: c.update(parents=c["parents"][:, :2].contiguous()), "parents must be"),
    (lambda c: c.update(loc=c["loc"][:, :1].contiguous()), "locations must be"),
    (lambda c: c.update(cos=c["cos"].half()), "float32"),
    (lambda c: c.update(sin=c["sin"][..., :8].contiguous()), "cosines/sines"),
    (lambda c: c.update(dk=c["dk"][:, :, :2].contiguous()), "draft_keys must be"),
    (lambda c: c.update(dv=c["dv"].cpu()), "CUDA"),
    (lambda c: c.update(bt=c["bt"][:1].contiguous()), "block_tables"),
    (lambda c: c.update(L=c["L"][:1].contiguous()), "fragment_lengths"),
    (lambda c: c.update(vc=c["vc"][:, :, :1].contiguous()), "v_cache"),
])
def test_refusals(change, word):
    c = on_gpu(make([[10, 4], [3, 3]], 3, 4, 2, 64, 32, 16, F16, seed=14))
    change(c)
    with pytest.raises(RuntimeError, match=word):
        dvattn_b200.dvattn_tree_sdpa(c["q"], c["parents"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"],
                                     c["dk"], c["dv"], c["scale"], out=torch.empty((2, 4, 3, 64), dtype=F16, device=DEV))


def test_append_refusals():
    W, Hkv, S, E = 2, 2, 4, 64
    t = dict(k_cache=torch.zeros((4, 16, Hkv, E), dtype=F16), v_cache=torch.zeros((4, 16, Hkv, E), dtype=F16),
             draft_keys=torch.zeros((W, Hkv, S, E), dtype=F16), draft_values=torch.zeros((W, Hkv, S, E), dtype=F16),
             cosines=torch.zeros((W, S, 32)), sines=torch.zeros((W, S, 32)), block_tables=torch.zeros((W, 2), dtype=torch.int32),
             positions=torch.zeros(W, dtype=torch.int32), accepted=torch.zeros((W, 3), dtype=torch.int32))
    t = {k: v.to(DEV) for k, v in t.items()}
    for name, bad, word in [("accepted", t["accepted"].long(), "int32"), ("accepted", t["accepted"][:1], r"accepted \[W, A\]"),
                            ("cosines", t["cosines"][:, :2].contiguous(), "cosines/sines"), ("draft_values", t["draft_values"].float(), "dtype"),
                            ("v_cache", t["v_cache"][:2], "v_cache"), ("draft_keys", t["draft_keys"].mT, "contiguous")]:
        with pytest.raises(RuntimeError, match=word):
            dvattn_b200.dvattn_tree_append(**{**t, name: bad})
