"""The 8-bit paged cache at its edges: pools past 4 GB, refusals of the torch ops, replayed appends, calls on several streams at
once, page tables that sequences share."""
import pytest
import torch

import dvattn_b200
import plain_q8
import test_q8_gpu as q8
from dvattn_b200 import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
F8 = torch.float8_e4m3fn


def high(c, pages):
    """The call with its cache's pages moved to the top of a pool of `pages`, the bytes below NaN."""
    NB = c["kc"].size(0)
    out = dict(c, bt=torch.where(c["bt"] >= 0, c["bt"] + (pages - NB), c["bt"]))
    for name in ("kc", "vc"):
        big = torch.full((pages,) + c[name].shape[1:], 0x7f, dtype=torch.uint8, device=DEV)
        big[pages - NB:] = c[name].view(torch.uint8)
        out[name] = big.view(F8)
    for name in ("ks", "vs"):
        big = torch.full((pages, c[name].size(1)), float("nan"), device=DEV)
        big[pages - NB:] = c[name]
        out[name] = big
    return out


@pytest.mark.parametrize("BS", [16, 6])  # pages by TMA, row by row
def test_offsets_past_32_bits(BS):
    """Bitwise what the same pages give in a small pool: decode, packed prefill and append at byte offsets above 2^32."""
    Hkv, E = 2, 128
    pages = (1 << 32) // (BS * Hkv * E) + 500
    c = q8.on_gpu(q8.make([[200, 77], [40, 500]], 2, 8, Hkv, E, 64, BS, BF16))
    v = q8.on_gpu(q8.make_varlen([[50, 9], [120, 40]], [3, 20], 8, Hkv, E, 32, BS, BF16))
    for data, call in ((c, q8.call), (v, q8.call_varlen)):
        small = call(data)
        big = high(data, pages)
        for x, y in zip(small, call(big)):
            assert torch.equal(x, y)
        del big
    g = torch.Generator(device=DEV).manual_seed(0)
    new = torch.randn((2, Hkv, 9, E), generator=g, device=DEV, dtype=BF16)
    ang = torch.rand((2, 9, 64), generator=g, device=DEV)
    at = torch.tensor([270, 533], dtype=torch.int32, device=DEV)
    big = high(c, pages)
    for d in (c, big):
        dvattn_b200.dvattn_paged_append_q8(d["kc"], d["vc"], d["ks"], d["vs"], new, -new, ang, ang, d["bt"], at)
    NB = c["kc"].size(0)
    for name in ("kc", "vc"):
        assert torch.equal(big[name][pages - NB:].view(torch.uint8), c[name].view(torch.uint8))
        assert bool((big[name][:pages - NB].view(torch.uint8) == 0x7f).all())
    for name in ("ks", "vs"):
        assert torch.equal(big[name][pages - NB:], c[name]) and bool(torch.isnan(big[name][:pages - NB]).all())


def test_refusals_of_the_ops():
    c = q8.on_gpu(q8.make([[20, 7]], 1, 4, 2, 64, 32, 16, F16))
    good = [c["q"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"]]
    dvattn_b200.dvattn_paged_sdpa_q8(*good, c["scale"])
    bad = {0: [c["q"].double(), c["q"][0], c["q"].expand(2, -1, -1, -1)], 1: [c["loc"].long(), c["loc"][:1]], 2: [c["cos"].half(), c["cos"][..., :20]],
           4: [c["L"].long(), c["L"][:1], c["L"].cpu()], 5: [c["kc"].view(torch.uint8), c["kc"].float(), c["kc"].to(torch.float8_e5m2), c["kc"][..., :32]],
           6: [c["vc"].view(torch.uint8), c["vc"][:, :8], c["vc"].transpose(1, 2)],
           7: [c["ks"].double(), c["ks"][:, :1], c["ks"][:1], c["ks"][:, 0], c["ks"].t().contiguous().t(), c["ks"].cpu()], 8: [c["vs"].half(), c["vs"][..., None]],
           9: [c["bt"].long(), c["bt"][0], c["bt"].expand(3, -1)]}
    for i, values in bad.items():
        for x in values:
            args = list(good)
            args[i] = x
            with pytest.raises(Exception):
                dvattn_b200.dvattn_paged_sdpa_q8(*args, c["scale"])
    i32 = dict(dtype=torch.int32, device=DEV)
    new, ang, at = torch.zeros((1, 2, 3, 64), dtype=F16, device=DEV), torch.zeros((1, 3, 32), device=DEV), torch.zeros(1, **i32)
    put = [c["kc"], c["vc"], c["ks"], c["vs"], new, new, ang, ang, c["bt"], at]
    for i, values in {0: [c["kc"].view(torch.uint8), c["kc"].half()], 2: [c["ks"][:1], c["ks"].half()], 4: [new.float(), new[:, :1], new.transpose(1, 2)],
                      6: [ang[..., :16], ang.half(), ang[:, :2]], 8: [c["bt"].long(), c["bt"].expand(2, -1)], 9: [at.long(), at[:0]]}.items():
        for x in values:
            args = list(put)
            args[i] = x
            with pytest.raises(Exception):
                dvattn_b200.dvattn_paged_append_q8(*args)
    bt, free, count = torch.full((2, 4), -1, **i32), torch.arange(8, **i32), torch.tensor([8], **i32)
    two = torch.ones(2, **i32)
    for args in ([bt.long(), free, count, two, two], [bt, free.long(), count, two, two], [bt, free, count.long(), two, two], [bt, free, count, two[:1], two],
                 [bt, free, count, two, two.long()], [bt.t(), free, count, two, two], [bt, free[None], count, two, two], [bt.cpu(), free, count, two, two],
                 [bt, free, torch.zeros(2, **i32), two, two]):
        with pytest.raises(Exception):
            dvattn_b200.dvattn_assign_pages(*args, 16)
        with pytest.raises(Exception):
            dvattn_b200.dvattn_release_pages(*args[:4 if args[4] is two else 3], *([] if args[4] is two else [two.long()]), 16)
    for size in (0, -1, 1 << 32):
        with pytest.raises(Exception):
            dvattn_b200.dvattn_assign_pages(bt, free, count, two, two, size)
    for slots in (torch.zeros((2, 3), **i32), torch.zeros((1, 3), dtype=torch.int64, device=DEV), torch.zeros(6, dtype=torch.int64, device=DEV)):
        with pytest.raises(Exception):
            dvattn_b200.dvattn_assign_pages(bt, free, count, two, two, 16, slots=slots)
    assert int(count) == 8 and bool((bt == -1).all())


def test_append_replayed_at_other_positions():
    """One captured append, its inputs written anew between replays; the same as calls of their own."""
    c = q8.make_append(3, 2, 2, 64, 32, 16, BF16, [0, 7, 30], 4)
    d = {k: x.to(DEV) if torch.is_tensor(x) else x for k, x in c.items()}
    names = ("kc", "vc", "ks", "vs")
    start = {n: d[n].clone() for n in names}

    def put(x):
        dvattn_b200.dvattn_paged_append_q8(x["kc"], x["vc"], x["ks"], x["vs"], x["k"], x["v"], x["cos"], x["sin"], x["bt"], x["positions"])

    put(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        put(d)
    own = {**d, **{n: start[n].clone() for n in names}, "k": d["k"].clone(), "v": d["v"].clone(), "positions": d["positions"].clone()}
    for n in names:
        d[n].copy_(start[n])
    for step in range(5):
        graph.replay()
        put(own)
        for x in (d, own):
            x["positions"] += 2
            x["k"] *= 1.7
            x["v"] *= -1.3
    torch.cuda.synchronize()
    for n in names:
        assert torch.equal(d[n].view(torch.uint8), own[n].view(torch.uint8)), n


def test_two_streams_at_once():
    """Two calls that overlap, each with a workspace of its own: each result is that of the call alone."""
    cs = [q8.on_gpu(q8.make([[3000, 500 * i], [40, 2000]], 1, 16, 2, 128, 64, 16, BF16, seed=i)) for i in (1, 2)]
    alone = [q8.call(c) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                got[i].append(q8.call(c))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x[0], alone[i][0]) and torch.equal(x[1], alone[i][1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sequences_that_share_pages(dtype):
    """A prompt's pages in three sequences' tables, and a page twice in one table."""
    c = q8.make([[64, 20], [64, 33], [64, 5]], 1, 8, 2, 64, 32, 16, dtype)
    c["bt"][1:, :4] = c["bt"][0, :4]
    c["bt"][2, 1] = c["bt"][2, 0]
    q8.check(c)


@pytest.mark.parametrize("W,BS,maxb,longest", [(9000, 4, 4, 16), (9000, 4, 4, 1), (200, 16, 300, 4800), (100, 2, 200, 400), (2, 16, 5000, 80000),
                                               (128, 16, 33, 500), (129, 16, 33, 500), (256, 8, 64, 3), (257, 8, 64, 512), (85, 16, 1, 16)])
@pytest.mark.parametrize("spare", [7, 0, -1, -300])
def test_pages_by_rows_and_by_parts(W, BS, maxb, longest, spare):
    """Several chunks of sequences to a warp, several warps to a sequence, long rows, and too few pages with each."""
    q8.test_pages(W, BS, maxb, longest, spare)


def test_append_tiles_at_the_border_of_a_warp():
    """Pages whose tile one warp can just hold, cannot, and that four warps cannot hold either; each type."""
    for dtype, E, sizes in ((BF16, 128, (16, 17, 64, 65, 200)), (F16, 64, (32, 33, 130)), (F32, 128, (8, 9, 33, 70)), (BF16, 256, (8, 9, 33))):
        for BS in sizes:
            for R in (0, E // 2, E):
                q8.check_append(q8.make_append(2, 2, 2 * BS + 3, E, R, BS, dtype, [0, BS // 2], 4, seed=BS, magnitude=1.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_ranges_of_the_split(dtype):
    """Windows in numbers around the CTAs', turns of one key, and turns that are empty for some sequences."""
    for turns in ([[1] * 6] * 9, [[1, 0, 33, 0, 0, 1], [0, 0, 0, 0, 0, 0], [0, 700, 0, 1, 0, 0]], [[5000, 1, 1, 4000]], [[64 * 148]], [[64 * 297, 1]],
                  [[1, 64 * 300], [0, 1]]):
        q8.check(q8.make(turns, 1, 8, 1, 64, 32, 16, dtype))


@pytest.mark.parametrize("dtype,E,Hq,Hkv", [(F32, 64, 6, 2), (F32, 256, 5, 1), (F16, 64, 48, 3), (BF16, 256, 8, 2), (BF16, 128, 3, 3)])
@pytest.mark.parametrize("BS", [16, 6])
def test_packed_row_tiles(dtype, E, Hq, Hkv, BS):
    """Row tiles of packed tokens: groups that do not divide a tile, sequences of no, one and many tokens, several turns."""
    q8.check_varlen(q8.make_varlen([[50, 9], [0, 0], [0, 0], [120, 40], [3, 3], [1, 300]], [5, 1, 0, 37, 2, 64], Hq, Hkv, E, E // 2, BS, dtype, seed=E + BS))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_packed_in_several_launches(dtype):
    """More row tiles than a launch takes; the same as each sequence in a call of its own."""
    c = q8.on_gpu(q8.make_varlen([[40], [17], [300]], [3000, 3, 1400], 16, 1, 64, 32, 16, dtype))
    out, lse = q8.call_varlen(c)
    assert c["q"].size(0) * 16 // 32 > 2048 and bool(torch.isfinite(out.float()).all())
    cu = c["cu"].tolist()
    for w in range(3):
        at = slice(cu[w], cu[w + 1])
        one = dict(c, q=c["q"][at].contiguous(), loc=c["loc"][:, at].contiguous(), cos=c["cos"][:, at].contiguous(), sin=c["sin"][:, at].contiguous(),
                   bt=c["bt"][w:w + 1].contiguous(), cu=torch.tensor([0, cu[w + 1] - cu[w]], dtype=torch.int32, device=DEV))
        o, l = q8.call_varlen(one)
        # the split of the keys differs: both are within the bounds of the definition
        ref = plain_q8.varlen({k: x.cpu() if torch.is_tensor(x) else x for k, x in dict(one, q=one["q"][:40], loc=one["loc"][:, :40], cos=one["cos"][:, :40],
                                                                                        sin=one["sin"][:, :40], cu=one["cu"].clamp(max=40)).items()})
        q8.close(one, o[:40], l[:40], *ref)
        q8.close(one, out[at][:40], lse[at][:40], *ref)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_packed_tokens_outside_the_sequences(dtype):
    """cu that begins behind the first token or ends before the last one: those tokens have the first sequence's table, in the 16-bit
    attention as here; cu of no order reads nothing outside."""
    c = q8.make_varlen([[60], [33]], [20, 12], 8, 2, 64, 32, 16, dtype)
    for cu in ([3, 20, 30], [0, 0, 0], [0, 32, 32], [9, 9, 40]):
        q8.check_varlen(dict(c, cu=torch.tensor(cu, dtype=torch.int32)))
    for cu in ([5, -3, 1000], [32, 16, 0], [-7, 1 << 30, 4]):
        q8.call_varlen(q8.on_gpu(dict(c, cu=torch.tensor(cu, dtype=torch.int32))))
    torch.cuda.synchronize()
    with pytest.raises(Exception):  # tokens and no sequence: the tables are empty, a null pointer, as in the 16-bit attention
        q8.call_varlen(q8.on_gpu(dict(c, bt=c["bt"][:0], cu=torch.zeros(1, dtype=torch.int32))))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_most_rows_of_a_sequence(dtype):
    """2048 tokens of 16 query heads to a KV head: as many row tiles as a launch takes, a sequence a launch."""
    q8.check(q8.make([[2100], [2060]], 2048, 16, 1, 64, 32, 16, dtype))


@pytest.mark.parametrize("W", [1, 2, 129, 160, 200, 255])
def test_pages_of_blocks_without_sequences(W):
    """Whole blocks of the page kernels' cluster without a sequence, which reach the exchange of counts before the others have walked
    theirs (or begun): every one of many calls gives what the first does, and the pages come back as they were."""
    BS, maxb = 16, 60
    i32 = dict(dtype=torch.int32, device=DEV)
    starts = torch.arange(W, **i32) % 7 * 13
    counts = torch.arange(W, **i32) % 5 * 101 + 1
    bt, count = torch.full((W, maxb), -1, **i32), torch.tensor([W * maxb], **i32)
    free = torch.arange(W * maxb, **i32)
    ref = plain_q8.assign(bt.cpu(), free.cpu(), W * maxb, starts.cpu(), counts.cpu(), BS)
    before = bt.clone(), free.clone(), count.clone()
    zero = torch.zeros_like(starts)
    for _ in range(300):
        granted = dvattn_b200.dvattn_assign_pages(bt, free, count, starts, counts, BS)
        assert torch.equal(bt.cpu(), ref[0]) and int(count) == ref[1] and torch.equal(granted.cpu(), ref[2])
        dvattn_b200.dvattn_release_pages(bt, free, count, zero, BS)
        assert torch.equal(bt, before[0]) and torch.equal(count, before[2]) and torch.equal(free, before[1])


def paged_workspace(c):
    a = capi.paged_args(c["q"], c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"])
    return capi.lib().dvattn_paged_sdpa_q8_workspace_size(a)


def varlen_workspace(c):
    a = capi.varlen_args(c["q"], c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"], c["cu"])
    return capi.lib().dvattn_varlen_paged_sdpa_q8_workspace_size(a)


def test_most_bytes_of_rotated_queries():
    """256 MB of rotated queries and what else a workspace holds (partial results of all CTAs: under 64 MB), however large the call: a
    sequence's row tiles, and the packed tokens', go to as many launches as that takes."""
    c = q8.make([[40, 7, 0, 30], [3, 50, 20, 1]], 600, 128, 8, 256, 32, 16, F32)
    d = q8.on_gpu(c)
    assert 600 * 2 * 4 * 8 * 16448 > 512 << 20 and 256 << 20 < paged_workspace(d) < 320 << 20
    out, lse = q8.call(d)
    q8.close(c, out, lse, *plain_q8.paged(c))
    turns = [[(w + f) % 4 for f in range(64)] for w in range(3)]
    c = q8.make_varlen(turns, [300, 1, 400], 8, 8, 256, 32, 16, F32)
    d = q8.on_gpu(c)
    assert 256 << 20 < varlen_workspace(d) < 320 << 20
    out, lse = q8.call_varlen(d)
    q8.close(c, out, lse, *plain_q8.varlen(c))
    # sizes that are not run: 2048 tokens of a sequence, 4 turns; one row tile of 4096 turns is more than 256 MB
    a = capi.PagedArgs()
    for k, v in dict(dtype=capi.DVATTN_FLOAT32, F=4, W=2, Hq=128, Hkv=8, E=256, Ev=256, S=2048, R=32, block_size=16, max_blocks_per_seq=8, num_blocks=8).items():
        setattr(a, k, v)
    assert 0 < capi.lib().dvattn_paged_sdpa_q8_workspace_size(a) < 320 << 20
    a.F, a.S = 4096, 1
    assert 4096 * 8 * 16448 < capi.lib().dvattn_paged_sdpa_q8_workspace_size(a) < 4096 * 8 * 16448 + (64 << 20)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("E", [64, 128, 256])
def test_value_scales_as_far_apart_as_they_may_be(dtype, E):
    """Scales of V 2^100 apart in one sequence and head, the least that the append writes among them: the keys of every page count."""
    c = q8.make([[300, 40], [5000, 3]], 2, 8, 2, E, 32, 16, dtype)
    c["vs"][::2], c["vs"][1::2] = 2.0 ** -60, 2.0 ** 40
    q8.check(c)
    c["vs"][:], c["vs"][c["bt"][0, 3]] = 2.0 ** 26, 2.0 ** 126 / 448
    q8.check(c)
