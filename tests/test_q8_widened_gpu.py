"""Which way the packed prefill over an 8-bit cache takes, and its widening path: the pages that the tokens see widened in the workspace
and given to the tensor-core prefill.  Small calls are sent there with DVATTN_PREFILL=1, and the workspace's size shows that they went."""
import pytest
import torch

import dvattn_b200
import plain64
import plain_q8
import test_q8_gpu as q8
import test_q8_limits_gpu as limits
from dvattn_b200 import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def workspace(c):
    """Bytes that the call asks for, and those of the widened pages of both caches."""
    a = capi.varlen_args(c["q"], c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"], c["cu"])
    NB, BS, Hkv, E = c["kc"].shape
    return capi.lib().dvattn_varlen_paged_sdpa_q8_workspace_size(a), 2 * 2 * min(NB, c["bt"].numel()) * BS * Hkv * E


def check(c):
    """Against the definition, on the widening path."""
    d = q8.on_gpu(c)
    size, pages = workspace(d)
    assert pages <= size < pages + (1 << 20)
    out, lse = q8.call_varlen(d)
    torch.cuda.synchronize()
    q8.close(c, out, lse, *plain_q8.varlen(c), wide=True)
    return out, lse


@pytest.fixture
def widened(monkeypatch):
    monkeypatch.setenv("DVATTN_PREFILL", "1")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("extra_pages", [0, 90])
def test_fragment_lengths_below_zero_and_past_the_table(widened, dtype, extra_pages):
    """A turn of a length below zero is empty, and a sum of lengths past 2^31 ends at the table's end: the same bits as with lengths that
    say so plainly."""
    c = q8.make_varlen([[60, 0, 45], [33, 0, 20]], [9, 30], 8, 2, 128, 32, 16, dtype, extra_pages=extra_pages)
    positions = c["bt"].size(1) * 16
    for odd, plain in (([64, -20, 75], [64, 0, 75]), ([-5, -2147483648, 75], [0, 0, 75]), ([2147483647, 2147483647, 64], [positions, 0, 0]),
                       ([40, 2147483647, 2147483647], [40, positions, 0])):
        ref = dict(c, L=torch.tensor(plain, dtype=torch.int32), loc=c["loc"].clone())
        ref["loc"][1] = ref["loc"][2] - 3  # the turn in the middle has keys, where it has a length
        want = check(ref)
        got = q8.call_varlen(q8.on_gpu(dict(ref, L=torch.tensor(odd, dtype=torch.int32))))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_locations(widened, dtype):
    """Locations of any order and sign, beyond the turn (the largest of all among them), and tokens that see nothing."""
    c = q8.make_varlen([[60, 45], [33, 20]], [9, 30], 8, 2, 128, 32, 16, dtype)
    c["loc"][0, ::3], c["loc"][0, 1::4], c["loc"][1, ::5] = 2147483647, -7, 500
    c["loc"][:, 4], c["loc"][:, 20] = -1, torch.tensor([-2147483648, 2147483647], dtype=torch.int32)
    out, lse = check(c)
    assert not out[4].any() and bool((lse[4] == -torch.inf).all())


@pytest.mark.parametrize("W", [2047, 2048, 2100])
def test_sequences_that_the_prefill_can_sort(widened, W):
    """2047 sequences are sorted by the tensor-core prefill; with more the call runs without it, over a 16-bit cache, too."""
    new = [0 if w % 3 == 1 else 2 + w % 2 for w in range(W)]
    c = q8.make_varlen([[w % 40] for w in range(W)], new, 4, 1, 128, 32, 16, BF16)
    d = q8.on_gpu(c)
    size, pages = workspace(d)
    assert (pages <= size < pages + (1 << 20)) == (W < 2048)
    out, lse = q8.call_varlen(d)
    q8.close(c, out, lse, *plain_q8.varlen(c), wide=W < 2048)
    k, v = [plain_q8.values(c[x], c[y]).to(BF16).to(DEV) for x, y in (("kc", "ks"), ("vc", "vs"))]
    wide = dvattn_b200.dvattn_varlen_paged_sdpa(d["q"], d["loc"], d["cos"], d["sin"], d["L"], k, v, d["bt"], d["cu"], None, d["scale"])
    q8.close(c, wide, lse, *plain_q8.varlen(c), wide=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("new,widens", [([1] * 600, False), ([8] * 74, False), ([16] * 37, True), ([1] * 200 + [400], False), ([1] * 20 + [600], True)])
def test_rows_of_a_sequence_decide(dtype, new, widens):
    """64 / 8 heads, enough tokens in all for the tensor-core prefill: pages are widened from 128 query rows (16 tokens) of a KV head in a
    sequence on average."""
    c = q8.make_varlen([[w % 30] for w in range(len(new))], new, 64, 8, 128, 32, 16, dtype)
    d = q8.on_gpu(c)
    size, pages = workspace(d)
    assert (pages <= size < pages + (1 << 20)) == widens
    out, lse = q8.call_varlen(d)
    q8.close(c, out, lse, *plain_q8.varlen(c), wide=widens)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("E,Hq,Hkv", [(64, 16, 2), (128, 16, 1), (128, 15, 3), (256, 8, 8)])
@pytest.mark.parametrize("new", [[1] * 70, [0, 1, 0, 0, 1], [1] * 40 + [25], [2] * 9 + [1]])
def test_few_rows_of_a_sequence(dtype, E, Hq, Hkv, new):
    """Packed sequences of 16 query rows or fewer on average: tiles of 16 rows, a chunk's and a single token's."""
    c = q8.make_varlen([[17 * w % 90, w % 3] for w in range(len(new))], new, Hq, Hkv, E, 32, 16, dtype, seed=E + len(new))
    out, lse = q8.call_varlen(q8.on_gpu(c))
    q8.close(c, out, lse, *plain_q8.varlen(c))


def far(c, pages, maxb):
    """The call (two turns, of which the first is not seen) with its last turn at the end of tables of `maxb` entries, its pages at the
    top of a pool of `pages`."""
    h = limits.high(c, pages)
    BS, W = c["kc"].size(1), c["bt"].size(0)
    n = c["bt"].size(1)
    maxb -= (maxb - n) * BS % 128 // BS  # windows begin at the same places
    bt = torch.full((W, maxb), -1, dtype=torch.int32, device=DEV)
    bt[:, maxb - n:] = h["bt"]
    L = c["L"].clone()
    L[0] += (maxb - n) * BS
    return dict(h, bt=bt, L=L)


def two_turns(dtype, seed=0):
    """Two sequences of two turns, the first of them unseen."""
    c = q8.make_varlen([[32, 45], [32, 120]], [9, 30], 8, 2, 128, 32, 16, dtype, seed=seed)
    c["loc"][0] = -1
    return c


@pytest.mark.parametrize("pages,maxb", [(700000, 300004), (590000, 300004)])  # a table in the workspace; the batch's own
def test_widened_pages_past_4_gb(widened, pages, maxb):
    """Widened caches of more than 4 GB each: bitwise what the same pages give in a small pool."""
    c = two_turns(BF16)
    want = check(c)
    d = far(q8.on_gpu(c), pages, maxb)
    size, widened_bytes = workspace(d)
    assert size >= widened_bytes > 8 << 30
    got = q8.call_varlen(d)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_most_bytes_of_widened_pages(widened, monkeypatch):
    """A pool whose widened pages would take more than 16 GB: the call runs on the row tiles, in a small workspace."""
    c = q8.on_gpu(two_turns(F16))
    pages = (1 << 32) // (16 * 2 * 128) + 500
    d = far(c, pages, pages)
    size, widened_bytes = workspace(d)
    assert size < 1 << 28 and widened_bytes > 16 << 30
    got = q8.call_varlen(d)
    monkeypatch.setenv("DVATTN_PREFILL", "0")
    want = q8.call_varlen(c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_last_positions_of_32_bits(widened, monkeypatch):
    """A table of 2^31 positions: those up to 2^31 - 256 are seen, as in the other calls over such a cache."""
    c = q8.make_varlen([[112, 144]], [5], 8, 2, 128, 32, 128, BF16)
    c["loc"][0], c["loc"][1] = -1, torch.tensor([10, 143, 200, 299, 500], dtype=torch.int32)
    c["bt"] = c["bt"][:, :2].contiguous()
    c["L"][1] = 300
    d = q8.on_gpu(c)
    bt = torch.full((1, 1 << 24), -1, dtype=torch.int32, device=DEV)
    bt[0, -4:-2] = d["bt"][0]
    bt[0, -2:] = d["bt"][0]  # positions that are not seen
    big = dict(d, bt=bt, L=d["L"] + torch.tensor([(1 << 31) - 512, 0], dtype=torch.int32, device=DEV))
    got = q8.call_varlen(big)
    q8.close(c, *got, *plain_q8.varlen(c))
    monkeypatch.setenv("DVATTN_PREFILL", "0")
    want = q8.call_varlen(big)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


# ---- what the short calls of the other files do not reach any more, on the widening path ------------------------
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("extra_pages", [0, 90])
def test_tables(widened, dtype, extra_pages):
    """A table in the workspace and the batch's own, three turns, pages outside the pool, a token behind the last sequence (the first
    one's), an empty sequence and one without keys."""
    c = q8.make_varlen([[50, 9, 17], [30, 11, 0], [0, 0, 0], [120, 40, 260]], [3, 2, 1, 90], 8, 2, 128, 32, 16, dtype, extra_pages=extra_pages)
    assert (c["kc"].size(0) > c["bt"].numel()) == (extra_pages > 0)
    check(c)
    c["bt"][2, 1], c["bt"][0, 0], c["bt"][3, 7] = -1, c["kc"].size(0), 2147483647
    check(c)
    c["cu"] = torch.tensor([0, 3, 3, 6, 90], dtype=torch.int32)
    check(c)


@pytest.mark.parametrize("BS", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("Hq,Hkv,R", [(3, 3, 0), (15, 3, 16), (32, 2, 128)])
def test_page_sizes_and_heads(widened, BS, Hq, Hkv, R):
    """Every page size that the tensor-core prefill takes, groups that do not divide its tiles, no and full rotary."""
    check(q8.make_varlen([[131, 200], [300, 1], [0, 17]], [40, 1, 17], Hq, Hkv, 128, R, BS, BF16, seed=BS + Hq, extra_pages=BS))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_scales(widened, dtype, monkeypatch):
    """Scales that are no powers of two (a widened value is rounded once more), of different magnitudes in every page."""
    # That rounding is off by UNIT of a key's element at most, and so q . k by UNIT * sum |q_i k_i| <= UNIT |q| |k| (Cauchy and Schwarz):
    # a term of the scaled score's error that keys with a power of two as their scale do not have.  (A value's is in `wide`.)
    exact = plain_q8.score_error

    def score_error(c):
        norm = [float(x.norm(dim=-1).max()) for x in (c["q"].double(), torch.nan_to_num(plain_q8.values(c["kc"], c["ks"])))]
        return exact(c) + plain64.UNIT[dtype] * abs(c["scale"]) * norm[0] * norm[1]
    monkeypatch.setattr(plain_q8, "score_error", score_error)
    c = q8.make_varlen([[50, 9], [120, 40]], [30, 60], 8, 2, 128, 32, 16, dtype, extra_pages=40)
    g = torch.Generator().manual_seed(3)
    for name, least, most in (("ks", 0.6, 1.0), ("vs", 0.3, 1.7)):
        c[name] = c[name] * (least + (most - least) * torch.rand(c[name].shape, generator=g))
    check(c)
    unseen = torch.ones(c["kc"].size(0), dtype=torch.bool)
    unseen[c["bt"].flatten().long()] = False
    c["ks"][unseen], c["vs"][unseen] = float("nan"), float("nan")
    check(c)


def test_values_past_f16(widened, monkeypatch):
    """f16: widened values past the type's largest number are taken for that number."""
    c = q8.make_varlen([[50], [120]], [30, 60], 8, 2, 128, 32, 16, F16)
    c["vs"][::2] = 1024.0
    exact = plain_q8.values
    assert float(exact(c["vc"], c["vs"]).abs().max()) > 65504
    monkeypatch.setattr(plain_q8, "values", lambda cache, scales: exact(cache, scales).clamp(-65504, 65504))
    check(c)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_nan_behind_the_keys(widened, dtype):
    """Bytes that no token sees, in the last seen page and in pages behind it, are not numbers."""
    c = q8.make_varlen([[75], [20]], [9, 30], 8, 2, 128, 32, 16, dtype, extra_pages=4)
    keys = c["loc"][0].tolist()
    for w, last in enumerate((max(keys[:9]), max(keys[9:]))):
        for p in range(last + 1, c["bt"].size(1) * 16):
            for t in (c["kc"], c["vc"]):
                t.view(torch.uint8)[int(c["bt"][w, p // 16]), p % 16] = 0x7F
    # Bytes that nobody sees have a weight of 0, so that zeros in their place change no result of the definition.  They give its bound the
    # sum of p |v| that the weights' rounding is relative to; with a NaN among the values the definition has |sum of p v| there, which is less.
    zeros = dict(c, **{n: torch.where(c[n].view(torch.uint8) == 0x7F, 0, c[n].view(torch.uint8)).view(c[n].dtype) for n in ("kc", "vc")})
    ref, odd = plain_q8.varlen(zeros), plain_q8.varlen(c)
    assert bool(((ref[0] - odd[0]).abs() <= 1e-12 * ref[2]).all()) and bool(((ref[1] - odd[1]).abs() <= 1e-12).all())
    d = q8.on_gpu(c)
    assert workspace(d)[0] >= workspace(d)[1]
    out, lse = q8.call_varlen(d)
    q8.close(zeros, out, lse, *ref, wide=True)
    same = q8.call_varlen(q8.on_gpu(zeros))
    assert torch.equal(same[0], out) and torch.equal(same[1], lse)


@pytest.mark.parametrize("extra_pages", [0, 90])
def test_stale_workspace_and_graph(widened, extra_pages):
    """The workspace's content from other calls does not matter; a captured call follows new contents of the cache and its tables."""
    c = q8.on_gpu(q8.make_varlen([[50, 30], [30, 70]], [40, 25], 8, 2, 128, 32, 16, BF16, extra_pages=extra_pages))
    size, pages = workspace(c)
    assert size >= pages
    ref, _ = q8.call_varlen(c)
    out = torch.zeros_like(ref)
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)

    def go():
        capi.varlen_paged_sdpa_q8(out, c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"], c["cu"],
                                  workspace=ws)
    for byte in (0x7F, 0xFF, 0x00):
        ws.fill_(byte)
        go()
        assert torch.equal(out, ref)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        go()
    c["vs"].mul_(2.0)
    ws.fill_(0x7F)
    g.replay()
    torch.cuda.synchronize()
    second = out.clone()
    assert torch.equal(second, q8.call_varlen(c)[0]) and not torch.equal(second, ref)
    c["bt"].copy_(c["bt"].flip(1).clone())
    c["cu"][1] -= 7
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, q8.call_varlen(c)[0]) and not torch.equal(out, second)
    assert capi.workspace_status(ws) == 0


def test_on_another_stream(widened):
    """Two widening calls at once on streams of their own: each result is that of the call alone."""
    cs = [q8.on_gpu(q8.make_varlen([[500 * i, 40], [30, 700]], [90, 200], 16, 2, 128, 32, 16, F16, seed=i, extra_pages=60 * i)) for i in (1, 2)]
    alone = [q8.call_varlen(c) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (c, s) in enumerate(zip(cs, streams)):
            with torch.cuda.stream(s):
                got[i].append(q8.call_varlen(c))
    torch.cuda.synchronize()
    for i in range(2):
        for x in got[i]:
            assert torch.equal(x[0], alone[i][0]) and torch.equal(x[1], alone[i][1])


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_row_tiles_keep_the_decode_bound(dtype, monkeypatch):
    """Packed calls on the row tiles, whose weights are f16 next to V in every type: the other files' cases, held to the decode's bound."""
    def narrow(c):
        d = q8.on_gpu(c)
        assert workspace(d)[0] > 0
        out, lse = q8.call_varlen(d)
        q8.close(c, out, lse, *plain_q8.varlen(c))
    monkeypatch.setattr(q8, "check_varlen", narrow)
    monkeypatch.setenv("DVATTN_PREFILL", "0")
    for E, BS in ((64, 16), (128, 16), (128, 6), (256, 64)):
        q8.test_varlen(dtype, E, BS)
    q8.test_varlen_tables(dtype)
    q8.test_serving_loop(dtype)
    for E, Hq, Hkv, BS in ((64, 48, 3, 16), (256, 8, 2, 6), (128, 3, 3, 16)):
        limits.test_packed_row_tiles(dtype, E, Hq, Hkv, BS)
    limits.test_packed_tokens_outside_the_sequences(dtype)
