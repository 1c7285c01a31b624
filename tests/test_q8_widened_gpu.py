"""Which way the packed prefill over an 8-bit cache takes, and its widening path: the pages that the tokens see widened in the workspace
and given to the tensor-core prefill.  Small calls are sent there with DVATTN_PREFILL=1, and the workspace's size shows that they went."""
import pytest
import torch

import dvattn_b200
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
