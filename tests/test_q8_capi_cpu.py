"""Refusals of the 8-bit paged cache's and the page assignment's entry points, without a GPU: through the C ABI, where
every call here answers before anything is launched, and of the torch ops."""
import ctypes

import pytest
import torch

import dvattn_b200
from dvattn_b200 import capi

LIB = capi.lib()
OK, INVALID, UNSUPPORTED = capi.DVATTN_OK, capi.DVATTN_ERR_INVALID_ARGUMENT, capi.DVATTN_ERR_UNSUPPORTED
SCALES = capi.Q8Scales()


def fill(a, base, kw):
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


def paged(**kw):
    return fill(capi.PagedArgs(), dict(dtype=capi.DVATTN_BFLOAT16, F=2, W=2, Hq=32, Hkv=2, E=128, Ev=128, S=1, R=64,
                                       block_size=16, max_blocks_per_seq=4, num_blocks=8, scale=0.1), kw)


def varlen(**kw):
    return fill(capi.VarlenArgs(), dict(dtype=capi.DVATTN_FLOAT16, F=1, W=2, Hq=32, Hkv=2, E=128, Ev=128, T=9, R=64,
                                        block_size=16, max_blocks_per_seq=4, num_blocks=8, scale=0.1), kw)


def append(**kw):
    return fill(capi.AppendArgs(), dict(dtype=capi.DVATTN_FLOAT32, W=2, Hkv=2, E=64, Ev=64, n=3, R=32, block_size=16,
                                        max_blocks_per_seq=4, num_blocks=8), kw)


def assign(**kw):
    return fill(capi.AssignArgs(), dict(W=2, block_size=16, max_blocks_per_seq=4, free_size=8, n=0), kw)


def release(**kw):
    return fill(capi.ReleaseArgs(), dict(W=2, block_size=16, max_blocks_per_seq=4, free_size=8), kw)


COMMON = [(dict(dtype=7), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED), (dict(E=96, Ev=96), UNSUPPORTED), (dict(Ev=64), UNSUPPORTED),
          (dict(Hq=64), UNSUPPORTED), (dict(Hq=33), INVALID), (dict(Hkv=0), INVALID), (dict(R=130), INVALID), (dict(R=63), INVALID),
          (dict(block_size=0), INVALID), (dict(W=-1), INVALID), (dict(F=-1), INVALID), (dict(num_blocks=-1), INVALID),
          (dict(max_blocks_per_seq=-1), INVALID), (dict(), INVALID)]


@pytest.mark.parametrize("name,make,kw,status",
                         [("dvattn_paged_sdpa_q8", paged, kw, st) for kw, st in COMMON + [(dict(S=-1), INVALID), (dict(S=2049), UNSUPPORTED), (dict(F=1 << 20, S=1 << 11), UNSUPPORTED)]] +
                         [("dvattn_varlen_paged_sdpa_q8", varlen, kw, st) for kw, st in COMMON + [
                             (dict(T=-1), INVALID), (dict(F=65536), UNSUPPORTED), (dict(T=1 << 28), UNSUPPORTED), (dict(W=(1 << 30) + 1, max_blocks_per_seq=1), UNSUPPORTED),
                             (dict(W=1 << 16, max_blocks_per_seq=1 << 16), UNSUPPORTED)]])
def test_attention(name, make, kw, status):
    """dict(): sizes in order, but null pointers."""
    a = make(**kw)
    assert getattr(LIB, name)(ctypes.byref(a), ctypes.byref(SCALES), None, 0, None) == status
    if kw:
        assert getattr(LIB, name + "_workspace_size")(ctypes.byref(a)) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=9), UNSUPPORTED), (dict(E=0), INVALID), (dict(E=36), UNSUPPORTED), (dict(Ev=4), UNSUPPORTED), (dict(R=33), INVALID),
    (dict(R=66), INVALID), (dict(n=-1), INVALID), (dict(W=-1), INVALID), (dict(Hkv=0), INVALID), (dict(block_size=0), INVALID),
    (dict(num_blocks=-1), INVALID), (dict(max_blocks_per_seq=-1), INVALID), (dict(block_size=1 << 20, max_blocks_per_seq=1 << 11), UNSUPPORTED),
    (dict(block_size=1 << 25), UNSUPPORTED), (dict(W=1 << 20, n=1 << 11), UNSUPPORTED), (dict(), INVALID)])
def test_append(kw, status):
    assert LIB.dvattn_paged_append_q8(ctypes.byref(append(**kw)), ctypes.byref(SCALES), None) == status


@pytest.mark.parametrize("name,make", [("dvattn_assign_pages", assign), ("dvattn_release_pages", release)])
@pytest.mark.parametrize("kw,status", [
    (dict(W=-1), INVALID), (dict(block_size=0), INVALID), (dict(max_blocks_per_seq=-1), INVALID), (dict(free_size=-1), INVALID),
    (dict(W=1 << 16, max_blocks_per_seq=1 << 15), UNSUPPORTED), (dict(block_size=1 << 16, max_blocks_per_seq=1 << 15), UNSUPPORTED),
    (dict(), INVALID)])
def test_pages(name, make, kw, status):
    assert getattr(LIB, name)(ctypes.byref(make(**kw)), None) == status


def test_slots_of_a_negative_number_of_tokens():
    assert LIB.dvattn_assign_pages(ctypes.byref(assign(n=-1)), None) == INVALID


def test_null_arguments_and_empty_calls():
    for name, make in (("dvattn_paged_sdpa_q8", paged), ("dvattn_varlen_paged_sdpa_q8", varlen)):
        call = getattr(LIB, name)
        assert call(None, ctypes.byref(SCALES), None, 0, None) == INVALID
        assert call(ctypes.byref(make()), None, None, 0, None) == INVALID
        assert getattr(LIB, name + "_workspace_size")(None) == 0
    for a in (paged(W=0), paged(S=0), paged(Hq=0)):
        assert LIB.dvattn_paged_sdpa_q8(ctypes.byref(a), ctypes.byref(SCALES), None, 0, None) == OK
    for a in (varlen(T=0), varlen(Hq=0)):
        assert LIB.dvattn_varlen_paged_sdpa_q8(ctypes.byref(a), ctypes.byref(SCALES), None, 0, None) == OK
    assert LIB.dvattn_paged_append_q8(None, ctypes.byref(SCALES), None) == INVALID
    assert LIB.dvattn_paged_append_q8(ctypes.byref(append()), None, None) == INVALID
    for a in (append(W=0), append(n=0)):
        assert LIB.dvattn_paged_append_q8(ctypes.byref(a), ctypes.byref(SCALES), None) == OK
    assert LIB.dvattn_assign_pages(None, None) == INVALID and LIB.dvattn_release_pages(None, None) == INVALID
    assert LIB.dvattn_assign_pages(ctypes.byref(assign(W=0)), None) == OK
    for a in (release(W=0), release(max_blocks_per_seq=0)):
        assert LIB.dvattn_release_pages(ctypes.byref(a), None) == OK


def test_misaligned_pointers():
    """Addresses that are never read: the refusal comes before."""
    ok = dict(out=256, queries=256, locations=256, fragment_lengths=256, cosines=256, sines=256, k_cache=256, v_cache=256, block_tables=256)
    sc = capi.Q8Scales(256, 256)
    for bad in ("out", "queries", "k_cache", "v_cache", "out_f32"):
        assert LIB.dvattn_paged_sdpa_q8(ctypes.byref(paged(**{**ok, bad: 264})), ctypes.byref(sc), None, 0, None) == INVALID
        assert LIB.dvattn_varlen_paged_sdpa_q8(ctypes.byref(varlen(**{**ok, "cu_seqlens_q": 256, bad: 264})), ctypes.byref(sc), None, 0, None) == INVALID
    put = dict(k_cache=256, v_cache=256, keys=256, values=256, cosines=256, sines=256, block_tables=256, positions=256)
    for bad in ("k_cache", "v_cache", "keys", "values"):
        assert LIB.dvattn_paged_append_q8(ctypes.byref(append(**{**put, bad: 264})), ctypes.byref(sc), None) == INVALID
    for gone in ok:
        if gone != "out":
            assert LIB.dvattn_paged_sdpa_q8(ctypes.byref(paged(**{**ok, gone: None})), ctypes.byref(sc), None, 0, None) == INVALID
    for gone in put:
        assert LIB.dvattn_paged_append_q8(ctypes.byref(append(**{**put, gone: None})), ctypes.byref(sc), None) == INVALID
    for k, v in ((None, 256), (256, None)):
        half = capi.Q8Scales(k, v)
        assert LIB.dvattn_paged_sdpa_q8(ctypes.byref(paged(**ok)), ctypes.byref(half), None, 0, None) == INVALID
        assert LIB.dvattn_varlen_paged_sdpa_q8(ctypes.byref(varlen(**ok, cu_seqlens_q=256)), ctypes.byref(half), None, 0, None) == INVALID
        assert LIB.dvattn_paged_append_q8(ctypes.byref(append(**put)), ctypes.byref(half), None) == INVALID


def test_the_python_calls_want_gpu_tensors():
    """A tensor of the host is refused, not read from a kernel."""
    f8, i32 = torch.float8_e4m3fn, torch.int32
    kc, ks, bt = torch.zeros((4, 16, 2, 64), dtype=f8), torch.ones((4, 2)), torch.zeros((1, 2), dtype=i32)
    q, ang, loc, L = torch.zeros((1, 2, 1, 64)), torch.zeros((1, 1, 1, 64)), torch.zeros((1, 1, 1), dtype=i32), torch.ones(1, dtype=i32)
    new, at = torch.zeros((1, 2, 3, 64)), torch.zeros(1, dtype=i32)
    calls = [
        lambda: dvattn_b200.dvattn_paged_sdpa_q8(q, loc, ang, ang, L, kc, kc, ks, ks, bt, 0.1),
        lambda: dvattn_b200.dvattn_varlen_paged_sdpa_q8(q[:, :, 0], loc[:, 0], ang[:, 0, :, :32], ang[:, 0, :, :32], L, kc, kc, ks, ks, bt,
                                                        torch.tensor([0, 1], dtype=i32), None, 0.1),
        lambda: dvattn_b200.dvattn_paged_append_q8(kc, kc.clone(), ks, ks.clone(), new, new, torch.zeros((1, 3, 64)), torch.zeros((1, 3, 64)), bt, at),
        lambda: dvattn_b200.dvattn_assign_pages(bt, torch.arange(4, dtype=i32), torch.tensor([4], dtype=i32), at, at, 16),
        lambda: dvattn_b200.dvattn_release_pages(bt, torch.arange(4, dtype=i32), torch.tensor([0], dtype=i32), at, 16),
    ]
    for call in calls:
        with pytest.raises(Exception):
            call()


@pytest.mark.parametrize("name,make", [("dvattn_assign_pages", assign), ("dvattn_release_pages", release)])
def test_tables_that_a_walk_would_step_past_32_bits(name, make):
    """A walk's step behind the last of 2^31 - 1 entries does not fit in 32 bits; 1024 entries fewer do (null pointers: refused next)."""
    for W, most in ((1, 0x7fffffff), (7, 0x7fffffff // 7), (1, 0x7fffffff - 1023)):
        assert getattr(LIB, name)(ctypes.byref(make(W=W, max_blocks_per_seq=most, block_size=1)), None) == UNSUPPORTED
    assert getattr(LIB, name)(ctypes.byref(make(W=1, max_blocks_per_seq=0x7fffffff - 1024, block_size=1)), None) == INVALID


@pytest.mark.parametrize("at", [256, 260, 252])
@pytest.mark.parametrize("name", ["starts", "counts"])
def test_granted_counts_over_the_requests(name, at):
    """Granted counts written where starts or counts are still read (a free list without pages: nothing else would be refused)."""
    ok = dict(block_tables=4096, free_pages=4096, free_count=4096, starts=1024, counts=2048, granted=256)
    assert LIB.dvattn_assign_pages(ctypes.byref(assign(**{**ok, name: at})), None) == INVALID
