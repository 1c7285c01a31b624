"""Argument validation of the draft-tree and bounded-cache entry points through the C ABI,
without a GPU: every call here answers before anything is launched."""
import ctypes

import pytest

from dvattn_b200 import capi

LIB = capi.lib()
OK, INVALID, UNSUPPORTED = capi.DVATTN_OK, capi.DVATTN_ERR_INVALID_ARGUMENT, capi.DVATTN_ERR_UNSUPPORTED


def fill(a, base, kw):
    for k, v in {**base, **kw}.items():
        setattr(a, k, v)
    return a


def tree(**kw):
    return fill(capi.TreeArgs(), dict(dtype=capi.DVATTN_BFLOAT16, F=2, W=2, Hq=32, Hkv=2, E=128, Ev=128, S=8, R=64,
                                      block_size=16, max_blocks_per_seq=4, num_blocks=8, scale=0.1), kw)


def mass(**kw):
    return fill(capi.MassArgs(), dict(dtype=capi.DVATTN_FLOAT16, F=1, W=2, Hq=32, Hkv=2, E=128, S=1, R=64, block_size=16,
                                      max_blocks_per_seq=4, num_blocks=8, positions=64, scale=0.1), kw)


def evict(**kw):
    return fill(capi.EvictArgs(), dict(dtype=capi.DVATTN_FLOAT32, W=2, Hkv=2, E=64, Ev=64, block_size=16, max_blocks_per_seq=4,
                                       sink=0, recent=0, num_blocks=8, positions=64), kw)


def append(**kw):
    return fill(capi.TreeAppendArgs(), dict(dtype=capi.DVATTN_FLOAT16, W=2, Hkv=2, E=64, Ev=64, S=8, A=4, R=32, block_size=16,
                                            max_blocks_per_seq=4, num_blocks=8), kw)


CASES = [
    ("dvattn_tree_sdpa", tree, [(dict(dtype=7), UNSUPPORTED), (dict(E=96, Ev=96), UNSUPPORTED), (dict(Ev=64), UNSUPPORTED),
                                (dict(Hq=64), UNSUPPORTED), (dict(Hq=33), INVALID), (dict(R=130), INVALID), (dict(R=63), INVALID),
                                (dict(block_size=0), INVALID), (dict(Hkv=0), INVALID), (dict(F=0), INVALID), (dict(S=-1), INVALID),
                                (dict(S=1025), UNSUPPORTED), (dict(W=-1), INVALID), (dict(), INVALID)]),
    ("dvattn_paged_mass", mass, [(dict(dtype=-1), UNSUPPORTED), (dict(E=96), UNSUPPORTED), (dict(Hq=66), UNSUPPORTED),
                                 (dict(Hq=33), INVALID), (dict(positions=-1), INVALID), (dict(S=1 << 20), UNSUPPORTED), (dict(), INVALID)]),
    ("dvattn_paged_evict", evict, [(dict(dtype=3), UNSUPPORTED), (dict(E=0), INVALID), (dict(E=6), UNSUPPORTED), (dict(sink=-1), INVALID),
                                   (dict(recent=-1), INVALID), (dict(positions=-1), INVALID), (dict(positions=1 << 31), UNSUPPORTED),
                                   (dict(W=40000), UNSUPPORTED), (dict(), INVALID)]),
]


@pytest.mark.parametrize("name,make,kw,status", [(n, m, kw, st) for n, m, cs in CASES for kw, st in cs])
def test_validation(name, make, kw, status):
    """The last entry of each list: sizes in order, but null pointers."""
    a = make(**kw)
    assert getattr(LIB, name)(ctypes.byref(a), None, 0, None) == status
    if kw:
        assert getattr(LIB, name + "_workspace_size")(ctypes.byref(a)) == 0


@pytest.mark.parametrize("kw,status", [(dict(dtype=9), UNSUPPORTED), (dict(A=-1), INVALID), (dict(S=-1), INVALID), (dict(R=33), INVALID),
                                       (dict(E=36), UNSUPPORTED), (dict(), INVALID)])
def test_append_validation(kw, status):
    assert LIB.dvattn_tree_append(ctypes.byref(append(**kw)), None) == status


def test_null_arguments_and_empty_calls():
    for name in ("dvattn_tree_sdpa", "dvattn_paged_mass", "dvattn_paged_evict"):
        assert getattr(LIB, name)(None, None, 0, None) == INVALID
        assert getattr(LIB, name + "_workspace_size")(None) == 0
    assert LIB.dvattn_tree_append(None, None) == INVALID
    for a in (tree(W=0), tree(S=0), tree(Hq=0)):
        assert LIB.dvattn_tree_sdpa(ctypes.byref(a), None, 0, None) == OK
    for a in (mass(W=0), mass(S=0), mass(F=0), mass(positions=0), mass(num_blocks=0)):
        assert LIB.dvattn_paged_mass(ctypes.byref(a), None, 0, None) == OK
    for a in (evict(W=0), evict(positions=0)):
        assert LIB.dvattn_paged_evict(ctypes.byref(a), None, 0, None) == OK
    for a in (append(W=0), append(S=0), append(A=0)):
        assert LIB.dvattn_tree_append(ctypes.byref(a), None) == OK
