"""Bounded waits that run out in the 8-bit decode attention are reported: the call's error word is set, its outputs are NaN,
the torch op raises with DVATTN_CHECK_STATUS=1, and the context stays usable.  As in test_status_gpu.py the failing case
faults nothing: DVATTN_TEST_STALL_TILE makes the first CTA never hand over one window (read once per process, hence the
child processes)."""
import os
import subprocess
import sys

import pytest
import torch

import test_q8_gpu as q8

from dvattn_b200 import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_CHILD = r"""
import sys
import torch
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/tests"]
import dvattn_b200
import test_q8_gpu as q8
from dvattn_b200 import capi
what, S, BS = sys.argv[2], int(sys.argv[3]), int(sys.argv[4])
c = q8.on_gpu(q8.make([[60000, 77], [40, 80000]], S, 32, 4, 128, 64, BS, torch.bfloat16))
out, lse = torch.zeros_like(c["q"]), torch.zeros(c["q"].shape[:3], device="cuda:0")
if what == "capi":
    ws = capi.paged_sdpa_q8(out, c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"], lse=lse)
    word = capi.workspace_status(ws)
    assert word != 0, "error word not set"
    assert torch.isnan(out.float()).all() and torch.isnan(lse).all(), "outputs not marked invalid"
else:
    try:
        dvattn_b200.dvattn_paged_sdpa_q8(c["q"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"], c["scale"])
    except RuntimeError as e:
        assert "bounded wait" in str(e), str(e)
        word = "raised"
    else:
        raise SystemExit("the op did not raise")
assert torch.arange(10, device="cuda:0").sum().item() == 45  # the context is still usable
print(what, word)
"""


@pytest.mark.parametrize("S, BS", [(1, 16), (5, 6)])  # one row tile and TMA boxes, several and gathered rows
@pytest.mark.parametrize("tile", [0, 1])              # a CTA's first window, or a later one
@pytest.mark.parametrize("what", ["capi", "op"])
def test_stalled_wait_is_reported(what, tile, S, BS):
    env = dict(os.environ, DVATTN_TEST_STALL_TILE=str(tile), DVATTN_CHECK_STATUS="1")
    r = subprocess.run([sys.executable, "-c", _CHILD, ROOT, what, str(S), str(BS)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout[-2000:], r.stderr[-3000:])
    assert r.stdout.startswith(what), r.stderr[-2000:]


def test_status_zero_after_completed_calls():
    c = q8.on_gpu(q8.make([[300, 77], [40, 500]], 1, 16, 2, 128, 64, 16, torch.bfloat16))
    out, ws = torch.zeros_like(c["q"]), None
    for _ in range(2):  # a workspace is used again as it is
        ws = capi.paged_sdpa_q8(out, c["scale"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["ks"], c["vs"], c["bt"],
                                workspace=ws)
        assert capi.workspace_status(ws) == 0
