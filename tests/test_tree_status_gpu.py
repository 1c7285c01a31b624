"""Bounded waits that run out in the draft-tree attention and the attention mass are reported:
the call's error word is set, the tree attention's outputs are NaN, the torch ops raise with
DVATTN_CHECK_STATUS=1, and the context stays usable.  As in test_status_gpu.py the failing case
faults nothing: DVATTN_TEST_STALL_TILE makes the first CTA never hand over one key tile (read
once per process, hence the child processes)."""
import os
import subprocess
import sys

import pytest
import torch

import test_tree_gpu as tree

from dvattn_b200 import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

_CHILD = r"""
import sys
import torch
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/tests"]
import dvattn_b200
import test_tree_gpu as tree
from dvattn_b200 import capi
what, S, BS = sys.argv[2], int(sys.argv[3]), int(sys.argv[4])
c = tree.on_gpu(tree.make([[300, 77], [40, 500]], S, 16, 2, 128, 64, BS, torch.bfloat16))
mass = torch.zeros((2, 2, 640), device="cuda:0")
lse = torch.zeros((2, 16, S), device="cuda:0")
out = torch.zeros_like(c["q"])
if what == "tree":
    ws = capi.tree_sdpa(out, c["scale"], c["parents"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"],
                        c["dk"], c["dv"], lse=lse)
    word = capi.workspace_status(ws)
    assert word != 0, "error word not set"
    assert torch.isnan(out.float()).all() and torch.isnan(lse).all(), "outputs not marked invalid"
elif what == "mass":
    ws = capi.paged_mass(mass, c["scale"], c["loc"], c["q"], lse, c["cos"], c["sin"], c["L"], c["kc"], c["bt"])
    word = capi.workspace_status(ws)
    assert word != 0, "error word not set"
else:
    try:
        if what == "tree_op":
            dvattn_b200.dvattn_tree_sdpa(c["q"], c["parents"], c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"],
                                         c["dk"], c["dv"], c["scale"])
        else:
            dvattn_b200.dvattn_paged_mass(mass, c["q"], lse, c["loc"], c["cos"], c["sin"], c["L"], c["kc"], c["bt"], c["scale"])
    except RuntimeError as e:
        assert "bounded wait" in str(e), str(e)
        word = "raised"
    else:
        raise SystemExit("the op did not raise")
assert torch.arange(10, device="cuda:0").sum().item() == 45  # the context is still usable
print(what, word)
"""


@pytest.mark.parametrize("S, BS", [(4, 16), (40, 6)])  # one row tile and TMA boxes, several and gathered rows
@pytest.mark.parametrize("what", ["tree", "tree_op", "mass", "mass_op"])
def test_stalled_wait_is_reported(what, S, BS):
    env = dict(os.environ, DVATTN_TEST_STALL_TILE="0", DVATTN_CHECK_STATUS="1")
    r = subprocess.run([sys.executable, "-c", _CHILD, ROOT, what, str(S), str(BS)], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout[-2000:], r.stderr[-3000:])
    assert r.stdout.startswith(what), r.stderr[-2000:]


def test_status_zero_after_completed_calls():
    c = tree.on_gpu(tree.make([[300, 77], [40, 500]], 4, 16, 2, 128, 64, 16, torch.bfloat16))
    out, lse = torch.zeros_like(c["q"]), torch.zeros((2, 16, 4), device=DEV)
    mass = torch.zeros((2, 2, 640), device=DEV)
    ws = mws = None
    for _ in range(2):  # a workspace is used again as it is
        ws = capi.tree_sdpa(out, c["scale"], c["parents"], c["loc"], c["q"], c["cos"], c["sin"], c["L"], c["kc"], c["vc"], c["bt"],
                            c["dk"], c["dv"], lse=lse, workspace=ws)
        assert capi.workspace_status(ws) == 0
        mws = capi.paged_mass(mass, c["scale"], c["loc"], c["q"], lse, c["cos"], c["sin"], c["L"], c["kc"], c["bt"], workspace=mws)
        assert capi.workspace_status(mws) == 0
