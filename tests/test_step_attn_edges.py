"""Edges of the step attention that its other tests leave out."""
import ctypes

import pytest
import torch

import hcp_ring_amd as H
from test_step_attn import AT, DESC, POOL, Step


# ---------------------------------------------------------------------------------
# a step without tokens
# ---------------------------------------------------------------------------------
@pytest.mark.parametrize("prefixes", [0, 3])
def test_an_empty_step_has_sizes_and_needs_no_workspace(hcp, prefixes):
    """0 is the answer for a bad shape, and a step of no tokens is none: its sizes are positive, and
    the call takes any workspace, or none."""
    L, d = H.lib(), H.DecodeDesc(**DESC)
    assert L.hcp_step_attn_plan_size(ctypes.byref(d), 0, prefixes) > 0
    assert L.hcp_step_attn_workspace_size(ctypes.byref(d), 0, prefixes) > 0
    shard = ctypes.byref(H.DecodeShard(AT, 3, 3, AT, 0))
    for ws, size in ((None, 0), (AT, 0), (AT, 1 << 20)):
        assert L.hcp_step_attn(ctypes.byref(d), ctypes.byref(H.PagedPool(*POOL)), 0, 1, H.View(0, 0, 0), AT, prefixes, shard, AT, 1 << 30,
                               2, H.View(0, 0, 0), None, ws, size, None) == 0, H.last_error()
    x = Step([0, 0], [3, 4], 4, 2, 64, ids=[0, -1], plens=[5]).device("cpu")
    assert H.step_attn_plan_size(x["q"], x["pool"], x["tables"], x["ptables"]) > 0
    assert H.step_attn_workspace_size(x["q"], x["pool"], x["tables"], x["ptables"]) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("prefix", [False, True])
def test_an_empty_step_runs(gpu, prefix):
    """No sequence has a new token: the plan and the call of every layer still go through."""
    step = Step([0, 0, 0], [3, 40, 0], 8, 2, 64, ids=[0, -1, 0] if prefix else None, plens=[37] if prefix else ())
    out, lse = step.run()
    assert out.shape == (8, 0, 64) and lse.shape == (8, 0)
    assert H.fetch_device_errors() == 0
