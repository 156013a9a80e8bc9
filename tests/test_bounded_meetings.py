"""The two softmax warps of 32 rows meet at a hardware barrier, which has no
time limit: a warp that gives up a wait of its own must let the other go."""

import os
import re
import time

import pytest
import torch

from pir2_b200 import _lib

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")


@pytest.mark.parametrize("name", ["attention_tile.cuh", "attention_few.cuh", "kv_cache.cuh"])
def test_ragged_kernels_meet_only_where_a_warp_can_leave(name):
    """Between roles they wait through mbar_wait (bounded) and
    PairMeeting; whole CTAs and clusters meet where every thread comes."""
    with open(os.path.join(CSRC, name)) as f:
        code = re.sub(r"//.*", "", f.read())
    assert not re.search(r"named_barrier|bar\.sync|bar\.red|bar\.arrive|barrier\.cta|barrier\.sync", code)
    # Every wait of a softmax warp that runs out is followed by leave().
    if name == "attention_tile.cuh":
        softmax = code[code.index("PairMeeting pair{") : code.index("kIdescO")]
        assert softmax.count("mbar_wait(") == softmax.count("pair.leave()") == 2


@pytest.mark.gpu
def test_a_warp_that_gives_up_lets_the_other_go():
    assert _lib.device_status() == 0
    result = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    begin = time.perf_counter()
    _lib.wait_probe(result)
    torch.cuda.synchronize()
    assert time.perf_counter() - begin < 30.0
    assert result.item() == 0            # neither the wait nor the meeting succeeded
    assert _lib.device_status() == _lib.STATUS_TIMEOUT_PROBE
