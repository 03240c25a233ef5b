"""Two proxied EP buffers in a process, world 2 via subprocesses on one device."""

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("requires GPU", allow_module_level=True)

REPO = Path(__file__).resolve().parent.parent


def test_two_buffers_share_lane_streams():
    """Each rank's two proxies have 6 lanes on 2 streams (4 hardware queues):
    a lane waits for its own copies, and every payload arrives."""
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT="29483",
               WORLD_SIZE="2", PYTHONPATH=str(REPO), UCCL_EP_FORCE_PROXY="1",
               GPU_MAX_HW_QUEUES="4")
    worker = str(REPO / "tests" / "workers" / "ep_two_buffers_worker.py")
    ps = [subprocess.Popen([sys.executable, "-u", worker],
                           env=dict(env, RANK=str(r)), stdout=subprocess.PIPE,
                           stderr=subprocess.STDOUT) for r in range(2)]
    outs = []
    for p in ps:
        try:
            outs.append(p.communicate(timeout=110)[0].decode())
        except subprocess.TimeoutExpired:
            p.kill()
            outs.append(p.communicate()[0].decode() + "\nTIMEOUT")
    joined = "\n=====\n".join(outs)
    assert all(p.returncode == 0 for p in ps), joined
    assert joined.count("TWO BUFFERS OK") == 2, joined
