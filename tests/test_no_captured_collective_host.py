"""The averaged step refuses to be captured with its collectives inside (without a GPU: the capture is a stand-in)."""
import os
import subprocess
import sys

import pytest
import torch
import torch.distributed as dist

from conftest import REPO
from nextou_amd import ddp


@pytest.fixture()
def averager():
    ddp.init_single_process_group("gloo")
    net = torch.nn.Linear(4, 3)
    a = ddp.BucketedGradientAverager(net)
    yield net, a
    a.remove_hooks()
    dist.destroy_process_group()


def test_a_capture_of_the_collectives_is_refused(averager, monkeypatch):
    net, a = averager
    x = torch.randn(5, 4)
    a.zero_grad()
    net(x).sum().backward()
    a.finalize()
    want = net.weight.grad.clone()
    monkeypatch.setattr(ddp, "_capturing", lambda device: True, raising=False)
    with pytest.raises(RuntimeError, match="not captured"):
        a.zero_grad()                              # the step's first call: nothing has been recorded
    assert net.weight.grad is not None
    a.defer_collectives = True                     # the buckets are filled inside the capture, the collectives wait for the eager call
    a.zero_grad()
    net(x).sum().backward()
    a.fill_missing()
    with pytest.raises(RuntimeError, match="not captured"):
        a.reduce_all()
    monkeypatch.setattr(ddp, "_capturing", lambda device: False, raising=False)
    a.reduce_all()
    a.wait_all()
    a.finish_local()
    assert torch.equal(net.weight.grad, want)


def test_bench_refuses_one_graph_with_a_process_group():
    for args in (["--force-averager"], ["--gpus", "2"]):
        out = subprocess.run([sys.executable, os.path.join(REPO, "bench.py"), "--graph", "on"] + args, capture_output=True, text=True, timeout=300)
        assert out.returncode == 2 and "--graph on" in out.stderr and out.stdout == ""
