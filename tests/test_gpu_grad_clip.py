"""clip_grad_norm_ on the GPU: gradients that go to torch's implementation, and the trainer's step that calls it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def optim():
    from nextou_amd import _lib, optim
    _lib.lib()
    assert "libnextou_hip.so" in open("/proc/self/maps").read(), "HIP extension not loaded into this process"
    return optim


def _with_grads(*grads):
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return params


@pytest.mark.parametrize("what", ["float64", "float64 among others", "two devices"])
def test_what_the_kernels_do_not_take_is_clipped_by_torch(optim, what):
    g = torch.Generator().manual_seed(3)
    make = lambda n, t, d: torch.randn(n, generator=g).to(t).to(d)  # noqa: E731
    grads = {"float64": [make(50, torch.float64, DEV), make(7, torch.float64, DEV)],
             "float64 among others": [make(50, torch.float32, DEV), make(7, torch.float64, DEV)],
             "two devices": [make(50, torch.float32, DEV), make(7, torch.float32, "cpu")]}[what]
    want = math.sqrt(sum(float((v.double() ** 2).sum()) for v in grads))
    before = [v.double().cpu() for v in grads]
    params = _with_grads(*grads)
    norm = optim.clip_grad_norm_(params, 1.0)
    # torch's float32 sums of 57 squares: at most 60 roundings of 2^-24, then the factor's three and the product's one
    assert abs(float(norm) - want) <= 64 * 2.0 ** -24 * want
    for p, b in zip(params, before):
        assert float((p.grad.double().cpu() - b / (want + 1e-6)).abs().max()) <= 72 * 2.0 ** -24 * float(b.abs().max()) / want


@pytest.mark.parametrize("t", [torch.float32, torch.float64], ids=str)
def test_train_step_with_another_optimizer(optim, t):
    """StandaloneTrainerBase.train_step with an optimizer that has no clip of its own: the update is 12 long"""
    from nextou_amd import harness
    g = torch.Generator().manual_seed(5)
    net = torch.nn.Linear(8, 5).to(t).to(DEV)
    trainer = object.__new__(harness.StandaloneTrainerBase)
    trainer.network, trainer.optimizer = net, torch.optim.SGD(net.parameters(), 0.5)
    trainer.loss = lambda out, target: ((out - target) ** 2).sum() * 1e3
    x, target = torch.randn(6, 8, generator=g).to(t).to(DEV), torch.randn(6, 5, generator=g).to(t).to(DEV)
    before = [p.detach().clone() for p in net.parameters()]
    loss = trainer.train_step(x, target)
    assert bool(torch.isfinite(loss))
    moved = torch.cat([((a - b).double() / 0.5).flatten() for a, b in zip(before, [p.detach() for p in net.parameters()])])
    # a value moves by up to 6 and is of that size: its rounding and the clip's are below 2^-20 of it
    assert abs(float(moved.norm()) - 12.0) <= 12.0 * 2.0 ** -18
