"""grad_norm / clip_grad_norm_ without a GPU: what reaches the kernels, and what goes to torch's implementation.  Device tensors are host
tensors that say is_cuda; the library is a stand-in on host memory."""
import ctypes
import math

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

from nextou_amd import _lib, optim


class _StandInLib:
    """nextou_multi_norm / nextou_multi_clip on host memory, as include/nextou_hip.h describes them (float32)."""

    def __init__(self):
        self.calls = 0

    def nextou_multi_norm_workspace(self, n, out):
        out._obj.value = 64
        return 0

    def _run(self, table, n, max_norm, out, scale):
        self.calls += 1
        rows = np.ctypeslib.as_array(ctypes.cast(table, ctypes.POINTER(ctypes.c_int64)), (n, 3))
        vals = [np.ctypeslib.as_array(ctypes.cast(int(p), ctypes.POINTER(ctypes.c_float)), (int(c),)) for p, c, _ in rows]
        norm = math.sqrt(sum(float((v.astype(np.float64) ** 2).sum()) for v in vals))
        factor = min(1.0, max_norm / (norm + 1e-6))
        np.ctypeslib.as_array(ctypes.cast(out, ctypes.POINTER(ctypes.c_float)), (2,))[:] = [norm, factor]
        for v in vals if scale else ():
            v *= np.float32(factor)
        return 0

    def nextou_multi_norm(self, table, n, norm, max_norm, ws, ws_bytes, out, stream):
        return self._run(table, n, max_norm, out, False)

    def nextou_multi_clip(self, table, n, norm, max_norm, ws, ws_bytes, out, stream):
        return self._run(table, n, max_norm, out, True)


@pytest.fixture()
def kernels(monkeypatch):
    """The GPU path on host tensors"""
    import contextlib
    fake = _StandInLib()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))
    monkeypatch.setattr(optim, "_current_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(optim, "_raw_stream", lambda index: 0)
    optim._multi_norm_bytes.cache_clear()
    yield fake
    optim._multi_norm_bytes.cache_clear()


def _with_grads(*grads):
    params = [torch.nn.Parameter(torch.zeros(g.shape, dtype=g.dtype)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    return params


def test_plain_gradients_reach_the_kernels(kernels):
    params = _with_grads(torch.full((4,), 3.0), torch.full((3, 2), 2.0))
    norm = math.sqrt(4 * 9 + 6 * 4)
    assert abs(float(optim.grad_norm([p.grad for p in params])) - norm) < 1e-6 and kernels.calls == 1
    assert abs(float(optim.clip_grad_norm_(params, 1.0)) - norm) < 1e-6 and kernels.calls == 2
    assert torch.allclose(params[1].grad, torch.full((3, 2), 2.0 / norm))


@pytest.mark.filterwarnings("ignore::DeprecationWarning")
def test_a_trace_holds_the_norm_and_the_clip(kernels):
    def clipped(a, b):
        a, b = a * 1.0, b * 1.0
        norm = optim.clip_grad_norm_(_with_grads(a, b), 1.0)
        return norm, a, b

    def example(seed):
        g = torch.Generator().manual_seed(seed)
        return torch.randn(5, generator=g), torch.randn(2, 3, generator=g)

    norm = torch.jit.trace(lambda a, b: optim.grad_norm([a, b]), example(1), check_trace=False)
    clip = torch.jit.trace(clipped, example(1), check_trace=False)
    for seed in (1, 2, 3):
        a, b = example(seed)
        want = torch.cat([a, b.flatten()]).norm()
        assert torch.allclose(norm(a, b), want)
        got, ca, cb = clip(a, b)
        assert torch.allclose(got, want) and torch.allclose(ca, a / want, atol=1e-5) and torch.allclose(cb, b / want, atol=1e-5)
    assert kernels.calls == 0


def test_a_tangent_is_not_dropped(kernels):
    with fwAD.dual_level():
        a = fwAD.make_dual(torch.randn(5), torch.randn(5))
        for call in (lambda: optim.grad_norm([a]), lambda: optim.clip_grad_norm_(_with_grads(a), 1.0)):
            try:
                out = call()
            except RuntimeError:                 # torch's own operator has no such derivative
                continue
            assert fwAD.unpack_dual(out).tangent is not None
    assert kernels.calls == 0


def _as_torch_clips(grads, max_norm=1.0):
    """(norm, gradients) of torch's clip on copies of the same layout"""
    params = _with_grads(*[torch.empty_strided(g.shape, g.stride(), dtype=g.dtype).copy_(g) for g in grads])
    return torch.nn.utils.clip_grad_norm_(params, max_norm), [p.grad for p in params]


@pytest.mark.parametrize("what", ["float64", "float64 among others", "sparse"])
@pytest.mark.parametrize("error_if_nonfinite", [False, True])
def test_what_the_kernels_do_not_take_is_clipped_by_torch(kernels, what, error_if_nonfinite):
    grads = {"float64": [torch.randn(5).double(), torch.randn(2, 3).double()],
             "float64 among others": [torch.randn(6), torch.randn(5).double(), torch.randn(4, 6)[:, :3]],
             "sparse": [torch.eye(4).to_sparse().coalesce()]}[what]
    if what == "sparse":
        params = _with_grads(grads[0].clone())
        try:
            want = torch.nn.utils.clip_grad_norm_(_with_grads(grads[0].clone()), 1.0)
        except Exception as refused:             # as torch has it
            with pytest.raises(type(refused)):
                optim.clip_grad_norm_(params, 1.0, error_if_nonfinite=error_if_nonfinite)
        else:
            assert float(optim.clip_grad_norm_(params, 1.0, error_if_nonfinite=error_if_nonfinite)) == float(want)
    else:
        want, clipped = _as_torch_clips(grads)
        params = _with_grads(*grads)
        norm = optim.clip_grad_norm_(params, 1.0, error_if_nonfinite=error_if_nonfinite)
        assert torch.equal(norm, want) and all(torch.equal(p.grad, c) for p, c in zip(params, clipped))
    assert kernels.calls == 0


def test_a_distributed_gradient_is_clipped_by_torch(kernels):
    """A tensor of several processes has no address of its own."""
    import torch.distributed as dist
    from nextou_amd import ddp
    from torch.distributed.tensor import Shard, distribute_tensor, init_device_mesh
    ddp.init_single_process_group("gloo")
    try:
        g = torch.randn(6, 4)
        d = distribute_tensor(g, init_device_mesh("cpu", (1,)), [Shard(0)])
        p = torch.nn.Parameter(torch.zeros_like(d))
        p.grad = d.clone()
        optim.clip_grad_norm_([p], 1.0)
        assert torch.allclose(p.grad.full_tensor(), g / g.norm(), atol=1e-6)
        with pytest.raises(TypeError):
            optim.grad_norm([d])
    finally:
        dist.destroy_process_group()
    assert kernels.calls == 0


def test_train_step_clips_float64_parameters_with_another_optimizer(kernels):
    """The trainer's step of an optimizer without a clip of its own, as it ran on torch's clip"""
    from nextou_amd import harness
    net = torch.nn.Linear(4, 3).double()
    trainer = object.__new__(harness.StandaloneTrainerBase)
    trainer.network, trainer.optimizer = net, torch.optim.SGD(net.parameters(), 0.5)
    trainer.loss = lambda out, target: ((out - target) ** 2).sum() * 1e3
    x, t = torch.randn(6, 4).double(), torch.randn(6, 3).double()
    before = [p.detach().clone() for p in net.parameters()]
    trainer.train_step(x, t)
    moved = torch.cat([((a - b) / 0.5).flatten() for a, b in zip(before, [p.detach() for p in net.parameters()])])
    assert abs(float(moved.norm()) - 12.0) < 1e-4


def test_strided_gradients_that_share_an_element_are_refused(kernels):
    base = torch.randn(12, 16)
    apart = [
        [base[:, :4], base[:, 4:8], base[:, 8:]], [base[::2, :4], base[1::2, :4]], [base[:6, ::2], base[:6, 1::2]], [base[2:5, 3:6], base[5:9, 3:6]],
        [base[:, :4], base[3, 4:16]], [base[:, 1], base[:, 2]], [base.t()[:4], base[:, 4:]], [base[:, :4], base[:, 5:6], torch.randn(3)],
        [base[:, 14:], base.view(-1)[16:30]], [base.view(-1)[0:64:4], base.view(-1)[1:64:4]],
    ]
    share = [
        [base[:, :4], base[:, 2:6]], [base[:, :4], base[::3, 3:5]], [base[:, :4], base], [base[:, 4:8], base.view(-1)[7:9]], [base[1:, :4], base[:-1, :4]],
        [base[:, :4].t(), base[:, 3]], [base.view(-1)[0:64:4], base.view(-1)[2:64:6]], [base[:, :4], torch.randn(3), base[:, :4]],
        [base[:, :4], base[0, 0]], [base.view(torch.bfloat16)[:, 1:4], base[:, 1:3]],
    ]
    for views in apart:
        grads = [v.clone() for v in views]
        want = math.sqrt(sum(float((v.double() ** 2).sum()) for v in grads))
        optim.clip_grad_norm_(_with_grads(*views), want / 2)
        assert all(torch.allclose(v, g / 2, rtol=1e-5) for v, g in zip(views, grads))
    before = base.clone()
    for views in share:
        for order in (views, views[::-1]):
            with pytest.raises(RuntimeError, match="share memory"):
                optim.clip_grad_norm_(_with_grads(*order), 1e-3)
    assert torch.equal(base, before)
    assert float(optim.grad_norm([base[:, :4], base[:, 2:6]])) > 0          # a norm only reads


def test_interleaved_dimensions_without_a_common_element_are_taken(kernels):
    base = torch.randn(12)
    view = base.as_strided((2, 3), (3, 2))                     # elements 0, 2, 4, 3, 5, 7
    want, around = view.clone(), base[[1, 6, 8, 9, 10, 11]].clone()
    optim.clip_grad_norm_(_with_grads(view), float(want.norm()) / 2)
    assert torch.allclose(view, want / 2, rtol=1e-5) and torch.equal(base[[1, 6, 8, 9, 10, 11]], around)
    with pytest.raises(ValueError, match="overlaps itself"):
        optim.clip_grad_norm_(_with_grads(base.as_strided((2, 3), (4, 2))), 1.0)


@pytest.mark.parametrize("strided", [False, True])
def test_a_graph_that_saved_a_gradient_notices_the_clip(kernels, strided):
    x = torch.randn(6, 4, requires_grad=True)
    (g,) = torch.autograd.grad((x ** 3).sum(), (x,), create_graph=True)
    if strided:
        g = torch.cat([g, g], 1)[:, 1:5]
    penalty = (g ** 2).sum()                                   # saves g
    params = _with_grads(g.detach())
    optim.grad_norm([p.grad for p in params])                  # only reads
    penalty.backward(retain_graph=True)
    optim.clip_grad_norm_(params, 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        penalty.backward()


def test_a_graph_that_saved_a_parameter_notices_the_step(monkeypatch):
    """ClipSGD's own kernels, over two parameter groups"""
    from test_linear_act_host import _StandInLib as StepLib
    fake = StepLib()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    a, b = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(4))
    opt = optim.ClipSGD([{"params": [a], "lr": 0.5}, {"params": [b], "lr": 0.25}], 0.1)
    opt._device_type = "cpu"
    loss = (a * b).sum()
    loss.backward(retain_graph=True)
    opt.clip_and_step(1.0)
    assert opt.last_path == "own"
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
