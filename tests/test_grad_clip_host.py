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
