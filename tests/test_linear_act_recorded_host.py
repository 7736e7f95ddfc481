"""linear_act where torch records its operations without any tensor requiring a gradient (a trace, forward-mode derivatives), over a backend
that writes its result through the output's address, as the kernels do."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from nextou_amd import graph_ops
from oracle.ref_ops import TorchRefBackend


class _ByAddress(TorchRefBackend):
    @staticmethod
    def linear_act_fwd(x, w, bias, residual, act, slope, groups, want_pre):
        with torch.inference_mode():
            copies = [None if t is None else torch.frombuffer(bytearray(bytes(t.contiguous().numpy().tobytes())), dtype=t.dtype).view(t.shape)
                      for t in (x.detach(), w.detach(), bias if bias is None else bias.detach(), residual if residual is None else residual.detach())]
            value = TorchRefBackend.linear_act_fwd(*copies, act, slope, groups, False)[0].contiguous()
        y = x.new_empty((x.shape[0], w.shape[0]))
        ctypes.memmove(y.data_ptr(), value.data_ptr(), 4 * value.numel())
        return y, None


@pytest.fixture()
def by_address():
    graph_ops.install_cpu_checker(_ByAddress)
    yield
    graph_ops.install_cpu_checker(None)


def _inputs(seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g) for s in ((6, 4), (3, 4), (3,), (6, 3))]


@pytest.mark.parametrize("which", range(4))
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_never_dropped(by_address, which, grad):
    ts = _inputs(1)
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        plain = graph_ops.linear_act(*ts, act="gelu")                  # no tangent: the value
        assert torch.allclose(plain, torch.nn.functional.gelu(ts[0] @ ts[1].t() + ts[2]) + ts[3], atol=1e-5)
        ts[which] = fwAD.make_dual(ts[which], torch.ones_like(ts[which]))
        with pytest.raises(NotImplementedError):
            graph_ops.linear_act(*ts, act="gelu")


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("grad", [True, False])
def test_a_trace_holds_the_operator(by_address, grad):
    with torch.set_grad_enabled(grad):
        traced = torch.jit.trace(lambda *t: graph_ops.linear_act(*t, act="relu"), _inputs(1), check_trace=False)
        for seed in (1, 2, 3):
            ts = _inputs(seed)
            assert torch.allclose(traced(*ts), torch.relu(ts[0] @ ts[1].t() + ts[2]) + ts[3], atol=1e-5)
