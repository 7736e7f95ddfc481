"""K10 (csrc/linear_act.hip) at the ends of its ranges: values near the largest of a type, and sizes that a launch cannot hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    from nextou_amd import _lib, graph_ops
    _lib.lib()
    assert "libnextou_hip.so" in open("/proc/self/maps").read(), "HIP extension not loaded into this process"
    return graph_ops


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("act", ["none", "relu", "leakyrelu", "gelu", "hswish"])
@pytest.mark.parametrize("rows,width", [(8, 1), (70, 1), (8, 40), (300, 40)])
def test_activations_of_the_largest_values(ops, t, act, rows, width):
    """One column of x reaches the sum with weight one, so z is x exactly, and every activation of a large z is z or (leaky ReLU: a part of z) 0."""
    top = torch.finfo(t).max
    values = torch.tensor([top, -top, top / 2, -top / 2, top / 5, -top / 5, 100.0, -100.0], dtype=t, device=DEV)
    x = torch.zeros(rows, width, dtype=t, device=DEV)
    x[:, width - 1] = values.repeat((rows + 7) // 8)[:rows]
    w = torch.zeros(12, width, dtype=t, device=DEV)
    w[:, width - 1] = 1.0
    z = x[:, width - 1:].double()
    want = {"none": z, "leakyrelu": torch.where(z > 0, z, z * 0.25)}.get(act, z.clamp_min(0)).expand(rows, 12)
    with torch.no_grad():
        y = ops.linear_act(x, w, act=act, negative_slope=0.25)
    assert torch.equal(y.double(), want)
