"""K11 (csrc/grad_norm.hip) on the GPU: the global norm of a gradient list and the clip, against the formula in float64.

The norm is a float64 sum rounded to float32 at the end: off by 2^-24 relative (the maximum is exact).  The clip factor is three float32
operations (1.5 * 2^-23), a clipped value one more rounding: half a step of its type."""
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


def _params(sizes, types, seed=0, scale=1.0, gap=0):
    """Parameters whose gradients are views into one flat buffer per type (odd offsets), NaN in the ``gap`` elements between them."""
    g = torch.Generator().manual_seed(seed)
    out, flats = [], {}
    for t in dict.fromkeys(types):
        total = sum(n + gap for n, s in zip(sizes, types) if s == t)
        flats[t] = [torch.full((total,), float("nan"), dtype=t, device=DEV), 0]
    for n, t in zip(sizes, types):
        flat, at = flats[t]
        p = torch.nn.Parameter(torch.empty(n, dtype=t, device=DEV))
        p.grad = flat[at:at + n]
        p.grad.copy_((torch.randn(n, generator=g) * scale).to(DEV))
        flats[t][1] = at + n + gap
        out.append(p)
    return out, [f for f, _ in flats.values()]


def _norm64(grads, p):
    parts = [g.double().abs() for g in grads if g.numel()]
    if p == math.inf:
        return max(float(a.max()) for a in parts)
    return sum(float((a ** p).sum()) for a in parts) ** (1 / p)


_LISTS = [
    ([1], ["f"]), ([3], ["b"]), ([7, 1, 9], ["h", "f", "b"]), ([16], ["b"]), ([8192, 8193, 4095, 4097], ["b", "b", "f", "f"]),
    ([33, 66, 132, 264, 1296] * 50, ["f", "b", "h", "b", "f"] * 50),                       # 250 tensors: the table is written to memory
    ([5, 700, 20000, 1] * 170, ["f", "f", "b", "h"] * 170), ([3_000_001, 17, 65536], ["b", "f", "h"]), ([40_000_003], ["f"]),
]
_T = {"f": torch.float32, "b": torch.bfloat16, "h": torch.float16}


@pytest.mark.parametrize("sizes,types", _LISTS, ids=[str(i) for i in range(len(_LISTS))])
@pytest.mark.parametrize("p", [2.0, 1.0, math.inf])
def test_norm_and_clip(optim, sizes, types, p):
    types = [_T[t] for t in types]
    params, flats = _params(sizes, types, seed=len(sizes), gap=3)
    grads = [q.grad.clone() for q in params]
    want = _norm64(grads, p)
    norm = optim.grad_norm([q.grad for q in params], p)
    assert norm.dtype == torch.float32 and norm.dim() == 0 and abs(float(norm) - want) <= 2.0 ** -23 * want
    assert all(torch.equal(a, q.grad) for a, q in zip(grads, params))
    for max_norm in (want * 2, want / 7):
        before = [f.clone() for f in flats]
        got = optim.clip_grad_norm_(params, max_norm, p)
        assert torch.equal(got, norm)
        c = min(1.0, max_norm / (want + 1e-6))
        for a, q in zip(grads, params):
            w = a.double() * c
            room = (2.0 ** -22 + torch.finfo(a.dtype).eps / 2) * w.abs() + torch.finfo(a.dtype).smallest_normal * torch.finfo(a.dtype).eps
            assert bool(((q.grad.double() - w).abs() <= (room if c < 1 else 0)).all())
        for f, b in zip(flats, before):                     # the gaps between the gradients are nobody's
            assert torch.equal(torch.isnan(f), torch.isnan(b))


def test_against_torch(optim):
    params, _ = _params([100, 5000, 33], [torch.float32] * 3, 4)
    others = [torch.nn.Parameter(q.detach().clone()) for q in params]
    for a, b in zip(params, others):
        b.grad = a.grad.clone()
    n1, n2 = optim.clip_grad_norm_(params, 0.5), torch.nn.utils.clip_grad_norm_(others, 0.5)
    assert abs(float(n1) - float(n2)) <= 1e-6 * float(n2)
    assert all(torch.allclose(a.grad, b.grad, rtol=1e-6, atol=0) for a, b in zip(params, others))


@pytest.mark.parametrize("t", list(_T.values()), ids=str)
def test_non_finite_large_and_tiny_values(optim, t):
    for p in (2.0, 1.0, math.inf):
        params, _ = _params([40, 9], [t, t], 3)
        params[1].grad[8] = float("nan")
        assert math.isnan(float(optim.grad_norm([q.grad for q in params], p)))
        with pytest.raises(RuntimeError, match="non-finite"):
            optim.clip_grad_norm_(params, 1.0, p, error_if_nonfinite=True)
        assert not bool(torch.isnan(params[0].grad).any())             # raised before anything was scaled
        optim.clip_grad_norm_(params, 1.0, p)
        assert all(bool(torch.isnan(q.grad).all()) for q in params)
        params, _ = _params([40, 9], [t, t], 3)
        params[0].grad[1] = -float("inf")
        assert float(optim.clip_grad_norm_(params, 1.0, p)) == math.inf
        assert bool(torch.isnan(params[0].grad[1])) and float(params[1].grad.abs().max()) == 0.0
    big = torch.finfo(t).max
    g = torch.full((3,), big, dtype=t, device=DEV)
    assert abs(float(optim.grad_norm([g[:1]])) / big - 1) <= 2.0 ** -23         # the squares leave float32's range, not float64's
    assert float(optim.grad_norm([g], math.inf)) == big
    tiny = torch.full((4,), torch.finfo(t).smallest_normal, dtype=t, device=DEV)
    assert abs(float(optim.grad_norm([tiny])) / (2 * torch.finfo(t).smallest_normal) - 1) <= 2.0 ** -23
    zero, _ = _params([12], [t])
    zero[0].grad.zero_()
    assert float(optim.clip_grad_norm_(zero, 1.0)) == 0.0 and float(zero[0].grad.abs().max()) == 0.0
    some, _ = _params([12], [t])
    optim.clip_grad_norm_(some, 0.0)
    assert float(some[0].grad.abs().max()) == 0.0


def test_layouts_and_refusals(optim):
    last = torch.nn.Parameter(torch.randn(4, 6, 3, 3, 3, device=DEV).contiguous(memory_format=torch.channels_last_3d))
    last.grad = torch.randn_like(last)
    wide = torch.randn(20, 30, device=DEV)
    part = torch.nn.Parameter(torch.empty(20, 7, device=DEV))
    part.grad = wide[:, 3:10]
    none, empty = torch.nn.Parameter(torch.empty(3, device=DEV)), torch.nn.Parameter(torch.empty(0, device=DEV))
    empty.grad = torch.empty(0, device=DEV)
    before, around = [last.grad.clone(), part.grad.clone()], wide.clone()
    want = _norm64(before, 2)
    norm = optim.clip_grad_norm_((q for q in (last, none, part, empty)), 1.0)
    assert abs(float(norm) - want) <= 2.0 ** -22 * want
    assert torch.allclose(last.grad, before[0] / want, rtol=1e-5) and torch.allclose(part.grad, before[1] / want, rtol=1e-5)
    around[:, 3:10] = wide[:, 3:10]
    assert torch.equal(around, wide)
    assert float(optim.clip_grad_norm_([empty], 1.0)) == 0.0 and float(optim.grad_norm(empty.grad)) == 0.0
    assert abs(float(optim.grad_norm(torch.ones(1, 5, device=DEV).expand(4, 5), 1.0)) - 20) == 0
    with pytest.raises(RuntimeError, match="overlap"):
        optim.clip_grad_norm_([last, last], 1.0)
    assert torch.allclose(last.grad, before[0] / want, rtol=1e-5)        # refused before anything ran
    with pytest.raises(ValueError, match="overlaps itself"):
        part.grad = torch.ones(1, 7, device=DEV).expand(20, 7)
        optim.clip_grad_norm_([part], 1.0)
    with pytest.raises(TypeError):
        optim.grad_norm([torch.randn(3, device=DEV, dtype=torch.float64)])
    with pytest.raises(ValueError, match="gradients on"):
        optim.grad_norm([torch.randn(3, device=DEV), torch.randn(3)])


def test_captured_clip_on_another_stream(optim):
    for count in (5, 400):
        sizes, types = [1 + 37 * (i % 11) for i in range(count)], [[torch.float32, torch.bfloat16][i % 2] for i in range(count)]
        params, flats = _params(sizes, types, 1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            optim.clip_grad_norm_(params, 1.0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = optim.clip_grad_norm_(params, 1.0)
        for seed in (2, 3, 4):
            fresh, new = _params(sizes, types, seed)
            for f, n in zip(flats, new):
                f.copy_(n)
            graph.replay()
            eager = optim.clip_grad_norm_(fresh, 1.0)
            torch.cuda.synchronize()
            assert torch.equal(norm, eager) and all(torch.equal(a.grad, b.grad) for a, b in zip(params, fresh))


def test_clip_sgd_over_two_groups(optim):
    g = torch.Generator().manual_seed(6)
    make = lambda: [torch.nn.Parameter(torch.randn(n, generator=g).to(DEV)) for n in (300, 7, 5000)]  # noqa: E731
    own_p = make()
    ref_p = [torch.nn.Parameter(q.detach().clone()) for q in own_p]
    groups = lambda ps: [{"params": ps[:2], "lr": 0.1}, {"params": ps[2:], "lr": 0.02, "momentum": 0.5, "nesterov": False}]  # noqa: E731
    own, ref = optim.ClipSGD(groups(own_p), 0.1, momentum=0.9, nesterov=True), torch.optim.SGD(groups(ref_p), 0.1, momentum=0.9, nesterov=True)
    for step in range(3):
        for a, b in zip(own_p, ref_p):
            b.grad = torch.randn(a.shape, generator=g).to(DEV)
            a.grad = b.grad.clone()
        norm = own.clip_and_step(3.0)
        want = torch.nn.utils.clip_grad_norm_(ref_p, 3.0)
        ref.step()
        assert own.last_path == "own" and abs(float(norm) - float(want)) <= 1e-6 * float(want)
        assert all(torch.allclose(a, b, rtol=2e-6, atol=1e-6) for a, b in zip(own_p, ref_p))


def test_layer_then_clip_as_in_a_step(optim):
    """The operators together: a 16-bit point-wise block with a float32 bias, its gradients, one clip over both types — eager and captured."""
    from nextou_amd import graph_ops
    g = torch.Generator().manual_seed(8)
    w1 = torch.nn.Parameter((torch.randn(96, 40, generator=g) * 0.2).bfloat16().to(DEV))
    w2 = torch.nn.Parameter((torch.randn(40, 96, generator=g) * 0.2).bfloat16().to(DEV))
    b1, b2 = torch.nn.Parameter(torch.zeros(96, device=DEV)), torch.nn.Parameter(torch.zeros(40, device=DEV))
    params = [w1, b1, w2, b2]
    x, gy = (torch.randn(500, 40, generator=g).bfloat16().to(DEV) for _ in range(2))

    def step():
        h = graph_ops.linear_act(x, w1, b1, act="gelu")
        y = graph_ops.linear_act(h, w2, b2, residual=x)
        for p, v in zip(params, torch.autograd.grad(y, params, gy)):
            p.grad = v
        return optim.clip_grad_norm_(params, 1.0)

    xd, wd = x.double(), [w1.detach().double().requires_grad_(True), w2.detach().double().requires_grad_(True)]
    h = torch.nn.functional.gelu(xd @ wd[0].t())
    grads64 = torch.autograd.grad(h @ wd[1].t() + xd, wd, gy.double())
    norm = step()
    total = math.sqrt(sum(float((q.grad.double() ** 2).sum()) for q in params))
    assert abs(total - 1.0) < 2.0 ** -8                        # every value half a bfloat16 step off at most
    for q, want in zip((w1, w2), grads64):                     # h, dz and the gradient are each rounded to bfloat16: four roundings in norm
        d = q.grad.double() * float(norm) - want
        assert float(d.norm()) <= 4 * 2.0 ** -8 * float(want.norm())
    eager = [q.grad.clone() for q in params]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, norm) and all(torch.equal(a, q.grad) for a, q in zip(eager, params))
