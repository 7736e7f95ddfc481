"""linear_act / pointwise_act and the gradient norm without a GPU: refusals, the autograd plumbing over the float64 checker (against torch's
autograd of the formula and against differences), the C entries' argument checks, ClipSGD's clip over several groups."""
import ctypes
import math

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from nextou_amd import _lib, graph_ops, optim

_ACTS = {"none": lambda z: z, "relu": F.relu, "leakyrelu": lambda z: F.leaky_relu(z, 0.2), "gelu": F.gelu, "hswish": F.hardswish}


def _formula(x, w, b, r, act, groups):
    xg = x.reshape(-1, groups, w.shape[1])
    wg = w.reshape(groups, -1, w.shape[1])
    z = torch.stack([xg[:, g] @ wg[g].t() for g in range(groups)], 1).reshape(x.shape[:-1] + (w.shape[0],))
    y = _ACTS[act](z if b is None else z + b)
    return y if r is None else y + r


@pytest.mark.parametrize("act", sorted(_ACTS))
@pytest.mark.parametrize("groups", [1, 3])
def test_gradients_are_the_formulas_and_the_differences(torch_ref_checker, act, groups):
    g = torch.Generator().manual_seed(groups)
    x, w = torch.randn(2, 5, 4 * groups, generator=g), torch.randn(3 * groups, 4, generator=g)
    b, r = torch.randn(3 * groups, generator=g), torch.randn(2, 5, 3 * groups, generator=g)
    gy = torch.randn(2, 5, 3 * groups, generator=g)
    leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
    y = graph_ops.linear_act(x, w, b, r, act, 0.2, groups)
    got = torch.autograd.grad(y, leaves, gy)
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    want_y = _formula(*wide, act, groups)
    want = torch.autograd.grad(want_y, wide, gy.double())
    assert float((y - want_y).detach().abs().max()) < 1e-5
    for a, c in zip(got, want):
        assert a.dtype == torch.float32 and a.shape == c.shape and float((a - c).abs().max()) < 1e-5 * max(1.0, float(c.abs().max()))
    # a difference along a random direction (float64 formula): d/dt f(v + t u) = <grad, u>
    us = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in wide]
    h = 1e-6
    with torch.no_grad():
        ends = [(_formula(*[t + s * h * u for t, u in zip(wide, us)], act, groups) * gy.double()).sum() for s in (1, -1)]
    slope = float(ends[0] - ends[1]) / (2 * h)
    assert abs(slope - sum(float((a.double() * u).sum()) for a, u in zip(got, us))) < 1e-4 * max(1.0, abs(slope))


def test_only_the_wanted_gradients_and_no_rows(torch_ref_checker):
    x, w, b = torch.randn(6, 4), torch.randn(3, 4, requires_grad=True), torch.randn(3)
    (gw,) = torch.autograd.grad(graph_ops.linear_act(x, w, b, act="gelu").sum(), (w,))
    assert gw.shape == w.shape
    r = torch.randn(1, 3, requires_grad=True)               # a broadcast shortcut: expand's own gradient sums it
    (gr,) = torch.autograd.grad(graph_ops.linear_act(x, w.detach(), None, r.expand(6, 3)).sum(), (r,))
    assert torch.equal(gr, torch.full((1, 3), 6.0))
    x0, bb = torch.randn(0, 4, requires_grad=True), torch.randn(3, requires_grad=True)
    y = graph_ops.linear_act(x0, w, bb, act="relu")
    assert y.shape == (0, 3)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x0, w, bb))
    assert gx.shape == (0, 4) and float(gw.abs().sum()) == 0 and float(gb.abs().sum()) == 0
    with torch.no_grad():
        assert not graph_ops.linear_act(x, w, b).requires_grad


def test_pointwise_act_is_the_convolution(torch_ref_checker):
    g = torch.Generator().manual_seed(4)
    x, w, b = torch.randn(2, 6, 3, 4, 5, generator=g), torch.randn(8, 3, 1, 1, 1, generator=g), torch.randn(8, generator=g)
    r = torch.randn(2, 8, 3, 4, 5, generator=g)
    want = F.leaky_relu(F.conv3d(x, w, b, groups=2), 0.01) + r
    for xi in (x, x.contiguous(memory_format=torch.channels_last_3d)):
        y = graph_ops.pointwise_act(xi, w, b, r, "leakyrelu", groups=2)
        assert y.shape == want.shape and y.is_contiguous(memory_format=torch.channels_last_3d)
        assert float((y - want).abs().max()) < 1e-5
    with pytest.raises(ValueError, match="kernel-1"):
        graph_ops.pointwise_act(x, torch.randn(8, 6, 3, 3, 3))


def test_linear_act_refuses_what_does_not_fit(torch_ref_checker):
    x, w = torch.randn(4, 6), torch.randn(8, 3)
    for bad in (dict(groups=1), dict(groups=3), dict(groups=0)):
        with pytest.raises(ValueError, match="do not fit"):
            graph_ops.linear_act(x, w, **bad)
    with pytest.raises(ValueError, match="bias"):
        graph_ops.linear_act(x, w, torch.randn(7), groups=2)
    with pytest.raises(ValueError, match="residual"):
        graph_ops.linear_act(x, w, None, torch.randn(1, 8), groups=2)
    with pytest.raises(ValueError, match="act 'tanh'"):
        graph_ops.linear_act(x, w, groups=2, act="tanh")
    with pytest.raises(TypeError):
        graph_ops.linear_act(x.double(), w.double(), groups=2)
    with pytest.raises(TypeError):
        graph_ops.linear_act(x.bfloat16(), w, groups=2)
    with pytest.raises(TypeError):
        graph_ops.linear_act(x, w, torch.randn(8).bfloat16(), groups=2)
    y = graph_ops.linear_act(x.requires_grad_(True), w, groups=2, act="gelu")
    (gx,) = torch.autograd.grad(y.sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()                                   # no double backward


def test_there_is_no_cpu_implementation():
    with pytest.raises(RuntimeError, match="MI355X"):
        graph_ops.linear_act(torch.randn(2, 3), torch.randn(4, 3))


def test_c_entries_check_their_arguments():
    L, n = _lib.lib(), ctypes.c_size_t(0)
    fwd = lambda **k: L.nextou_linear_act_fwd(*[{**dict(x=16, w=16, b=None, r=None, y=16, pre=None, P=1, N=1, K=1, g=1, ldx=1,  # noqa: E731
                                                        ldr=0, ldy=1, dt=0, bf=0, act=0, s=0.0, st=None), **k}[i] for i in
                                                "x w b r y pre P N K g ldx ldr ldy dt bf act s st".split()])
    assert fwd(x=None) == -1 and b"null" in L.nextou_last_error()
    assert fwd(P=0) == -1 and fwd(N=0) == -1 and fwd(K=-1) == -1 and fwd(g=0) == -1 and fwd(dt=3) == -1 and fwd(act=5) == -1
    assert fwd(N=4, ldy=3) == -1 and b"stride" in L.nextou_last_error()
    assert fwd(ldx=-1) == -1 and fwd(g=70000) == -1
    assert fwd(P=1 << 30) == -1 and b"16 bytes" in L.nextou_last_error()
    bwd = lambda **k: L.nextou_linear_act_bwd(*[{**dict(gy=16, x=16, w=16, sv=None, kind=0, gx=16, gw=None, gb=None, ws=None, wsb=0, P=1, N=1,  # noqa: E731
                                                        K=1, g=1, ldg=1, ldx=1, dt=0, gbf=0, act=0, s=0.0, st=None), **k}[i] for i in
                                                "gy x w sv kind gx gw gb ws wsb P N K g ldg ldx dt gbf act s st".split()])
    assert bwd(gx=None) == -1 and bwd(act=1) == -1 and bwd(kind=1) == -1 and bwd(act=2, kind=1) == -1
    assert bwd(act=3, kind=2, sv=16) == -1 and b"sign" in L.nextou_last_error()
    assert bwd(act=2, kind=2, sv=16, s=-0.5) == -1
    assert bwd(act=3, kind=1, sv=16) == -2 and b"workspace" in L.nextou_last_error()
    assert L.nextou_linear_act_bwd_workspace(4, 4, 4, 1, 9, 0, 1, 1, 1, ctypes.byref(n)) == -1
    assert L.nextou_linear_act_bwd_workspace(1 << 30, 8, 7, 1, 1, 0, 1, 1, 1, ctypes.byref(n)) == -1
    assert L.nextou_linear_act_bwd_workspace(1 << 30, 8, 8, 1, 1, 0, 1, 1, 1, ctypes.byref(n)) == 0

    assert L.nextou_multi_norm_workspace(0, ctypes.byref(n)) == -1
    assert L.nextou_multi_norm_workspace(3, ctypes.byref(n)) == 0 and n.value >= 8
    room = n.value
    tab = lambda *rows: (ctypes.c_int64 * (3 * len(rows)))(*[v for r in rows for v in r])  # noqa: E731
    norm = lambda t, k, code=2, mx=1.0, ws=16, wsb=room, out=16: L.nextou_multi_norm(t, k, code, mx, ws, wsb, out, None)  # noqa: E731
    ok = (4096, 4, 0)
    assert norm(None, 1) == -1 and norm(tab(ok), 0) == -1 and norm(tab(ok), 1, code=3) == -1 and norm(tab(ok), 1, out=None) == -1
    assert norm(tab(ok), 1, mx=-1.0) == -1 and norm(tab(ok), 1, mx=float("nan")) == -1
    assert norm(tab(ok), 1, wsb=8) == -2 and norm(tab(ok), 1, ws=None) == -2
    for bad in ((0, 4, 0), (4098, 4, 0), (4097, 4, 1), (4096, 0, 0), (4096, -3, 2), (4096, 4, 3), (4096, 1 << 37, 1)):
        assert norm(tab(ok, bad), 2) == -1, bad
    assert b"tensor 1" in L.nextou_last_error()
    clip = lambda t, k: L.nextou_multi_clip(t, k, 2, 1.0, 16, room, 16, None)  # noqa: E731
    assert clip(tab(ok, ok), 2) == -1 and b"overlap" in L.nextou_last_error()
    assert clip(tab((4108, 8, 1), (4096, 4, 0)), 2) == -1 and b"overlap" in L.nextou_last_error()


def test_gradient_norm_refusals_and_cpu_gradients():
    p = torch.nn.Parameter(torch.randn(5))
    p.grad = torch.tensor([3.0, 4.0, 0.0, 0.0, 0.0])
    for bad in (3.0, 0.5, -math.inf, 0.0):
        with pytest.raises(ValueError, match="norm"):
            optim.clip_grad_norm_([p], 1.0, bad)
        with pytest.raises(ValueError, match="norm"):
            optim.grad_norm([p.grad], bad)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            optim.clip_grad_norm_([p], bad)
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.randn(3))], 1.0)) == 0.0 and float(optim.grad_norm([])) == 0.0
    assert float(optim.grad_norm([p.grad, p.grad], 1.0)) == 14.0
    assert float(optim.clip_grad_norm_((q for q in [p]), 1.0)) == 5.0 and abs(float(p.grad.norm()) - 1.0) < 1e-6
    # what the kernels' table refuses, before anything is launched (host tensors stand in for device ones)
    rows = lambda ts, in_place=True: optim._norm_rows(ts, in_place)  # noqa: E731
    with pytest.raises(TypeError):
        rows([torch.randn(3).double()])
    with pytest.raises(TypeError):
        rows([torch.randn(3, 3).to_sparse()])
    with pytest.raises(ValueError, match="overlaps itself"):
        rows([torch.randn(1, 3).expand(4, 3)])
    with pytest.raises(ValueError, match="overlaps itself"):
        rows([torch.randn(9).as_strided((3, 4), (2, 1))])
    vals, copies = rows([torch.randn(1, 3).expand(4, 3), torch.randn(0), torch.randn(8)[::2]], False)
    assert len(vals) == 6 and len(copies) == 2 and vals[1] == 12 and vals[4] == 4
    last = torch.randn(2, 3, 4, 5).contiguous(memory_format=torch.channels_last)
    vals, copies = rows([last, torch.randn(3, 4).t(), torch.randn(2, 3, 1).bfloat16()])
    assert not copies and list(vals)[0] == last.data_ptr() and list(vals)[8] == 1


class _StandInLib:
    """nextou_multi_norm and the two step kernels on host memory, as include/nextou_hip.h describes them."""

    def __init__(self):
        self.calls = []

    @staticmethod
    def _f32(ptr, n):
        return np.ctypeslib.as_array(ctypes.cast(ptr, ctypes.POINTER(ctypes.c_float)), (n,))

    def nextou_device_write_i64(self, dst, host_values, n, stream):
        ctypes.memmove(dst, host_values, 8 * n)
        return 0

    def nextou_multi_norm_workspace(self, n, out):
        out._obj.value = 64
        return 0

    def nextou_multi_norm(self, table, n, norm, max_norm, ws, ws_bytes, out, stream):
        self.calls.append("norm")
        t = np.ctypeslib.as_array(ctypes.cast(table, ctypes.POINTER(ctypes.c_int64)), (n, 3))
        s = math.sqrt(sum(float((self._f32(int(p), int(c)).astype(np.float64) ** 2).sum()) for p, c, _ in t))
        self._f32(out, 2)[:] = [s, min(1.0, max_norm / (s + 1e-6))]
        return 0

    def nextou_clip_sgd_update(self, table, n, chunks, n_chunks, chunk, total, coef, lr, lr_dev, momentum, wd, nesterov, stream):
        self.calls.append("update")
        t = np.ctypeslib.as_array(ctypes.cast(table, ctypes.POINTER(ctypes.c_int64)), (n, 4))
        for p, g, m, c in t:
            pv, gv = self._f32(int(p), int(c)), self._f32(int(g), int(c))
            gv *= self._f32(coef, 2)[1]
            pv -= np.float32(lr) * gv
        return 0


def test_a_strided_gradient_listed_twice_is_refused():
    base = torch.randn(6, 8)
    left, right = base[:, :4], base[:, 4:]
    assert len(optim._norm_rows([left, right, torch.randn(3)], True)[1]) == 2          # interleaved, nothing shared
    with pytest.raises(RuntimeError, match="share memory"):
        optim._norm_rows([left, right, left], True)
    assert len(optim._norm_rows([left, right, left], False)[1]) == 3                    # a norm only reads


def test_clip_sgd_clips_over_several_groups(monkeypatch):
    fake = _StandInLib()
    monkeypatch.setattr(_lib, "lib", lambda: fake)
    a, b = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(3, 2))
    opt = optim.ClipSGD([{"params": [a], "lr": 0.5}, {"params": [b], "lr": 0.25}], 0.1)
    opt._device_type = "cpu"
    a.grad, b.grad = torch.full((4,), 3.0), torch.full((3, 2), 2.0)
    norm = opt.clip_and_step(1.0)
    want = math.sqrt(4 * 9 + 6 * 4)
    assert opt.last_path == "own" and fake.calls == ["norm", "update", "update"]
    assert abs(float(norm) - want) < 1e-6
    assert torch.allclose(a.detach(), torch.full((4,), 1 - 0.5 * 3 / want)) and torch.allclose(b.detach(), torch.full((3, 2), 1 - 0.25 * 2 / want))
    assert torch.allclose(b.grad, torch.full((3, 2), 2 / want))
