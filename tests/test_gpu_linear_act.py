"""K10 (csrc/linear_act.hip) on the GPU against the formula in float64.

Tolerances count roundings: a float32 sum of n terms is off by at most (n + 8) 2^-23 times the sum of absolute products (n steps, in any order, of a
unit that may truncate), an output by half a step of its type (eps / 2), the activation's own evaluation by 4e-7 relative + 3e-7 |z| (exp
and the error function), dz in 16 bits by half a step, a saved z of 16-bit rows by half a step of float16.  The activations whose slope
jumps are given inputs whose sums are exact in every type, ties included, so that the slope is the formula's."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = 2.0 ** -23


@pytest.fixture(scope="module")
def ops():
    from nextou_amd import _lib, graph_ops
    _lib.lib()
    assert "libnextou_hip.so" in open("/proc/self/maps").read(), "HIP extension not loaded into this process"
    return graph_ops


def _half(t):
    return torch.finfo(t).eps / 2


def _floor(t):       # half of the smallest step: what rounding leaves of a value too small for the type
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def _act64(z, act, slope):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "leakyrelu":
        return torch.where(z > 0, z, z * slope), torch.where(z > 0, 1.0, slope).double()
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return z * (z + 3).clamp(0, 6) / 6, torch.where(z <= -3, 0.0, torch.where(z >= 3, 1.0, (2 * z + 3) / 6))


def _mm(a, b, groups):
    """per group a_g b_g^T in float64: (P, G*K), (G*N, K) -> (P, G*N)"""
    k, n = a.shape[1] // groups, b.shape[0] // groups
    return torch.cat([a[:, g * k:(g + 1) * k] @ b[g * n:(g + 1) * n].t() for g in range(groups)], 1)


def _wt(w, groups):
    n, k = w.shape[0] // groups, w.shape[1]
    return w.view(groups, n, k).transpose(1, 2).reshape(groups * k, n)


def _outer(dz, x, groups):
    n, k = dz.shape[1] // groups, x.shape[1] // groups
    return torch.cat([dz[:, g * n:(g + 1) * n].t() @ x[:, g * k:(g + 1) * k] for g in range(groups)])


def _expect(x, w, b, r, gy, act, slope, groups, exact_z=False):
    """{name: (value, allowed error)} in float64"""
    t = x.dtype
    X, W = x.detach().double(), w.detach().double()
    B = torch.zeros(w.shape[0], device=x.device, dtype=torch.float64) if b is None else b.detach().double()
    K, N, P = w.shape[1], w.shape[0] // groups, x.shape[0]
    z = _mm(X, W, groups) + B
    ez = torch.zeros_like(z) if exact_z else (K + 8) * U * (_mm(X.abs(), W.abs(), groups) + B.abs())
    v, s = _act64(z, act, slope)
    y = v if r is None else v + r.detach().double()
    ev = 1.6 * ez + (0 if act in ("none", "relu") else 4e-7 * v.abs() + 3e-7 * z.abs())
    out = {"y": (y, (ev + U * y.abs()) * 1.01 + _half(t) * y.abs() + _floor(t))}
    if gy is None:
        return out
    G = gy.double()
    dz = G * s
    edz = torch.zeros_like(z)
    if act in ("gelu", "hswish") and not exact_z:      # the slope's own slope is at most 0.8 (gelu); float16 keeps z of 16-bit rows
        edz = G.abs() * (0.8 * (ez + (0 if t == torch.float32 else _half(torch.float16) * z.abs() + _floor(torch.float16))) + 1e-6)
    elif act != "none":
        edz = G.abs() * 1e-6
    sums = edz.clone()
    if act != "none" and t != torch.float32:
        edz = edz + _half(t) * dz.abs() + _floor(t)
    wt, wta = _wt(W, groups), _wt(W.abs(), groups)
    gx, ax = _mm(dz, wt, groups), _mm(dz.abs() + edz, wta, groups)
    out["gx"] = (gx, (N + 8) * U * ax + _mm(edz, wta, groups) + _half(t) * gx.abs() + _floor(t))
    gw, aw = _outer(dz, X, groups), _outer(dz.abs() + edz, X.abs(), groups)
    out["gw"] = (gw, (P + 8) * U * aw + _outer(edz, X.abs(), groups) + _half(t) * gw.abs() + _floor(t))
    if b is not None:
        gb = dz.sum(0)
        out["gb"] = (gb, (P + 8) * U * (dz.abs() + sums).sum(0) + sums.sum(0) + _half(b.dtype) * gb.abs() + _floor(b.dtype))
    if r is not None:
        out["gr"] = (G, torch.zeros_like(G))
    return out


def _check(got, expect):
    for name, value in got.items():
        want, room = expect[name]
        assert value.shape == want.shape, name
        over = (value.double() - want).abs() / room.clamp_min(1e-300)
        assert float(over.max()) <= 1.0, "%s: %.3g times the allowed error" % (name, float(over.max()))


def _inputs(P, K, N, groups, t, seed, coarse=False, bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)

    def make(*shape, scale=1.0):
        v = torch.randn(shape, generator=g) * scale
        if coarse:       # small multiples of 1/4: products are multiples of 1/16 and every sum of them is exact, also in float16
            v = (v * 4 / scale).round().clamp(-3, 3) / 4
        return v.to(t).to(DEV)

    x, w = make(P, groups * K), make(groups * N, K, scale=K ** -0.5)
    if coarse and K > 16:       # sparse rows keep |z| small enough for float16 to hold it exactly
        w = w * (torch.rand(w.shape, generator=g) < 12.0 / K).to(DEV)
    b = make(groups * N, scale=0.3) if bias else None
    r = make(P, groups * N) if residual else None
    return x, w, b, r, make(P, groups * N)


def _run(ops, x, w, b, r, gy, act, slope, groups):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    xs, ws = next(it), next(it)
    bs = next(it) if b is not None else None
    rs = next(it) if r is not None else None
    y = ops.linear_act(xs, ws, bs, rs, act, slope, groups)
    grads = torch.autograd.grad(y, leaves, gy)
    names = ["gx", "gw"] + (["gb"] if b is not None else []) + (["gr"] if r is not None else [])
    return dict(zip(["y"] + names, (y.detach(),) + grads))


_SHAPES = [
    # P, K, N, groups
    (1, 1, 1, 1), (1, 5, 3, 1), (2, 33, 66, 1), (3, 1, 70, 1), (5, 2, 3, 7), (7, 132, 44, 1), (8, 1024, 512, 1), (16, 640, 33, 1), (17, 8, 11, 6), (15, 999, 333, 1),
    (33, 260, 4, 1), (63, 31, 65, 1), (64, 64, 64, 1), (65, 129, 127, 1), (96, 2048, 80, 1), (128, 256, 128, 1), (129, 100, 36, 4), (257, 44, 44, 6), (300, 1296, 324, 1), (336, 324, 1296, 1),
    (512, 512, 512, 1), (513, 72, 40, 1), (1000, 3, 1100, 1), (2, 4099, 7, 1), (4097, 40, 33, 1), (2050, 136, 520, 1), (6000, 264, 256, 1), (31, 4096, 256, 1),
]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("P,K,N,groups", _SHAPES)
def test_values_and_gradients(ops, P, K, N, groups, t):
    i = _SHAPES.index((P, K, N, groups))
    bias, residual = i % 3 != 1, i % 2 == 0
    act = ["gelu", "none", "gelu"][i % 3]
    x, w, b, r, gy = _inputs(P, K, N, groups, t, 100 + i, bias=bias, residual=residual)
    _check(_run(ops, x, w, b, r, gy, act, 0.01, groups), _expect(x, w, b, r, gy, act, 0.01, groups))


_MANY = [
    # P, K, N, groups: the weight in LDS (every register size, panels of several groups and of parts of one group, odd widths) and the largest tiles
    (65536, 9, 5, 1), (65552, 44, 44, 6), (65537, 20, 33, 3), (65542, 132, 72, 1), (70000, 100, 529, 1), (65599, 200, 264, 1), (65536, 264, 96, 1),
    (65550, 266, 700, 1), (65553, 393, 40, 1), (65536, 528, 132, 1), (66000, 17, 1, 40), (68000, 67, 131, 2), (20000, 44, 44, 6), (16385, 132, 72, 1),
    (8200, 200, 4104, 1), (260, 4104, 3080, 1),
]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("P,K,N,groups", _MANY)
def test_many_rows_and_large_weights(ops, P, K, N, groups, t):
    i = _MANY.index((P, K, N, groups))
    bias, residual = i % 3 != 1, i % 2 == 0
    act = ["gelu", "none", "gelu"][(i + 1) % 3]
    x, w, b, r, gy = _inputs(P, K, N, groups, t, 300 + i, bias=bias, residual=residual)
    _check(_run(ops, x, w, b, r, gy, act, 0.01, groups), _expect(x, w, b, r, gy, act, 0.01, groups))
    with torch.no_grad():
        y = ops.linear_act(x, w, b, r, "none", groups=groups)
    _check({"y": y}, _expect(x, w, b, r, None, "none", 0.01, groups))


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("act,slope", [("relu", 0.01), ("leakyrelu", 0.01), ("leakyrelu", 0.0), ("leakyrelu", -0.5), ("leakyrelu", 1.5), ("hswish", 0.01), ("none", 0.0)])
@pytest.mark.parametrize("P,K,N,groups,residual", [(70, 12, 9, 1, False), (70, 12, 9, 1, True), (300, 16, 72, 2, False), (6, 200, 136, 1, True), (260, 256, 256, 1, False)])
def test_activations_with_kinks(ops, P, K, N, groups, residual, act, slope, t):
    x, w, b, r, gy = _inputs(P, K, N, groups, t, 7, coarse=True, residual=residual)
    z = _mm(x.double(), w.double(), groups) + b.double()
    assert int((z == 0).sum()) > 0 and float(z.abs().max()) <= 64          # multiples of 1/16: exact in float16 as well
    _check(_run(ops, x, w, b, r, gy, act, slope, groups), _expect(x, w, b, r, gy, act, slope, groups, exact_z=True))


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_forward_alone_gives_the_training_forward(ops, t):
    for P, K, N, groups, act in ((5, 300, 70, 1, "gelu"), (700, 100, 130, 1, "hswish"), (129, 64, 32, 3, "leakyrelu")):
        x, w, b, r, gy = _inputs(P, K, N, groups, t, 3)
        with torch.no_grad():
            y = ops.linear_act(x, w, b, r, act, groups=groups)
        assert torch.equal(y, _run(ops, x, w, b, r, gy, act, 0.01, groups)["y"])


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_repeats_are_bit_identical(ops, t):
    for P, K, N, groups in ((4097, 264, 132, 1), (300, 40, 24, 6), (9, 1030, 250, 1)):
        x, w, b, r, gy = _inputs(P, K, N, groups, t, 5)
        one, two = (_run(ops, x, w, b, r, gy, "gelu", 0.01, groups) for _ in range(2))
        assert all(torch.equal(one[k], two[k]) for k in one)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("P,K,N,groups", [(6, 136, 200, 1), (300, 99, 187, 1), (20000, 44, 44, 2), (20000, 132, 72, 1), (700, 331, 130, 1)])
def test_many_calls_give_one_result(ops, P, K, N, groups, t):
    """Rows that end inside a 16-byte piece or a stage, two hundred calls in a row (whole numbers: the sums are exact, so is the comparison)."""
    g = torch.Generator().manual_seed(K)
    x = torch.randint(-3, 4, (P, groups * K), generator=g).to(t).to(DEV)
    w = torch.randint(-3, 4, (groups * N, K), generator=g).to(t).to(DEV)
    want = _mm(x.double(), w.double(), groups).to(t)
    with torch.no_grad():
        wrong = sum((ops.linear_act(x, w, groups=groups) != want).any().int() for _ in range(200))
    assert int(wrong) == 0


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("P,K,N", [(37, 50, 35), (150, 128, 72), (260, 264, 136), (3, 515, 129)])
def test_strides_offsets_and_surroundings(ops, P, K, N, t):
    """Rows inside wider tensors at odd offsets, transposed operands, expanded rows; everything around the operands is NaN, so a value read from
    there would show; what surrounds nothing but is written is checked by the outputs being whole tensors of their own."""
    x, w, b, r, gy = _inputs(P, K, N, 1, t, 11)

    def inside(v, left, right):
        wide = torch.full((v.shape[0] + 2, v.shape[1] + left + right), float("nan"), dtype=t, device=DEV)
        wide[1:-1, left:left + v.shape[1]] = v
        return wide[1:-1, left:left + v.shape[1]]

    want = _run(ops, x, w, b, r, gy, "gelu", 0.01, 1)
    _check(want, _expect(x, w, b, r, gy, "gelu", 0.01, 1))
    for left, right in ((1, 0), (3, 2), (8, 8), (4, 5)):
        leaves = [inside(v, left, right).requires_grad_(True) for v in (x, r)]
        y = ops.linear_act(leaves[0], w, b, leaves[1], "gelu")
        gx, gr = torch.autograd.grad(y, leaves, inside(gy, left, right))
        _check({"y": y.detach(), "gx": gx, "gr": gr}, _expect(x, w, b, r, gy, "gelu", 0.01, 1))
        # the weight inside a NaN-filled buffer, one element off any 16-byte boundary
        flat = torch.full((N * K + 9,), float("nan"), dtype=t, device=DEV)
        wv = flat[left:left + N * K].view(N, K)
        wv.copy_(w)
        wl = wv.requires_grad_(True)
        y = ops.linear_act(x, wl, b, r, "gelu")
        (gw,) = torch.autograd.grad(y, (wl,), gy)
        _check({"y": y.detach(), "gw": gw}, _expect(x, w, b, r, gy, "gelu", 0.01, 1))
    xt, wt, gt = x.t().contiguous().t(), w.t().contiguous().t(), gy.t().contiguous().t()
    got = _run(ops, xt, wt, b, r, gt, "gelu", 0.01, 1)
    assert all(torch.equal(got[k], want[k]) for k in want)
    one = x[:1]
    y = ops.linear_act(one.expand(P, K), w, b, r[:1].expand(P, N), "none")
    _check({"y": y}, _expect(one.expand(P, K), w, b, r[:1].expand(P, N), None, "none", 0.01, 1))
    assert torch.equal(y, y[:1].expand(P, N))


@pytest.mark.parametrize("t", TYPES, ids=str)
def test_non_finite_values_stay_in_their_rows(ops, t):
    """A row with NaN or infinity, or with the type's largest values, changes no other row (padding is never multiplied in)."""
    for P, K, N in ((200, 70, 45), (6, 300, 37), (300, 256, 128)):
        x, w, b, r, gy = _inputs(P, K, N, 1, t, 13)
        want = _run(ops, x, w, b, r, gy, "relu", 0.01, 1)
        bad = x.clone()
        bad[1, K - 1], bad[2, 0], bad[3] = float("nan"), float("inf"), torch.finfo(t).max
        with torch.no_grad():
            y = ops.linear_act(bad, w, b, r, "relu")
        keep = [i for i in range(P) if i not in (1, 2, 3)]
        assert torch.equal(y[keep], want["y"][keep])
        assert bool(torch.isnan(y[1]).all()) and bool((torch.isinf(y[2]) | (y[2] == r[2]) | torch.isnan(y[2])).all())
        gbad = gy.clone()
        gbad[4, 0] = float("nan")
        got = _run(ops, x, w, b, r, gbad, "none", 0.01, 1)
        assert bool(torch.isnan(got["gx"][4]).all()) and not bool(torch.isnan(got["gx"][[i for i in range(P) if i != 4]]).any())
        assert bool(torch.isnan(got["gw"][0]).all()) and not bool(torch.isnan(got["gw"][1:]).any())
        assert bool(torch.isnan(got["gb"][0])) and not bool(torch.isnan(got["gb"][1:]).any())


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("slope", [0.0, 0.01, 1.0, 1.5, -0.5])
def test_leaky_relu_of_infinities(ops, slope, t):
    # one column of ones: z is x, exactly
    x = torch.tensor([[float("inf")], [float("-inf")], [float("nan")], [0.0], [-2.0], [2.0]], device="cuda", dtype=t)
    with torch.no_grad():
        y = ops.linear_act(x, torch.ones(8, 1, device="cuda", dtype=t), None, None, "leakyrelu", slope)
    torch.testing.assert_close(y, torch.nn.functional.leaky_relu(x, slope).expand(-1, 8), rtol=0, atol=0, equal_nan=True)


def test_small_positive_values_keep_their_sign(ops):
    """float16: z = 2^-30 rounds to 0, its ReLU gradient is still 1."""
    x = torch.tensor([[2.0 ** -14], [-2.0 ** -14]], dtype=torch.float16, device=DEV).requires_grad_(True)
    w = torch.tensor([[2.0 ** -14]], dtype=torch.float16, device=DEV)
    for act, want in (("relu", [1.0, 0.0]), ("leakyrelu", [1.0, 0.25])):
        y = ops.linear_act(x, w, act=act, negative_slope=0.25)
        (gx,) = torch.autograd.grad(y, (x,), torch.full((2, 1), 2.0 ** 12, dtype=torch.float16, device=DEV))
        assert torch.equal(gx[:, 0].float().cpu(), torch.tensor(want) * 2.0 ** -2)


def test_float32_bias_beside_16_bit_rows_and_autocast(ops):
    for t in (torch.bfloat16, torch.float16):
        x, w, b, r, gy = _inputs(90, 70, 50, 1, t, 17)
        b = (torch.randn(50, generator=torch.Generator().manual_seed(1)) * 0.3).to(DEV)
        got = _run(ops, x, w, b, r, gy, "gelu", 0.01, 1)
        assert got["gb"].dtype == torch.float32
        _check(got, _expect(x, w, b, r, gy, "gelu", 0.01, 1))
    x32, w32 = torch.randn(40, 24, device=DEV, requires_grad=True), torch.randn(16, 24, device=DEV, requires_grad=True)
    with torch.autocast("cuda", torch.bfloat16):
        y = ops.linear_act(x32, w32, act="relu")
    assert y.dtype == torch.bfloat16
    assert torch.equal(y, ops.linear_act(x32.detach().bfloat16(), w32.detach().bfloat16(), act="relu"))
    gx, gw = torch.autograd.grad(y.float().sum(), (x32, w32))
    assert gx.dtype == gw.dtype == torch.float32 and gx.shape == x32.shape


def test_no_rows_and_refusals(ops):
    w = torch.randn(6, 5, device=DEV, requires_grad=True)
    x = torch.randn(0, 5, device=DEV, requires_grad=True)
    y = ops.linear_act(x, w, act="gelu")
    gx, gw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (0, 6) and gx.shape == (0, 5) and float(gw.abs().max()) == 0.0
    with pytest.raises(ValueError, match="tensors on"):
        ops.linear_act(torch.randn(4, 5, device=DEV), torch.randn(6, 5))
    with pytest.raises(TypeError):
        ops.linear_act(torch.randn(4, 5, device=DEV), w.detach().half())
    y = ops.linear_act(torch.randn(2, 3, 5, device=DEV), w, torch.randn(6, device=DEV), torch.randn(2, 3, 6, device=DEV))
    assert y.shape == (2, 3, 6)


def test_another_stream_and_a_captured_step(ops):
    """Work queued on a side stream; then forward + backward captured once and replayed with new contents, eager work in between."""
    cases = [(900, 100, 68, 1, torch.bfloat16, "gelu"), (5, 515, 129, 1, torch.float16, "none"), (260, 48, 40, 3, torch.float32, "leakyrelu")]
    for P, K, N, groups, t, act in cases:
        x, w, b, r, gy = _inputs(P, K, N, groups, t, 23)
        want = _run(ops, x, w, b, r, gy, act, 0.01, groups)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _run(ops, x, w, b, r, gy, act, 0.01, groups)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(got[k], want[k]) for k in want)
        static = [v.clone() for v in (x, w, b, r, gy)]
        with torch.cuda.stream(side):
            _run(ops, *static, act, 0.01, groups)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _run(ops, *static, act, 0.01, groups)
        for seed in (31, 37, 41):
            fresh = _inputs(P, K, N, groups, t, seed)
            for s, f in zip(static, fresh):
                s.copy_(f)
            graph.replay()
            eager = _run(ops, *fresh, act, 0.01, groups)
            torch.cuda.synchronize()
            assert all(torch.equal(out[k], eager[k]) for k in eager)


def test_pointwise_act_on_a_channels_last_volume(ops):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 36, 3, 5, 7, generator=g).to(DEV).contiguous(memory_format=torch.channels_last_3d).requires_grad_(True)
    w = (torch.randn(30, 6, 1, 1, 1, generator=g) * 0.4).to(DEV).requires_grad_(True)
    b, r = torch.randn(30, generator=g).to(DEV), torch.randn(2, 30, 3, 5, 7, generator=g).to(DEV)
    y = ops.pointwise_act(x, w, b, r, "gelu", groups=6)
    gy = torch.randn(y.shape, generator=g).to(DEV)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    rows = lambda v: v.detach().permute(0, 2, 3, 4, 1).reshape(-1, v.shape[1])  # noqa: E731
    want = _expect(rows(x), w.detach().flatten(1), b, rows(r), rows(gy), "gelu", 0.01, 6)
    assert y.is_contiguous(memory_format=torch.channels_last_3d) and gw.shape == w.shape
    _check({"y": rows(y), "gx": rows(gx), "gw": gw.flatten(1)}, want)


def test_rows_beyond_two_billion_elements(ops):
    """Offsets past 32 bits: 2^25 + 3 rows of 72 bfloat16 columns, a few rows checked against the formula."""
    P, K, N = (1 << 25) + 3, 72, 8
    x = torch.empty(P, K, dtype=torch.bfloat16, device=DEV).normal_()
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    with torch.no_grad():
        y = ops.linear_act(x, w, act="relu")
    at = torch.tensor([0, 1, (1 << 25) - 1, 1 << 25, P - 1, 31_000_001], device=DEV)
    _check({"y": y[at]}, _expect(x[at], w, None, None, None, "relu", 0.01, 1))
