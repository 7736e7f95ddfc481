"""K10 (csrc/linear_act.hip): values and gradients over small whole numbers, where every float32 sum is exact, so that each output is the formula's
rounded once, bit for bit: a row, a stage, a row block or a split that is lost or counted twice shows whatever the number of rows.

Exactness: products of values up to 3 are up to 9; the longest sum has 65 599 of them (or 4.2 million of products up to 1), below 2^24."""
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


def _whole(gen, top, rows, cols, t, pad=0):
    """(rows, cols) of whole numbers; ``pad``: inside wider rows, ``pad`` columns from their start, NaN around"""
    v = torch.randint(-top, top + 1, (rows, cols), generator=gen, device=DEV, dtype=torch.int8).to(t)
    if not pad:
        return v
    wide = torch.full((rows, cols + 2 * pad), float("nan"), dtype=t, device=DEV)
    wide[:, pad:pad + cols] = v
    return wide[:, pad:pad + cols]


def _mm(a, b, groups):
    k, n = a.shape[1] // groups, b.shape[0] // groups
    return torch.cat([a[:, g * k:(g + 1) * k] @ b[g * n:(g + 1) * n].t().contiguous() for g in range(groups)], 1)


def _expect(x, w, b, r, gy, act, groups):
    X, W, G = x.detach().double(), w.detach().double(), gy.double()
    n, k = w.shape[0] // groups, w.shape[1]
    z = _mm(X, W, groups)
    if b is not None:
        z = z + b.detach().double()
    y, dz = (z, G) if act == "none" else (z.clamp_min(0), G * (z > 0))
    if r is not None:
        y = y + r.detach().double()
    gx = _mm(dz, W.view(groups, n, k).transpose(1, 2).reshape(groups * k, n), groups)
    gw = torch.cat([dz[:, g * n:(g + 1) * n].t().contiguous() @ X[:, g * k:(g + 1) * k] for g in range(groups)])
    out = {"y": y.to(x.dtype), "gx": gx.to(x.dtype), "gw": gw.to(x.dtype)}
    if b is not None:
        out["gb"] = dz.sum(0).to(b.dtype)
    return out


_SHAPES = [
    # P, K, N, groups: ragged row counts around the splits, row blocks and panels; aligned and unaligned widths; one and many groups
    (257, 264, 96, 1), (1025, 99, 187, 1), (4999, 99, 187, 1), (5000, 300, 64, 1), (16385, 132, 72, 1), (16385, 264, 1056, 1), (20000, 44, 44, 6), (20000, 33, 7, 2),
    (21503, 5, 3, 1), (40001, 528, 132, 1), (65537, 264, 96, 1), (65537, 20, 33, 3), (65599, 100, 529, 1), (65599, 8, 8, 1), (65536, 44, 44, 6),
    (1000, 4096, 3080, 1), (2111, 2048, 6152, 1),
]


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("P,K,N,groups", _SHAPES)
def test_every_row_is_in_every_sum(ops, P, K, N, groups, t):
    gen = torch.Generator(device=DEV).manual_seed(P + K)
    for act, pad, wide_bias in (("none", 0, False), ("relu", 0, False), ("none", 1, True), ("relu", 3, True)):
        x, gy = _whole(gen, 3, P, groups * K, t, pad), _whole(gen, 3, P, groups * N, t, pad)
        w, b = _whole(gen, 3, groups * N, K, t), _whole(gen, 3, 1, groups * N, torch.float32 if wide_bias else t)[0].clone()
        r = _whole(gen, 3, P, groups * N, t) if act == "relu" and pad else None      # (with a shortcut z is saved, without one the output's sign)
        leaves = [v.detach().requires_grad_(True) for v in (x, w, b)]
        y = ops.linear_act(*leaves, r, act, 0.01, groups)
        got = dict(zip(("y", "gx", "gw", "gb"), (y.detach(),) + torch.autograd.grad(y, leaves, gy)))
        for name, want in _expect(x, w, b, r, gy, act, groups).items():
            assert torch.equal(got[name], want), (name, act, pad, int((got[name] != want).sum()))


@pytest.mark.parametrize("t,P,K,N,residual", [(torch.bfloat16, (1 << 22) + 3, 520, 516, False), (torch.float16, (1 << 22) + 3, 520, 516, True),
                                              (torch.float32, (1 << 21) + 3, 1032, 1028, False)], ids=["bfloat16", "float16", "float32"])
def test_gradients_beyond_two_billion_elements(ops, t, P, K, N, residual):
    """Offsets past 32 bits in x, y, the incoming gradient, its product with the activation's slope and the gradient of x, in rows too long for the
    panel kernel: the weight's and the bias's gradient against the whole sum, the rest at some rows."""
    torch.cuda.empty_cache()
    gen = torch.Generator(device=DEV).manual_seed(K)

    def whole(rows, cols):
        v = torch.empty(rows, cols, dtype=t, device=DEV)
        for at in range(0, rows, 1 << 18):
            v[at:at + (1 << 18)] = torch.randint(-1, 2, (min(1 << 18, rows - at), cols), generator=gen, device=DEV, dtype=torch.int8)
        return v

    x, gy, w, b = whole(P, K), whole(P, N), whole(N, K), whole(1, N)[0].clone()
    r = whole(P, N) if residual else None
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    y = ops.linear_act(*leaves, r, "relu")
    gx, gw, gb = torch.autograd.grad(y, leaves, gy)
    x, w, b, y = x.detach(), w.detach(), b.detach(), y.detach()
    want_w, want_b = torch.zeros(N, K, dtype=torch.float64, device=DEV), torch.zeros(N, dtype=torch.float64, device=DEV)
    W = w.double()
    for at in range(0, P, 1 << 17):
        X, G = x[at:at + (1 << 17)].double(), gy[at:at + (1 << 17)].double()
        z = X @ W.t().contiguous() + b.double()
        dz = G * (z > 0)
        want_w += dz.t().contiguous() @ X
        want_b += dz.sum(0)
        if at in (0, (P >> 18) << 17, (P - 1) >> 17 << 17):             # the first rows, those in the middle, the last
            v = z.clamp_min(0)
            if residual:
                v = v + r[at:at + (1 << 17)].double()
            assert torch.equal(y[at:at + (1 << 17)], v.to(t)) and torch.equal(gx[at:at + (1 << 17)], (dz @ W).to(t))
    assert float(want_w.abs().max()) < 2 ** 24
    assert torch.equal(gw, want_w.to(t)) and torch.equal(gb, want_b.to(t))
    del x, gy, y, gx, r, leaves
    torch.cuda.empty_cache()
