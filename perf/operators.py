"""The point-wise layer with its epilogue (forward, and forward + backward) and the global gradient norm with the clip, as cases that
can be timed: in a plain form of elementary torch operations, and through the framework's own entry points (``own``).

A ``linear`` case is ``y = act(x w^T + b) [+ residual]`` over rows, in ``groups`` independent channel groups; ``train`` cases also
return the gradients of x, w, b and of the residual.  A ``clip`` case scales the gradients of a parameter list to a global norm,
a ``norm`` case only takes the norm.  The gradients of a list lie back to back in one flat buffer per type, as the data-parallel buckets hold them.
"""
import math
import random

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_SLOPE = 0.01


def _linear(name, rows, k, n, dtype, act, residual=False, train=False, groups=1):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "groups": groups, "dtype": dtype, "act": act,
            "residual": residual, "train": train}


def listed():
    return [
        # one row through a layer: what a single token, or the pooled feature of one image, costs; the weights' bytes and the launch
        _linear("one row bf16", 1, 1024, 4096, "bf16", "gelu"),
        # the bottleneck of a 3-D patch in a batch of two: 336 points, the second product of the feed-forward block
        _linear("336 rows bf16 residual", 336, 1296, 324, "bf16", "none", residual=True),
        # the widest graph stage of the 3-D plans at batch 2 (172 032 points): the feed-forward block's two products when a case is predicted in 16 bits
        _linear("172032 rows bf16 leaky", 172032, 132, 528, "bf16", "leakyrelu"),
        _linear("172032 rows fp16 residual", 172032, 528, 132, "fp16", "none", residual=True),
        # the graph convolution's grouped product in float32 (six groups of 44 channels), with an activation and no norm
        _linear("172032 rows fp32 6 groups", 172032, 44, 44, "fp32", "relu", groups=6),
        # a large square-ish product: bound by the matrix units
        _linear("8192 rows fp16 hardswish", 8192, 4096, 4096, "fp16", "hardswish"),
        # training: the next graph stage (21 504 points); odd channel counts in float32; a wide feed-forward layer.  (The activations
        # with a kink are left to the forward cases: where a sum's last bit decides the sign, the gradient of one point jumps.)
        _linear("train 21504 rows bf16", 21504, 264, 1056, "bf16", "gelu", train=True),
        _linear("train 4999 rows fp32 odd", 4999, 99, 187, "fp32", "gelu", residual=True, train=True),
        _linear("train 16384 rows bf16 wide", 16384, 2048, 8192, "bf16", "gelu", train=True),
        # the clip of the 3-D network's 358 trainable tensors (30.7 M float32 values)
        {"name": "clip 358 fp32", "op": "clip", "tensors": 358, "values": 30_700_000, "dtype": "fp32", "max_norm": 1.0, "p": 2.0},
        # a model of a billion parameters: large 16-bit tensors, small ones in float32
        {"name": "clip 610 bf16 and fp32", "op": "clip", "tensors": 610, "values": 1_000_000_000, "dtype": "mixed", "max_norm": 1.0, "p": 2.0},
        # the largest gradient of a small model, as a monitor asks for it every step: latency
        {"name": "max norm 12 fp16", "op": "norm", "tensors": 12, "values": 9_001, "dtype": "fp16", "max_norm": 0.0, "p": math.inf},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["forward", "forward", "train", "train", "clip"])
    if kind == "clip":
        op = rng.choice(["clip", "clip", "norm"])
        tensors = _log_int(rng, 1, 600)
        return {"op": op, "tensors": tensors, "values": max(40 * tensors, _log_int(rng, 5_000, 500_000_000)),
                "dtype": rng.choice(["fp32", "bf16", "fp16", "mixed"]), "max_norm": 1.0 if op == "clip" else 0.0,
                "p": 2.0 if op == "clip" else rng.choice([1.0, 2.0, math.inf])}
    train = kind == "train"
    while True:
        rows = _log_int(rng, 256 if train else 1, 200_000)
        k, n = _log_int(rng, 33, 4608), _log_int(rng, 33, 4608)
        groups = rng.choice([1, 1, 1, 1, 4, 6])
        if groups > 1:
            k, n = max(8, k // groups), max(8, n // groups)
        if train and groups * k * n < 2000:
            continue
        if rows * groups * max(k, n) <= 120_000_000 and rows * groups * k * n <= 1.0e11:
            break
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if dtype == "fp32" and rows * groups * k * n > 3.0e10:
        rows = max(256, rows // 8)
    act = rng.choice(["none", "gelu"]) if train else rng.choice(["none", "relu", "leakyrelu", "gelu", "hardswish"])
    return {"op": "linear", "rows": rows, "k": k, "n": n, "groups": groups, "dtype": dtype, "act": act,
            "residual": rng.random() < 0.5, "train": train}


def _sizes(case):
    """Element counts of a parameter list: half of the tensors are vectors of a few dozen to a few hundred values (norms, biases), the
    rest filters whose sizes spread over a factor of a thousand and fill the list up to ``values``."""
    rng = random.Random(case["tensors"] * 7919 + 17)
    count, total = case["tensors"], case["values"]
    small = [rng.randint(1, 33) if total < 40_000 else rng.randint(17, 1296) for _ in range(count // 2)]
    while sum(small) > total // 2:
        small = [max(1, s // 2) for s in small]
    large = count - len(small)
    shares = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(large)]
    left = total - sum(small)
    sizes = [max(1, int(left * s / sum(shares))) for s in shares]
    sizes[-1] = max(1, left - sum(sizes[:-1]))
    out = []
    for i in range(max(len(small), len(sizes))):      # a filter, then its vector, as a network lists them
        if i < len(sizes):
            out.append((sizes[i], "fp32" if case["dtype"] == "fp32" else ("bf16" if case["dtype"] == "mixed" else case["dtype"])))
        if i < len(small):
            out.append((small[i], "fp32" if case["dtype"] in ("fp32", "mixed") else case["dtype"]))
    return out


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def prepare(case, seed):
    g = _generator(seed)

    def normal(shape, scale, dtype):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)

    if case["op"] == "linear":
        dt = _TYPES[case["dtype"]]
        p, k, n, groups = case["rows"], case["k"], case["n"], case["groups"]
        x = normal((p, groups * k), 1.0, dt)
        w = normal((groups * n, k), 1.0 / math.sqrt(k), dt)
        b = normal((groups * n,), 0.2, dt)
        r = normal((p, groups * n), 1.0, dt) if case["residual"] else None
        state = {"case": case, "x": x, "w": w, "b": b, "r": r}
        if case["train"]:
            state["gy"] = normal((p, groups * n), 1.0, dt)
            for t in (x, w, b, r):
                if t is not None:
                    t.requires_grad_(True)
        return state

    sizes = _sizes(case)
    flat, values, params = {}, {}, []
    for kind in dict.fromkeys(s[1] for s in sizes):
        total = sum(s[0] for s in sizes if s[1] == kind)
        flat[kind] = torch.empty(total, dtype=_TYPES[kind], device="cuda").normal_(0.0, 0.05, generator=g)
        values[kind] = torch.empty(total, dtype=_TYPES[kind], device="cuda")
    at = dict.fromkeys(flat, 0)
    for count, kind in sizes:
        p = torch.nn.Parameter(values[kind][at[kind]:at[kind] + count])
        p.grad = flat[kind][at[kind]:at[kind] + count]
        params.append(p)
        at[kind] += count
    return {"case": case, "params": params, "flat": flat}


# ---- the framework's calls -----------------------------------------------------------------------------------------------------
def _run_own(state):
    case = state["case"]
    if case["op"] == "linear":
        from nextou_amd.graph_ops import linear_act
        x, w, b, r = state["x"], state["w"], state["b"], state["r"]
        y = linear_act(x, w, b, residual=r, act=case["act"], negative_slope=_SLOPE, groups=case["groups"])
        if not case["train"]:
            return y
        leaves = [x, w, b] if r is None else [x, w, b, r]
        return [y.detach()] + list(torch.autograd.grad(y, leaves, state["gy"]))
    from nextou_amd.optim import clip_grad_norm_, grad_norm
    if case["op"] == "norm":
        return grad_norm([p.grad for p in state["params"]], case["p"])
    return [clip_grad_norm_(state["params"], case["max_norm"], case["p"])] + list(state["flat"].values())


# ---- the plain form ------------------------------------------------------------------------------------------------------------
def _by_group(t, groups):
    """(P, groups * C) -> (groups, P, C)"""
    return t.view(t.shape[0], groups, -1).transpose(0, 1).contiguous() if groups > 1 else t.unsqueeze(0)


def _joined(t):
    """(groups, P, C) -> (P, groups * C)"""
    return t.transpose(0, 1).reshape(t.shape[1], -1) if t.shape[0] > 1 else t[0]


def _activation(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "leakyrelu":
        return torch.where(z > 0, z, z * _SLOPE)
    if act == "gelu":
        return z * (0.5 + 0.5 * torch.erf(z * math.sqrt(0.5)))
    return z * (z + 3.0).clamp(0.0, 6.0) / 6.0


def _activation_slope(z, act):
    """d act / dz of the activations that the training cases use."""
    return 0.5 + 0.5 * torch.erf(z * math.sqrt(0.5)) + z * torch.exp(z * z * -0.5) * (1.0 / math.sqrt(2.0 * math.pi))


def _run_plain(state):
    case = state["case"]
    if case["op"] == "linear":
        dt, groups, act = _TYPES[case["dtype"]], case["groups"], case["act"]
        x, w = state["x"].detach().float(), state["w"].detach().float()
        xg, wg = _by_group(x, groups), w.view(groups, case["n"], case["k"])
        z = _joined(torch.matmul(xg, wg.transpose(1, 2).contiguous())) + state["b"].detach().float()
        y = _activation(z, act)
        if state["r"] is not None:
            y = y + state["r"].detach().float()
        y = y.to(dt)
        if not case["train"]:
            return y
        dz = state["gy"].float()
        if act != "none":
            dz = dz * _activation_slope(z, act)
        zg = _by_group(dz, groups)
        gx = _joined(torch.matmul(zg, wg)).to(dt)
        gw = torch.matmul(zg.transpose(1, 2).contiguous(), xg).reshape(w.shape).to(dt)
        out = [y, gx, gw, dz.sum(0).to(dt)]
        return out if state["r"] is None else out + [state["gy"]]

    grads = [p.grad for p in state["params"]]
    if case["p"] == math.inf:
        norm = torch.stack([g.abs().max().float() for g in grads]).max()
    elif case["p"] == 1.0:
        norm = torch.stack([g.double().abs().sum() for g in grads]).sum().float()
    else:
        norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt().float()
    if case["op"] == "norm":
        return norm
    factor = (case["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
    [g.copy_(g.float() * factor) for g in grads]
    return [norm] + list(state["flat"].values())


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- sizes and the definition in 64 bits ------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "linear":
        e, p, g = _BYTES[case["dtype"]], case["rows"], case["groups"]
        xs, ws, ys, bs = p * g * case["k"], g * case["n"] * case["k"], p * g * case["n"], g * case["n"]
        numbers = xs + ws + bs + ys * (2 if case["residual"] else 1)
        flops = 2.0 * p * ws
        if case["train"]:      # the incoming gradient read; the gradients of x, w, b written (the residual's is the incoming one)
            numbers += ys + xs + ws + bs
            flops *= 3.0
        return {"bytes": float(numbers * e), "flops": flops}
    size = sum(count * _BYTES[kind] for count, kind in _sizes(case))
    return {"bytes": float(size * (2 if case["op"] == "clip" else 1)), "flops": (3.0 if case["op"] == "clip" else 2.0) * case["values"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "linear":
        d = {kind: t.double() for kind, t in s["flat"].items()}
        if case["p"] == math.inf:
            norm = max(t.abs().amax() for t in d.values())
        else:
            norm = sum((t.abs() ** case["p"]).sum() for t in d.values()) ** (1.0 / case["p"])
        if case["op"] == "norm":
            return norm
        for t in d.values():
            t.mul_(min(1.0, case["max_norm"] / (float(norm) + 1e-6)))
        return [norm] + list(d.values())
    k, n, act = case["k"], case["n"], case["act"]
    x, w, b = (s[i].detach().double() for i in ("x", "w", "b"))
    gy = s["gy"].double() if case["train"] else None
    ys, gxs, gws, gbs = [], [], [], []
    for i in range(case["groups"]):
        xi, wi = x[:, i * k:(i + 1) * k], w[i * n:(i + 1) * n]
        z = torch.addmm(b[i * n:(i + 1) * n], xi, wi.t())
        if act == "gelu":
            tail = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
            y, slope = z * tail, tail + z * torch.exp(-0.5 * z ** 2) / math.sqrt(2.0 * math.pi)
        else:
            slope = torch.ones_like(z)
            y = {"none": lambda: z, "relu": lambda: torch.maximum(z, torch.zeros_like(z)),
                 "leakyrelu": lambda: torch.maximum(z, z * _SLOPE),
                 "hardswish": lambda: torch.where(z <= -3, 0.0 * z, torch.where(z >= 3, z, z * (z + 3) / 6))}[act]()
        ys.append(y)
        if gy is not None:
            dz = gy[:, i * n:(i + 1) * n] * slope
            gxs.append(dz @ wi)
            gws.append(dz.t() @ xi)
            gbs.append(dz.sum(0))
    y = torch.cat(ys, 1)
    if s["r"] is not None:
        y = y + s["r"].detach().double()
    if gy is None:
        return y
    out = [y, torch.cat(gxs, 1), torch.cat(gws, 0), torch.cat(gbs, 0)]
    return out if s["r"] is None else out + [gy]
