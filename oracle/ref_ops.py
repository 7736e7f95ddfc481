"""The reference's op sequence for the graph hot path, restated in PyTorch-CPU.  TEST
INFRASTRUCTURE ONLY (see oracle/__init__.py).

Where ``nextou_oracle.c`` fixes the arithmetic to a canonical form, this file keeps the *ops* the
reference executes, in its order, so that (a) it can be compared value-for-value with golden
vectors made from the reference itself and (b) timing it on the host is a fair stand-in for the
reference's CPU path (bench.py ``cpu_baseline.kind = "port"``; the reference's Python cannot
travel to the GPU box).  Each function cites the reference lines it follows.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def knn_graph_ref(x, y=None, relpos=None, k=9, normalize=True):
    """torch_edge.py:151-163 (normalize) + :58-110 (distance, += relative_pos, topk(-dist)).
    x (B,C,N), y (B,C,M)|None, relpos (N,M)|None -> int64 (B,N,k) in torch.topk's order."""
    with torch.no_grad():
        if normalize:
            x = F.normalize(x, p=2.0, dim=1)
            y = None if y is None else F.normalize(y, p=2.0, dim=1)
        xt = x.transpose(2, 1)                                    # (B,N,C)            :66 / :103
        yt = xt if y is None else y.transpose(2, 1)
        inner = -2 * torch.matmul(xt, yt.transpose(2, 1))         # :20 / :52
        x_sq = torch.sum(torch.mul(xt, xt), dim=-1, keepdim=True)  # :21 / :53
        y_sq = torch.sum(torch.mul(yt, yt), dim=-1, keepdim=True)
        dist = x_sq + inner + y_sq.transpose(2, 1)                # :22 / :55
        if relpos is not None:
            dist += relpos.unsqueeze(0)                           # :79 / :86 / :107
        _, nn_idx = torch.topk(-dist, k=k)                        # :87 / :108
    return nn_idx


def pairwise_ref(x, y=None, row_start=0, row_end=None):
    """torch_edge.py:12-23 / :26-39 / :42-55 on channel-major inputs."""
    xt = x.transpose(2, 1)
    yt = xt if y is None else y.transpose(2, 1)
    row_end = xt.shape[1] if row_end is None else row_end
    xp = xt[:, row_start:row_end]
    inner = -2 * torch.matmul(xp, yt.transpose(2, 1))
    return (xp * xp).sum(-1, keepdim=True) + inner + (yt * yt).sum(-1, keepdim=True).transpose(2, 1)


def batched_index_select_ref(x, idx):
    """torch_nn.py:94-115 — x (B,C,M), idx (B,N,k) int64 -> (B,C,N,k) via the flat (B*M, C) gather."""
    B, C, M = x.shape
    _, N, k = idx.shape
    base = torch.arange(0, B, device=idx.device).view(-1, 1, 1) * M
    flat = (idx + base).contiguous().view(-1)
    feat = x.transpose(2, 1).contiguous().view(B * M, -1)[flat, :]
    return feat.view(B, N, k, C).permute(0, 3, 1, 2).contiguous()


def mr_aggregate_ref(x, nn_idx, y=None, center_idx=None):
    """NexToU_Encoder_Decoder.py:401-409 — x (B,C,N), nn_idx (B,N,k) -> (B,2C,N), differentiable."""
    B, C, N = x.shape
    nn_idx = nn_idx.to(torch.int64)
    if center_idx is None:
        center_idx = torch.arange(N, device=x.device).view(1, N, 1).expand_as(nn_idx)
    x_i = batched_index_select_ref(x, center_idx.to(torch.int64))
    x_j = batched_index_select_ref(x if y is None else y, nn_idx)
    x_j, _ = torch.max(x_j - x_i, -1, keepdim=True)               # :407
    out = torch.cat([x.unsqueeze(2).unsqueeze(-1), x_j.unsqueeze(2)], dim=2)  # :409
    return out.reshape(B, 2 * C, N)


def bti_critical_ref(P, interactions, dim, connectivity, min_thick=1):
    """loss/bti_loss.py:76-117 with the kernel of :52-73 — the float64 conv formulation.
    P: float64 label map (B,1,*sp); interactions: list of (is_inclusion, A tensor, C tensor)."""
    import numpy as np
    k = 2 * min_thick + 1
    if dim == 2:
        kern = np.array([[0, 1, 0], [1, 1, 1], [0, 1, 0]]) if connectivity == 4 else np.ones((k, k))
        conv = F.conv2d
    else:
        if connectivity == 6:
            kern = np.zeros((3, 3, 3))
            kern[1, 1, :] = 1
            kern[1, :, 1] = 1
            kern[:, 1, 1] = 1
        else:
            kern = np.ones((k, k, k))
        conv = F.conv3d
    kernel = torch.from_numpy(kern[None, None]).double()
    critical = None
    for inclusion, lab_a, lab_c in interactions:
        mask_a = torch.isin(P, lab_a).double()
        mask_c = torch.isin(P, lab_c).double()
        if inclusion:
            mask_c = torch.logical_not(torch.logical_or(mask_c, mask_a)).double()
        nb_c = (conv(mask_c, kernel, padding='same') >= 1.0).double()
        nb_a = (conv(mask_a, kernel, padding='same') >= 1.0).double()
        viol = ((nb_c * mask_a + nb_a * mask_c) >= 1.0).double()
        critical = viol if critical is None else torch.logical_or(critical, viol).double()
    return critical


def _norm_act_ref(x, weight, bias, running_mean, running_var, training, momentum, eps, slope, period):
    """The reference op sequence: batch_norm | instance_norm -> leaky_relu (torch_nn.py:84-90).

    x (B,C,S); ``period`` > 0 means x is (1, B*period, S) holding an instance norm (weight index c % period).
    """
    F = torch.nn.functional
    if period:
        z = F.instance_norm(x.view(-1, period, x.shape[-1]), None, None, weight, bias, True, momentum, eps).view_as(x)
    else:
        z = F.batch_norm(x, running_mean, running_var, weight, bias, training, momentum, eps)
    return z if slope == 1.0 else F.leaky_relu(z, slope)


def norm_act_fwd_ref(x, weight, bias, running_mean, running_var, training, momentum, eps, slope, period,
                     pre_bias=None):
    if pre_bias is not None:    # the reference adds the conv bias to the tensor itself (conv -> norm)
        reps = x.shape[1] // pre_bias.numel()
        x = x + pre_bias.repeat(reps).view(1, -1, 1)
    with torch.no_grad():
        y = _norm_act_ref(x, weight, bias, running_mean, running_var, training, momentum, eps, slope, period)
        if training:
            xd = x.double()
            mean = xd.mean(dim=(0, 2))
            invstd = 1.0 / torch.sqrt(xd.var(dim=(0, 2), unbiased=False) + eps)
        else:
            mean, invstd = running_mean.double(), 1.0 / torch.sqrt(running_var.double() + eps)
        if pre_bias is not None:   # the backward protocol works on the bias-free tensor: fold b into the saved mean
            mean = mean - pre_bias.double().repeat(x.shape[1] // pre_bias.numel())
    return y, mean.float(), invstd.float()


def norm_act_bwd_ref(x, gy, weight, bias, save_mean, save_invstd, training, slope, period, eps):
    """autograd of the reference op sequence; inference mode rebuilds the running statistics it was given."""
    with torch.enable_grad():
        xr = x.detach().requires_grad_(True)
        C = x.shape[1]
        npar = period if period else C
        w = (torch.ones(npar) if weight is None else weight.detach().clone()).requires_grad_(True)
        b = (torch.zeros(npar) if bias is None else bias.detach().clone()).requires_grad_(True)
        if training:
            y = _norm_act_ref(xr, w, b, None, None, True, 0.0, eps, slope, period)
        else:
            z = (xr - save_mean.view(1, -1, 1)) * save_invstd.view(1, -1, 1) * w.view(1, -1, 1) + b.view(1, -1, 1)
            y = z if slope == 1.0 else torch.nn.functional.leaky_relu(z, slope)
        gx, gw, gb = torch.autograd.grad(y, (xr, w, b), gy)
    if period:  # the backend protocol returns per-normalised-channel sums; the caller folds them
        B = C // period
        with torch.no_grad():
            xh = (x - save_mean.view(1, -1, 1)) * save_invstd.view(1, -1, 1)
            wv = (torch.ones(npar) if weight is None else weight).repeat(B).view(1, -1, 1)
            bv = (torch.zeros(npar) if bias is None else bias).repeat(B).view(1, -1, 1)
            dz = torch.where(xh * wv + bv > 0, gy, gy * slope)
            return gx, (dz * xh).sum(dim=(0, 2)), dz.sum(dim=(0, 2))
    return gx, gw, gb


def _act64(z, act, slope):
    """value and slope of nextou_linear_act's activations (0 none, 1 relu, 2 leaky relu, 3 gelu, 4 hardswish) in float64"""
    if act == 1:
        return torch.where(z <= 0, torch.zeros_like(z), z), (z > 0).double()
    if act == 2:
        return torch.where(z > 0, z, z * slope), torch.where(z > 0, 1.0, float(slope)).double()
    if act == 3:
        phi = 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == 4:
        return z * (z + 3).clamp(0, 6) / 6, torch.where(z <= -3, 0.0, torch.where(z >= 3, 1.0, (2 * z + 3) / 6))
    return z, torch.ones_like(z)


def _grouped64(a, b, groups):
    """(P, groups*A), (groups*B, A) -> (P, groups*B): a_g b_g^T per group"""
    ag, bg = a.double().reshape(a.shape[0], groups, -1), b.double().reshape(groups, b.shape[0] // groups, -1)
    return torch.stack([ag[:, g] @ bg[g].t() for g in range(groups)], 1).reshape(a.shape[0], -1)


def linear_act_fwd_ref(x, w, bias, residual, act, slope, groups, want_pre):
    """float64 restatement of nextou_linear_act_fwd -> (y in x's type, z in float64 | None)"""
    z = _grouped64(x, w, groups)
    if bias is not None:
        z = z + bias.double()
    y = _act64(z, act, slope)[0]
    if residual is not None:
        y = y + residual.double()
    return y.to(x.dtype), z if want_pre else None


def linear_act_bwd_ref(gy, x, w, saved, saved_kind, act, slope, groups, want_gx, want_gw, gb_dtype):
    """float64 restatement of nextou_linear_act_bwd"""
    dz = gy.double()
    if saved_kind:
        dz = dz * _act64(saved.double(), act, slope)[1]
    n, k = w.shape[0] // groups, w.shape[1]
    wt = w.reshape(groups, n, k).transpose(1, 2).reshape(groups * k, n)
    gx = _grouped64(dz, wt, groups).to(x.dtype) if want_gx else None
    gw = None
    if want_gw:
        dg, xg = dz.reshape(-1, groups, n), x.double().reshape(-1, groups, k)
        gw = torch.cat([dg[:, g].t() @ xg[:, g] for g in range(groups)]).to(w.dtype)
    return gx, gw, None if gb_dtype is None else dz.sum(0).to(gb_dtype)


class TorchRefBackend:
    """Backend protocol of nextou_amd.graph_ops with the reference's op sequence (CPU baseline)."""

    name = "oracle-torch-ref"

    @staticmethod
    def window_gather(x, window, shift):
        return window_gather_ref(x, window, shift)

    @staticmethod
    def window_scatter(src, residual, spatial, window, shift):
        return window_scatter_ref(src, residual, spatial, window, shift)

    @staticmethod
    def pool_rows(x, pool):
        return pool_rows_ref(x, pool)

    @staticmethod
    def cell_gather(x, cell, pool):
        return cell_gather_ref(x, cell, pool)

    @staticmethod
    def cell_scatter(src, cell, spatial, pool):
        return cell_scatter_ref(src, cell, spatial, pool)

    @staticmethod
    def knn_graph(x, y, relpos, k_total, algo=0, normalize=True):
        return knn_graph_ref(x, y, relpos, k_total, normalize).to(torch.int32)

    @staticmethod
    def pairwise_distance(x, y, row_start, row_end):
        return pairwise_ref(x, y, row_start, row_end)

    @staticmethod
    def edge_index(nn_idx, dilation):
        from . import CanonicalBackend
        return CanonicalBackend.edge_index(nn_idx, dilation)

    # mr_fwd / mr_bwd as a pair through autograd of the reference op sequence
    @staticmethod
    def mr_has_arg(B, C, N, M, K):
        return False    # the reference has no such side output: backward re-runs its autograd

    @staticmethod
    def mr_fwd(x, y, nn_idx, center, K, idx_step, want_arg=False):
        idx = nn_idx[:, :, ::idx_step][:, :, :K]
        ctr = None if center is None else center[:, :, ::idx_step][:, :, :K]
        with torch.no_grad():
            return mr_aggregate_ref(x, idx, y, ctr), None

    @staticmethod
    def mr_bwd(gout, x, y, nn_idx, center, K, idx_step):
        idx = nn_idx[:, :, ::idx_step][:, :, :K]
        ctr = None if center is None else center[:, :, ::idx_step][:, :, :K]
        with torch.enable_grad():
            xg = x.detach().requires_grad_(True)
            yg = None if y is None else y.detach().requires_grad_(True)
            out = mr_aggregate_ref(xg, idx, yg, ctr)
            grads = torch.autograd.grad(out, [xg] if yg is None else [xg, yg], gout)
        return grads[0], (None if yg is None else grads[1])

    @staticmethod
    def gather_fwd(src, idx):
        return batched_index_select_ref(src, idx.to(torch.int64))

    @staticmethod
    def gather_bwd(gout, idx, M):
        from . import CanonicalBackend
        return CanonicalBackend.gather_bwd(gout, idx, M)

    @staticmethod
    def argmax_labels(logits):
        return torch.argmax(F.softmax(logits, 1), dim=1).to(torch.uint8)   # bti_loss.py:132-133

    @staticmethod
    def bti_critical(labels, lut_a, lut_c, connectivity, min_thick):
        from . import CanonicalBackend
        return CanonicalBackend.bti_critical(labels, lut_a, lut_c, connectivity, min_thick)

    @staticmethod
    def bti_ce_fwd(logits, target, critical):
        from . import CanonicalBackend
        return CanonicalBackend.bti_ce_fwd(logits, target, critical)

    @staticmethod
    def bti_ce_bwd(logits, target, critical, scale):
        from . import CanonicalBackend
        return CanonicalBackend.bti_ce_bwd(logits, target, critical, scale)

    @staticmethod
    def norm_act_fwd(x, weight, bias, running_mean, running_var, training, momentum, eps, slope, period,
                     pre_bias=None):
        return norm_act_fwd_ref(x, weight, bias, running_mean, running_var, training, momentum, eps, slope, period,
                                pre_bias)

    @staticmethod
    def norm_act_bwd(x, gy, weight, bias, save_mean, save_invstd, training, slope, period, eps):
        return norm_act_bwd_ref(x, gy, weight, bias, save_mean, save_invstd, training, slope, period, eps)

    @staticmethod
    def channel_sum(x, channels_last=False):
        return x.double().sum(dim=[0] + list(range(2, x.dim()))).float()

    linear_act_fwd = staticmethod(linear_act_fwd_ref)
    linear_act_bwd = staticmethod(linear_act_bwd_ref)


# ----------------------------------------------------------------------------------------------
# K3 / K4 checkers: the reference's own op sequences for the window / pool data movement
# (NexToU_Encoder_Decoder.py:781-790 + :634-660, :807-817 + :662-693, :524-549), in PyTorch-CPU.
# ----------------------------------------------------------------------------------------------
def _partition(x, window):
    """'b (s p1) (h p2) (w p3) c -> (b s h w) p1 p2 p3 c' of the channel-last permutation, permuted back (:634-660)."""
    import einops
    if x.dim() == 4:
        w = einops.rearrange(x.permute(0, 2, 3, 1), 'b (h p1) (w p2) c -> (b h w) p1 p2 c', p1=window[0], p2=window[1])
        return w.permute(0, 3, 1, 2)
    w = einops.rearrange(x.permute(0, 2, 3, 4, 1), 'b (s p1) (h p2) (w p3) c -> (b s h w) p1 p2 p3 c',
                         p1=window[0], p2=window[1], p3=window[2])
    return w.permute(0, 4, 1, 2, 3)


def _reverse(windows, window, spatial):
    import einops
    if windows.dim() == 4:
        H, W = spatial
        b = int(windows.shape[0] / (H * W / window[0] / window[1]))
        x = einops.rearrange(windows.permute(0, 2, 3, 1), '(b h w) p1 p2 c -> b (h p1) (w p2) c', p1=window[0],
                             p2=window[1], b=b, h=H // window[0], w=W // window[1])
        return x.permute(0, 3, 1, 2)
    S, H, W = spatial
    b = int(windows.shape[0] / (S * H * W / window[0] / window[1] / window[2]))
    x = einops.rearrange(windows.permute(0, 2, 3, 4, 1), '(b s h w) p1 p2 p3 c -> b (s p1) (h p2) (w p3) c',
                         p1=window[0], p2=window[1], p3=window[2], b=b, s=S // window[0], h=H // window[1],
                         w=W // window[2])
    return x.permute(0, 4, 1, 2, 3)


def window_gather_ref(x, window, shift):
    dims = tuple(range(2, x.dim()))
    if max(shift) > 0:
        x = torch.roll(x, shifts=tuple(-s for s in shift), dims=dims)
    w = _partition(x, window)
    return w.reshape(w.shape[0], w.shape[1], -1).contiguous()


def window_scatter_ref(src, residual, spatial, window, shift):
    dims = tuple(range(2, 2 + len(spatial)))
    x = _reverse(src.reshape(src.shape[0], src.shape[1], *window), window, spatial)
    if max(shift) > 0:
        x = torch.roll(x, shifts=tuple(shift), dims=dims)
    return (x if residual is None else x + residual).contiguous()


def _pool_fn(dim):
    import torch.nn.functional as F
    return (F.max_pool2d, F.max_unpool2d) if dim == 2 else (F.max_pool3d, F.max_unpool3d)


def pool_rows_ref(x, pool):
    from nextou_amd.graph_ops import flat_indices_to_cells
    pool_fn, _ = _pool_fn(x.dim() - 2)
    values, indices = pool_fn(x, pool, pool, return_indices=True)
    return values.reshape(values.shape[0], values.shape[1], -1).contiguous(), flat_indices_to_cells(indices, x.shape[2:], pool)


def cell_scatter_ref(src, cell, spatial, pool):
    """MaxUnpool(out, cat(indices, indices)) (:536-549)."""
    from nextou_amd.graph_ops import cells_to_flat_indices
    _, unpool_fn = _pool_fn(len(spatial))
    indices = cells_to_flat_indices(cell, spatial, pool)
    pooled = [s // p for s, p in zip(spatial, pool)]
    reps = src.shape[1] // indices.shape[1]
    idx = torch.cat([indices] * reps, 1)
    return unpool_fn(src.reshape(src.shape[0], src.shape[1], *pooled), idx, pool, pool, output_size=list(spatial))


def cell_gather_ref(x, cell, pool):
    from nextou_amd.graph_ops import cells_to_flat_indices
    indices = cells_to_flat_indices(cell, x.shape[2:], pool)
    reps = x.shape[1] // indices.shape[1]
    idx = torch.cat([indices] * reps, 1)
    return x.flatten(2).gather(2, idx.flatten(2)).contiguous()


def depth_unroll_ref(x):
    """(B, C, D, H, W) -> (B*D, 3C, H, W): channel kd*C + c of depth slice d is x[:, c, d + kd - 1] (zero outside) — the three depth
    taps a [3,k,k] 'same' convolution of the reference's plain stages (NexToU_Encoder_Decoder.py:125-136) reads for output slice d."""
    b, c, d, h, w = x.shape
    padded = torch.nn.functional.pad(x, (0, 0, 0, 0, 1, 1))                       # zero slices before and after the depth axis
    taps = torch.stack([padded[:, :, kd:kd + d] for kd in range(3)], 1)           # (B, 3, C, D, H, W)
    return taps.permute(0, 3, 1, 2, 4, 5).reshape(b * d, 3 * c, h, w)
