"""``ClipSGD``: nnU-Net's optimizer step — ``clip_grad_norm_(parameters, 12)`` then ``torch.optim.SGD(momentum, nesterov,
weight_decay).step()`` — on this library's step-glue kernels (csrc/step_glue.hip, ABI v13).

The reference sets no optimizer of its own (nnUNetTrainer_NexToU.py:17-91 overrides only build_network_architecture and inherits nnUNetTrainer's ``configure_optimizers`` and
``train_step``); the plug-ins' step therefore ends with torch's multi-tensor clip and SGD — a few dozen launches of a few dozen workgroups
each for the 358 trainable tensors of a cfg-2 network (575 us replayed, profiles/r05_step_glue2.md).  ``ClipSGD`` IS a ``torch.optim.SGD`` (same constructor, ``param_groups``,
``state`` with ``momentum_buffer`` tensors, ``state_dict`` / ``load_state_dict``, LR schedulers) whose ``step()`` names its
tensors to the kernels through a table in device memory: one launch for the update, two more for the clip
(:meth:`clip_and_step`), whatever the tensor count.

Same update rule and operation order as ``torch.optim.SGD(foreach=True)``; results agree to the last bit or two (a fused
multiply-add here, a separately rounded product there — the same spread as between torch's own foreach / fused / single-tensor
variants).  Anything the kernels do not take (CPU or non-float32 parameters, sparse gradients, dampening, maximize) goes through
torch's implementation, unchanged — ``last_path`` / ``last_reason`` say which ran and why; a gradient stored in another element order
than its parameter is copied into the parameter's order first.

``clip_grad_norm_`` and ``grad_norm`` are the clip alone, for any optimizer: gradients of float32, bfloat16 and float16 in one list, the 2-, 1-
or maximum norm, two launches and one more for every 224 tensors of a list longer than that (csrc/grad_norm.hip, ABI v15).
"""
from __future__ import annotations

import array
import ctypes
import functools
import math
import operator
import os
from typing import Iterable, List, Optional, Union

import numpy as np
import torch

from . import _lib
from .graph_ops import _current_device, _raw_stream, _recorded

__all__ = ["ClipSGD", "clip_grad_norm_", "grad_norm"]

_CHUNK = 16384          # elements per workgroup (64 KB of each tensor)


def _same_dense_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Same element order in memory: equal shapes and equal strides in every dimension LONGER THAN ONE.  (The stride of a size-1
    dimension is arbitrary — autograd's layout contract for ``.grad`` ignores it too — and the gradients of (N, K, 1, 1, 1) filters
    routinely arrive with other values there than the parameter has.)"""
    if a.shape != b.shape:
        return False
    sa, sb = a.stride(), b.stride()
    return sa == sb or all(x == y for x, y, n in zip(sa, sb, a.shape) if n > 1)


def _dense(p: torch.Tensor) -> bool:
    """True when ``p``'s elements occupy exactly ``numel`` consecutive slots in some dimension order (contiguous, channels-last ...):
    the tensor can be walked as a flat array."""
    dims = sorted((d for d in range(p.dim()) if p.shape[d] > 1), key=lambda d: p.stride(d))
    expect = 1
    for d in dims:
        if p.stride(d) != expect:
            return False
        expect *= p.shape[d]
    return True


def _stream_of(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream if device.type == "cuda" else 0


def _capturing(device: torch.device) -> bool:
    return device.type == "cuda" and torch.cuda.is_current_stream_capturing()


class _on_device:
    def __init__(self, device):
        self._ctx = torch.cuda.device(device) if device.type == "cuda" else None

    def __enter__(self):
        if self._ctx is not None:
            self._ctx.__enter__()

    def __exit__(self, *exc):
        if self._ctx is not None:
            self._ctx.__exit__(*exc)
        return False


_NORM_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_NORM_CODES = {math.inf: 0, 1.0: 1, 2.0: 2}
_LAST = {4: torch.channels_last, 5: torch.channels_last_3d}
_DTYPE, _DEVICE = operator.attrgetter("dtype"), operator.attrgetter("device")
_GRAD = operator.attrgetter("grad")


class _NotTaken(Exception):
    """Tensors that the kernels do not take and torch's implementation may."""


class _OtherTypes(_NotTaken, TypeError):
    pass


class _OtherDevices(_NotTaken, ValueError):
    pass


def _norm_code(norm_type) -> int:
    code = _NORM_CODES.get(float(norm_type))
    if code is None:
        raise ValueError("the norm of gradients is the 1-, 2- or maximum (inf) norm, not %r" % (norm_type,))
    return code


def _flat_run(t: torch.Tensor) -> bool:
    return t.is_contiguous() or (t.dim() in _LAST and t.is_contiguous(memory_format=_LAST[t.dim()])) or _dense(t)


def _norm_rows(tensors: List[torch.Tensor], in_place: bool):
    """(host table, [(tensor, its dense copy)]) of the tensors that have elements; everything the kernels do not take is refused here."""
    try:
        # the usual list, attribute by attribute (a few hundred tensors: the loop below costs more than the kernels)
        if all(map(torch.Tensor.is_contiguous, tensors)):
            counts, types = list(map(torch.Tensor.numel, tensors)), list(map(_NORM_TYPES.get, map(_DTYPE, tensors)))
            if None not in types and 0 not in counts and len(set(map(_DEVICE, tensors))) == 1:
                at = array.array("q", map(torch.Tensor.data_ptr, tensors))              # (a tensor without storage raises here, or has address 0)
                if 0 not in at:
                    vals = array.array("q", bytes(24 * len(tensors)))
                    vals[0::3], vals[1::3], vals[2::3] = at, array.array("q", counts), array.array("q", types)
                    return vals, []
    except (RuntimeError, NotImplementedError):
        pass
    device, vals, copies = tensors[0].device, array.array("q"), []
    for t in tensors:
        code = _NORM_TYPES.get(t.dtype)
        if code is None or t.layout is not torch.strided:
            raise _OtherTypes("gradient norm: dense float32, bfloat16 or float16 gradients, got %s %s" % (t.layout, t.dtype))
        if t.device != device:
            raise _OtherDevices("gradient norm: gradients on %s and %s" % (device, t.device))
        n = t.numel()
        if n == 0:
            continue
        if not t.data_ptr():
            raise _OtherTypes("gradient norm: a %s without memory of its own" % type(t).__name__)
        if not _flat_run(t):
            if in_place and any(a < b for a, b in _strides_and_reach(t)) and _overlaps_itself(t):
                raise ValueError("gradient norm: a gradient of shape %s and strides %s overlaps itself" % (tuple(t.shape), t.stride()))
            copies.append((t, t.contiguous()))
            vals.extend((copies[-1][1].data_ptr(), n, code))
        else:
            vals.extend((t.data_ptr(), n, code))
    if in_place and copies:                   # (the library compares the dense ones)
        _check_strided_apart(tensors, copies)
    return vals, copies


def _check_strided_apart(tensors: List[torch.Tensor], copies) -> None:
    """RuntimeError where an element of a strided gradient is another gradient's as well."""
    strided = {id(t) for t, _ in copies}
    spans = sorted(((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum(s * (n - 1) for s, n in zip(t.stride(), t.shape))), i, t)
                    for i, t in enumerate(tensors) if t.numel()), key=operator.itemgetter(0, 1, 2))
    open_spans = []
    for lo, hi, _, t in spans:
        open_spans = [(h, o) for h, o in open_spans if h > lo]
        for _, o in open_spans:
            if (id(t) in strided or id(o) in strided) and _share_memory(t, o):
                raise RuntimeError("gradient norm: two of the gradients share memory (the same one listed twice?)")
        open_spans.append((hi, t))


def _share_memory(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors whose spans meet have a byte in common.  Column blocks of one wide tensor are told apart by their addresses modulo
    the row's length; anything else element by element."""
    row = max([s * t.element_size() for t in (a, b) for s, n in zip(t.stride(), t.shape) if n > 1], default=1)
    blocks = []
    for t in (a, b):
        size = t.element_size()
        lo = t.data_ptr() % row
        blocks.append((lo, lo + size + sum(s * size * (n - 1) for s, n in zip(t.stride(), t.shape) if s * size % row)))
    (lo_a, hi_a), (lo_b, hi_b) = blocks
    if max(hi_a, hi_b) <= row and (hi_a <= lo_b or hi_b <= lo_a):
        return False
    return bool(np.intersect1d(_addresses(a), _addresses(b)).size)


def _addresses(t: torch.Tensor) -> np.ndarray:
    """Of every pair of bytes of a float32, bfloat16 or float16 tensor"""
    size = t.element_size()
    at = np.arange(t.data_ptr(), t.data_ptr() + size, 2, dtype=np.int64)
    for s, n in zip(t.stride(), t.shape):
        at = (at[:, None] + np.arange(n, dtype=np.int64) * (s * size)).reshape(-1)
    return at


def _overlaps_itself(t: torch.Tensor) -> bool:
    return any(s == 0 and n > 1 for s, n in zip(t.stride(), t.shape)) or np.unique(_addresses(t)).size * 2 != t.numel() * t.element_size()


def _strides_and_reach(t: torch.Tensor):
    """Per dimension longer than one, by ascending stride: (stride, elements that the smaller dimensions span); a stride below the span may overlap."""
    reach = 1
    for stride, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        yield stride, reach
        reach += stride * (n - 1)


@functools.lru_cache(maxsize=64)
def _multi_norm_bytes(n: int) -> int:
    need = ctypes.c_size_t(0)
    _lib.check(_lib.lib().nextou_multi_norm_workspace(n, ctypes.byref(need)), "multi_norm_workspace")
    return need.value


def _multi_norm(tensors: List[torch.Tensor], code: int, max_norm: float, scale: bool) -> torch.Tensor:
    """float32 (norm, clip factor) of device tensors; ``scale`` multiplies them by the factor in place."""
    first = tensors[0]
    device = first.device
    with _current_device(device):
        vals, copies = _norm_rows(tensors, scale)
        if not vals:
            return torch.zeros(2, device=device)          # only empty tensors
        n, L = len(vals) // 3, _lib.lib()
        need = _multi_norm_bytes(n)
        ws, out = first.new_empty((need,), dtype=torch.uint8), first.new_empty((2,), dtype=torch.float32)
        call = L.nextou_multi_clip if scale else L.nextou_multi_norm
        rc = call(vals.buffer_info()[0], n, code, max_norm, ws.data_ptr(), need, out.data_ptr(), _raw_stream(device.index))
        if rc:
            _lib.check(rc, "multi_clip" if scale else "multi_norm")
        if scale:
            for t, dense in copies:
                t.copy_(dense)
            torch.autograd.graph.increment_version(tensors)      # written by address: a graph that saved one of them has to notice
    return out


@torch.no_grad()
def grad_norm(tensors: Union[torch.Tensor, Iterable[torch.Tensor]], norm_type: float = 2.0) -> torch.Tensor:
    """The ``norm_type``-norm (1, 2 or inf) of all elements of ``tensors`` taken together, as a 0-dim float32 tensor on their device (no host
    synchronisation): what ``torch.nn.utils.get_total_norm`` returns, for float32 / bfloat16 / float16 tensors in one list, with float64 sums
    in a fixed order.  NaN if any element is.  An empty list gives 0.  TypeError / ValueError for other types and mixed devices.  CPU tensors,
    and what a trace or a forward-mode derivative records, go through torch's implementation."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    code = _norm_code(norm_type)
    if not tensors:
        return torch.tensor(0.0)
    if not tensors[0].is_cuda or _recorded():
        return torch.nn.utils.get_total_norm(tensors, float(norm_type)).float()
    return _multi_norm(tensors, code, math.inf, False)[0]


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False, foreach: Optional[bool] = None) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for gradients on the GPU in two launches (and one for every 224 of more than 224 tensors): every gradient times ``min(1, max_norm / (norm + 1e-6))``, in place,
    rounded once; returns the norm before the clip (0-dim float32, no host synchronisation unless ``error_if_nonfinite``).

    Gradients may be float32, bfloat16 and float16 in one list, of any dense layout (others are copied and written back).  A norm that is
    infinite or NaN scales as in torch: to zeros and NaN.  No two gradients may share memory (a parameter listed twice: RuntimeError).
    What the kernels do not take — CPU gradients, other types, sparse and distributed ones, several devices, a trace, a forward-mode derivative — goes
    through torch's implementation, for the same three norms; ``foreach`` is accepted for its signature.  Capturable: the gradients' addresses and
    ``max_norm`` are those of the capture."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    code, max_norm = _norm_code(norm_type), float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError("clip_grad_norm_: max_norm %g" % max_norm)
    grads = [g for g in map(_GRAD, parameters) if g is not None]
    if not grads:
        return torch.tensor(0.0)
    if grads[0].is_cuda and not _recorded():
        try:
            if error_if_nonfinite:
                norm = _multi_norm(grads, code, max_norm, False)[0]
                if not math.isfinite(norm.item()):
                    raise RuntimeError("The total norm of order %s for gradients from `parameters` is non-finite, so it cannot be clipped." % norm_type)
            return _multi_norm(grads, code, max_norm, True)[0]
        except _NotTaken:                     # (raised before anything is launched)
            pass
    return torch.nn.utils.clip_grad_norm_(parameters, max_norm, norm_type, error_if_nonfinite, foreach)


class _Table:
    """Device table + chunk list + workspace of one set of (parameter, gradient, buffer) tensors.  Immutable once built: the values
    travel as kernel arguments (nextou_device_write_i64), so a captured hipGraph keeps rewriting — and its kernels keep reading — the
    table it was captured with; nothing on the host is read at replay and no pinned allocation happens inside a capture."""

    def __init__(self, rows: List[tuple], device: torch.device):
        flat, chunks, total = [], [], 0
        for i, (p, g, m, n) in enumerate(rows):
            flat.extend((p, g, m, n))
            for c in range((n + _CHUNK - 1) // _CHUNK):
                chunks.append(i | (c << 32))              # int32 pair (row, chunk) as one little-endian int64
            total += n
        self.n_tensors, self.n_chunks, self.total = len(rows), len(chunks), total
        self.table = torch.empty((len(flat),), dtype=torch.int64, device=device)
        self.chunks = torch.empty((len(chunks),), dtype=torch.int64, device=device)
        L = _lib.lib()
        with _on_device(device):
            stream = _stream_of(device)
            for dst, vals in ((self.table, flat), (self.chunks, chunks)):
                host = (ctypes.c_int64 * len(vals))(*vals)
                _lib.check(L.nextou_device_write_i64(dst.data_ptr(), ctypes.cast(host, ctypes.c_void_p), len(vals), stream),
                           "device_write_i64")
        self.partial = torch.empty((self.n_chunks,), dtype=torch.float64, device=device)
        self.norm_coef = torch.empty((2,), dtype=torch.float32, device=device)


class ClipSGD(torch.optim.SGD):
    """``torch.optim.SGD`` with the step (and, through :meth:`clip_and_step`, the gradient clip) on own kernels."""

    def __init__(self, params, lr=1e-3, momentum=0.0, dampening=0.0, weight_decay=0.0, nesterov=False, *, maximize=False,
                 foreach=None, differentiable=False, fused=None):
        # torch.optim.SGD's constructor, keyword for keyword: `foreach` / `fused` choose what the FALLBACK path runs (torch's
        # default on the GPU is foreach); the own kernels do not need either
        super().__init__(params, lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay, nesterov=nesterov,
                         maximize=maximize, foreach=foreach, differentiable=differentiable, fused=fused)
        self._clip_request = None        # clip_and_step() -> step(): the max norm of this one step
        self._clip_norm = None
        self._tables = {}
        self._retired = []
        self._static = {}
        self._device_type = "cuda"       # (the CPU tests of the table plumbing run the same code on host tensors against a stand-in library)
        self.last_path = None            # "own" | "torch": which implementation the last step took (tests, bench line)
        self.last_reason = None          # why torch's implementation took it

    def __setstate__(self, state):
        # torch.optim.Optimizer pickles defaults / state / param_groups only: the tables (device pointers of another process) start empty
        super().__setstate__(state)
        self._tables, self._retired, self._static = {}, [], {}
        self.__dict__.setdefault("_device_type", "cuda")
        self.__dict__.setdefault("last_path", None)
        self.__dict__.setdefault("last_reason", None)
        self.__dict__.setdefault("_clip_request", None)
        self.__dict__.setdefault("_clip_norm", None)

    # ---------------------------------------------------------------------------------------------------------------
    def _plan(self, group):
        """(rows, device) of one param group for the kernels, or a string — why torch's implementation has to run it."""
        if os.environ.get("NEXTOU_CLIP_SGD", "1") == "0":
            return "NEXTOU_CLIP_SGD=0"
        if group["dampening"] != 0 or group["maximize"] or group.get("differentiable", False):
            return "dampening / maximize / differentiable"
        if group["nesterov"] and group["momentum"] <= 0:
            return "nesterov without momentum"
        lr = group["lr"]
        if isinstance(lr, torch.Tensor) and not (lr.device.type == self._device_type and lr.dtype == torch.float32 and lr.numel() == 1):
            return "learning-rate tensor not a float32 scalar on the device"
        rows, device = [], None
        f32, want_m, state, static = torch.float32, group["momentum"] != 0, self.state, self._static
        for p in group["params"]:
            g = p.grad
            if g is None:
                continue
            ptr = p.data_ptr()
            rec = static.get(id(p))
            if rec is None or rec[0] != ptr:
                # what does not change from step to step (checked again when the parameter's storage moves): (pointer, strides, count, device)
                if not (p.device.type == self._device_type and p.dtype == f32 and _dense(p)):
                    return "parameter %s %s on %s, strides %s: not a dense float32 %s tensor" % (
                        tuple(p.shape), p.dtype, p.device, p.stride(), self._device_type)
                rec = static[id(p)] = (ptr, p.stride(), p.numel(), p.device, p.shape)
            if device is None:
                device = rec[3]
            if g.dtype != f32 or g.is_sparse or g.device != device or g.shape != rec[4]:
                return "gradient %s %s on %s of parameter %s" % (tuple(g.shape), g.dtype, g.device, tuple(p.shape))
            if g.stride() != rec[1] and not _same_dense_layout(p, g):
                # a gradient in another element order than its parameter (autograd's layout contract makes this rare: a .grad assigned
                # by hand, bucket views of another layout): one copy into the parameter's order, then it is walked flat like the rest
                g = torch.empty_like(p, memory_format=torch.preserve_format).copy_(g)
                p.grad = g
            m = 0
            if want_m:
                st = state[p]
                buf = st.get("momentum_buffer")
                if buf is None:
                    # zeros: momentum * 0 + d = d is torch's "buf = clone(d)" of the first step
                    buf = st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                if buf.dtype != f32 or buf.device != device or buf.shape != rec[4]:
                    return "momentum buffer %s %s on %s of parameter %s" % (tuple(buf.shape), buf.dtype, buf.device, tuple(p.shape))
                if buf.stride() != rec[1] and not _same_dense_layout(p, buf):
                    buf = st["momentum_buffer"] = torch.empty_like(p, memory_format=torch.preserve_format).copy_(buf)
                m = buf.data_ptr()
            if rec[2]:
                rows.append((ptr, g.data_ptr(), m, rec[2]))
        if not rows:
            return "no gradients"
        return rows, device

    def _table(self, gi: int, rows, device) -> _Table:
        key = tuple(rows)
        cached = self._tables.get(gi)
        if cached is not None and cached[0] == key:
            t = cached[1]
        else:
            t = _Table(rows, device)
            self._tables[gi] = (key, t)
        if _capturing(device) and not any(r is t for r in self._retired):
            self._retired.append(t)               # the captured graph's kernels keep reading this table after a later step replaced it
        return t

    @staticmethod
    def _norm_of_groups(rows, device, max_norm):
        vals = array.array("q", [v for _, g, _, n in rows for v in (g, n, 0)])
        L, need = _lib.lib(), ctypes.c_size_t(0)
        with _on_device(device):
            _lib.check(L.nextou_multi_norm_workspace(len(rows), ctypes.byref(need)), "multi_norm_workspace")
            ws = torch.empty((need.value,), dtype=torch.uint8, device=device)
            out = torch.empty((2,), dtype=torch.float32, device=device)
            _lib.check(L.nextou_multi_norm(vals.buffer_info()[0], len(rows), 2, float(max_norm), ws.data_ptr(), need.value, out.data_ptr(),
                                           _stream_of(device)), "multi_norm")
        return out

    # ---------------------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def _own_step(self, max_norm: Optional[float]):
        """The whole step on the kernels; returns the total-norm tensor (None without a clip), or NotImplemented when any group
        needs torch's implementation (nothing but zero-filled momentum buffers has been created then — torch's update of a
        zero buffer is its first-step ``buf = clone(d)``)."""
        groups_with_grads = [gi for gi, g in enumerate(self.param_groups) if any(p.grad is not None for p in g["params"])]
        if not groups_with_grads:
            self.last_reason = None
            return None if max_norm is None else torch.zeros(())
        plans = {gi: self._plan(self.param_groups[gi]) for gi in groups_with_grads}
        why = [pl for pl in plans.values() if isinstance(pl, str)]
        if not why and max_norm is not None and len({device for _, device in plans.values()}) != 1:
            why = ["the clip's norm spans several devices"]
        self.last_reason = why[0] if why else None
        if why:
            return NotImplemented
        live = sorted(plans.items())
        L = _lib.lib()
        norm = shared = None
        if max_norm is not None and len(live) > 1:      # one norm over all groups (K11); each group's update reads its factor
            shared = self._norm_of_groups([r for _, (rows, _) in live for r in rows], live[0][1][1], max_norm)
            norm = shared[0]
        for gi, (rows, device) in live:
            group = self.param_groups[gi]
            t = self._table(gi, rows, device)
            lr = group["lr"]
            lr_dev = lr.data_ptr() if isinstance(lr, torch.Tensor) else None
            with _on_device(device):
                stream = _stream_of(device)
                if max_norm is not None and shared is None:
                    _lib.check(L.nextou_grad_norm_clip_coef(t.table.data_ptr(), t.n_tensors, t.chunks.data_ptr(), t.n_chunks, _CHUNK,
                                                            t.total, t.partial.data_ptr(), float(max_norm), t.norm_coef.data_ptr(),
                                                            stream), "grad_norm_clip_coef")
                    norm = t.norm_coef[0]
                coef = None if max_norm is None else (t.norm_coef if shared is None else shared)
                _lib.check(L.nextou_clip_sgd_update(t.table.data_ptr(), t.n_tensors, t.chunks.data_ptr(), t.n_chunks, _CHUNK, t.total,
                                                    coef.data_ptr() if coef is not None else None,
                                                    0.0 if lr_dev else float(lr), lr_dev, float(group["momentum"]),
                                                    float(group["weight_decay"]), int(bool(group["nesterov"])), stream),
                           "clip_sgd_update")
        written = [p for gi, _ in live for p in self.param_groups[gi]["params"] if p.grad is not None]
        torch.autograd.graph.increment_version(written + [p.grad for p in written])      # written by address: graphs that saved them notice
        return norm

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        max_norm, self._clip_request = self._clip_request, None
        norm = self._own_step(max_norm)
        if norm is NotImplemented:
            self.last_path = "torch"
            if max_norm is not None:
                params = [p for g in self.param_groups for p in g["params"]]
                norm = torch.nn.utils.clip_grad_norm_(params, max_norm)
            else:
                norm = None
            super().step()
        else:
            self.last_path = "own"
        self._clip_norm = norm
        return loss

    def clip_and_step(self, max_norm: float) -> torch.Tensor:
        """``torch.nn.utils.clip_grad_norm_(all parameters of this optimizer, max_norm)`` followed by :meth:`step` — through ``self.step``,
        i.e. with the optimizer's step pre / post hooks, the profiler's record and the LR schedulers' bookkeeping; returns the
        total norm (a 0-dim tensor, no host synchronisation).  The gradients are left scaled, as the clip leaves them.  The returned
        tensor is the caller's own copy outside a stream capture; inside one it is the table's buffer, rewritten by every replay."""
        self._clip_request = float(max_norm)
        try:
            self.step()
        finally:
            self._clip_request = None
        norm, self._clip_norm = self._clip_norm, None
        if isinstance(norm, torch.Tensor) and norm.is_cuda and not _capturing(norm.device):
            norm = norm.clone()
        return norm
