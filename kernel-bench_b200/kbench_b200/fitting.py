"""The fitting step: the global norm of a list of gradients, clipping by it, and the Adam update.

A solve has two gradients, ``grad_theta`` [S, 3] and ``grad_col`` [S].  A caller that fits several solves with
rates of their own under one norm passes the gradients of all of them in one list.  There is no
reference counterpart of these kernels (the reference's fits run torch optimisers).

    opt = fitting.Adam([theta], lr=0.05, max_norm=1.0)
    grad_theta, grad_col = runtime.run_backward(static, theta, col_weights, saved)
    norm = opt.step([grad_theta])              # a device scalar; nothing waits for the GPU

Tensors are on one CUDA device; gradients are fp32, bf16 or fp16 (each its own), parameters and
moments fp32.  Written tensors must each fill a block of memory (any order of dimensions) and share
it with no other; gradients that are only read may have any strides.  What a call writes gets a new
version, as after any in-place operation.
"""

from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from . import _lib
from .scoring import _DTYPES

_OTHER_DEVICE, _OTHER_DTYPE, _STRIDED, _NOT_F32 = 1, 2, 4, 8  # csrc/kb_host.cpp: gather's flags
_KINDS = {2: 2, 2.0: 2, "max": 0}


def _kind(kind) -> int:
    try:
        return _KINDS[kind]
    except (KeyError, TypeError):
        raise ValueError(f"kind must be 2 or 'max' (got {kind!r})") from None


def _max_norm(max_norm) -> float:
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be non-negative (got {max_norm})")
    return max_norm


def _sequence(tensors):
    return tensors if isinstance(tensors, (list, tuple)) else list(tensors)


def _dense(t) -> bool:
    """Whether the entries of ``t`` fill one block of memory, in some order of its dimensions."""
    if t.is_contiguous():
        return True
    step = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != step:
            return False
        step *= size
    return True


def _same_layout(a, b) -> bool:
    """Whether equal indexes of two dense tensors of one shape are equally far into their memory."""
    return a.is_contiguous() and b.is_contiguous() or \
        all(s == t for s, t, n in zip(a.stride(), b.stride(), a.shape) if n != 1)


def _device(name: str, tensors):
    if not tensors:
        raise ValueError(f"{name} must hold at least one tensor")
    device = tensors[0].device
    if device.type != "cuda":
        raise RuntimeError(f"{name} requires CUDA tensors")
    return device


class _Lists:
    """What the C entry points take of lists of tensors on one device: the first ``n_written`` are
    written, the others read (``in_place``: written tensor i may be read tensor i itself)."""

    def __init__(self, names, lists, device, n_written: int, in_place: bool):
        self.described, self.flags, same, meet = _lib.host().gather(lists, device.index, n_written, in_place)
        self.counts = self.described[-1]
        for name, tensors, flags in zip(names, lists, self.flags):
            if not same:
                _check_shapes(name, tensors, names[0], lists[0])
            if flags & (_OTHER_DEVICE | _OTHER_DTYPE):
                _refuse(name, tensors, device)
        for name, tensors, flags in zip(names[:n_written], lists, self.flags):
            if flags & _STRIDED:
                for t in tensors:
                    if not _dense(t):
                        raise ValueError(f"{name} must each fill one block of memory "
                                         f"(got strides {t.stride()} of {tuple(t.shape)})")
        self.meet = meet
        self.written = ", ".join(names[:n_written])

    def apart(self):
        """Refuses written tensors that share memory."""
        if self.meet:
            raise ValueError(f"{self.written} must not share memory with one another or with what is read")
        return self


def _refuse(name: str, tensors, device):
    for t in tensors:
        if t.device != device:
            raise RuntimeError(f"{name} must be on one CUDA device (got {t.device} beside {device})")
        if t.dtype not in _DTYPES:
            raise RuntimeError(f"{name} supports fp32, bf16 and fp16 tensors only (got {t.dtype})")
    raise RuntimeError(f"{name} must be strided CUDA tensors")


def _check_shapes(name: str, tensors, like_name: str, like):
    if len(tensors) != len(like):
        raise ValueError(f"{name} must have {len(like)} tensors, as {like_name} (got {len(tensors)})")
    for t, u in zip(tensors, like):
        if t.shape != u.shape:
            raise ValueError(f"{name}: shape {tuple(t.shape)} beside {tuple(u.shape)} of {like_name}")


def _in_layout_of(t, like):
    """``t`` with its entries in memory in the order of ``like``'s (a copy where they are not)."""
    return t if _same_layout(t, like) else torch.empty_like(like, dtype=t.dtype).copy_(t)


@lru_cache(maxsize=None)
def _workspace_bytes(n: int) -> int:
    size = ctypes.c_longlong()
    _lib.call("kb_fit_workspace", n, ctypes.byref(size))
    return size.value


def _clip(source, destination, counts, n: int, kind: int, max_norm: float, like):
    size = _workspace_bytes(n)
    norm, ws = _lib.host().fit_buffers(like, size)
    addresses, dtypes = source
    _lib.call_on(like.device, "kb_clip_gradients", addresses, destination, counts, dtypes, n, kind, max_norm,
                 norm.data_ptr(), ws.data_ptr(), size)
    return norm


def gradient_norm(grads, *, kind=2) -> torch.Tensor:
    """The norm of all entries of ``grads`` as one vector, a device scalar: the square root of the sum
    of squares (``kind=2``) or the largest magnitude (``kind="max"``).  It is returned in fp32 (infinite past
    its range); clipping goes by the value in 64 bits."""
    kind = _kind(kind)
    grads = _sequence(grads)
    device = _device("grads", grads)
    norm = _lib.call_host("clip", "kb_clip_gradients", device, grads, None, False, kind, 0.0, _workspace_bytes(len(grads)))
    if norm is not None:
        return norm
    lists = _Lists(("grads",), (grads,), device, 0, False)
    if lists.flags[0] & _STRIDED:
        grads = [t if _dense(t) else t.contiguous() for t in grads]
        lists = _Lists(("grads",), (grads,), device, 0, False)
    return _clip(lists.described[0], None, lists.counts, len(grads), kind, 0.0, grads[0])


def clip_gradients(grads, max_norm, *, kind=2, out=None) -> torch.Tensor:
    """Scales ``grads`` by ``min(1, max_norm / (norm + 1e-6))`` in place, or into the tensors ``out`` (same
    shapes and dtypes), and returns the norm before it (a device scalar)."""
    kind, max_norm = _kind(kind), _max_norm(max_norm)
    grads = _sequence(grads)
    device = _device("grads", grads)
    out = None if out is None else _sequence(out)
    norm = _lib.call_host("clip", "kb_clip_gradients", device, grads, out, True, kind, max_norm,
                          _workspace_bytes(len(grads)))
    if norm is not None:
        return norm
    if out is None:
        lists = _Lists(("grads",), (grads,), device, 1, False).apart()
        source = lists.described[0]
        norm = _clip(source, source[0], lists.counts, len(grads), kind, max_norm, grads[0])
        _lib.host().written(grads)
        return norm
    lists = _Lists(("out", "grads"), (out, grads), device, 1, True)
    if lists.described[0][1] != lists.described[1][1]:
        raise RuntimeError("out must have the gradients' dtypes")
    if (lists.flags[0] | lists.flags[1]) & _STRIDED:
        grads = [_in_layout_of(g, o) for g, o in zip(grads, out)]
        lists = _Lists(("out", "grads"), (out, grads), device, 1, True)
    (destination, _), source = lists.apart().described[:2]
    norm = _clip(source, destination, lists.counts, len(grads), kind, max_norm, grads[0])
    _lib.host().written(out)
    return norm


def adam_step(params, grads, exp_avg, exp_avg_sq, step: int, *, lr: float, beta1: float = 0.9, beta2: float = 0.999,
              eps: float = 1e-8, weight_decay: float = 0.0, max_norm=None, kind=2):
    """Adam's update number ``step`` (from 1) of ``params`` and the moments in place, with decoupled
    weight decay; with ``max_norm`` the gradients count as clipped by their global norm, which is
    returned (a device scalar; ``None`` without).  ``grads`` are not changed.

    The bias corrections of ``step`` are taken on the host: a captured call replays that step's, whatever
    the replay's number, so capture one only where they no longer change (late steps).  As with any graph,
    a replay gives the written tensors no new version."""
    step = int(step)
    if step < 1:
        raise ValueError(f"step counts from 1 (got {step})")
    if not (0.0 <= beta1 < 1.0 and 0.0 <= beta2 < 1.0):
        raise ValueError(f"beta1 and beta2 must be in [0, 1) (got {beta1}, {beta2})")
    if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0):
        raise ValueError("lr, eps and weight_decay must be non-negative")
    kind = -1 if max_norm is None else _kind(kind)
    limit = 0.0 if max_norm is None else _max_norm(max_norm)
    params, grads, exp_avg, exp_avg_sq = map(_sequence, (params, grads, exp_avg, exp_avg_sq))
    device = _device("params", params)
    size = _workspace_bytes(len(grads))
    correction1, correction2 = 1.0 - beta1 ** step, 1.0 - beta2 ** step
    norm = _lib.call_host("adam", "kb_adam_step", device, params, grads, exp_avg, exp_avg_sq, lr, beta1, beta2, eps,
                          weight_decay, correction1, correction2, kind, limit, size)
    if norm is not None:
        return None if max_norm is None else norm
    names = ("params", "exp_avg", "exp_avg_sq", "grads")
    lists = _Lists(names, (params, exp_avg, exp_avg_sq, grads), device, 3, False)
    for name, flags in zip(names[:3], lists.flags):
        if flags & _NOT_F32:
            raise RuntimeError(f"{name} must be fp32")
    if any(flags & _STRIDED for flags in lists.flags):
        for name, ts in (("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq)):
            for t, p in zip(ts, params):
                if not _same_layout(t, p):
                    raise ValueError(f"{name} must have the parameters' strides (got {t.stride()} beside {p.stride()})")
        grads = [_in_layout_of(g, p) for g, p in zip(grads, params)]
        lists = _Lists(names, (params, exp_avg, exp_avg_sq, grads), device, 3, False)
    (p, _), (m, _), (v, _), (g, dtypes) = lists.apart().described[:4]
    norm, ws = _lib.host().fit_buffers(params[0], size)
    _lib.call_on(device, "kb_adam_step", p, g, m, v, lists.counts, dtypes, len(grads), lr, beta1, beta2, eps,
                 weight_decay, correction1, correction2, kind, limit, norm.data_ptr(), ws.data_ptr(), size)
    for tensors in (params, exp_avg, exp_avg_sq):
        _lib.host().written(tensors)
    return None if max_norm is None else norm


class Adam:
    """Adam with decoupled weight decay over fp32 parameters, updated in place; ``max_norm`` clips the
    gradients of each step by their global norm."""

    def __init__(self, params, *, lr: float, beta1: float = 0.9, beta2: float = 0.999, eps: float = 1e-8,
                 weight_decay: float = 0.0, max_norm=None, kind=2):
        self.params = list(params)
        self.options = {"lr": lr, "beta1": beta1, "beta2": beta2, "eps": eps, "weight_decay": weight_decay,
                        "max_norm": max_norm, "kind": kind}
        self.exp_avg = [torch.zeros_like(p) for p in self.params]
        self.exp_avg_sq = [torch.zeros_like(p) for p in self.params]
        self.steps = 0

    def step(self, grads):
        """One update by ``grads`` (one a parameter); the norm before clipping, or ``None``."""
        norm = adam_step(self.params, grads, self.exp_avg, self.exp_avg_sq, self.steps + 1, **self.options)
        self.steps += 1
        return norm
