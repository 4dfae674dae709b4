"""Updates scaled to a bound on their norm, on device tensors.

    norm = sqrt(sum of squares over everything listed), in 64 bits
    f    = scale * (1 if norm <= max_norm else max_norm / norm)

A client bounds its gradients on the way into its update buffers
(:class:`GradPlan`: any number of tensors, two launches); the server bounds the
sum of its clients' deltas on the way into the master table
(:func:`apply_updates_clipped`, beside rowops.apply_updates).  A norm over several
lists, tables or ranks: add up their sums of squares (``sum_squares``, a float64
device value) and pass the total as ``total``.

C-ABI calls (gp_grad_*, gp_bucket_sum_clipped / _squares, include/gp_reduce.h) on
the caller's current HIP stream; nothing waits for the device, and every call can
be captured into a HIP graph.  The same inputs give the same bits.
"""
from __future__ import annotations

import ctypes
from typing import Sequence

import torch

from . import native
from .native import check
from .routing import _On, _TYPES, _current_device, _current_stream


def _bound(max_norm, scale, skip_nonfinite):
    max_norm, scale = float(max_norm), float(scale)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative or NaN, got {max_norm}")
    if scale - scale != 0.0:
        raise ValueError(f"scale must be finite, got {scale}")
    return max_norm, scale, native.GP_CLIP_SKIP if skip_nonfinite else native.GP_CLIP_PROPAGATE


def _flat(t, name, dtype=None, device=None) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA (HIP) tensor")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on another device")


def _total(total, device):
    if total is None:
        return None
    if (not isinstance(total, torch.Tensor) or total.device != device or total.dtype != torch.float64
            or total.numel() != 1):
        raise ValueError("total must be one float64 value on the tensors' device")
    return total.data_ptr()


def _workspace(like):
    """A call's workspace, on a float32 tensor's device.  The caller holds it until
    the call has returned: another thread may allocate on the same stream."""
    return like.new_empty(native.GP_CLIP_WORKSPACE_BYTES // 4)


class GradPlan:
    """A list of gradients and of the buffers that their scaled values go to,
    compiled once (gp_grad_plan_create, outside of any graph capture), for buffers
    that stay in place from step to step.  ``outs`` (default: the gradients themselves) are of the gradients'
    types or float32, and overlap nothing but, each, its own gradient.  The plan
    keeps the tensors and their storages.  A tensor whose memory was replaced since
    (``t.data = ...``, ``module.half()``, ``resize_``) makes every call raise
    ValueError; it takes a new plan.  A captured graph of the plan's calls needs the
    plan, which holds the table of buffers on the device and their memory, for as
    long as it is replayed; a replay checks nothing, so its tensors keep their
    memory until then."""

    def __init__(self, grads: Sequence[torch.Tensor], outs: Sequence[torch.Tensor] | None = None):
        self._h = ctypes.c_void_p()
        self.grads = list(grads)
        self.outs = self.grads if outs is None else list(outs)
        if not self.grads:
            raise ValueError("no gradients")
        if len(self.outs) != len(self.grads):
            raise ValueError("one output per gradient")
        self.device = getattr(self.grads[0], "device", None)
        for i, (g, o) in enumerate(zip(self.grads, self.outs)):
            _flat(g, f"grads[{i}]", device=self.device)
            if o is not g:
                _flat(o, f"outs[{i}]", device=self.device)
                if o.numel() != g.numel():
                    raise ValueError(f"outs[{i}] has {o.numel()} values, its gradient {g.numel()}")
                if o.dtype not in (g.dtype, torch.float32):
                    raise ValueError(f"outs[{i}] must be {g.dtype} or float32, got {o.dtype}")
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise ValueError("a plan cannot be made while a graph is captured: its table is copied to the device")
            # what a call allocates: the norm and a workspace, each call's own
            self._like = (torch.empty((), dtype=torch.float32, device=self.device),
                          torch.empty(native.GP_CLIP_WORKSPACE_BYTES // 4, dtype=torch.float32, device=self.device))
        # what the table points at: it must not be given to other tensors, and must be what the tensors still hold
        self._tensors = (*self.grads, *(() if outs is None else self.outs))
        self._storages = [t.untyped_storage() for t in self._tensors]
        facts = native.tensor_facts()
        n = len(self.grads)
        ptrs, ints, sizes = ctypes.c_void_p * n, ctypes.c_int * n, ctypes.c_size_t * n
        with torch.cuda.device(self.device):
            check(native.lib().gp_grad_plan_create(
                ctypes.byref(self._h), n, ptrs(*[g.data_ptr() for g in self.grads]),
                ints(*[_TYPES[g.dtype] for g in self.grads]), ptrs(*[o.data_ptr() for o in self.outs]),
                ints(*[_TYPES[o.dtype] for o in self.outs]), sizes(*[g.numel() for g in self.grads])),
                "gp_grad_plan_create")
        # (after data_ptr(), which gives a copy-on-write clone memory of its own)
        self._facts, self._moved = facts.facts(self._tensors), facts.moved

    def _open(self):
        if not self._h:
            raise ValueError("the plan is closed")
        moved = self._moved(self._tensors, self._facts)
        if moved >= 0:
            n = len(self.grads)
            name = f"grads[{moved}]" if moved < n else f"outs[{moved - n}]"
            raise ValueError(f"{name} is not where it was when the plan was made, or of another length or type")

    def sum_squares(self, stream=None) -> torch.Tensor:
        """The sum of the gradients' squares: one float64 value."""
        self._open()
        if stream is not None or self.device.index != _current_device():
            with _On(self.device, stream):
                return self.sum_squares()
        total = torch.empty((), dtype=torch.float64, device=self.device)
        workspace = torch.empty_like(self._like[1])
        check(native.lib().gp_grad_sum_squares(self._h, total.data_ptr(), workspace.data_ptr(),
                                               _current_stream(self.device.index)), "gp_grad_sum_squares")
        return total

    def norm(self, stream=None) -> torch.Tensor:
        """The gradients' norm: one float32 value (infinity past float32's range)."""
        self._open()
        with _On(self.device, stream):
            return self.sum_squares().sqrt().float()

    def clip(self, max_norm: float, scale: float = 1.0, total: torch.Tensor | None = None,
             skip_nonfinite: bool = False, stream=None) -> torch.Tensor:
        """``outs[i] = f * grads[i]`` in 32 bits, rounded once; returns the norm, one
        float32 value.  ``total``: the sum of squares to go by instead of these
        gradients' own.  A norm that is infinite or NaN goes into the outputs, or,
        with ``skip_nonfinite``, makes them zeros."""
        self._open()
        max_norm, scale, mode = _bound(max_norm, scale, skip_nonfinite)
        given = _total(total, self.device)
        if stream is not None or self.device.index != _current_device():
            with _On(self.device, stream):
                return self.clip(max_norm, scale, total, skip_nonfinite)
        norm, workspace = torch.empty_like(self._like[0]), torch.empty_like(self._like[1])
        check(native.lib().gp_grad_clip(self._h, max_norm, scale, mode, given, norm.data_ptr(), workspace.data_ptr(),
                                        _current_stream(self.device.index)), "gp_grad_clip")
        return norm

    def close(self) -> None:
        if self._h:
            native.lib().gp_grad_plan_destroy(self._h)
            self._h = ctypes.c_void_p()
        self.grads = self.outs = self._tensors = self._storages = ()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def _buckets(updates, n, device):
    ptrs = (ctypes.c_void_p * max(1, len(updates)))()
    for k, b in enumerate(updates):
        _flat(b, f"updates[{k}]", torch.float32, device)
        if b.numel() < n:
            raise ValueError(f"updates[{k}] smaller than the master")
        ptrs[k] = b.data_ptr()
    return ptrs


def _scratch(scratch, count, n, device):
    if scratch is not None:
        _flat(scratch, "scratch", torch.float32, device)
        if scratch.numel() < n:
            raise ValueError("scratch smaller than the master")
        return scratch
    return torch.empty(n, dtype=torch.float32, device=device) if count > 2 else None


def sum_updates_squares(updates: Sequence[torch.Tensor], scratch: torch.Tensor | None = None,
                        stream=None) -> torch.Tensor:
    """The sum of squares of ``u = updates[0] + updates[1] + ...`` (float32 tensors
    of one length, added in order): one float64 value.  From three updates on
    ``scratch`` is left holding u, for apply_updates_clipped with ``total``."""
    if not updates:
        raise ValueError("no updates")
    _flat(updates[0], "updates[0]", torch.float32)
    device, n = updates[0].device, updates[0].numel()
    if stream is not None or device.index != _current_device():
        with _On(device, stream):
            return sum_updates_squares(updates, scratch)
    ptrs = _buckets(updates, n, device)
    scratch = _scratch(scratch, len(updates), n, device)
    total, workspace = torch.empty((), dtype=torch.float64, device=device), _workspace(updates[0])
    check(native.lib().gp_bucket_sum_squares(None if scratch is None else scratch.data_ptr(), ptrs, len(updates), n,
                                             total.data_ptr(), workspace.data_ptr(),
                                             _current_stream(device.index)), "gp_bucket_sum_squares")
    return total


def apply_updates_clipped(master: torch.Tensor, updates: Sequence[torch.Tensor], max_norm: float, scale: float = 1.0,
                          out: torch.Tensor | None = None, scratch: torch.Tensor | None = None,
                          total: torch.Tensor | None = None, skip_nonfinite: bool = False,
                          stream=None) -> torch.Tensor:
    """``out = master + f * u`` for ``u = updates[0] + updates[1] + ...`` (in 32
    bits, in order) with u's norm bounded; returns the norm, one float32 value
    (infinity past float32's range; f goes by the 64-bit norm).
    ``out`` defaults to the master.  ``scratch`` (as long as the master) holds u
    between the passes from three updates on; it is allocated when not given.
    ``total``: the sum of squares to go by, over all tables or ranks; u is then
    taken from ``scratch`` as sum_updates_squares left it.  A norm that is infinite
    or NaN goes into the table, or, with ``skip_nonfinite``, leaves it unchanged."""
    _flat(master, "master", torch.float32)
    device, n = master.device, master.numel()
    if stream is not None or device.index != _current_device():
        with _On(device, stream):
            return apply_updates_clipped(master, updates, max_norm, scale, out, scratch, total, skip_nonfinite)
    if out is None:
        out = master
    else:
        _flat(out, "out", torch.float32, device)
        if out.numel() < n:
            raise ValueError("out smaller than the master")
    max_norm, bound_scale, mode = _bound(max_norm, scale, skip_nonfinite)
    ptrs = _buckets(updates, n, device)
    given = _total(total, device)
    if given is not None and scratch is None and len(updates) > 2:
        raise ValueError("total needs the scratch that sum_updates_squares left")
    scratch = _scratch(scratch, len(updates), n, device)
    norm, workspace = master.new_empty(()), _workspace(master)
    check(native.lib().gp_bucket_sum_clipped(out.data_ptr(), master.data_ptr(), ptrs, len(updates), n,
                                             None if scratch is None else scratch.data_ptr(), max_norm, bound_scale, mode,
                                             given, norm.data_ptr(), workspace.data_ptr(),
                                             _current_stream(device.index)), "gp_bucket_sum_clipped")
    return norm
