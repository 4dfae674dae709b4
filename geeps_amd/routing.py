"""Expert row routing on device tensors: a router's (token, choice) pairs grouped
by expert, the tokens' rows moved there, the groups' rows brought back with
weights, and the gradients of both moves.

The row operations of :mod:`geeps_amd.rowops` move rows through an index that the
caller has; these make the index on the device from the router's choices and use
it in the same step.  One C-ABI call each (gp_route_*, include/gp_reduce.h) on
the caller's current HIP stream; nothing waits for the device, and no size comes
back from it: the grouped layout has a fixed number of rows.

    route = sort_tokens(ids, num_experts, align=16)      # places
    rows = dispatch(x, route)                            # (route.order.numel(), width)
    # ... the experts' products over rows[offsets[e]:offsets[e] + counts[e]] ...
    y = combine(rows, route, weights)                    # (tokens, width)

    d_rows, d_weights = combine_grad(dy, rows, route, weights)
    dx = dispatch_grad(d_rows, route)

Outputs carry no gradient: the calls for it are the two above, for a manual
backward pass or an autograd.Function of them.  A tensor that requires one is
refused while gradients are recorded, rather than cut off from its graph; under
torch.no_grad() or inside a Function's forward it is taken.

Every call can be captured into a HIP graph.  Rows are float32, bfloat16 or
float16, one contiguous row after another or with a row stride; sums are kept in
32 bits.  An id outside [0, num_experts) is a choice with no row (padding, or an
expert of another rank): it gets no place, adds nothing, and its weight's
gradient is 0, whatever its weight holds.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import native
from .native import check

MAX_CHOICES = 64     # choices per token
MAX_EXPERTS = 1024

_TYPES = {torch.float32: native.GP_F32, torch.bfloat16: native.GP_BF16, torch.float16: native.GP_F16}


class Route(NamedTuple):
    """Where the choices of (tokens, k) ids lie in the rows grouped by expert
    (int32 tensors of one device)."""

    position: torch.Tensor  # (tokens, k): row of a choice, or -1
    order: torch.Tensor     # (rows,): flat choice t * k + c in a row, or -1
    counts: torch.Tensor    # (experts,): choices of an expert
    offsets: torch.Tensor   # (experts + 1,): first row of an expert's group; the end of the last


_current_device = torch._C._cuda_getDevice
_current_stream = torch._C._cuda_getCurrentRawStream  # (device index) -> hipStream_t, without a Stream object


class _On:
    """The device and stream of a call as the current ones, so that its outputs and
    temporaries are allocated on the stream that uses them.  The calls below enter
    it, and call themselves again, unless both are current already."""

    def __init__(self, device, stream):
        self.guard = [torch.cuda.device(device)]
        if stream is not None:
            if not hasattr(stream, "cuda_stream"):  # a raw hipStream_t: 0 is the device's null stream
                handle = int(stream)
                stream = (torch.cuda.ExternalStream(handle, device=device) if handle
                          else torch.cuda.default_stream(device))
            if stream.device != device:
                raise ValueError("stream of another device than the tensors")
            self.guard.append(torch.cuda.stream(stream))

    def __enter__(self):
        for g in self.guard:
            g.__enter__()

    def __exit__(self, *exc):
        for g in reversed(self.guard):
            g.__exit__(*exc)


def _no_gradient(t, name):
    if isinstance(t, torch.Tensor) and t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which the result would not carry: call this under "
                         "torch.no_grad() or in an autograd.Function, with combine_grad and dispatch_grad for its "
                         "backward pass")


def _rows2d(t, name, dtype=None, device=None, width=None) -> int:
    """The row stride of a (rows, width) tensor, checked."""
    _no_gradient(t, name)
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA (HIP) tensor")
    if t.dim() != 2:
        raise ValueError(f"{name} must have shape (rows, width)")
    if dtype is None:
        if t.dtype not in _TYPES:
            raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    elif t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on another device")
    n, w = t.shape
    if width is not None and w != width:
        raise ValueError(f"{name} must have rows of {width} values, got {w}")
    stride, inner = t.stride()
    if n <= 1:
        stride = w
    if (w > 1 and inner != 1) or stride < w:
        raise ValueError(f"{name} must have contiguous rows that do not overlap")
    return stride


def _route(route, device):
    """(tokens, k, rows) of a route; device: a GPU's."""
    position, order = route.position, route.order
    for t, name in ((position, "route.position"), (order, "route.order")):
        if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 CUDA tensor")
        if t.device != device:
            raise ValueError(f"{name} is on another device")
    if position.dim() != 2 or order.dim() != 1:
        raise ValueError("route.position must have shape (tokens, k) and route.order (rows,)")
    return *position.shape, order.shape[0]


def _out(out, name, shape, like):
    if out is None:
        return like.new_empty(shape), shape[1]
    stride = _rows2d(out, name, like.dtype, like.device, shape[1])
    if out.shape[0] < shape[0]:
        raise ValueError(f"{name} has {out.shape[0]} rows, {shape[0]} are written")
    return out, stride


def _ids(expert_ids, num_experts, align):
    if not isinstance(expert_ids, torch.Tensor) or not expert_ids.is_cuda:
        raise ValueError("expert_ids must be a CUDA (HIP) tensor")
    if expert_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expert_ids must be int32 or int64, got {expert_ids.dtype}")
    if expert_ids.dim() != 2 or not expert_ids.is_contiguous():
        raise ValueError("expert_ids must be a contiguous tensor of shape (tokens, k)")
    tokens, k = expert_ids.shape
    return tokens, k, group_rows(tokens, k, num_experts, align)


def group_rows(tokens: int, k: int, num_experts: int, align: int = 1) -> int:
    """Rows of the grouped layout: every choice, and align - 1 for each expert
    that can have one, rounded down to whole groups."""
    if not 1 <= k <= MAX_CHOICES:
        raise ValueError(f"1 to {MAX_CHOICES} choices per token, got {k}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts, got {num_experts}")
    if not 1 <= align <= 1 << 20:
        raise ValueError(f"align must be 1 to 2^20, got {align}")
    n = tokens * k
    rows = n + min(num_experts, n) * (align - 1)
    if tokens < 0 or rows >= 1 << 31:
        raise ValueError("tokens * choices and the grouped rows must be under 2^31")
    return rows // align * align


def _new_route(tokens, k, rows, num_experts, device):
    """The route's tensors and the sort's workspace, of one allocation."""
    sizes, size = [tokens * k, rows, num_experts, num_experts + 1], 0
    if sizes[0] > native.GP_ROUTE_UNCOUNTED:
        need = ctypes.c_size_t()
        check(native.lib().gp_route_workspace(tokens, k, num_experts, ctypes.byref(need)), "gp_route_workspace")
        size = need.value
        sizes.append(size // 4)
    parts = torch.empty(sum(sizes), dtype=torch.int32, device=device).split_with_sizes(sizes)
    route = Route(parts[0].view(tokens, k), parts[1], parts[2], parts[3])
    return route, parts[4].data_ptr() if size else None, size


def sort_tokens(expert_ids: torch.Tensor, num_experts: int, align: int = 1, stream=None) -> Route:
    """The places of (tokens, k) ``expert_ids`` (int32 or int64) in rows grouped by
    expert, tokens in order inside a group, every group rounded up to whole
    multiples of ``align`` rows."""
    tokens, k, rows = _ids(expert_ids, num_experts, align)
    device = expert_ids.device
    if stream is not None or device.index != _current_device():
        with _On(device, stream):
            return sort_tokens(expert_ids, num_experts, align)
    route, scratch, size = _new_route(tokens, k, rows, num_experts, device)
    check(native.lib().gp_route_sort(expert_ids.data_ptr(), 8 * expert_ids.element_size(), tokens, k, num_experts,
                                     align, route.position.data_ptr(), route.order.data_ptr(),
                                     route.counts.data_ptr(), route.offsets.data_ptr(), scratch, size,
                                     _current_stream(device.index)), "gp_route_sort")
    return route


def dispatch(x: torch.Tensor, route: Route, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """``rows[r] = x[route.order[r] // k]``, zeros where a row holds no choice.
    With ``out`` given, its rows behind the layout are left as they were."""
    stride = _rows2d(x, "x")
    device = x.device
    tokens, k, rows = _route(route, device)
    if x.shape[0] != tokens:
        raise ValueError(f"x has {x.shape[0]} rows, the route {tokens} tokens")
    if stream is not None or device.index != _current_device():
        with _On(device, stream):
            return dispatch(x, route, out)
    width = x.shape[1]
    out, out_stride = _out(out, "out", (rows, width), x)
    check(native.lib().gp_route_dispatch(out.data_ptr(), out_stride, x.data_ptr(), stride, _TYPES[x.dtype],
                                         route.position.data_ptr(), route.order.data_ptr(), tokens, k, rows, width,
                                         _current_stream(device.index)), "gp_route_dispatch")
    return out


def sort_and_dispatch(x: torch.Tensor, expert_ids: torch.Tensor, num_experts: int, align: int = 1,
                      out: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, Route]:
    """``sort_tokens`` and ``dispatch`` in one call (one launch for few choices):
    (rows, route)."""
    stride = _rows2d(x, "x")
    tokens, k, rows = _ids(expert_ids, num_experts, align)
    device = x.device
    if device != expert_ids.device:
        raise ValueError("x is on another device")
    if x.shape[0] != tokens:
        raise ValueError(f"x has {x.shape[0]} rows, expert_ids {tokens} tokens")
    if stream is not None or device.index != _current_device():
        with _On(device, stream):
            return sort_and_dispatch(x, expert_ids, num_experts, align, out)
    width = x.shape[1]
    route, scratch, size = _new_route(tokens, k, rows, num_experts, device)
    out, out_stride = _out(out, "out", (rows, width), x)
    check(native.lib().gp_route_sort_dispatch(out.data_ptr(), out_stride, x.data_ptr(), stride, _TYPES[x.dtype],
                                              expert_ids.data_ptr(), 8 * expert_ids.element_size(), tokens, k,
                                              num_experts, align, width, route.position.data_ptr(),
                                              route.order.data_ptr(), route.counts.data_ptr(),
                                              route.offsets.data_ptr(), scratch, size,
                                              _current_stream(device.index)), "gp_route_sort_dispatch")
    return out, route


def _weights(weights, tokens, k, like) -> int:
    _no_gradient(weights, "weights")
    if not isinstance(weights, torch.Tensor) or weights.device != like.device or not weights.is_contiguous():
        raise ValueError("weights must be a contiguous tensor on the rows' device")
    if weights.dtype not in (torch.float32, like.dtype):
        raise ValueError(f"weights must be float32 or {like.dtype}, got {weights.dtype}")
    if tuple(weights.shape) != (tokens, k):
        raise ValueError(f"weights must have shape {(tokens, k)}, got {tuple(weights.shape)}")
    return _TYPES[weights.dtype]


def combine(rows: torch.Tensor, route: Route, weights: torch.Tensor | None = None, out: torch.Tensor | None = None,
            stream=None) -> torch.Tensor:
    """``y[t] = sum over c of weights[t, c] * rows[route.position[t, c]]``, choices
    in order, in 32 bits, rounded once; choices without a row are left out, and a
    token with none gets zeros.  ``weights`` (tokens, k) are float32 or of the
    rows' type; without them every weight is 1."""
    stride = _rows2d(rows, "rows")
    device = rows.device
    tokens, k, n = _route(route, device)
    if rows.shape[0] < n:
        raise ValueError(f"rows has {rows.shape[0]} rows, the route {n}")
    wtype = native.GP_F32 if weights is None else _weights(weights, tokens, k, rows)
    if stream is not None or device.index != _current_device():
        with _On(device, stream):
            return combine(rows, route, weights, out)
    width = rows.shape[1]
    out, out_stride = _out(out, "out", (tokens, width), rows)
    check(native.lib().gp_route_combine(out.data_ptr(), out_stride, rows.data_ptr(), stride, _TYPES[rows.dtype],
                                        route.position.data_ptr(), None if weights is None else weights.data_ptr(),
                                        wtype, tokens, k, n, width, _current_stream(device.index)),
          "gp_route_combine")
    return out


def dispatch_grad(d_rows: torch.Tensor, route: Route, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The gradient of ``dispatch`` by x: every token's rows of ``d_rows`` summed."""
    return combine(d_rows, route, None, out, stream)


def combine_grad(dy: torch.Tensor, rows: torch.Tensor, route: Route, weights: torch.Tensor,
                 out: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The gradients of ``combine`` with weights by its rows and its weights:
    ``d_rows[r] = weights.flat[order[r]] * dy[order[r] // k]`` (zeros where a row
    holds no choice) and ``d_weights[t, c] = dy[t] . rows[position[t, c]]`` (0 where
    a choice has no row).  ``out``, if given, takes d_rows; its rows behind the
    layout are left as they were."""
    dy_stride = _rows2d(dy, "dy")
    row_stride = _rows2d(rows, "rows", dy.dtype, dy.device, dy.shape[1])
    tokens, k, n = _route(route, dy.device)
    if dy.shape[0] != tokens:
        raise ValueError(f"dy has {dy.shape[0]} rows, the route {tokens} tokens")
    if rows.shape[0] < n:
        raise ValueError(f"rows has {rows.shape[0]} rows, the route {n}")
    wtype = _weights(weights, tokens, k, dy)
    device = dy.device
    if stream is not None or device.index != _current_device():
        with _On(device, stream):
            return combine_grad(dy, rows, route, weights, out)
    width = dy.shape[1]
    out, out_stride = _out(out, "out", (n, width), dy)
    d_weights = torch.empty_like(weights)
    check(native.lib().gp_route_combine_grad(out.data_ptr(), out_stride, d_weights.data_ptr(), dy.data_ptr(),
                                             dy_stride, rows.data_ptr(), row_stride, _TYPES[dy.dtype],
                                             route.position.data_ptr(), route.order.data_ptr(), weights.data_ptr(),
                                             wtype, tokens, k, n, width, _current_stream(device.index)),
          "gp_route_combine_grad")
    return out, d_weights
