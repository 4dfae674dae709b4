"""Expert row routing (geeps_amd.routing) against plain definitions in 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

from geeps_amd import native, routing

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # a rounding, relative
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}  # ... of a subnormal
U = 2.0 ** -24
TYPES = list(HALF)


# -- plain definitions --------------------------------------------------------
def places(ids, experts, align):
    """(position, order, counts, offsets) choice by choice."""
    tokens, k = ids.shape
    n = tokens * k
    rows = (n + min(experts, n) * (align - 1)) // align * align
    flat = ids.reshape(-1)
    groups = [np.nonzero(flat == e)[0] for e in range(experts)]
    position, order = np.full(n, -1, np.int64), np.full(rows, -1, np.int64)
    counts, offsets = [], [0]
    for g in groups:
        at = offsets[-1] + np.arange(len(g))
        position[g] = at
        order[at] = g
        counts.append(len(g))
        offsets.append(offsets[-1] + -(-len(g) // align) * align)
    return position.reshape(ids.shape), order, np.array(counts), np.array(offsets)


def same_route(route, want):
    for got, exp in zip(route, want):
        assert np.array_equal(got.cpu().numpy(), exp)


def choices(tokens, k, experts, seed, drop=0.0, dtype=torch.int64):
    r = np.random.default_rng(seed)
    ids = r.random((tokens, experts)).argsort(1)[:, :k] if tokens else np.zeros((0, k), np.int64)
    if drop and tokens:
        ids[r.random(ids.shape) < drop] = -1
        ids[tokens - int(tokens * drop / 2):] = experts + 3
    return torch.from_numpy(np.ascontiguousarray(ids)).to(dtype)


def held_rows(values, position):
    """(tokens, k, width) rows in 64 bits, zeros where a choice has none."""
    p = position.long()
    r = values.double()[p.clamp(min=0)]
    return torch.where((p >= 0)[..., None], r, torch.zeros((), dtype=torch.float64, device=r.device))


def within(got, want, bound, dtype):
    """|got - want| <= bound before the last rounding, and that rounding."""
    bound = bound + HALF[dtype] * (want.abs() + bound) + TINY[dtype]
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


def check_combine(y, rows, position, weights):
    r = held_rows(rows, position)
    w = torch.ones_like(position, dtype=torch.float64) if weights is None else weights.double()
    w = torch.where(position >= 0, w, 0.0)
    terms = w[..., None] * r
    # k multiply-adds in 32 bits: each rounds a partial sum that is at most sum |w r|
    within(y, terms.sum(1), position.shape[1] * U * 1.01 * terms.abs().sum(1), y.dtype)


def check_combine_grad(d_rows, d_weights, dy, rows, route, weights):
    position, order = route.position, route.order.long()
    k, width = position.shape[1], dy.shape[1]
    at = order.clamp(min=0)
    want = weights.double().reshape(-1)[at][:, None] * dy.double()[at // k]
    want = torch.where((order >= 0)[:, None], want, 0.0)
    within(d_rows[:len(order)], want, U * want.abs(), dy.dtype)  # one product in 32 bits
    terms = held_rows(rows, position) * dy.double()[:, None]
    # a lane adds `per` values for every 64 * per of the row, then the wave's 6 steps and 3 more joins
    per = 16 // dy.element_size()
    depth = per * -(-width // (64 * per)) + 9
    within(d_weights, terms.sum(2), depth * U * 1.01 * terms.abs().sum(2), d_weights.dtype)


def as_device(shape, dtype, dev, seed, layout="plain"):
    """Random rows; "wide": the middle of wider rows, at an odd element."""
    g = torch.Generator().manual_seed(seed)
    n, w = shape
    if layout == "wide":
        return torch.randn(n, w + 9, generator=g).to(dtype).to(dev)[:, 3:3 + w]
    return torch.randn(n, w, generator=g).to(dtype).to(dev)


# -- refusals (no device) -----------------------------------------------------
def test_group_rows():
    assert routing.group_rows(0, 2, 8, 16) == 0
    assert routing.group_rows(1, 1, 1024, 16) == 16
    assert routing.group_rows(5, 2, 3, 4) == 16
    assert routing.group_rows(7, 3, 4) == 21
    rows = ctypes.c_size_t()
    for args in ((0, 2, 8, 16), (1, 1, 1024, 16), (5, 2, 3, 4), (7, 3, 4, 1), (1 << 20, 8, 512, 128)):
        assert native.lib().gp_route_rows(*args, ctypes.byref(rows)) == 0
        assert rows.value == routing.group_rows(*args)
    for bad in ((4, 0, 8, 1), (4, 65, 80, 1), (4, 2, 0, 1), (4, 2, 1025, 1), (4, 2, 8, 0), (4, 2, 8, (1 << 20) + 1),
                (1 << 30, 2, 8, 1), (1 << 29, 4, 8, 1), ((1 << 31) - 20, 1, 8, 4)):
        with pytest.raises(ValueError):
            routing.group_rows(*bad)
        assert native.lib().gp_route_rows(*bad, ctypes.byref(rows)) == native.GP_ERR_INVALID, bad


def test_tensors_refused_without_device():
    ids, x = torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 8)
    route = routing.Route(*(torch.zeros(s, dtype=torch.int32) for s in ((4, 2), 8, 3, 4)))
    for call in (lambda: routing.sort_tokens(ids, 3), lambda: routing.dispatch(x, route),
                 lambda: routing.sort_and_dispatch(x, ids, 3), lambda: routing.combine(x, route),
                 lambda: routing.combine_grad(x, x, route, torch.zeros(4, 2))):
        with pytest.raises(ValueError):
            call()


def test_c_calls_refused_without_device():
    L, p, n = native.lib(), ctypes.c_void_p, native
    a, b, c, d = (p(1 << 20), p(2 << 20), p(3 << 20), p(4 << 20))

    def refused(rc, word):
        assert rc == n.GP_ERR_INVALID and word in L.gp_last_error(), L.gp_last_error()

    refused(L.gp_route_sort(a, 16, 4, 2, 8, 1, b, c, d, d, None, 0, None), b"32 or 64")
    refused(L.gp_route_sort(a, 64, 4, 2, 2000, 1, b, c, d, d, None, 0, None), b"experts")
    refused(L.gp_route_sort(None, 64, 4, 2, 8, 1, b, c, d, d, None, 0, None), b"null")
    refused(L.gp_route_sort(a, 64, 4, 2, 8, 1, b, c, None, d, None, 0, None), b"null")
    need = ctypes.c_size_t()
    assert L.gp_route_workspace(100000, 8, 256, ctypes.byref(need)) == 0 and need.value > 0
    refused(L.gp_route_sort(a, 64, 100000, 8, 256, 1, b, c, d, d, None, 0, None), b"workspace")
    refused(L.gp_route_sort(a, 64, 100000, 8, 256, 1, b, c, d, d, a, need.value - 1, None), b"workspace")

    def move(out=a, os=8, x=b, xs=8, t=0, tokens=4, k=2, rows=8, width=8):
        return L.gp_route_dispatch(out, os, x, xs, t, c, d, tokens, k, rows, width, None)

    refused(move(t=3), b"type")
    refused(move(os=7), b"stride")
    refused(move(xs=7), b"stride")
    refused(move(out=None), b"null")
    refused(move(x=a), b"overlaps")
    refused(move(x=p((1 << 20) + 8 * 8 * 4 - 4)), b"overlaps")
    refused(move(k=65), b"choices")
    refused(move(width=(1 << 24) + 1, os=1 << 25, xs=1 << 25), b"width")
    assert move(rows=0) == 0 and move(width=0) == 0

    def back(y=a, r=b, t=0, w=c, wt=0, tokens=4):
        return L.gp_route_combine(y, 8, r, 8, t, d, w, wt, tokens, 2, 8, 8, None)

    refused(back(t=1, wt=2), b"weights")
    refused(back(y=None), b"null")
    refused(back(r=a), b"overlaps")
    assert back(tokens=0) == 0

    def grad(dr=a, dw=c, dy=b, r=p(5 << 20), w=c, t=0, wt=0):
        return L.gp_route_combine_grad(dr, 8, dw, dy, 8, r, 8, t, d, d, w, wt, 4, 2, 8, 8, None)

    refused(grad(t=2, wt=1), b"weights")
    refused(grad(w=None), b"null")
    refused(grad(dr=b), b"overlaps dy")
    refused(grad(r=a), b"overlaps the rows")


# -- places -------------------------------------------------------------------
SORTS = [(0, 2, 8, 4, 0.0), (1, 1, 1, 1, 0.0), (1, 8, 256, 16, 0.0), (3, 2, 5, 4, 0.5), (17, 3, 60, 8, 0.2),
         (64, 1, 2, 1, 0.0), (65, 4, 7, 128, 0.1), (341, 3, 33, 1, 0.0), (1000, 8, 64, 16, 0.0), (1025, 8, 64, 1, 0.05),
         (2049, 4, 1024, 2, 0.3), (5001, 7, 129, 64, 0.0), (40000, 8, 256, 16, 0.05), (300001, 4, 512, 1, 0.0),
         (200, 64, 100, 1, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,k,experts,align,drop", SORTS)
@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_places(dev, tokens, k, experts, align, drop, dtype):
    r = np.random.default_rng(tokens + k)
    ids = r.integers(0, experts, (tokens, k)) if tokens > 20000 else choices(tokens, k, experts, 3, drop).numpy()
    if tokens > 20000 and drop:
        ids[r.random(ids.shape) < drop] = -7
    route = routing.sort_tokens(torch.from_numpy(ids).to(dtype).to(dev), experts, align)
    same_route(route, places(ids, experts, align))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 63, 100, 9000])
def test_places_of_lopsided_ids(dev, n):
    for fill in (0, 6, -1, 7, 1 << 40, -(1 << 40), (1 << 32) + 2):
        ids = torch.full((n, 2), fill, dtype=torch.int64)
        same_route(routing.sort_tokens(ids.to(dev), 7, 4), places(ids.numpy(), 7, 4))
    ids = torch.arange(2 * n).view(n, 2) % 7  # the same expert may be chosen twice
    ids[:, 1] = ids[:, 0]
    same_route(routing.sort_tokens(ids.to(dev), 7, 3), places(ids.numpy(), 7, 3))


# -- moves --------------------------------------------------------------------
MOVES = [  # tokens, k, experts, width, align, drop
    (1, 1, 1, 1, 1, 0.0), (1, 8, 16, 4096, 1, 0.0), (2, 2, 4, 7, 4, 0.0), (5, 3, 4, 8, 8, 0.5), (16, 4, 64, 2048, 1, 0.0),
    (33, 2, 9, 513, 16, 0.3), (64, 9, 12, 1000, 1, 0.1), (127, 6, 33, 777, 4, 0.2), (300, 15, 40, 130, 1, 0.0),
    (1021, 5, 64, 96, 16, 1.0), (6000, 2, 8, 260, 1, 0.02), (4500, 11, 64, 33, 1, 0.1), (9, 64, 80, 70, 2, 0.1)]


def routed(dev, tokens, k, experts, align, drop, seed=5):
    ids = choices(tokens, k, experts, seed, drop).to(dev)
    return ids, routing.sort_tokens(ids, experts, align)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["plain", "wide"])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,k,experts,width,align,drop", MOVES)
def test_moves(dev, tokens, k, experts, width, align, drop, dtype, layout):
    ids, route = routed(dev, tokens, k, experts, align, drop)
    same_route(route, places(ids.cpu().numpy(), experts, align))
    n = route.order.numel()
    x = as_device((tokens, width), dtype, dev, 1, layout)
    out = as_device((n + 3, width), dtype, dev, 2, layout)
    tail = out[n:].clone()
    got = routing.dispatch(x, route, out=out)
    assert got is out and torch.equal(out[n:], tail)  # rows behind the layout: as they were
    at = route.order.long().clamp(min=0)
    want = torch.where((route.order >= 0)[:, None], x[at // k], torch.zeros((), dtype=dtype, device=dev))
    assert torch.equal(out[:n], want)
    rows2, route2 = routing.sort_and_dispatch(x, ids, experts, align)
    assert torch.equal(rows2, want) and all(torch.equal(p, q) for p, q in zip(route, route2))

    rows = as_device((n, width), dtype, dev, 3, layout)
    rows[route.order < 0] = float("nan")  # a row that holds no choice is not read
    w = torch.rand(tokens, k, generator=torch.Generator().manual_seed(4)).to(dev) - 0.3
    w[route.position < 0] = float("nan")  # nor is the weight of a choice without a row
    for weights in (w, w.to(dtype), None):
        check_combine(routing.combine(rows, route, weights), rows, route.position, weights)
    check_combine(routing.dispatch_grad(rows, route), rows, route.position, None)
    y = as_device((tokens, width), dtype, dev, 6, layout)
    assert routing.combine(rows, route, w, out=y) is y
    assert torch.equal(y, routing.combine(rows, route, w))

    dy = as_device((tokens, width), dtype, dev, 7, layout)
    out = as_device((n + 2, width), dtype, dev, 8, layout)
    tail = out[n:].clone()
    for weights in (w, w.to(dtype)):
        d_rows, d_weights = routing.combine_grad(dy, rows, route, weights, out=out)
        assert d_rows is out and torch.equal(out[n:], tail)
        check_combine_grad(d_rows, d_weights, dy, rows, route, weights)
        assert bool((d_weights[route.position < 0] == 0).all())


@pytest.mark.gpu
def test_gradients_against_differences(dev):
    """combine is linear in its rows and in its weights, so a central difference
    is its derivative but for the 32-bit roundings of the two sums."""
    _, route = routed(dev, 6, 3, 5, 2, 0.2)
    n, width = route.order.numel(), 5
    rows, w = as_device((n, width), torch.float32, dev, 1), torch.rand(6, 3).to(dev)
    dy = as_device((6, width), torch.float32, dev, 2)
    d_rows, d_weights = routing.combine_grad(dy, rows, route, w)

    def loss(r, v):
        return float((routing.combine(r, route, v).double() * dy.double()).sum())

    # two sums of at most 18 * 5 terms, each under 2 * 4 * 4 = 32 in size, roundings 3 * 2^-24 of it, over 2h = 1
    tol = 2 * 90 * 32 * 3 * U
    for i in range(w.numel()):
        up, down = w.clone(), w.clone()
        up.view(-1)[i] += 0.5
        down.view(-1)[i] -= 0.5
        step = float(up.view(-1)[i].double() - down.view(-1)[i].double())
        assert abs((loss(rows, up) - loss(rows, down)) / step - float(d_weights.view(-1)[i])) < tol
    for i in range(rows.numel()):
        up, down = rows.clone(), rows.clone()
        up.view(-1)[i] += 0.5
        down.view(-1)[i] -= 0.5
        step = float(up.view(-1)[i].double() - down.view(-1)[i].double())
        assert abs((loss(up, w) - loss(down, w)) / step - float(d_rows.view(-1)[i])) < tol


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_round_trip_and_its_gradient(dev, dtype):
    """dispatch, a product per expert, combine, and back, as a layer of experts
    runs them, against autograd through the plain formulas in 64 bits."""
    tokens, k, experts, width, align = 75, 3, 6, 48, 8
    ids, _ = routed(dev, tokens, k, experts, align, 0.1)
    x, w = as_device((tokens, width), dtype, dev, 1), torch.rand(tokens, k).to(dev)
    gain = as_device((experts, width), dtype, dev, 2)
    rows, route = routing.sort_and_dispatch(x, ids, experts, align)
    expert = torch.searchsorted(route.offsets[1:].long(), torch.arange(len(rows), device=dev), right=True)
    expert = expert.clamp(max=experts - 1)
    scaled = (rows.float() * gain.float()[expert]).to(dtype)
    y = routing.combine(scaled, route, w)
    dy = as_device((tokens, width), dtype, dev, 3)
    d_scaled, d_w = routing.combine_grad(dy, scaled, route, w)
    d_rows = (d_scaled.float() * gain.float()[expert]).to(dtype)
    dx = routing.dispatch_grad(d_rows, route)

    x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
    good = (ids >= 0) & (ids < experts)
    chosen = x64[:, None] * gain.double()[torch.where(good, ids, 0)] * good[..., None]
    y64 = (w64[..., None] * chosen).sum(1)
    y64.backward(dy.double())
    u = HALF[dtype] + 2 * U
    # y: the rounded rows, then the sum's own rounding; terms bounded by their absolute sum
    size = (w64[..., None] * chosen).abs().sum(1).detach()
    assert bool(((y.double() - y64.detach()).abs() <= 2.1 * u * size + (k + 2) * U * size + TINY[dtype] * 4).all())
    terms = (chosen.detach() * dy.double()[:, None]).abs().sum(2)
    assert bool(((d_w.double() - w64.grad).abs() <= (1.1 * u + 32 * U) * terms + 1e-30).all())
    size = (w64.detach()[..., None] * dy.double()[:, None] * gain.double()[torch.where(good, ids, 0)]
            * good[..., None]).abs().sum(1)
    assert bool(((dx.double() - x64.grad).abs() <= 3.1 * u * size + (k + 2) * U * size + TINY[dtype] * 8).all())


@pytest.mark.gpu
def test_infinities_stay_in_their_rows(dev):
    _, route = routed(dev, 20, 2, 4, 1, 0.0)
    x = torch.ones(20, 24, device=dev)
    x[3] = float("inf")
    x[4, 5] = float("nan")
    y = routing.combine(routing.dispatch(x, route), route, torch.full((20, 2), 0.5, device=dev))
    assert torch.equal(torch.isfinite(y), torch.isfinite(x)) and bool((y[3] == float("inf")).all())
    assert bool(torch.isnan(y[4, 5]))


@pytest.mark.gpu
def test_past_32_bit_offsets(dev):
    """More than 2^32 values in the grouped rows."""
    tokens, width = 262_149, 16_400
    ids = (torch.arange(tokens, device=dev) * 7919 % 3).view(-1, 1)
    x = torch.randint(-100, 100, (tokens, width), dtype=torch.int8, device=dev).to(torch.bfloat16)
    rows, route = routing.sort_and_dispatch(x, ids, 3)
    assert rows.numel() > 1 << 32
    pick = torch.cat([torch.arange(64), torch.arange(tokens - 64, tokens), torch.arange(0, tokens, 997)]).to(dev)
    assert torch.equal(rows[pick], x[route.order[pick].long()])
    y = routing.combine(rows, route)
    assert torch.equal(y[pick], x[pick]) and bool((y == x).all())


@pytest.mark.gpu
def test_streams_and_repeats(dev):
    """Calls on two streams at once, each with its own data, and the same bits again."""
    cases = []
    for seed in (1, 2):
        ids = choices(3000, 4, 32, seed, 0.1).to(dev)
        x = as_device((3000, 200), torch.bfloat16, dev, seed)
        w = torch.rand(3000, 4, generator=torch.Generator().manual_seed(seed)).to(dev)
        cases.append((ids, x, w))

    def whole(ids, x, w, stream=None):
        rows, route = routing.sort_and_dispatch(x, ids, 32, 16, stream=stream)
        y = routing.combine(rows, route, w, stream=stream)
        return (rows, *route, y, *routing.combine_grad(x, rows, route, w, stream=stream))

    want = [whole(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        got = [whole(*c, stream=s) for c, s in zip(cases, streams)]
        raw = whole(*cases[0], stream=streams[1].cuda_stream)
        torch.cuda.synchronize()
        for g, e in zip(got + [raw], want + want[:1]):
            assert all(torch.equal(a, b) for a, b in zip(g, e))


@pytest.mark.gpu
def test_captured_and_replayed(dev):
    """A graph of the whole pass, replayed on new inputs between eager work."""
    tokens, k, experts, width = 2600, 4, 24, 136
    ids, x = choices(tokens, k, experts, 1, 0.1).to(dev), as_device((tokens, width), torch.float16, dev, 1)
    w, dy = torch.rand(tokens, k).to(dev), as_device((tokens, width), torch.float16, dev, 2)

    def whole():
        rows, route = routing.sort_and_dispatch(x, ids, experts, 8)
        y = routing.combine(rows, route, w)
        d_rows, d_w = routing.combine_grad(dy, rows, route, w)
        return (rows, *route, y, d_rows, d_w, routing.dispatch_grad(d_rows, route))

    whole()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = whole()
    for seed in (1, 2, 3, 4):
        ids.copy_(choices(tokens, k, experts, seed, 0.2 * (seed - 1)))
        x.copy_(as_device((tokens, width), torch.float16, dev, 10 + seed))
        w.copy_(torch.rand(tokens, k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, whole())), seed


@pytest.mark.gpu
def test_refusals(dev):
    ids, route = routed(dev, 8, 2, 4, 1, 0.0)
    x = torch.zeros(8, 16, device=dev)
    rows = torch.zeros(16, 16, device=dev)
    w = torch.ones(8, 2, device=dev)
    bad = [
        lambda: routing.sort_tokens(ids.float(), 4), lambda: routing.sort_tokens(ids.t(), 4),
        lambda: routing.sort_tokens(ids[0], 4), lambda: routing.sort_tokens(ids, 0),
        lambda: routing.dispatch(x.double(), route), lambda: routing.dispatch(x.t(), route),
        lambda: routing.dispatch(x[:7], route), lambda: routing.dispatch(x, route, out=rows[:15]),
        lambda: routing.dispatch(x, route, out=rows.half()), lambda: routing.dispatch(x[:1].expand(8, 16), route),
        lambda: routing.dispatch(x, route, out=torch.zeros(16, 17, device=dev)),
        lambda: routing.dispatch(x, route._replace(order=route.order.long())),
        lambda: routing.sort_and_dispatch(x[:7], ids, 4),
        lambda: routing.combine(rows[:15], route, w), lambda: routing.combine(rows, route, w.double()),
        lambda: routing.combine(rows, route, w[:7]), lambda: routing.combine(rows, route, w.cpu()),
        lambda: routing.combine(rows, route, w, out=x[:, :8]),
        lambda: routing.combine_grad(x, rows.half(), route, w), lambda: routing.combine_grad(x[:7], rows, route, w),
        lambda: routing.combine_grad(x, rows[:, :8], route, w),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    both = torch.zeros(24, 16, device=dev)
    with pytest.raises(native.GpError, match="overlaps"):
        routing.dispatch(both[:8], route, out=both[4:20])
    with pytest.raises(native.GpError, match="overlaps"):
        routing.combine(both[:16], route, w, out=both[10:18])
    with pytest.raises(native.GpError, match="overlaps"):
        routing.combine_grad(x, rows, route, w, out=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,k,experts,align,width", [
    (0, 3, 5, 4, 16), (1, 1, 1024, 64, 40), (16, 64, 64, 1, 24), (128, 8, 1024, 3, 9), (205, 5, 300, 16, 130),
    (1024, 1, 3, 8, 8), (1025, 1, 3, 8, 8), (40, 2, 7, 1, 0)])
def test_sort_and_dispatch_few_choices(dev, id_type, tokens, k, experts, align, width):
    """The one-launch form up to 1024 choices and the first sizes past it."""
    r = np.random.default_rng(tokens)
    for kind in ("any", "one", "none"):
        ids = r.integers(-2, experts + 2, (tokens, k)) if kind == "any" else np.full((tokens, k), 0 if kind == "one" else -1)
        want = places(np.where((ids >= 0) & (ids < experts), ids, -1), experts, align)
        x = as_device((tokens, width), torch.bfloat16, dev, 1)
        out = as_device((len(want[1]) + 5, width), torch.bfloat16, dev, 2)
        tail = out[len(want[1]):].clone()
        rows, route = routing.sort_and_dispatch(x, torch.from_numpy(ids).to(id_type).to(dev), experts, align, out=out)
        assert rows is out and torch.equal(out[len(want[1]):], tail)
        same_route(route, want)
        assert torch.equal(out[:len(want[1])], routing.dispatch(x, route))
        held = route.order >= 0
        assert torch.equal(out[:len(want[1])][held], x[route.order[held].long() // k])
        assert not bool(out[:len(want[1])][~held].any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tokens,k,experts,align,width", [
    (torch.bfloat16, 17, 64, 64, 1, 24), (torch.float32, 1025, 1, 1, 64, 1), (torch.float16, 513, 3, 1024, 3, 130),
    (torch.bfloat16, 5461, 3, 60, 16, 128), (torch.float32, 16385, 1, 300, 8, 33), (torch.bfloat16, 6001, 3, 1024, 1, 64),
    (torch.float16, 9001, 7, 5, 32, 72), (torch.bfloat16, 600, 2, 9, 1, 5001)])
def test_sort_and_dispatch_more_choices(dev, dtype, tokens, k, experts, align, width):
    """Places and moves in one launch: with every block's own count, and past 16384 choices with counts in runs."""
    r = np.random.default_rng(tokens)
    for kind in ("any", "last first", "one", "none"):
        if kind == "any":
            ids = r.integers(-2, experts + 2, (tokens, k))
        elif kind == "last first":  # the groups' order is the tokens' backwards
            ids = np.sort(r.integers(0, experts, (tokens, k)), axis=0)[::-1].copy()
        else:
            ids = np.full((tokens, k), experts - 1 if kind == "one" else experts)
        want = places(np.where((ids >= 0) & (ids < experts), ids, -1), experts, align)
        n = len(want[1])
        x = as_device((tokens, width), dtype, dev, 1)
        wide = as_device((n + 5, width + 3), dtype, dev, 2)  # rows of another stride, at an odd place
        before, out = wide.clone(), wide[:, 2:2 + width]
        rows, route = routing.sort_and_dispatch(x, torch.from_numpy(ids).to(dev), experts, align, out=out)
        plain, again = routing.sort_and_dispatch(x, torch.from_numpy(ids).int().to(dev), experts, align)
        same_route(route, want)
        same_route(again, want)
        held = route.order >= 0
        assert torch.equal(plain[held], x[route.order[held].long() // k]) and not bool(plain[~held].any())
        assert rows is out and torch.equal(out[:n], plain)
        before[:n, 2:2 + width] = plain
        assert torch.equal(wide, before)


@pytest.mark.gpu
def test_more_waves_than_a_grid_holds(dev):
    """2^26 tokens: more than 2^32 lanes."""
    tokens = (1 << 26) + 1003
    ids = (torch.arange(tokens, device=dev, dtype=torch.int32) * 7919 % 5 - 1).view(-1, 1)
    x = (torch.arange(tokens, device=dev, dtype=torch.int32) % 2039).to(torch.float16).view(-1, 1)
    rows, route = routing.sort_and_dispatch(x, ids, 4)
    p = route.position.view(-1)
    held = p >= 0
    assert torch.equal(held, (ids >= 0).view(-1)) and int(route.counts.sum()) == int(held.sum())
    at = route.order.long().clamp(min=0)
    assert torch.equal(rows.view(-1), torch.where(route.order >= 0, x.view(-1)[at], torch.zeros((), dtype=x.dtype, device=dev)))
    y = routing.combine(rows, route)
    assert torch.equal(y.view(-1), torch.where(held, x.view(-1), torch.zeros((), dtype=x.dtype, device=dev)))
    w = torch.full((tokens, 1), 2.0, device=dev)
    d_rows, d_w = routing.combine_grad(x, rows, route, w)
    assert torch.equal(d_rows, 2 * rows)
    assert torch.equal(d_w.view(-1), torch.where(held, x.view(-1).float() ** 2, torch.zeros((), device=dev)))
