"""Expert row routing and autograd: no gradient is lost without a word, and a Function of the calls carries it."""
import pytest
import torch

from geeps_amd import routing


def wanted(*shape, dev="cpu"):
    return torch.zeros(*shape, device=dev, requires_grad=True)


def calls(t, dev):
    """Every call that takes t-like rows or weights, with one tensor at a time made by t()."""
    z = lambda *shape: torch.zeros(*shape, device=dev)
    ids = torch.arange(8, device=dev).view(4, 2) % 3
    if dev == "cpu":
        route = routing.Route(*(torch.zeros(s, dtype=torch.int32) for s in ((4, 2), 8, 3, 4)))
    else:
        route = routing.sort_tokens(ids, 3)
    return [
        lambda: routing.dispatch(t(4, 8), route), lambda: routing.dispatch(z(4, 8), route, out=t(8, 8)),
        lambda: routing.sort_and_dispatch(t(4, 8), ids, 3), lambda: routing.sort_and_dispatch(z(4, 8), ids, 3, out=t(8, 8)),
        lambda: routing.combine(t(8, 8), route, z(4, 2)), lambda: routing.combine(z(8, 8), route, t(4, 2)),
        lambda: routing.combine(z(8, 8), route, out=t(4, 8)), lambda: routing.dispatch_grad(t(8, 8), route),
        lambda: routing.combine_grad(t(4, 8), z(8, 8), route, z(4, 2)),
        lambda: routing.combine_grad(z(4, 8), t(8, 8), route, z(4, 2)),
        lambda: routing.combine_grad(z(4, 8), z(8, 8), route, t(4, 2)),
        lambda: routing.combine_grad(z(4, 8), z(8, 8), route, z(4, 2), out=t(8, 8)),
    ]


@pytest.mark.parametrize("which", [0, 2, 4, 7, 8])  # those whose first tensor it is: before any device is asked for
def test_lost_gradients_are_refused_without_device(which):
    with pytest.raises(ValueError, match="requires a gradient"):
        calls(wanted, "cpu")[which]()
    with torch.no_grad(), pytest.raises(ValueError, match="must be a CUDA"):
        calls(wanted, "cpu")[which]()


@pytest.mark.gpu
def test_lost_gradients_are_refused(dev):
    for call in calls(lambda *s: wanted(*s, dev=dev), dev):
        with pytest.raises(ValueError, match="requires a gradient"):
            call()
        with torch.no_grad():
            call()
    for call in calls(lambda *s: torch.zeros(*s, device=dev), dev):
        call()


class Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, route):
        ctx.route = route
        return routing.dispatch(x, route)

    @staticmethod
    def backward(ctx, d_rows):
        return routing.dispatch_grad(d_rows.contiguous(), ctx.route), None


class Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, route, weights):
        ctx.route = route
        ctx.save_for_backward(rows, weights)
        return routing.combine(rows, route, weights)

    @staticmethod
    def backward(ctx, dy):
        rows, weights = ctx.saved_tensors
        d_rows, d_weights = routing.combine_grad(dy.contiguous(), rows, ctx.route, weights)
        return d_rows, None, d_weights


@pytest.mark.gpu
def test_a_function_of_the_calls_carries_the_gradient(dev):
    """Small whole numbers, so that every product and sum is exact whatever its order."""
    g = torch.Generator().manual_seed(1)
    tokens, k, experts, width = 50, 3, 7, 20
    ids = torch.randint(-1, experts, (tokens, k), generator=g).to(dev)
    small = lambda *s: torch.randint(-4, 5, s, generator=g).float().to(dev)
    x, w, scale = small(tokens, width).requires_grad_(), small(tokens, k).requires_grad_(), small(experts, width)
    route = routing.sort_tokens(ids, experts, 4)
    of_row = torch.zeros(route.order.numel(), width, device=dev)
    for e, (a, n) in enumerate(zip(route.offsets.tolist(), route.counts.tolist())):
        of_row[a:a + n] = scale[e]
    y = Combine.apply(Dispatch.apply(x, route) * of_row, route, w)
    (y * (y + 1)).sum().backward()
    got = x.grad.clone(), w.grad.clone()
    x.grad = w.grad = None
    held = (ids >= 0).float()
    rows = x[:, None, :] * scale[ids.clamp(min=0)]
    y = (rows * (w * held)[..., None]).sum(1)
    (y * (y + 1)).sum().backward()
    assert torch.equal(got[0], x.grad) and torch.equal(got[1], w.grad)
