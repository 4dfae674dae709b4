"""Streams given to the routing and clipping calls: a Stream, a raw handle, and 0, the device's null stream."""
import pytest
import torch

from geeps_amd import clipping, native, routing


@pytest.fixture
def streams_of_calls(monkeypatch):
    """The stream that every C call of the two families gets."""
    real, seen = native.lib(), []

    class Watched:
        def __getattr__(self, name):
            f = getattr(real, name)
            if not name.startswith(("gp_route_", "gp_grad_", "gp_bucket_")) or name in ("gp_route_workspace",
                                                                                       "gp_grad_plan_create",
                                                                                       "gp_grad_plan_destroy"):
                return f

            def call(*args):
                seen.append(args[-1])
                return f(*args)
            return call

    monkeypatch.setattr(native, "lib", lambda: Watched())
    return seen


@pytest.mark.gpu
def test_a_call_runs_on_the_stream_that_it_is_given(dev, streams_of_calls):
    ids = torch.arange(40, device=dev).view(20, 2) % 6
    x, w = torch.randn(20, 32, device=dev), torch.rand(20, 2, device=dev)
    grads, master = [torch.randn(100, device=dev)], torch.randn(100, device=dev)
    plan = clipping.GradPlan(grads, [torch.empty_like(grads[0])])
    route = routing.sort_tokens(ids, 6)
    rows = routing.dispatch(x, route)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    calls = [
        lambda s: routing.sort_tokens(ids, 6, stream=s).position, lambda s: routing.dispatch(x, route, stream=s),
        lambda s: routing.sort_and_dispatch(x, ids, 6, stream=s)[0], lambda s: routing.combine(rows, route, w, stream=s),
        lambda s: routing.dispatch_grad(rows, route, stream=s), lambda s: routing.combine_grad(x, rows, route, w, stream=s)[1],
        lambda s: plan.sum_squares(stream=s), lambda s: plan.norm(stream=s), lambda s: plan.clip(1.0, stream=s),
        lambda s: clipping.sum_updates_squares(grads * 3, stream=s),
        lambda s: clipping.apply_updates_clipped(master, grads * 3, 1.0, out=torch.empty_like(master), stream=s),
    ]
    for call in calls:
        want = call(None)
        torch.cuda.synchronize()
        for given, handle in ((0, 0), (torch.cuda.default_stream(), 0), (side, side.cuda_stream),
                              (side.cuda_stream, side.cuda_stream)):
            streams_of_calls.clear()
            got = call(given)
            assert streams_of_calls == [handle], given
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        # under another current stream 0 still is the null stream
        with torch.cuda.stream(side):
            streams_of_calls.clear()
            call(0), call(None)
            assert streams_of_calls == [0, side.cuda_stream]
        torch.cuda.synchronize()
