"""Expert row routing between columns of one buffer: rows of one stride that pass between each other."""
import ctypes

import pytest
import torch

from geeps_amd import native, routing

AT = 1 << 50  # nothing is read there: every call below is refused, for its rows if not for its overlap
ROWS, WIDTH = (1 << 31) - 1, 8192


def refused(call, a, a_stride, b, b_stride):
    L, p = native.lib(), ctypes.c_void_p
    a, b, other = p(a), p(b), p(1 << 60)
    rc = {"dispatch": lambda: L.gp_route_dispatch(a, a_stride, b, b_stride, 0, other, other, ROWS, 1, ROWS, WIDTH, None),
          "combine": lambda: L.gp_route_combine(a, a_stride, b, b_stride, 0, other, None, 0, ROWS, 1, ROWS, WIDTH, None),
          "dy": lambda: L.gp_route_combine_grad(a, a_stride, other, b, b_stride, other, WIDTH, 0, other, other, other, 0,
                                                ROWS, 1, ROWS, WIDTH, None),
          "rows": lambda: L.gp_route_combine_grad(a, a_stride, other, other, WIDTH, b, b_stride, 0, other, other, other, 0,
                                                  ROWS, 1, ROWS, WIDTH, None)}[call]()
    assert rc == native.GP_ERR_INVALID
    return L.gp_last_error()


@pytest.mark.parametrize("call", ["dispatch", "combine", "dy", "rows"])
def test_which_rows_overlap(call):
    """Rows that share no value are not refused for an overlap; these calls are for their number of rows."""
    row, s = WIDTH * 4, 2 * WIDTH + 10
    for apart in (row, row + 4, row + 40):
        for way in (apart, -apart, apart + 3 * s * 4, -apart - 3 * s * 4):
            assert b"too many rows" in refused(call, AT + way, s, AT, s), way
    for apart in (0, 4, row - 4, row + 44, 4 * s - 4):
        for way in (apart, -apart, apart + 3 * s * 4, -apart - 3 * s * 4):
            assert b"overlaps" in refused(call, AT + way, s, AT, s), way
    assert b"overlaps" in refused(call, AT + row, s, AT, s + 2)  # of two strides: by their spans
    assert b"too many rows" in refused(call, AT, s, AT + (ROWS * s) * 4, s + 2)
    assert b"overlaps" in refused(call, AT, WIDTH, AT + 4 * WIDTH * 5, WIDTH)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("tokens,k,experts,width", [(1, 1, 4, 40), (1, 3, 4, 40), (37, 2, 5, 130), (700, 4, 16, 1001)])
def test_columns_of_one_buffer(dev, dtype, tokens, k, experts, width):
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(-1, experts, (tokens, k), generator=g).to(dev)
    w = torch.rand(tokens, k, generator=g).to(dev)
    route = routing.sort_tokens(ids, experts)
    n = route.order.numel()

    def buffer(columns):
        return torch.randn(max(n, tokens), columns * width + 5, generator=g).to(dtype).to(dev)

    def column(b, i, rows):
        return b[:rows, i * width + 2:(i + 1) * width + 2]

    for first in (0, 1):
        b = buffer(2)
        before, x = b.clone(), column(b, first, tokens)
        want = routing.dispatch(x.clone(), route)
        out = column(b, 1 - first, n)
        assert routing.dispatch(x, route, out=out) is out and torch.equal(out, want)
        column(before, 1 - first, n).copy_(want)
        assert torch.equal(b, before)
        out.zero_()
        got, _ = routing.sort_and_dispatch(x, ids, experts, out=out)
        assert got is out and torch.equal(b, before)

        b = buffer(2)
        before, rows = b.clone(), column(b, first, n)
        want = routing.combine(rows.clone(), route, w)
        out = column(b, 1 - first, tokens)
        assert torch.equal(routing.combine(rows, route, w, out=out), want)
        column(before, 1 - first, tokens).copy_(want)
        assert torch.equal(b, before)

        b = buffer(3)
        before, dy, rows = b.clone(), column(b, first, tokens), column(b, 1 - first, n)
        want, want_w = routing.combine_grad(dy.clone(), rows.clone(), route, w)
        out = column(b, 2, n)
        got, got_w = routing.combine_grad(dy, rows, route, w, out=out)
        assert torch.equal(got, want) and torch.equal(got_w, want_w)
        column(before, 2, n).copy_(want)
        assert torch.equal(b, before)
