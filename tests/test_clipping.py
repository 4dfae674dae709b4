"""Updates scaled to a bound on their norm (geeps_amd.clipping) against plain
definitions in 64 bits."""
import ctypes
import math

import pytest
import torch

from geeps_amd import clipping, native

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
U = 2.0 ** -24
TYPES = list(HALF)
INF = float("inf")


def factor(square_sum, max_norm, scale=1.0):
    norm = math.sqrt(square_sum)
    return norm, scale * (1.0 if norm <= max_norm else max_norm / norm)


def squares(tensors):
    return math.fsum(float(t.double().square().sum()) for t in tensors)


def check_norm(got, want):
    assert got.dtype == torch.float32 and got.shape == ()
    # one rounding to 32 bits; the 64-bit sums are far below it
    assert abs(float(got) - want) <= 1.001 * U * want + 2.0 ** -150, (float(got), want)


def check_scaled(out, grad, f):
    """f's own rounding, the product's, the output's; f may be off by 2^-40 before."""
    want = grad.double() * f
    bound = (2 * U + 2.0 ** -30) * want.abs() + 2.0 ** -149
    bound = bound + HALF[out.dtype] * (want.abs() + bound) + TINY[out.dtype]
    assert bool(((out.double() - want).abs() <= bound).all())


def values(n, dtype, dev, seed, size=1.0):
    return (torch.randn(n, generator=torch.Generator().manual_seed(seed)) * size).to(dtype).to(dev)


# -- refusals (no device) -----------------------------------------------------
def plan_create(grads, outs, sizes, types=None, out_types=None):
    n = len(grads)
    h = ctypes.c_void_p()
    types = types or [0] * n
    rc = native.lib().gp_grad_plan_create(
        ctypes.byref(h), n, (ctypes.c_void_p * n)(*grads), (ctypes.c_int * n)(*types), (ctypes.c_void_p * n)(*outs),
        (ctypes.c_int * n)(*(out_types or types)), (ctypes.c_size_t * n)(*sizes))
    assert h.value is None or rc == 0
    if rc == 0:
        native.lib().gp_grad_plan_destroy(h)
    return rc, native.lib().gp_last_error()


def test_plans_refused_without_device():
    bad = [
        (([4096], [8192], [16], [3]), b"types"), (([4096], [8192], [16], [0], [1]), b"type or GP_F32"),
        (([4096], [8192], [16], [1], [2]), b"type or GP_F32"),
        (([None], [8192], [16]), b"null"), (([4096], [None], [16]), b"null"),
        (([4096, 1 << 20], [8192, 8192 + 60], [16, 16]), b"two outputs overlap"),
        (([4096, 4096], [4096, 4096], [16, 16]), b"listed twice"),
        (([4096], [4100], [16]), b"overlaps a gradient"),
        (([4096], [4096], [16], [1], [0]), b"overlaps a gradient"),       # in place, but wider
        (([4096, 8192], [16384, 4096], [16, 16]), b"overlaps a gradient"),  # another's gradient
        (([4096, 8192], [8192, 4096], [16, 16]), b"overlaps a gradient"),
    ]
    for args, word in bad:
        rc, msg = plan_create(*args)
        assert rc == native.GP_ERR_INVALID and word in msg, (args, msg)
    # nothing in it: no table, no device
    assert plan_create([], [], [])[0] == 0
    assert plan_create([None, 4096], [None, 4096], [0, 0])[0] == 0


def test_calls_refused_without_device():
    L, p = native.lib(), ctypes.c_void_p
    a, b, c, d = (p(1 << 20), p(2 << 20), p(3 << 20), p(4 << 20))

    def buckets(*at):
        return (ctypes.c_void_p * max(1, len(at)))(*at)

    def refused(rc, word):
        assert rc == native.GP_ERR_INVALID and word in L.gp_last_error(), L.gp_last_error()

    three = buckets(5 << 20, 6 << 20, 7 << 20)

    def clipped(out=a, src=b, bk=three, nb=3, scratch=c, max_norm=1.0, scale=1.0, mode=0, ws=d, n=16):
        return L.gp_bucket_sum_clipped(out, src, bk, nb, n, scratch, max_norm, scale, mode, None, None, ws, None)

    refused(clipped(max_norm=-1.0), b"max_norm")
    refused(clipped(max_norm=float("nan")), b"max_norm")
    refused(clipped(scale=INF), b"scale")
    refused(clipped(scale=float("nan")), b"scale")
    refused(clipped(mode=2), b"nonfinite")
    refused(clipped(ws=None), b"workspace")
    refused(clipped(scratch=None), b"scratch")
    refused(clipped(out=None), b"null")
    refused(clipped(nb=-1), b"negative")
    refused(clipped(bk=buckets(5 << 20, None, 7 << 20)), b"null bucket")
    refused(clipped(out=p((2 << 20) + 4)), b"out overlaps in")
    refused(clipped(out=p((6 << 20) + 60)), b"out overlaps a bucket")
    refused(clipped(scratch=a), b"scratch overlaps out")
    refused(clipped(scratch=b), b"scratch overlaps out")
    refused(clipped(scratch=p((7 << 20) - 60)), b"scratch overlaps a bucket")
    refused(L.gp_bucket_sum_squares(c, three, 3, 16, None, d, None), b"null sum")
    refused(L.gp_bucket_sum_squares(None, three, 3, 16, a, d, None), b"scratch")
    refused(L.gp_grad_clip(None, 1.0, 1.0, 0, None, None, d, None), b"null grad plan")
    refused(L.gp_grad_sum_squares(None, a, d, None), b"null grad plan")


def test_tensors_refused_without_device():
    t = torch.zeros(8)
    for call in (lambda: clipping.GradPlan([t]), lambda: clipping.GradPlan([]),
                 lambda: clipping.apply_updates_clipped(t, [t], 1.0), lambda: clipping.sum_updates_squares([t]),
                 lambda: clipping.sum_updates_squares([]), lambda: clipping.apply_updates_clipped(t, [t], -1.0),
                 lambda: clipping.apply_updates_clipped(t, [t], 1.0, scale=INF)):
        with pytest.raises(ValueError):
            call()


# -- gradients ----------------------------------------------------------------
LISTS = [[1], [0, 1, 0], [7, 8, 9, 1023, 1024, 1025], [2047, 2048, 2049, 5, 0, 4096], [100_003],
         [3] * 700, [1 << 20, 17, 65_537, 300_000], [40_000_000, 1, 12_345_679]]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", LISTS, ids=lambda s: f"{len(s)}x{max(s)}")
@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16", "mixed"])
@pytest.mark.parametrize("out", ["same", "float32", "in place"])
def test_clip(dev, sizes, kind, out):
    types = [TYPES[i % 3] if kind == "mixed" else getattr(torch, kind) for i in range(len(sizes))]
    grads = [values(n, t, dev, i, 0.3) for i, (n, t) in enumerate(zip(sizes, types))]
    want_in = [g.clone() for g in grads]
    outs = None if out == "in place" else [
        torch.full((n,), 7.0, device=dev, dtype=t if out == "same" else torch.float32) for n, t in zip(sizes, types)]
    plan = clipping.GradPlan(grads, outs)
    total = squares(want_in)
    assert abs(float(plan.sum_squares()) - total) <= 1e-12 * total
    check_norm(plan.norm(), math.sqrt(total))
    for max_norm, scale in ((0.5 * math.sqrt(total), 1.0), (INF, -0.125), (2 * math.sqrt(total), 1.0), (0.0, 1.0)):
        norm, f = factor(total, max_norm, scale)
        check_norm(plan.clip(max_norm, scale=scale), norm)
        for o, g in zip(plan.outs, want_in):
            check_scaled(o, g, f)
        if out == "in place":
            for g, w in zip(grads, want_in):
                g.copy_(w)
        else:
            assert all(torch.equal(g, w) for g, w in zip(grads, want_in))
    plan.close()
    with pytest.raises(ValueError, match="closed"):
        plan.clip(1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_clip_odd_places(dev, dtype):
    """Gradients and outputs that start at any element, and what lies around them."""
    base, to = values(20_000, dtype, dev, 1), torch.full((20_000,), 3.0, device=dev, dtype=dtype)
    cuts = [(1, 5), (7, 1000), (1011, 1012), (1500, 9001), (9002, 19_999)]
    plan = clipping.GradPlan([base[a:b] for a, b in cuts], [to[a - 1:b - 1] for a, b in cuts])
    total = squares([base[a:b] for a, b in cuts])
    norm, f = factor(total, 1.0)
    check_norm(plan.clip(1.0), norm)
    left = torch.ones(20_000, dtype=torch.bool, device=dev)
    for a, b in cuts:
        check_scaled(to[a - 1:b - 1], base[a:b], f)
        left[a - 1:b - 1] = False
    assert bool((to[left] == 3.0).all())


@pytest.mark.gpu
def test_clip_whole_range_of_values(dev):
    """Squares that no 32-bit float holds."""
    for size, dtype in ((1e30, torch.float32), (1e-30, torch.float32), (3e-42, torch.float32), (1e38, torch.bfloat16),
                        (1e-38, torch.bfloat16), (6e4, torch.float16), (1e-7, torch.float16)):
        g = (torch.randint(-3, 4, (5000,), generator=torch.Generator().manual_seed(1)).float() / 3 * size).to(dtype).to(dev)
        out = torch.zeros(5000, device=dev)
        plan = clipping.GradPlan([g], [out])
        norm, f = factor(squares([g]), 0.5)
        if norm < 3e38:
            check_norm(plan.clip(0.5), norm)
        else:
            assert float(plan.clip(0.5)) == INF  # past the float range; f is not
        # f is rounded to a float, and may be a subnormal one: half a step of 2^-149 times the value
        want = g.double() * f
        assert bool(((out.double() - want).abs() <= 3 * U * want.abs() + 2.0 ** -150 * g.double().abs() + 2.0 ** -149).all())


@pytest.mark.gpu
def test_zeros_and_no_numbers(dev):
    z = torch.zeros(3000, device=dev)
    plan = clipping.GradPlan([z])
    for max_norm in (0.0, 1.0, INF):
        assert float(plan.clip(max_norm)) == 0.0 and bool((z == 0).all())
    for bad in (INF, -INF, float("nan")):
        g, h = torch.ones(3000, device=dev), torch.ones(70, device=dev, dtype=torch.bfloat16)
        g[1234] = bad
        out, to = torch.empty_like(g), torch.empty_like(h)
        plan = clipping.GradPlan([g, h], [out, to])
        norm = float(plan.clip(1.0))
        if bad != bad:
            assert norm != norm and bool(out.isnan().all()) and bool(to.isnan().all())
        else:
            assert norm == INF and bool(out[1234].isnan()) and int(out.isnan().sum()) == 1
            assert float(out.nan_to_num().abs().sum()) == 0.0 and bool((to == 0).all())
        norm = float(plan.clip(1.0, skip_nonfinite=True))
        assert not math.isfinite(norm) and bool((out == 0).all()) and bool((to == 0).all())
    m, u = values(999, torch.float32, dev, 1), torch.ones(999, device=dev)
    u[5] = float("nan")
    for count in (1, 2, 4):
        out = torch.empty_like(m)
        norm = clipping.apply_updates_clipped(m, [u] * count, 1.0, out=out, skip_nonfinite=True)
        assert bool(norm.isnan()) and torch.equal(out, m)
        clipping.apply_updates_clipped(m, [u] * count, 1.0, out=out)
        assert bool(out.isnan().all())


@pytest.mark.gpu
def test_norm_over_several_lists(dev):
    a, b = [values(5000, torch.bfloat16, dev, 1), values(3, torch.float32, dev, 2)], [values(70_001, torch.float16, dev, 3)]
    updates = [values(4097, torch.float32, dev, 4 + i) for i in range(4)]
    plans = [clipping.GradPlan(x, [torch.empty_like(t) for t in x]) for x in (a, b)]
    scratch = torch.empty(4097, device=dev)
    total = plans[0].sum_squares() + plans[1].sum_squares() + clipping.sum_updates_squares(updates, scratch)
    u = updates[0] + updates[1] + updates[2] + updates[3]
    assert torch.equal(scratch, u)
    want = squares(a + b + [u])
    norm, f = factor(want, 1.0)
    for p, x in zip(plans, (a, b)):
        check_norm(p.clip(1.0, total=total), norm)
        for o, g in zip(p.outs, x):
            check_scaled(o, g, f)
    m = torch.zeros(4097, device=dev)
    check_norm(clipping.apply_updates_clipped(m, updates, 1.0, scratch=scratch, total=total), norm)
    check_scaled(m, u, f)


# -- the server's sum ---------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("clients", [1, 2, 3, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("n", [1, 3, 1023, 4096, 65_541, 3_000_001])
def test_apply_updates_clipped(dev, clients, n):
    base = values(n + 1, torch.float32, dev, 99)
    for at in (0, 1):  # aligned and not
        m = base[at:at + n]
        keep = m.clone()
        updates = [values(n + at, torch.float32, dev, i, 0.1)[at:] for i in range(clients)]
        u = updates[0].clone()
        for x in updates[1:]:
            u += x  # in 32 bits, in order: the bits the kernel sums to
        for share, scale in ((0.5, 1.0), (2.0, -0.5)):
            norm, f = factor(squares([u]), share * math.sqrt(squares([u])), scale)
            max_norm = share * norm
            out = torch.full_like(keep, 5.0)
            check_norm(clipping.apply_updates_clipped(m, updates, max_norm, scale=scale, out=out), norm)
            assert torch.equal(m, keep)
            add = u.double() * f
            want = keep.double() + add
            bound = (2 * U + 2.0 ** -30) * add.abs() + 1.001 * U * (want.abs() + 2 * U * add.abs()) + 2.0 ** -149
            assert bool(((out.double() - want).abs() <= bound).all())
            total = clipping.sum_updates_squares(updates, scratch := torch.empty_like(keep))
            again = torch.empty_like(keep)
            clipping.apply_updates_clipped(m, updates, max_norm, scale=scale, out=again, scratch=scratch, total=total)
            assert torch.equal(again, out)
            clipping.apply_updates_clipped(m, updates, max_norm, scale=scale)  # in place
            assert torch.equal(m, out)
            m.copy_(keep)
        assert torch.equal(base[at:at + n], keep)


@pytest.mark.gpu
def test_apply_nothing(dev):
    m = values(77, torch.float32, dev, 1)
    out = torch.empty_like(m)
    assert float(clipping.apply_updates_clipped(m, [], 1.0, out=out)) == 0.0 and torch.equal(out, m)
    empty = torch.empty(0, device=dev)
    assert float(clipping.apply_updates_clipped(empty, [empty] * 3, 1.0)) == 0.0
    assert float(clipping.sum_updates_squares([empty])) == 0.0


@pytest.mark.gpu
def test_apply_past_32_bit_offsets(dev):
    n = (1 << 32) // 2 + 4099  # over 2^31 values, 2^33 bytes
    m, u = torch.ones(n, device=dev), torch.full((n,), 0.25, device=dev)
    u[-1] = 2.0
    norm = clipping.apply_updates_clipped(m, [u], 1.0)
    check_norm(norm, math.sqrt((n - 1) / 16 + 4.0))
    f = 1.0 / math.sqrt((n - 1) / 16 + 4.0)
    lo, hi = float(m[:-1].min()), float(m[:-1].max())
    assert lo == hi and abs(lo - (1 + 0.25 * f)) <= 2 * U and abs(float(m[-1]) - (1 + 2 * f)) <= 2 * U


@pytest.mark.gpu
def test_clip_past_32_bit_offsets(dev):
    n = (1 << 32) + 2053
    g = torch.ones(n, device=dev, dtype=torch.bfloat16)
    g[-1] = 4.0
    plan = clipping.GradPlan([g])
    check_norm(plan.clip(1 << 15), math.sqrt(n - 1 + 16))  # norm 65536.1...: f just under 0.5
    half = torch.tensor(0.5 * 65536 / math.sqrt(n + 15)).to(torch.bfloat16)
    assert bool((g[:-1] == half).all()) and float(g[-1]) == 4 * float(half)


@pytest.mark.gpu
def test_streams_and_repeats(dev):
    lists = [[values(n, torch.bfloat16, dev, s * 10 + i) for i, n in enumerate((300_000, 77, 1_000_000))] for s in (1, 2)]
    updates = [[values(200_003, torch.float32, dev, s * 100 + i) for i in range(5)] for s in (1, 2)]
    m = values(200_003, torch.float32, dev, 7)
    plans = [clipping.GradPlan(x, [torch.empty_like(t) for t in x]) for x in lists]

    def whole(i, stream=None):
        out = torch.empty_like(m)
        a = plans[i].clip(1.0, stream=stream)
        b = clipping.apply_updates_clipped(m, updates[i], 1.0, out=out, stream=stream)
        return a, b, out

    want = [(*whole(i), *[o.clone() for o in plans[i].outs]) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in (0, 1)]
    for _ in range(3):
        got = [whole(i, s) for i, s in zip((0, 1), streams)]
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip((*got[i], *plans[i].outs), want[i]))


@pytest.mark.gpu
def test_captured_and_replayed(dev):
    grads = [values(n, t, dev, i) for i, (n, t) in enumerate(zip((70_000, 3, 5001), TYPES))]
    outs = [torch.empty_like(g) for g in grads]
    updates, m = [values(50_001, torch.float32, dev, 10 + i) for i in range(3)], values(50_001, torch.float32, dev, 9)
    plan = clipping.GradPlan(grads, outs)
    table = torch.empty_like(m)

    def whole():
        total = plan.sum_squares()
        return total, plan.clip(1.0), clipping.apply_updates_clipped(m, updates, 1.0, out=table)

    whole()
    other = clipping.GradPlan([updates[0]])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = whole()
        with pytest.raises(ValueError, match="captured"):
            clipping.GradPlan([updates[0]])
        del other  # a plan may be dropped meanwhile
    for seed in (1, 2, 3):
        for t in (*grads, *updates, m):
            t.copy_(values(t.numel(), t.dtype, dev, 50 * seed + t.numel() % 50, 0.5))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*held, *outs, table)]
        for t in (*outs, table):
            t.zero_()
        want = (*whole(), *outs, table)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


@pytest.mark.gpu
def test_sharded_reducer_bounds_its_update(dev):
    from geeps_amd.shard import ShardedReducer
    rows, width, clients = 300, 130, 4
    r = ShardedReducer(rows, width, clients, dev, max_norm=1.0)
    deltas = [values(rows * width, torch.float32, dev, i, 0.2) for i in range(clients)]
    u = deltas[0] + deltas[1] + deltas[2] + deltas[3]
    norm, f = factor(squares([u]), 1.0)
    for step in (1, 2):
        table = r.step(deltas)
        check_norm(r.norm, norm)
        want = step * f * u.double()
        assert bool(((table.double() - want).abs() <= 4 * step * U * want.abs() + 2.0 ** -149).all())
    with pytest.raises(ValueError):
        ShardedReducer(rows, width, clients, dev, max_norm=-1.0)


@pytest.mark.gpu
def test_refusals(dev):
    g, o = torch.zeros(8, device=dev), torch.zeros(8, device=dev)
    bad = [
        lambda: clipping.GradPlan([g.double()]), lambda: clipping.GradPlan([torch.zeros(4, 4, device=dev).t()]),
        lambda: clipping.GradPlan([g], [o[:7]]), lambda: clipping.GradPlan([g], [o, o]),
        lambda: clipping.GradPlan([g], [o.half()]), lambda: clipping.GradPlan([g, o.cpu()]),
        lambda: clipping.GradPlan([g.half()], [o.bfloat16()]),
        lambda: clipping.GradPlan([g]).clip(float("nan")), lambda: clipping.GradPlan([g]).clip(1.0, scale=INF),
        lambda: clipping.GradPlan([g]).clip(1.0, total=o[:1]),
        lambda: clipping.apply_updates_clipped(g, [o[:7]], 1.0),
        lambda: clipping.apply_updates_clipped(g, [o.half()], 1.0),
        lambda: clipping.apply_updates_clipped(g.half(), [o], 1.0),
        lambda: clipping.apply_updates_clipped(g, [o] * 3, 1.0, scratch=torch.zeros(7, device=dev)),
        lambda: clipping.apply_updates_clipped(g, [o] * 3, 1.0, total=torch.zeros(1, device=dev, dtype=torch.float64)),
        lambda: clipping.apply_updates_clipped(g, [o], 1.0, out=o[:7]),
    ]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    both = torch.zeros(64, device=dev)
    for call in (lambda: clipping.GradPlan([g, g]), lambda: clipping.GradPlan([both[:32]], [both[16:48]]),
                 lambda: clipping.GradPlan([g, o], [o, g]),
                 lambda: clipping.apply_updates_clipped(g, [g], 1.0),
                 lambda: clipping.apply_updates_clipped(both[:32], [o.repeat(4)], 1.0, out=both[8:40]),
                 lambda: clipping.apply_updates_clipped(g, [o] * 3, 1.0, scratch=o)):
        with pytest.raises(native.GpError, match="overlap"):
            call()


# -- over ranks (gloo, CPU; plain stand-ins for the device calls) --------------
def plain_squares(updates, scratch):
    u = updates[0].clone()
    for x in updates[1:]:
        u += x
    if scratch is not None:
        scratch.copy_(u)
    return u.double().square().sum()


def plain_clipped(master, updates, max_norm, scratch, total):
    u = updates[0] + updates[1] if len(updates) == 2 else updates[0] if scratch is None else scratch
    norm, f = factor(float(total), max_norm)
    master += u * torch.tensor(f, dtype=torch.float32)
    return torch.tensor(norm, dtype=torch.float32)


def run_bounded(rank, world, port, rows, width, clients, exchange, out_dir):
    import os

    import torch.distributed as dist
    os.environ.update({"MASTER_ADDR": "127.0.0.1", "MASTER_PORT": str(port)})
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        from geeps_amd.shard import ShardedReducer
        r = ShardedReducer(rows, width, clients, "cpu", exchange=exchange, max_norm=1.0,
                           clip_fns=(plain_squares, plain_clipped))
        for _ in range(2):
            table = r.step([values(rows * width, torch.float32, "cpu", c, 0.2) for c in r.hosted])
        torch.save({"norm": r.norm, "table": table[:rows * width].clone()}, os.path.join(out_dir, f"{rank}.pt"))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world,rows,width,clients,exchange", [
    (2, 64, 16, 4, "a2a"), (2, 37, 12, 2, "rs"), (4, 41, 8, 8, "a2a"), (4, 3, 5, 4, "a2a")])
def test_bound_is_over_all_shards(tmp_path, world, rows, width, clients, exchange):
    import socket

    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(run_bounded, args=(world, port, rows, width, clients, exchange, str(tmp_path)), nprocs=world, join=True)
    u = sum(values(rows * width, torch.float32, "cpu", c, 0.2).double() for c in range(clients))
    norm, f = factor(float(u.square().sum()), 1.0)
    got = [torch.load(tmp_path / f"{r}.pt", weights_only=True) for r in range(world)]
    size = sum(values(rows * width, torch.float32, "cpu", c, 0.2).double().abs() for c in range(clients))
    for g in got:
        assert torch.equal(g["table"], got[0]["table"]) and float(g["norm"]) == float(got[0]["norm"])
        # the sum's roundings (clients of them, of at most sum |b|), f's, the product's and two additions'
        assert abs(float(g["norm"]) - norm) <= 1.01 * (U * norm + clients * U * float(size.square().sum().sqrt()))
        bound = 2 * f * (2 * clients + 6) * U * (size + 2 * u.abs())
        assert bool(((g["table"].double() - 2 * f * u).abs() <= bound).all())


@pytest.mark.gpu
def test_workspace_is_held_while_a_call_runs(dev, monkeypatch):
    """No allocation of the same stream, made while a call runs, gets the call's workspace."""
    real = native.lib()
    sides = {"gp_grad_clip": 6, "gp_grad_sum_squares": 2, "gp_bucket_sum_clipped": 11, "gp_bucket_sum_squares": 5}
    seen = []

    class Watched:
        def __getattr__(self, name):
            f = getattr(real, name)
            if name not in sides:
                return f

            def call(*args):
                other = [torch.empty(native.GP_CLIP_WORKSPACE_BYTES, dtype=torch.uint8, device=dev) for _ in range(4)]
                assert args[sides[name]] not in [t.data_ptr() for t in other], name
                seen.append(name)
                return f(*args)
            return call

    grads = [torch.randn(1000, device=dev), torch.randn(3, device=dev)]
    plan = clipping.GradPlan(grads)
    updates = [torch.randn(5000, device=dev) for _ in range(3)]
    master = torch.zeros(5000, device=dev)
    monkeypatch.setattr(native, "lib", lambda: Watched())
    plan.clip(1.0)
    plan.sum_squares()
    clipping.apply_updates_clipped(master, updates, 1.0)
    clipping.sum_updates_squares(updates)
    assert sorted(seen) == sorted(sides)
