"""Measured cases of the expert row routing and of the clipped gradient updates.

``run`` makes one pass through an operator.  With ``own`` false it is the
operator's plain form, in elementary torch operations; with ``own`` true it is
the call a program makes of geeps_amd.routing or geeps_amd.clipping.

Five operators:

dispatch      rows sorted by expert: from the experts that a router chose for
              every token, the place of every (token, choice) among the rows
              grouped by expert, and the rows there.
combine       back to the tokens: a token's rows times their weights, summed.
              Without weights it is the gradient of dispatch.
combine_grad  the gradient of combine: of its rows and of its weights.
clip          the norm of a list of gradients, and the list scaled to a bound.
apply         the server's sum of the clients' deltas, scaled to a bound on
              its norm and added to the master table.
"""
import functools
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}

# The parameter blobs of the two tables that this repository's tests and
# benchmark use: AlexNet with grouped convolutions, and an Inception-style
# CIFAR-10 net.
ALEXNET = [96 * 3 * 11 * 11, 96, 256 * 48 * 5 * 5, 256, 384 * 256 * 3 * 3, 384,
           384 * 192 * 3 * 3, 384, 256 * 192 * 3 * 3, 256, 4096 * 9216, 4096,
           4096 * 4096, 4096, 1000 * 4096, 1000]


def _inception():
    blobs, cin = [64 * 3 * 3 * 3, 64], 64
    for b1, r3, b3, r5, b5, pp in [(32, 48, 64, 8, 16, 16), (64, 64, 96, 16, 48, 32),
                                   (96, 48, 104, 8, 24, 32), (80, 56, 112, 12, 32, 32),
                                   (64, 64, 128, 12, 32, 32), (112, 72, 144, 16, 32, 32)]:
        blobs += [b1 * cin, r3 * cin, b3 * r3 * 9, r5 * cin, b5 * r5 * 25, pp * cin,
                  b1, r3, b3, r5, b5, pp]
        cin = b1 + b3 + b5 + pp
    return blobs + [10 * cin, 10]


def _blobs(case):
    """The lengths of a clip case's gradients."""
    if case["table"] == "alexnet":
        return ALEXNET
    if case["table"] == "inception":
        return _inception()
    if case["table"] == "layers":  # a stack of blocks: two norms, four square matrices, a wide pair with biases
        w = case["width"]
        return [n for _ in range(case["layers"])
                for n in (w, w, w * w, w * w, w * w, w * w, w, 4 * w * w, 4 * w, 4 * w * w, w)]
    r = random.Random(case["tensors"] * 1000003 + case["top"])  # "ragged": any lengths, from one element up
    return [int(math.exp(r.uniform(0.0, math.log(case["top"])))) for _ in range(case["tensors"])]


def _blob_types(case, count):
    cycle = ["bfloat16", "float32", "float16"] if case["dtype"] == "mixed" else [case["dtype"]]
    return [cycle[i % len(cycle)] for i in range(count)]


def _slots(case):
    """Rows of the grouped layout: every choice, and each expert's padding to a whole group."""
    n, a = case["tokens"] * case["k"], case["align"]
    return (n + min(case["experts"], n) * (a - 1)) // a * a


def listed():
    def route(op, name, tokens, k, experts, width, dtype, align=1, drop=0.0, **more):
        return {"name": name, "op": op, "tokens": tokens, "k": k, "experts": experts, "width": width,
                "dtype": dtype, "align": align, "drop": drop, **more}

    return [
        # a batch of single tokens: all of it is latency
        route("dispatch", "dispatch-decode", 16, 4, 64, 4096, "bfloat16"),
        # a prompt batch, groups padded for a tiled product
        route("dispatch", "dispatch-prompt", 16384, 8, 128, 4096, "bfloat16", align=16),
        # odd sizes, padded tokens, experts of other ranks
        route("dispatch", "dispatch-ragged", 4099, 3, 60, 1001, "float32", align=8, drop=0.1),
        route("combine", "combine-decode", 32, 8, 256, 2048, "bfloat16", weighted=True),
        route("combine", "combine-prompt", 16384, 8, 128, 4096, "bfloat16", weighted=True),
        # the gradient of dispatch in a training step
        route("combine", "dispatch-grad", 8190, 2, 16, 1000, "float16", drop=0.02, weighted=False),
        route("combine_grad", "combine-grad-train", 8192, 8, 64, 2048, "bfloat16"),
        route("combine_grad", "combine-grad-ragged", 1021, 5, 33, 777, "float32", align=4, drop=0.2),
        # a small net's gradients, many of them a few hundred bytes
        {"name": "clip-inception", "op": "clip", "table": "inception", "dtype": "float32", "out": "same",
         "max_norm": 1.0},
        # a deep stack's, far past every cache
        {"name": "clip-layers", "op": "clip", "table": "layers", "layers": 12, "width": 2048,
         "dtype": "bfloat16", "out": "same", "max_norm": 1.0},
        # two clients' updates of a 1 K x 64 table
        {"name": "apply-small", "op": "apply", "rows": 1024, "width": 64, "clients": 2, "max_norm": 1.0},
        # eight clients' updates of the AlexNet table in 128-float rows
        {"name": "apply-alexnet", "op": "apply", "rows": 476292, "width": 128, "clients": 8, "max_norm": 1.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


MOST = 1.2e9  # bytes of a drawn case: less than the largest listed ones


def draw(rng):
    op = rng.choice(["dispatch", "combine", "combine_grad", "clip", "apply"])
    while True:
        if op == "clip":
            table = rng.choice(["alexnet", "layers", "layers", "ragged", "ragged"])
            case = {"op": op, "table": table, "dtype": rng.choice(["float32", "bfloat16", "float16", "mixed"]),
                    "out": rng.choice(["same", "float32"]), "max_norm": rng.choice([0.1, 1.0, 5.0, 1e6])}
            if table == "layers":
                case.update(layers=rng.randint(1, 24), width=_log(rng, 60, 1900))
            elif table == "ragged":
                case.update(tensors=rng.randint(1, 700), top=_log(rng, 100, 4000000))
        elif op == "apply":
            case = {"op": op, "rows": _log(rng, 1, 1000000), "width": rng.choice([1, 33, 64, 128, 500, 1024]),
                    "clients": rng.randint(1, 17), "max_norm": rng.choice([0.1, 1.0, 5.0, 1e6])}
        else:
            experts = _log(rng, 4, 512)
            case = {"op": op, "tokens": _log(rng, 1, 32768), "k": rng.randint(1, min(10, experts)),
                    "experts": experts,
                    "width": rng.choice([_log(rng, 32, 7168), 8 * _log(rng, 8, 896), 128 * _log(rng, 1, 56)]),
                    "dtype": rng.choice(["float32", "bfloat16", "float16"]),
                    "align": rng.choice([1, 1, 4, 16, 64]), "drop": rng.choice([0.0, 0.0, 0.05, 0.5])}
            if op == "combine":
                case["weighted"] = rng.random() < 0.7
        if work(case)["bytes"] <= MOST:
            return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _choices(case, g):
    """A router's choices: k different experts a token, some experts far more popular than others, int64 as
    topk gives them; -1 where a token is padding (the batch's end) or its expert belongs to another rank."""
    T, K, E = case["tokens"], case["k"], case["experts"]
    logits = torch.randn(T, E, device="cuda", generator=g) + 1.5 * torch.randn(E, device="cuda", generator=g)
    top, ids = logits.topk(K, dim=1)
    if case["drop"]:
        ids[torch.rand(T, K, device="cuda", generator=g) < case["drop"] / 2] = -1
        ids[T - int(T * case["drop"] / 2):] = -1
    return ids, top.softmax(1)


def _places(ids, experts, align, slots):
    """(position, order, counts, offsets) of the rows grouped by expert, tokens in order inside a group."""
    n = ids.numel()
    key = ids.reshape(-1)
    key = torch.where((key >= 0) & (key < experts), key, experts)
    order = torch.sort(key, stable=True).indices
    sorted_key = key[order]
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    counts.scatter_add_(0, key, torch.ones_like(key))
    padded = (counts[:experts] + align - 1) // align * align
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    offsets[1:] = padded.cumsum(0)
    first = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device)
    first[1:] = counts[:experts].cumsum(0)
    slot = offsets[sorted_key] + torch.arange(n, device=ids.device) - first[sorted_key]
    slot = torch.where(sorted_key < experts, slot, slots)
    position = torch.empty(n, dtype=torch.int64, device=ids.device)
    position[order] = torch.where(slot < slots, slot, -1)
    back = torch.full((slots + 1,), -1, dtype=torch.int64, device=ids.device)
    back[slot] = order
    back[slots] = -1
    return (position.view(ids.shape).int(), back[:slots].int(), counts[:experts].int(), offsets.int())


def prepare(case, seed):
    g = _generator(seed)
    op, state = case["op"], {"case": case}
    if op in ("dispatch", "combine", "combine_grad"):
        dtype, T, H = DTYPES[case["dtype"]], case["tokens"], case["width"]
        ids, weights = _choices(case, g)
        if op == "dispatch":
            state["ids"] = ids
            state["x"] = torch.randn(T, H, device="cuda", dtype=dtype, generator=g)
            return state
        # the places were made by the same step's dispatch
        state["places"] = _places(ids, case["experts"], case["align"], _slots(case))
        state["rows"] = torch.randn(_slots(case), H, device="cuda", dtype=dtype, generator=g)
        state["weights"] = weights if case.get("weighted", True) else None
        if op == "combine_grad":
            state["dy"] = torch.randn(T, H, device="cuda", dtype=dtype, generator=g)
        return state
    if op == "clip":
        sizes = _blobs(case)
        types = _blob_types(case, len(sizes))
        spread = (0.1 * torch.exp(1.5 * torch.randn(len(sizes), device="cuda", generator=g))).tolist()
        state["grads"] = [torch.randn(n, device="cuda", dtype=DTYPES[t], generator=g).mul_(s)
                          for n, t, s in zip(sizes, types, spread)]
        # the update buffers: one of each type, every gradient's update at a row of 128 values
        state["flat"], state["outs"] = _flat(sizes, [case["out"] if case["out"] != "same" else t for t in types])
        if own:  # a program's gradient and update buffers stay, and so does the plan over them
            from geeps_amd import clipping
            state["plan"] = clipping.GradPlan(state["grads"], state["outs"])
        return state
    n = case["rows"] * case["width"]
    state["master"] = torch.randn(n, device="cuda", generator=g).mul_(0.05)
    state["out"] = torch.zeros(n, device="cuda")  # the next version of the table, beside the published one
    state["updates"] = [torch.randn(n, device="cuda", generator=g).mul_(0.01) for _ in range(case["clients"])]
    return state


def _flat(sizes, types):
    """One zeroed buffer of each type, and in them a view of every length, at multiples of 128 values."""
    ends, at = {}, []
    for n, t in zip(sizes, types):
        at.append(ends.get(t, 0))
        ends[t] = at[-1] + -(-n // 128) * 128
    flat = {t: torch.zeros(n, device="cuda", dtype=DTYPES[t]) for t, n in ends.items()}
    return flat, [flat[t][a:a + n] for n, t, a in zip(sizes, types, at)]


def _factor(square_sum, max_norm):
    """(norm, scale) in 64 bits."""
    norm = square_sum.sqrt()
    return norm, torch.where(norm <= max_norm, torch.ones_like(norm), max_norm / norm)


def _taken(values, position):
    """(tokens, k, width) rows in 32 bits, zeros where a choice has no row."""
    rows = values.float()[position.long().clamp(min=0)]
    return torch.where((position >= 0)[..., None], rows, torch.zeros_like(rows[:1, :1]))


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from geeps_amd import clipping, routing
        if op == "dispatch":
            rows, route = routing.sort_and_dispatch(state["x"], state["ids"], case["experts"], align=case["align"])
            return {"rows": rows, "position": route.position, "order": route.order, "counts": route.counts,
                    "offsets": route.offsets}
        if op == "combine":
            return {"y": routing.combine(state["rows"], routing.Route(*state["places"]), state["weights"])}
        if op == "combine_grad":
            d_rows, d_weights = routing.combine_grad(state["dy"], state["rows"], routing.Route(*state["places"]),
                                                     state["weights"])
            return {"d_rows": d_rows, "d_weights": d_weights}
        if op == "clip":
            norm = state["plan"].clip(case["max_norm"])
            return {"norm": norm, "updates": state["flat"]}
        norm = clipping.apply_updates_clipped(state["master"], state["updates"], case["max_norm"], out=state["out"])
        return {"norm": norm, "master": state["out"]}
    if op == "dispatch":
        position, order, counts, offsets = _places(state["ids"], case["experts"], case["align"], _slots(case))
        x = state["x"]
        rows = torch.where((order >= 0)[:, None], x[order.clamp(min=0) // case["k"]], torch.zeros_like(x[:1]))
        return {"rows": rows, "position": position, "order": order, "counts": counts, "offsets": offsets}
    if op == "combine":
        taken = _taken(state["rows"], state["places"][0])
        if state["weights"] is not None:
            taken = taken * state["weights"][..., None]
        return {"y": taken.sum(1).to(state["rows"].dtype)}
    if op == "combine_grad":
        position, order = state["places"][:2]
        dy, weights = state["dy"].float(), state["weights"]
        d_weights = (_taken(state["rows"], position) * dy[:, None]).sum(2)
        at = order.clamp(min=0).long()
        d_rows = weights.reshape(-1)[at][:, None] * dy[at // case["k"]]
        d_rows = torch.where((order >= 0)[:, None], d_rows, torch.zeros_like(d_rows[:1]))
        return {"d_rows": d_rows.to(state["dy"].dtype), "d_weights": d_weights}
    if op == "clip":
        squares = torch.stack([x.float().square().sum(dtype=torch.float64) for x in state["grads"]])
        norm, factor = _factor(squares.sum(), case["max_norm"])
        factor = factor.float()
        _ = [torch.mul(x.float(), factor, out=o) for x, o in zip(state["grads"], state["outs"])]
        return {"norm": norm.float(), "updates": state["flat"]}
    total = functools.reduce(torch.add, state["updates"])
    norm, factor = _factor(total.square().sum(dtype=torch.float64), case["max_norm"])
    return {"norm": norm.float(), "master": state["master"] + total * factor.float()}


def work(case):
    op = case["op"]
    if op in ("dispatch", "combine", "combine_grad"):
        n, s = case["tokens"] * case["k"], SIZE[case["dtype"]]
        tokens, kept = case["tokens"] * case["width"] * s, n * (1 - case["drop"])
        rows = kept * case["width"] * s
        if op == "dispatch":  # choices and x in; every row of the grouped layout, both maps and the groups out
            return {"bytes": 8 * n + tokens + _slots(case) * (case["width"] * s + 4) + 4 * n + 8 * case["experts"],
                    "flops": 0}
        if op == "combine":
            return {"bytes": rows + tokens + 4 * n * (2 if case["weighted"] else 1), "flops": 2 * kept * case["width"]}
        return {"bytes": rows + _slots(case) * (case["width"] * s + 4) + tokens + 12 * n,
                "flops": 3 * kept * case["width"]}
    if op == "clip":
        sizes = _blobs(case)
        types = _blob_types(case, len(sizes))
        return {"bytes": sum(n * (SIZE[t] + (4 if case["out"] == "float32" else SIZE[t]))
                             for n, t in zip(sizes, types)), "flops": 3 * sum(sizes)}
    n = case["rows"] * case["width"]
    return {"bytes": 4 * n * (case["clients"] + 2), "flops": n * (case["clients"] + 4)}


def exact(case, seed):
    """What run() returns, from the definitions, in 64 bits: token by token sums, expert by expert places."""
    state, op = prepare(case, seed), case["op"]
    if op == "dispatch":
        ids, x = state["ids"].reshape(-1), state["x"]
        position = torch.full_like(ids, -1)
        order = torch.full((_slots(case),), -1, dtype=torch.int64, device="cuda")
        counts, offsets = [], [0]
        for e in range(case["experts"]):
            mine = (ids == e).nonzero().reshape(-1)
            at = offsets[-1] + torch.arange(len(mine), device="cuda")
            position[mine] = at
            order[at] = mine
            counts.append(len(mine))
            offsets.append(offsets[-1] + -(-len(mine) // case["align"]) * case["align"])
        rows = torch.zeros(_slots(case), case["width"], dtype=torch.float64, device="cuda")
        held = order >= 0
        rows[held] = x.double()[torch.div(order[held], case["k"], rounding_mode="floor")]
        return {"rows": rows, "position": position.view(state["ids"].shape), "order": order,
                "counts": torch.tensor(counts), "offsets": torch.tensor(offsets)}
    if op == "combine":
        y = torch.zeros(case["tokens"], case["width"], dtype=torch.float64, device="cuda")
        for k in range(case["k"]):
            p = state["places"][0][:, k].long()
            t = (p >= 0).nonzero().reshape(-1)
            r = state["rows"][p[t]].double()
            y[t] += r if state["weights"] is None else state["weights"][t, k].double()[:, None] * r
        return {"y": y}
    if op == "combine_grad":
        d_rows = torch.zeros(_slots(case), case["width"], dtype=torch.float64, device="cuda")
        d_weights = torch.zeros(case["tokens"], case["k"], dtype=torch.float64, device="cuda")
        for k in range(case["k"]):
            p = state["places"][0][:, k].long()
            t = (p >= 0).nonzero().reshape(-1)
            dy = state["dy"][t].double()
            d_rows[p[t]] = state["weights"][t, k].double()[:, None] * dy
            d_weights[t, k] = (state["rows"][p[t]].double() * dy).sum(1)
        return {"d_rows": d_rows, "d_weights": d_weights}
    if op == "clip":
        norm = math.sqrt(sum(float(x.double().square().sum()) for x in state["grads"]))
        factor = min(1.0, case["max_norm"] / norm) if norm else 1.0
        flat = {t: buffer.double() for t, buffer in state["flat"].items()}
        start = {t: buffer.data_ptr() for t, buffer in state["flat"].items()}
        for x, o in zip(state["grads"], state["outs"]):
            t = str(o.dtype).replace("torch.", "")
            a = (o.data_ptr() - start[t]) // o.element_size()
            flat[t][a:a + x.numel()] = x.double() * factor
        return {"norm": torch.tensor(norm, dtype=torch.float64), "updates": flat}
    total = torch.zeros_like(state["master"], dtype=torch.float64)
    for u in state["updates"]:
        total += u
    norm = float(total.square().sum().sqrt())
    return {"norm": torch.tensor(norm, dtype=torch.float64),
            "master": state["master"].double() + min(1.0, case["max_norm"] / norm) * total}
