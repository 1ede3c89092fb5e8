"""Operators over rows that are grouped by an index: tokens routed to experts and back, the experts'
products, and low-rank adapters of many requests, each with sizes that stand for its real use.

Every operator has a plain form here (elementary torch operations in 32 bits, rounded once at the end)
and the call that a program makes of this package. `run` takes either, by `own`.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def package():
    """The framework's Python binding (its folder is no importable package name)."""
    if "spmm_b200" not in sys.modules:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "sparse-matrix-multiplication_b200"))
    import spmm_b200

    return spmm_b200


# ------------------------------------------------------------------ cases


def listed():
    route = {"op": "route", "dtype": "bf16", "drop": 0.0}
    grad = {"op": "route_grad", "dtype": "bf16", "drop": 0.0}
    mm = {"op": "grouped", "dtype": "bf16", "out": "bf16", "skew": 0.5, "tail": 0}
    lora = {"op": "lora", "dtype": "bf16", "tail": 0, "none": 0.0, "base": True}
    return [
        # One token being answered, two experts of eight: nothing but latency.
        {**route, "name": "route one token", "tokens": 1, "topk": 2, "groups": 8, "hidden": 1024},
        # A packed batch of odd length in 32 bits, rows that start off a 16-byte boundary; a tenth of the pairs
        # belong to experts of another GPU and are left out.
        {**route, "name": "route odd f32", "tokens": 1021, "topk": 3, "groups": 60, "hidden": 1001, "dtype": "f32", "drop": 0.1},
        # A training or prefill batch over many experts.
        {**route, "name": "route large", "tokens": 16384, "topk": 8, "groups": 256, "hidden": 4096},
        # The backward pass of a small ragged batch, rows on 4-byte boundaries, pairs left out.
        {**grad, "name": "route grad odd f16", "tokens": 777, "topk": 4, "groups": 32, "hidden": 2050, "dtype": "f16", "drop": 0.1},
        # The backward pass of a training batch.
        {**grad, "name": "route grad large", "tokens": 16384, "topk": 8, "groups": 128, "hidden": 2048},
        # 32 tokens being answered, each with 8 of 128 experts: two rows an expert, the weights are read once.
        {**mm, "name": "grouped decode", "rows": 256, "groups": 128, "n": 1024, "k": 2048},
        # Prefill over many small experts with ragged lengths, some empty, and a buffer longer than its rows.
        {**mm, "name": "grouped ragged f16", "rows": 5003, "groups": 60, "n": 1000, "k": 1960, "dtype": "f16", "out": "f16", "skew": 1.2, "tail": 61},
        # A training batch on large experts.
        {**mm, "name": "grouped large", "rows": 32768, "groups": 8, "n": 4096, "k": 4096, "skew": 0.2},
        # Gradients of a small ragged batch, with the weights' gradient kept in 32 bits.
        {**mm, "op": "grouped_grad", "name": "grouped grad ragged", "rows": 3001, "groups": 16, "n": 520, "k": 776, "out": "f32", "skew": 1.0},
        # Gradients of a training batch.
        {**mm, "op": "grouped_grad", "name": "grouped grad large", "rows": 16384, "groups": 8, "n": 4096, "k": 2048, "skew": 0.2},
        # 64 requests being answered at once, one token each, of 32 adapters.
        {**lora, "name": "lora decode", "long": 0, "rows": 0, "single": 64, "adapters": 32, "rank": 16, "k": 4096, "n": 4096},
        # Four prompts and 100 answers in one batch, some without an adapter, and a buffer longer than its rows.
        {**lora, "name": "lora mixed", "long": 4, "rows": 8100, "single": 100, "adapters": 8, "rank": 64, "k": 4096, "n": 4096, "none": 0.1, "tail": 92},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _width(rng, low, high, odd):
    """A feature width: mostly whole 16-byte vectors, as models have them, else any number."""
    n = _log(rng, low, high)
    return n if rng.random() < odd else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["route", "route_grad", "grouped", "grouped_grad", "lora"])
    dtype = rng.choice(["f16", "bf16"])
    if op in ("route", "route_grad"):
        top = 16384 * 8 * 4096 if op == "route" else 16384 * 8 * 2048
        topk = rng.randint(1, 8)
        hidden = _width(rng, 64, 4096, 0.25)
        tokens = _log(rng, 1, 16384)
        dtype = rng.choice(["f16", "bf16", "f32"])
        if tokens * topk * hidden * BYTES[dtype] // 2 > top:
            dtype = "bf16"
        tokens = min(tokens, max(1, top // (topk * hidden)))
        return {"op": op, "tokens": tokens, "topk": topk, "groups": _log(rng, max(8, topk), 512), "hidden": hidden, "dtype": dtype,
                "drop": rng.choice([0.0, 0.0, 0.1, 0.5])}
    if op in ("grouped", "grouped_grad"):
        groups = _log(rng, 1, 128)
        n, k = _width(rng, 64, 4096, 0.1), _width(rng, 64, 4096, 0.1)
        top = 32768 * 4096 * 4096 if op == "grouped" else 16384 * 4096 * 2048
        groups = max(1, min(groups, 128 * 1024 * 2048 // (n * k)))
        rows = min(_log(rng, 1, 32768), top // (n * k))
        return {"op": op, "rows": rows, "groups": groups, "n": n, "k": k, "dtype": dtype, "out": rng.choice([dtype, "f32"]),
                "skew": rng.choice([0.0, 0.5, 1.0]), "tail": rng.choice([0, 0, rng.randint(1, 100)])}
    long = rng.choice([0, 0, rng.randint(1, 8)])
    return {"op": op, "long": long, "rows": _log(rng, 16, 8000) if long else 0, "single": _log(rng, 1, 128), "adapters": _log(rng, 1, 32),
            "rank": rng.choice([8, 16, 32, 64, 64, 128]), "k": max(64, _log(rng, 256, 4096) // 8 * 8), "n": max(64, _log(rng, 256, 4096) // 8 * 8),
            "dtype": dtype, "none": rng.choice([0.0, 0.1]), "base": rng.random() < 0.75, "tail": rng.choice([0, rng.randint(1, 64)])}


def _sizes(total, parts, skew):
    """`total` cut into `parts` whole numbers that fall like (i + 1)^-skew."""
    if not parts:
        return []
    weight = [(i + 1.0) ** -skew for i in range(parts)]
    size = [int(total * v / sum(weight)) for v in weight]
    for i in range(total - sum(size)):
        size[i % parts] += 1
    return size


# ------------------------------------------------------------------ inputs


def _generator(seed, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ids(g, case):
    """The experts of each token: distinct, some more wanted than others; -1 where the pair is another GPU's."""
    tokens, topk, groups = case["tokens"], case["topk"], case["groups"]
    wanted = torch.randn((1, groups), generator=g, device="cuda") * 0.5
    score = torch.randn((tokens, groups), generator=g, device="cuda") + wanted
    top = score.topk(topk, dim=1)
    ids = top.indices.to(torch.int32)
    weights = torch.softmax(top.values, dim=1).contiguous()
    if case["drop"]:
        ids = torch.where(torch.rand((tokens, topk), generator=g, device="cuda") < case["drop"], torch.full_like(ids, -1), ids)
    return ids.contiguous(), weights


def _lengths(case, seed):
    size = _sizes(case["rows"], case["long"], 0.5) + [1] * case["single"]
    order = torch.randperm(len(size), generator=_generator(seed, "cpu")).tolist()
    return [size[i] for i in order]


def _offsets(size):
    return torch.tensor([0] + size, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    op = case["op"]
    s = {"case": case}
    if op in ("route", "route_grad"):
        tokens, pairs, hidden = case["tokens"], case["tokens"] * case["topk"], case["hidden"]
        s["ids"], s["w"] = _ids(g, case)
        s["ys"] = _normal(g, (pairs, hidden), dtype)
        if op == "route":
            s["x"] = _normal(g, (tokens, hidden), dtype)
            s["offsets"] = torch.zeros(case["groups"] + 1, dtype=torch.int32, device="cuda")
            s["order"] = torch.zeros(pairs, dtype=torch.int32, device="cuda")
            s["pos"] = torch.zeros((tokens, case["topk"]), dtype=torch.int32, device="cuda")
            s["xs"], s["y"] = torch.zeros_like(s["ys"]), torch.zeros_like(s["x"])
        else:
            s["pos"] = _sort(s["ids"], case["groups"])[2]  # the forward pass left it
            s["dy"] = _normal(g, (tokens, hidden), dtype)
            s["dxs"] = _normal(g, (pairs, hidden), dtype)
            s["dys"], s["dx"] = torch.zeros_like(s["dxs"]), torch.zeros_like(s["dy"])
            s["dw"] = torch.zeros_like(s["w"])
        return s
    if op in ("grouped", "grouped_grad"):
        rows, groups, n, k = case["rows"], case["groups"], case["n"], case["k"]
        size = _sizes(rows, groups, case["skew"])
        order = torch.randperm(groups, generator=_generator(seed, "cpu")).tolist()
        s["offsets"], s["longest"] = _offsets([size[i] for i in order]), max(size)
        rows += case["tail"]
        s["x"] = _normal(g, (rows, k), dtype)
        s["w"] = _normal(g, (groups, n, k), dtype, k ** -0.5)
        if op == "grouped":
            s["y"] = torch.zeros((rows, n), dtype=DTYPES[case["out"]], device="cuda")
        else:
            s["dy"] = _normal(g, (rows, n), dtype)
            s["dx"] = torch.zeros((rows, k), dtype=dtype, device="cuda")
            s["dw"] = torch.zeros((groups, n, k), dtype=DTYPES[case["out"]], device="cuda")
        return s
    size = _lengths(case, seed)
    rows, rank, adapters = sum(size) + case["tail"], case["rank"], case["adapters"]
    s["offsets"] = _offsets(size)
    adapter = torch.randint(0, adapters, (len(size),), generator=g, device="cuda", dtype=torch.int32)
    none = torch.rand(len(size), generator=g, device="cuda") < case["none"]
    s["adapter"] = torch.where(none, torch.full_like(adapter, -1), adapter)
    s["x"] = _normal(g, (rows, case["k"]), dtype)
    s["a"] = _normal(g, (adapters, rank, case["k"]), dtype, case["k"] ** -0.5)
    s["b"] = _normal(g, (adapters, case["n"], rank), dtype, rank ** -0.5)
    s["scale"] = torch.rand(adapters, generator=g, device="cuda") + 0.5
    s["base"] = _normal(g, (rows, case["n"]), dtype) if case["base"] else None
    s["out"] = torch.zeros((rows, case["n"]), dtype=dtype, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms


def _sort(ids, groups):
    """The pairs in the order of their groups, pairs of one group in their own order, pairs without a group last."""
    flat = ids.reshape(-1).long()
    key = torch.where(flat >= 0, flat, groups)
    order = torch.sort(key, stable=True).indices
    pos = torch.empty_like(order)
    pos[order] = torch.arange(order.numel(), device=order.device)
    count = torch.zeros(groups + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, key, torch.ones_like(key))
    offsets = torch.cat([torch.zeros_like(count[:1]), count[:-1].cumsum(0)])
    order = torch.where(torch.arange(order.numel(), device=order.device) < offsets[-1], order, -1)
    pos = torch.where(flat >= 0, pos, -1).reshape(ids.shape)
    return offsets.int(), order.int(), pos.int()


def _to_groups(x, pos, weight=None):
    """Row pos[t, j] of the result is x[t], times weight[t, j]; rows that no pair has stay zero."""
    tokens, topk = pos.shape
    rows = x[:, None, :].expand(tokens, topk, x.shape[1])
    if weight is not None:
        rows = (rows.float() * weight[:, :, None]).to(x.dtype)
    spare = tokens * topk
    out = torch.zeros((spare + 1, x.shape[1]), dtype=x.dtype, device=x.device)
    out[torch.where(pos >= 0, pos.long(), spare).reshape(-1)] = rows.reshape(spare, -1)
    return out[:spare]


def _pairs(ys, pos):
    """Every pair's row in 32 bits, [tokens, topk, hidden], zero where it has none."""
    return torch.where(pos[:, :, None] >= 0, ys[pos.clamp(min=0).long()], 0).float()


def _blocks(offsets, longest, rows):
    """[groups, longest] row numbers of each group, the spare row `rows` behind its end."""
    at = offsets[:-1, None].long() + torch.arange(longest, device=offsets.device)
    return torch.where(at < offsets[1:, None], at, rows)


def _spare(x):
    """x in 32 bits with a row of zeros behind its last."""
    return torch.cat([x.float(), torch.zeros((1, x.shape[1]), device=x.device)])


def _back(blocks, at, rows, dtype):
    """The groups' rows at their places, the others zero."""
    out = torch.zeros((rows + 1, blocks.shape[2]), dtype=dtype, device=blocks.device)
    out[at.reshape(-1)] = blocks.to(dtype).reshape(-1, blocks.shape[2])
    return out[:rows]


def _row_adapter(offsets, adapter, rows):
    """Each row's request is real, and its adapter (-1: none)."""
    at = torch.arange(rows, device=offsets.device, dtype=torch.int32)
    request = torch.searchsorted(offsets, at, right=True) - 1
    real = (at >= offsets[0]) & (at < offsets[-1])
    return real, torch.where(real, adapter[request.clamp(0, adapter.numel() - 1)], -1).long()


def _plain(s):
    case, op = s["case"], s["case"]["op"]
    if op == "route":
        offsets, order, pos = _sort(s["ids"], case["groups"])
        y = (_pairs(s["ys"], pos) * s["w"][:, :, None]).sum(1).to(s["ys"].dtype)
        return {"offsets": offsets, "order": order, "pos": pos, "xs": _to_groups(s["x"], pos), "y": y}
    if op == "route_grad":
        dw = (_pairs(s["ys"], s["pos"]) * s["dy"].float()[:, None, :]).sum(2)
        dx = _pairs(s["dxs"], s["pos"]).sum(1).to(s["dy"].dtype)
        return {"dys": _to_groups(s["dy"], s["pos"], s["w"]), "dw": dw, "dx": dx}
    if op in ("grouped", "grouped_grad"):
        rows = s["x"].shape[0]
        at = _blocks(s["offsets"], s["longest"], rows)
        x, w = _spare(s["x"])[at], s["w"].float()
        if op == "grouped":
            return {"y": _back(torch.bmm(x, w.transpose(1, 2)), at, rows, s["y"].dtype)}
        dy = _spare(s["dy"])[at]
        return {"dx": _back(torch.bmm(dy, w), at, rows, s["dx"].dtype), "dw": torch.bmm(dy.transpose(1, 2), x).to(s["dw"].dtype)}
    # One product with every adapter, of which a row keeps its own: elementary, and two matrix products.
    x, a, b = s["x"].float(), s["a"].float(), s["b"].float()
    real, mine = _row_adapter(s["offsets"], s["adapter"], x.shape[0])
    adapters, rank, _ = a.shape
    keep = (mine[:, None] == torch.arange(adapters, device=x.device)) * s["scale"]
    u = (x @ a.reshape(adapters * rank, -1).T).reshape(-1, adapters, rank) * keep[:, :, None]
    y = u.reshape(-1, adapters * rank) @ b.transpose(1, 2).reshape(adapters * rank, -1)
    if s["base"] is not None:
        y = y + s["base"].float()
    return {"out": torch.where(real[:, None], y, 0).to(s["out"].dtype)}


# ------------------------------------------------------------------ the framework's calls


def _own(s):
    S = package()
    case, op = s["case"], s["case"]["op"]
    stream = torch.cuda.current_stream()
    if op == "route":
        S.route_build(s["ids"], case["groups"], s["offsets"], s["order"], s["pos"], stream=stream)
        S.route_gather(s["pos"], s["x"], s["xs"], stream=stream)
        S.route_combine(s["pos"], s["ys"], s["y"], s["w"], stream=stream)
        return {"offsets": s["offsets"], "order": s["order"], "pos": s["pos"], "xs": s["xs"], "y": s["y"]}
    if op == "route_grad":
        S.route_combine_grad(s["pos"], s["dy"], s["ys"], s["w"], s["dys"], s["dw"], stream=stream)
        S.route_combine(s["pos"], s["dxs"], s["dx"], stream=stream)  # the gather's gradient: the sum of a token's rows
        return {"dys": s["dys"], "dw": s["dw"], "dx": s["dx"]}
    if op == "grouped":
        S.grouped_mm(s["offsets"], s["x"], s["w"], s["y"], stream=stream)
        return {"y": s["y"]}
    if op == "grouped_grad":
        S.grouped_mm_dx(s["offsets"], s["dy"], s["w"], s["dx"], stream=stream)
        S.grouped_mm_dw(s["offsets"], s["dy"], s["x"], s["dw"], stream=stream)
        return {"dx": s["dx"], "dw": s["dw"]}
    S.lora(s["offsets"], s["adapter"], s["x"], s["a"], s["b"], s["out"], base=s["base"], scale=s["scale"], stream=stream)
    return {"out": s["out"]}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    op, e = case["op"], BYTES[case["dtype"]]
    if op in ("route", "route_grad"):
        tokens, pairs, hidden = case["tokens"], case["tokens"] * case["topk"], case["hidden"]
        kept = pairs * (1 - case["drop"])
        rows = 2 * (tokens + kept) * hidden * e  # route: x and the outputs' rows in, both out
        if op == "route":
            return {"bytes": int(rows + 12 * pairs + 4 * kept + 4 * case["groups"]), "flops": int(2 * kept * hidden)}
        return {"bytes": int(rows + kept * hidden * e + 4 * pairs + 8 * kept), "flops": int(4 * kept * hidden)}
    if op in ("grouped", "grouped_grad"):
        rows, n, k = case["rows"], case["n"], case["k"]
        used = sum(v > 0 for v in _sizes(rows, case["groups"], case["skew"]))
        o = BYTES[case["out"]]
        if op == "grouped":
            return {"bytes": rows * k * e + used * n * k * e + rows * n * o, "flops": 2 * rows * n * k}
        return {"bytes": rows * (n + 2 * k) * e + used * n * k * e + case["groups"] * n * k * o, "flops": 4 * rows * n * k}
    rows = case["rows"] + case["single"]
    with_one = rows * (1 - case["none"])
    used = min(case["adapters"], case["long"] + case["single"])
    k, n, rank = case["k"], case["n"], case["rank"]
    return {"bytes": int((with_one * k + rows * n * (2 if case["base"] else 1) + used * rank * (k + n)) * e), "flops": int(2 * with_one * rank * (k + n))}


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("route", "route_grad"):
        tokens, topk = s["ids"].shape
        pairs = tokens * topk
        ids = s["ids"].flatten().long()
        # A pair's row: the pairs of smaller groups, and those of its own that come before it, by one sort of distinct numbers.
        rank = torch.argsort(torch.argsort(torch.where(ids < 0, case["groups"], ids) * pairs + torch.arange(pairs, device="cuda")))
        has, token = ids >= 0, torch.arange(pairs, device="cuda") // topk
        pair = torch.nonzero(has).flatten()
        row, hidden = rank[pair], case["hidden"]
        w = s["w"].double().flatten()[pair, None]
        if op == "route":
            order = torch.full((pairs,), -1, device="cuda")
            order[row] = pair
            xs = torch.zeros((pairs, hidden), dtype=torch.float64, device="cuda")
            xs[row] = s["x"].double()[token[pair]]
            y = torch.zeros((tokens, hidden), dtype=torch.float64, device="cuda").index_add_(0, token[pair], w * s["ys"][row].double())
            count = torch.stack([(ids == v).sum() for v in range(case["groups"])])
            offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
            return {"offsets": offsets.int(), "order": order.int(), "pos": torch.where(has, rank, -1).reshape(tokens, topk).int(), "xs": xs, "y": y}
        dy = s["dy"].double()[token[pair]]
        dys = torch.zeros((pairs, hidden), dtype=torch.float64, device="cuda")
        dys[row] = w * dy
        dw = torch.zeros(pairs, dtype=torch.float64, device="cuda")
        dw[pair] = torch.einsum("ph,ph->p", dy, s["ys"][row].double())
        dx = torch.zeros((tokens, hidden), dtype=torch.float64, device="cuda").index_add_(0, token[pair], s["dxs"][row].double())
        return {"dys": dys, "dw": dw.reshape(tokens, topk), "dx": dx}
    if op in ("grouped", "grouped_grad"):
        at = s["offsets"].tolist()
        if op == "grouped":
            y = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
            for e, (i, j) in enumerate(zip(at, at[1:])):
                y[i:j] = s["x"][i:j].double() @ s["w"][e].double().T
            return {"y": y}
        dx = torch.zeros(s["dx"].shape, dtype=torch.float64, device="cuda")
        dw = torch.zeros(s["dw"].shape, dtype=torch.float64, device="cuda")
        for e, (i, j) in enumerate(zip(at, at[1:])):
            dx[i:j] = s["dy"][i:j].double() @ s["w"][e].double()
            dw[e] = s["dy"][i:j].double().T @ s["x"][i:j].double()
        return {"dx": dx, "dw": dw}
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    at = s["offsets"].tolist()
    for e, i, j in zip(s["adapter"].tolist(), at, at[1:]):
        if s["base"] is not None:
            out[i:j] = s["base"][i:j].double()
        if e >= 0:
            out[i:j] += s["scale"][e].double() * (s["x"][i:j].double() @ s["a"][e].double().T @ s["b"][e].double().T)
    return {"out": out}
