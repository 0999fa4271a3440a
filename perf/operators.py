"""What the routed 8-bit operators are measured on: vectors quantised by rows, products in 8-bit integers with a scale for
each row and channel, rows sorted by the expert (or root codeword) they were assigned to and back, and the gradient of that
exchange.

``run`` computes them in elementary torch operations, or, where ``own`` is true, through ``stlq_b200.Kernels``.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"
_KERNELS = None


def kernels():
    """The handle that a program keeps."""
    global _KERNELS
    if _KERNELS is None:
        import stlq_b200

        _KERNELS = stlq_b200.Kernels(0)
    return _KERNELS


# ---- cases -------------------------------------------------------------------------------------

def listed():
    return [
        # A projection of one token while serving: bound by reading the weights, and by latency.
        {"name": "linear 1 token", "op": "linear", "tokens": 1, "cols": 4096, "n": 4096, "dtype": "bf16", "bias": False},
        # A ragged batch of vectors with 960 dimensions (the large-dimension vector sets) into 1,000 channels.
        {"name": "linear ragged", "op": "linear", "tokens": 777, "cols": 960, "n": 1000, "dtype": "f16", "bias": True},
        # A projection over the tokens of many prompts: bound by the tensor cores.
        {"name": "linear prompts", "op": "linear", "tokens": 16384, "cols": 4096, "n": 4096, "dtype": "bf16", "bias": False},
        # Scores of a block of 8-bit vectors against the largest root codebook (65,536 codewords, 128 dimensions): bound
        # by writing them.
        {"name": "scores of 65536 roots", "op": "product", "tokens": 4096, "cols": 128, "n": 65536, "dtype": "f32", "bias": False},
        # The routing of one serving step: latency.
        {"name": "sort a step", "op": "sort", "tokens": 64, "topk": 8, "experts": 256, "ids": "i64", "drop": 0.1},
        # A block of a million vectors grouped by 16,384 roots.
        {"name": "sort a block by root", "op": "sort", "tokens": 1000000, "topk": 1, "experts": 16384, "ids": "i32", "drop": 0.0},
        # The exchange at an odd dimension and in 32 bits, with choices that capacity dropped.
        {"name": "exchange odd", "op": "exchange", "tokens": 333, "topk": 2, "experts": 10, "cols": 30, "dtype": "f32", "ids": "i32", "drop": 0.2},
        # The exchange of a large batch with fine experts.
        {"name": "exchange batch", "op": "exchange", "tokens": 16384, "topk": 8, "experts": 128, "cols": 2048, "dtype": "bf16", "ids": "i64", "drop": 0.0},
        # The gradient of both halves: a small ragged batch, and a large one.
        {"name": "gradient ragged", "op": "gradient", "tokens": 1000, "topk": 4, "experts": 33, "cols": 200, "dtype": "f16", "ids": "i64", "drop": 0.1},
        {"name": "gradient batch", "op": "gradient", "tokens": 16384, "topk": 4, "experts": 64, "cols": 4096, "dtype": "bf16", "ids": "i64", "drop": 0.05},
        # A routed layer while serving eight tokens: the weights of the experts that were chosen are read once.
        {"name": "experts 8 tokens", "op": "experts", "tokens": 8, "topk": 8, "experts": 128, "cols": 2048, "n": 1024, "dtype": "bf16", "ids": "i64", "drop": 0.0},
        # A routed layer over a batch of prompts.
        {"name": "experts prompts", "op": "experts", "tokens": 8192, "topk": 4, "experts": 64, "cols": 2048, "n": 2048, "dtype": "bf16", "ids": "i64", "drop": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "product", "sort", "exchange", "gradient", "experts", "experts"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    ids = rng.choice(["i32", "i64"])
    drop = rng.choice([0.0, 0.0, rng.uniform(0.0, 0.5)])
    while True:
        c = {"op": op}
        if op in ("linear", "product"):
            c |= {"tokens": _log(rng, 1, 16384), "cols": _log(rng, 24, 8192), "n": _log(rng, 24, 65536 if op == "product" else 8192), "dtype": dtype, "bias": rng.random() < 0.5}
            if c["tokens"] * c["n"] > 4096 * 65536 or c["n"] * c["cols"] > 8192 * 8192:
                continue
        elif op == "sort":
            c |= {"tokens": _log(rng, 16, 1000000), "topk": rng.choice([1, 1, 2, 4, 6, 8]), "experts": _log(rng, 2, 65536), "ids": ids, "drop": drop}
            if c["tokens"] * c["topk"] > 1000000 or (c["topk"] > 1 and c["tokens"] * c["experts"] > 1 << 26):
                continue
        else:
            c |= {"tokens": _log(rng, 1, 16384), "topk": rng.choice([1, 2, 4, 6, 8]), "experts": _log(rng, 8, 256), "cols": _log(rng, 24, 8192)}
            if op == "experts":
                c |= {"n": _log(rng, 24, 4096)}
                if c["experts"] * c["n"] * c["cols"] > 1 << 29:
                    continue
            c |= {"dtype": dtype, "ids": ids, "drop": drop}
            if c["tokens"] * c["topk"] * max(c["cols"], c.get("n", 0)) > 1 << 28:
                continue
        if work(c)["flops"] <= 2 * 16384 * 4096 * 4096 and work(c)["bytes"] <= 1.8e9:
            return c


# ---- inputs ------------------------------------------------------------------------------------

def _vectors(g, rows, cols, dtype):
    """Rows with norms of their own and some channels that stand out, as activations have them."""
    x = torch.randn(rows, cols, device=DEV, generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device=DEV, generator=g))
    x *= torch.where(torch.rand(1, cols, device=DEV, generator=g) < 0.01, 8.0, 1.0)
    return x.to(TYPES[dtype])


def _weights(g, rows, cols):
    """8-bit rows laid out once, each row on a 16-byte boundary, and a scale for each."""
    w = torch.randn(rows, (cols + 15) // 16 * 16, device=DEV, generator=g).mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)
    return w[:, :cols], (torch.rand(rows, device=DEV, generator=g) + 0.5) * (1.0 / (36.0 * math.sqrt(cols)))


def _ids(g, c):
    """Choices without repeats, some experts more popular than others; a dropped choice is -1."""
    t, k, e = c["tokens"], c["topk"], c["experts"]
    if k == 1:
        ids = (torch.rand(t, 1, device=DEV, generator=g).pow(1.5) * e).long().clamp_(max=e - 1)
    else:
        logits = torch.randn(t, e, device=DEV, generator=g) + 0.5 * torch.randn(1, e, device=DEV, generator=g)
        ids = logits.topk(min(k, e), dim=1).indices
        if k > e:
            ids = torch.cat([ids, torch.full((t, k - e), -1, device=DEV, dtype=torch.int64)], 1)
    if c["drop"]:
        ids = torch.where(torch.rand(t, k, device=DEV, generator=g) < c["drop"], -1, ids)
    return ids.to(torch.int32 if c["ids"] == "i32" else torch.int64).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    c, s = case, {"case": case}
    op, dtype = c["op"], c.get("dtype")
    if op in ("linear", "product", "experts"):
        s["x"] = _vectors(g, c["tokens"], c["cols"], "f32" if op == "product" else dtype)
        e = c.get("experts", 1)
        s["w"], s["ws"] = _weights(g, e * c["n"], c["cols"])
        if op == "experts":
            s["w"], s["ws"] = s["w"].unflatten(0, (e, c["n"])), s["ws"].view(e, c["n"])
        s["bias"] = 0.1 * torch.randn(c["n"], device=DEV, generator=g) if c.get("bias") else None
    if op == "product":  # rows that were quantised before
        s["x"], s["xs"] = _weights(g, c["tokens"], c["cols"])
    if op in ("sort", "exchange", "gradient", "experts"):
        s["ids"] = _ids(g, c)
    if op in ("exchange", "gradient", "experts"):
        s["mix"] = torch.softmax(torch.randn(c["tokens"], c["topk"], device=DEV, generator=g), 1)
    if op in ("exchange", "gradient"):
        pairs = c["tokens"] * c["topk"]
        s["x"] = _vectors(g, c["tokens"], c["cols"], dtype)  # also the gradient that comes back
        s["y"] = torch.randn(pairs, c["cols"], device=DEV, generator=g).to(TYPES[dtype])
        order, position, offsets = _sorted(s["ids"], c["experts"])
        s["y"][int(offsets[-1]):] = math.nan  # rows of dropped choices hold no result
        if op == "gradient":  # the forward pass left the routing and its own rows
            s["dxs"] = torch.randn(pairs, c["cols"], device=DEV, generator=g).to(TYPES[dtype])
            s["order"], s["position"], s["offsets"] = order, position, offsets
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _sorted(ids, experts):
    """(order, position, offsets) of the pairs, those without a valid expert last."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = torch.sort(key, stable=True).indices
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=DEV).index_add_(0, key, torch.ones_like(key))
    offsets = torch.cumsum(counts, 0) - counts
    return order.int(), position.view(ids.shape).int(), offsets.int()


def _quantised(x):
    x = x.float()
    amax = x.abs().amax(1, keepdim=True)
    q = torch.where(amax > 0, torch.round(x * 127 / torch.where(amax > 0, amax, 1.0)), 0.0)
    return q, (amax / 127)[:, 0]


def _scaled(acc, s, ws, bias):
    y = acc * s[..., None] * ws[..., None, :]
    return y if bias is None else y + bias


def _dispatched(x, order, offsets, topk):
    kept = torch.arange(order.numel(), device=DEV)[:, None] < offsets[-1]
    return torch.where(kept, x[order.long() // topk], torch.zeros((), dtype=x.dtype, device=DEV))


def _combined(y, mix, position, offsets):
    kept = (position < offsets[-1])[..., None]
    rows = torch.where(kept, y[position.long()].float(), 0.0)
    return (rows if mix is None else rows * mix[..., None]).sum(1)


def _experts(q, s, w, ws, order, offsets, topk):
    """Every expert's rows padded to the longest segment, one batched product, and back to the sorted order."""
    counts = offsets[1:] - offsets[:-1]
    longest = max(1, int(counts.max()))
    rows = order.numel()
    at = offsets[:-1, None].long() + torch.arange(longest, device=DEV)
    real = torch.arange(longest, device=DEV) < counts[:, None]
    token = order.long()[at.clamp(max=rows - 1)] // topk
    acc = torch.matmul(torch.where(real[..., None], q[token], 0.0), w.float().transpose(1, 2))
    y = _scaled(acc, s[token], ws, None)
    out = torch.zeros(rows + 1, w.shape[1], device=DEV)
    out[torch.where(real, at, rows).reshape(-1)] = y.flatten(0, 1)
    out[rows] = 0.0
    return out[:rows]


def _plain(s):
    c = s["case"]
    op = c["op"]
    if op == "sort":
        order, position, offsets = _sorted(s["ids"], c["experts"])
        return {"order": order, "position": position, "offsets": offsets}
    kind = TYPES[c["dtype"]]
    if op in ("linear", "product"):
        q, scale = _quantised(s["x"]) if op == "linear" else (s["x"].float(), s["xs"])
        return {"y": _scaled(torch.matmul(q, s["w"].float().t()), scale, s["ws"], s["bias"]).to(kind)}
    if op == "exchange":
        order, position, offsets = _sorted(s["ids"], c["experts"])
        return {"xs": _dispatched(s["x"], order, offsets, c["topk"]), "out": _combined(s["y"], s["mix"], position, offsets).to(kind)}
    if op == "gradient":
        order, position, offsets = s["order"].long(), s["position"], s["offsets"]
        dx = _combined(s["dxs"], None, position, offsets).to(kind)
        kept = torch.arange(order.numel(), device=DEV)[:, None] < offsets[-1]
        dy = torch.where(kept, s["x"][order // c["topk"]].float() * s["mix"].reshape(-1)[order][:, None], 0.0).to(kind)
        rows = torch.where((position < offsets[-1])[..., None], s["y"][position.long()].float(), 0.0)
        return {"dx": dx, "dy": dy, "dmix": (rows * s["x"].float()[:, None]).sum(-1)}
    order, position, offsets = _sorted(s["ids"], c["experts"])
    q, scale = _quantised(s["x"])
    y = _experts(q, scale, s["w"], s["ws"], order, offsets, c["topk"]).to(kind)
    return {"out": _combined(y, s["mix"], position, offsets).to(kind)}


# ---- the framework's operators -----------------------------------------------------------------

def _own(s):
    c, k = s["case"], kernels()
    op = c["op"]
    if op == "linear":
        q, scale = k.quantize_rows(s["x"])
        return {"y": k.matmul_i8(q, scale, s["w"], s["ws"], bias=s["bias"], out_dtype=s["x"].dtype)}
    if op == "product":
        return {"y": k.matmul_i8(s["x"], s["xs"], s["w"], s["ws"], bias=s["bias"], out_dtype=TYPES[c["dtype"]])}
    if op == "sort":
        r = k.sort_by_expert(s["ids"], c["experts"])
        return {"order": r.order, "position": r.position, "offsets": r.offsets}
    if op == "exchange":
        r = k.sort_by_expert(s["ids"], c["experts"])
        return {"xs": k.dispatch(s["x"], r), "out": k.combine(s["y"], s["mix"], r)}
    if op == "gradient":
        import stlq_b200

        r = stlq_b200.Routing(s["order"], s["position"], s["offsets"])
        dx = k.dispatch_backward(s["dxs"], r)
        dy, dmix = k.combine_backward(s["x"], s["y"], s["mix"], r)
        return {"dx": dx, "dy": dy, "dmix": dmix}
    r = k.sort_by_expert(s["ids"], c["experts"])
    q, scale = k.dispatch_i8(s["x"], r)
    y = k.matmul_i8_grouped(q, scale, s["w"], s["ws"], r.offsets, out_dtype=s["x"].dtype)
    return {"out": k.combine(y, s["mix"], r)}


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    c = case
    op, t = c["op"], c["tokens"]
    e = BYTES.get(c.get("dtype"), 0)
    if op in ("linear", "product"):
        x = t * c["cols"] * (e if op == "linear" else 1) + (0 if op == "linear" else 4 * t)
        b = x + c["n"] * c["cols"] + 4 * c["n"] * (2 if c["bias"] else 1) + t * c["n"] * e
        return {"bytes": b, "flops": 2 * t * c["cols"] * c["n"]}
    pairs = t * c["topk"]
    kept = pairs * (1.0 - c["drop"])
    ids = pairs * (4 if c["ids"] == "i32" else 8)
    if op == "sort":
        return {"bytes": ids + 8 * pairs + 4 * (c["experts"] + 1), "flops": 0}
    d = c["cols"]
    if op == "exchange":
        return {"bytes": ids + 4 * pairs + (2 * t + pairs + kept) * d * e, "flops": 2 * kept * d}
    if op == "gradient":  # dxs and y read once where kept, dout read, dx and dy written, weights and their gradient
        return {"bytes": (2 * kept + 2 * t + pairs) * d * e + 16 * pairs, "flops": 4 * kept * d}
    used = c["experts"] * (1.0 - (1.0 - 1.0 / c["experts"]) ** kept)  # experts that some row chose
    return {"bytes": ids + 4 * pairs + t * d * e + used * c["n"] * (d + 4) + t * c["n"] * e, "flops": 2 * kept * d * c["n"]}


# ---- the definition in 64 bits -----------------------------------------------------------------

def _exact_rows(x):
    x = x.double()
    top = x.abs().max(dim=1).values
    return torch.where(top[:, None] > 0, torch.round(127.0 * x / top[:, None]), 0.0), top / 127.0


def _exact_pairs(ids, experts):
    """The pairs that are kept, expert by expert, and how many each expert has."""
    flat = ids.reshape(-1).cpu().numpy().astype(np.int64)
    valid = np.nonzero((flat >= 0) & (flat < experts))[0]
    valid = valid[np.argsort(flat[valid], kind="stable")]
    return torch.from_numpy(valid).to(DEV), np.bincount(flat[valid], minlength=experts)


def exact(case, seed):
    c = case
    op = c["op"]
    if op == "sort":
        return None  # whole numbers
    s = prepare(case, seed)
    if op in ("linear", "product"):
        q, scale = _exact_rows(s["x"]) if op == "linear" else (s["x"].double(), s["xs"].double())
        y = (q * scale[:, None]) @ (s["w"].double() * s["ws"].double()[:, None]).t()
        return {"y": y if s["bias"] is None else y + s["bias"].double()}
    pairs, counts = _exact_pairs(s["ids"], c["experts"])
    kept = pairs.numel()
    token, mix = pairs // c["topk"], s["mix"].double().reshape(-1)[pairs][:, None]
    if op == "exchange":
        xs = torch.zeros(c["tokens"] * c["topk"], c["cols"], dtype=torch.float64, device=DEV)
        xs[:kept] = s["x"].double()[token]
        out = torch.zeros(c["tokens"], c["cols"], dtype=torch.float64, device=DEV).index_add_(0, token, s["y"][:kept].double() * mix)
        return {"xs": xs, "out": out}
    if op == "gradient":
        dx = torch.zeros(c["tokens"], c["cols"], dtype=torch.float64, device=DEV).index_add_(0, token, s["dxs"][:kept].double())
        dy = torch.zeros(c["tokens"] * c["topk"], c["cols"], dtype=torch.float64, device=DEV)
        dout = s["x"].double()[token]
        dy[:kept] = dout * mix
        dmix = torch.zeros(c["tokens"] * c["topk"], dtype=torch.float64, device=DEV)
        dmix[pairs] = (dout * s["y"][:kept].double()).sum(1)
        return {"dx": dx, "dy": dy, "dmix": dmix.view(c["tokens"], c["topk"])}
    q, scale = _exact_rows(s["x"])
    out = torch.zeros(c["tokens"], c["n"], dtype=torch.float64, device=DEV)
    first = 0
    for e, count in enumerate(counts.tolist()):
        if count:
            rows = token[first:first + count]
            y = (q[rows] @ s["w"][e].double().t()) * scale[rows][:, None] * s["ws"][e].double()
            out.index_add_(0, rows, y * mix[first:first + count])
        first += count
    return {"out": out}
