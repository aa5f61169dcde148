"""The expert operators at the sizes their users call them with.

A quantised mixture-of-experts feed-forward runs four operators: the router
(``route_experts``), the products of the rows sorted by expert
(``gemm_w8a8_grouped`` for int8 weights, ``matvec_w4`` for 4-bit weights and
few rows) and the weighted sum back into token order (``combine_experts``).
``matvec_w4`` also serves the plain few-row linears of an int4 model, such as
a block's modulation, whose rows are the batch's samples.

With ``own`` false, ``run`` computes each operator in elementary float32
torch operations; with ``own`` true it calls the framework.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
GROUP = 128  # k values that share a 4-bit weight scale, where a row has several


def _framework():
    """The package (its folder's name has dashes, as ComfyUI's node folders do)."""
    name = "comfyui_int8_fast_rocm_b200"
    if name not in sys.modules:
        folder = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "comfyui-int8-fast-rocm_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        module = importlib.util.module_from_spec(spec)
        sys.modules[name] = module
        spec.loader.exec_module(module)
    return sys.modules[name].ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # the router of a served model: one new token
        dict(name="route 1 token", op="route", tokens=1, experts=64, top=6, scoring="softmax", renorm=True,
             dtype="f32", masked=0),
        # a prompt (or an image's tokens over a batch) through fine-grained experts
        dict(name="route 16384 tokens", op="route", tokens=16384, experts=128, top=8, scoring="softmax", renorm=True,
             dtype="bf16", masked=0),
        # an odd number of tokens, some experts switched off, padding tokens that may choose none
        dict(name="route 1021 masked", op="route", tokens=1021, experts=60, top=4, scoring="sigmoid", renorm=False,
             dtype="f32", masked=7),
        # a few tokens in flight: every active expert has one row or a few, so the weights' bytes are the work
        dict(name="grouped decode", op="grouped", rows=32, spare=0, experts=64, n=2048, k=4096, dtype="bf16",
             gather=True, bias=False),
        # ragged everything: columns that fill no tile, a depth that ends inside a slab, rows that belong to no expert
        dict(name="grouped odd", op="grouped", rows=1237, spare=11, experts=12, n=1000, k=1328, dtype="f16",
             gather=False, bias=True),
        # 4096 tokens, two of eight experts each: the up projection, gathered from the tokens' rows
        dict(name="grouped prompt", op="grouped", rows=8192, spare=0, experts=8, n=12288, k=4096, dtype="bf16",
             gather=True, bias=False),
        # 4096 tokens, eight of 64 experts each: the down projection of fine-grained experts
        dict(name="grouped fine", op="grouped", rows=32768, spare=0, experts=64, n=2048, k=1536, dtype="bf16",
             gather=False, bias=False),
        # a block's modulation for one sample: six vectors of the hidden size
        dict(name="matvec modulation", op="matvec", rows=1, spare=0, experts=0, n=24576, k=4096, groups=True,
             dtype="bf16", gather=False, bias=True),
        # float32 embeddings of a small batch through a layer with one scale a row and odd sizes
        dict(name="matvec odd f32", op="matvec", rows=5, spare=0, experts=0, n=1111, k=1440, groups=False,
             dtype="f32", gather=False, bias=True),
        # sixteen tokens in flight, two of eight experts each
        dict(name="matvec experts", op="matvec", rows=32, spare=0, experts=8, n=8192, k=4096, groups=True,
             dtype="f16", gather=True, bias=False),
        # one token's experts added up
        dict(name="combine 1 token", op="combine", tokens=1, top=8, n=4096, dtype="bf16", residual=False, dropped=0),
        # a prompt's experts added up onto the residual stream
        dict(name="combine 4096 tokens", op="combine", tokens=4096, top=2, n=4096, dtype="bf16", residual=True,
             dropped=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["route", "grouped", "grouped", "matvec", "matvec", "combine"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "route":
        experts = _log(rng, 4, 256)
        return dict(op=op, tokens=_log(rng, 1, 32768), experts=experts, top=rng.randint(1, min(8, experts)),
                    scoring=rng.choice(["softmax", "sigmoid"]), renorm=rng.random() < 0.7, dtype=dtype,
                    masked=rng.choice([0, 0, experts // 3]))
    if op == "combine":
        return dict(op=op, tokens=_log(rng, 1, 8192), top=rng.randint(1, 8), n=_log(rng, 64, 8192), dtype=dtype,
                    residual=rng.random() < 0.5, dropped=rng.choice([0, 0, 3]))
    rows, experts, n = _log(rng, 1, 16384 if op == "grouped" else 48), _log(rng, 2, 128), _log(rng, 64, 12288)
    spare = rng.choice([0, 0, 0, rng.randint(1, 40)])
    common = dict(spare=spare, dtype=dtype, gather=rng.random() < 0.5, bias=rng.random() < 0.4)
    if op == "grouped":
        k = 16 * _log(rng, 8, 512)
        while experts > 2 and experts * n * k > 1.2e9:
            experts //= 2
        while rows > 64 and rows * n * k > 2e11:
            rows //= 2
        return dict(op=op, rows=rows, experts=experts, n=n, k=k, **common)
    groups = rng.random() < 0.7
    k = GROUP * _log(rng, 1, 128) if groups else 2 * _log(rng, 32, 8192)
    experts = rng.choice([0, experts])
    while experts > 2 and experts * n * k > 8e8:
        experts //= 2
    if not experts:
        common.update(spare=0, gather=False)
    return dict(op=op, rows=rows, experts=experts, n=n, k=k, groups=groups, **common)


def _counts(rows, experts):
    """Rows of each expert, most popular first: shares of 1 / (i + 4), as uneven as routers are."""
    share = [1.0 / (i + 4) for i in range(experts)]
    total, counts, left = sum(share), [], rows
    for i in range(experts):
        take = min(left, int(math.ceil(left * share[i] / total))) if i < experts - 1 else left
        counts.append(take)
        left, total = left - take, total - share[i]
    return counts


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 1000003 + 17)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] == "route":
        T, E = case["tokens"], case["experts"]
        logits = _randn(g, T, E) * 1.5 + _randn(g, E)
        if case["masked"]:  # experts switched off, and padding tokens without any
            logits[:, torch.randperm(E, generator=g, device="cuda")[:case["masked"]]] = -math.inf
            logits[torch.rand(T, generator=g, device="cuda") < 0.03] = -math.inf
        s["logits"] = logits.to(dt)
        return s
    if case["op"] == "combine":
        T, k, n = case["tokens"], case["top"], case["n"]
        s["y"] = _randn(g, T * k, n, dtype=dt)
        s["weights"] = torch.softmax(_randn(g, T, k), -1)
        s["pos"] = torch.randperm(T * k, generator=g, device="cuda").to(torch.int32).reshape(T, k)
        if case["dropped"]:
            gone = torch.rand(T, k, generator=g, device="cuda") < 1.0 / case["dropped"]
            s["pos"] = torch.where(gone, torch.full_like(s["pos"], -1), s["pos"])
            s["weights"] = torch.where(gone, torch.zeros_like(s["weights"]), s["weights"])
        s["residual"] = _randn(g, T, n, dtype=dt) if case["residual"] else None
        return s
    E, n, k, rows = case["experts"], case["n"], case["k"], case["rows"]
    total = rows + case["spare"]  # the spare rows lie behind the last expert's
    if E:
        counts = torch.tensor(_counts(rows, E), dtype=torch.int32)
        order = torch.randperm(E, generator=torch.Generator().manual_seed(seed))
        counts = counts[order]
        s["cap"] = int(counts.max())  # what a caller knows of its buffers: the plain form pads to it
        s["offsets"] = torch.cat((torch.zeros(1, dtype=torch.int32), counts.cumsum(0).to(torch.int32))).cuda()
    else:
        s["offsets"] = None
    lead = (E,) if E else ()
    sources = max(1, total // 2) if case["gather"] else total
    s["a_rows"] = torch.randint(0, sources, (total,), generator=g, device="cuda", dtype=torch.int32) \
        if case["gather"] else None
    s["bias"] = _randn(g, *lead, n, dtype=dt) if case["bias"] else None
    if case["op"] == "grouped":
        s["a"] = (_randn(g, sources, k) * 32).round().clamp(-127, 127).to(torch.int8)
        s["a_scale"] = torch.rand(sources, 1, generator=g, device="cuda") * 0.04 + 0.01
        w = torch.empty(E, n, k, dtype=torch.int8, device="cuda")
        for part in w.split(max(1, 2 ** 28 // (n * k))):
            part.copy_((_randn(g, *part.shape) * 32).round().clamp(-127, 127))
        s["w"] = w
        s["w_scale"] = torch.rand(E, n, generator=g, device="cuda") * 4e-4 + 1e-4
        return s
    x = _randn(g, sources, k)
    x[:, torch.rand(k, generator=g, device="cuda") < 0.001] *= 20  # the outlier channels of such activations
    s["x"] = x.to(dt)
    s["w"] = torch.randint(-128, 128, (*lead, n, k // 2), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
    scale = torch.rand(*lead, n, k // GROUP if case["groups"] else 1, generator=g, device="cuda") * 8e-3 + 2e-3
    s["w_scale"] = scale if case["groups"] else scale.squeeze(-1)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def run(s):
    case = s["case"]
    return {"route": _route, "combine": _combine, "grouped": _grouped, "matvec": _matvec}[case["op"]](s, case)


def _route(s, case):
    if own:
        return _framework().route_experts(s["logits"], case["top"], case["scoring"], case["renorm"])
    T, E, k = case["tokens"], case["experts"], case["top"]
    v = s["logits"].float()
    best, ids = torch.sort(v, dim=-1, descending=True, stable=True)  # ties: the lowest index first
    best, ids = best[:, :k], ids[:, :k]
    chosen = best > -math.inf
    if case["scoring"] == "softmax":
        m = v.amax(-1, keepdim=True)
        p = torch.exp(v - m)
        weights = torch.exp(best - m) / p.sum(-1, keepdim=True)
    else:
        weights = 1 / (1 + torch.exp(-best))
    weights = torch.where(chosen, weights, torch.zeros_like(weights))
    if case["renorm"]:
        weights = torch.where(chosen, weights / weights.sum(-1, keepdim=True), torch.zeros_like(weights))
    ids = torch.where(chosen, ids, torch.full_like(ids, -1))
    key = torch.where(chosen, ids, torch.full_like(ids, E)).reshape(-1)
    order = torch.argsort(key, stable=True)
    counts = (key[:, None] == torch.arange(E, device="cuda")).sum(0)
    offsets = torch.cat((torch.zeros_like(counts[:1]), counts.cumsum(0)))
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device="cuda")
    pos = torch.where(chosen, place.reshape(T, k), torch.full_like(ids, -1))
    rows = torch.where(torch.arange(T * k, device="cuda") < offsets[-1], order // k, torch.full_like(order, -1))
    whole = [t.to(torch.int32) for t in (ids, offsets, rows, pos)]
    return whole[0], weights, whole[1], whole[2], whole[3]


def _combine(s, case):
    if own:
        return _framework().combine_experts(s["y"], s["weights"], s["pos"], s["residual"])
    taken = s["pos"] >= 0
    y = s["y"].float()[s["pos"].clamp(min=0).long()]
    out = (torch.where(taken, s["weights"], torch.zeros_like(s["weights"]))[..., None] * y).sum(1)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(DTYPES[case["dtype"]])


def _by_expert(x, w, offsets, cap):
    """[R, N] products of the rows with their experts' weights [E, N, K], the experts padded to `cap` rows each; zeros
    where a row has no expert."""
    R, E = x.shape[0], w.shape[0]
    r = torch.arange(R, device="cuda", dtype=torch.int32)
    e = torch.searchsorted(offsets[1:].contiguous(), r, right=True)
    slot = torch.where(e < E, e * cap + r - offsets[e.clamp(max=E)], E * cap).long()
    padded = torch.zeros(E * cap + 1, x.shape[1], device="cuda")
    padded[slot] = x
    y = torch.bmm(padded[:-1].reshape(E, cap, -1), w.transpose(1, 2)).reshape(E * cap, -1)
    return torch.cat((y, y.new_zeros(1, y.shape[1])))[slot], e


def _add_bias(y, bias, e):
    if bias is None:
        return y
    if e is None:
        return y + bias.float()
    padded = torch.cat((bias.float(), torch.zeros(1, bias.shape[1], device="cuda")))
    return y + padded[e]


def _grouped(s, case):
    if own:
        return _framework().gemm_w8a8_grouped(s["a"], s["a_scale"], s["w"], s["w_scale"], s["offsets"], s["a_rows"],
                                              s["bias"], DTYPES[case["dtype"]])
    a, scale = s["a"].float(), s["a_scale"]
    if s["a_rows"] is not None:
        a, scale = a[s["a_rows"].long()], scale[s["a_rows"].long()]
    y, e = _by_expert(a, s["w"].float(), s["offsets"], s["cap"])
    columns = torch.cat((s["w_scale"], torch.zeros(1, case["n"], device="cuda")))[e]
    return _add_bias(y * scale * columns, s["bias"], e).to(DTYPES[case["dtype"]])


def _matvec(s, case):
    if own:
        return _framework().matvec_w4(s["x"], s["w"], s["w_scale"], s["bias"], s["offsets"], s["a_rows"])
    low, high = s["w"] << 4 >> 4, s["w"] >> 4  # signed nibbles, the low one at the even k
    w = torch.stack((low, high), -1).flatten(-2).float()
    if case["groups"]:
        w = (w.unflatten(-1, (-1, GROUP)) * s["w_scale"][..., None]).flatten(-2)
    else:
        w = w * s["w_scale"][..., None]
    x, e = s["x"].float(), None
    if s["offsets"] is None:
        y = x @ w.T
    else:
        y, e = _by_expert(x if s["a_rows"] is None else x[s["a_rows"].long()], w, s["offsets"], s["cap"])
    return _add_bias(y, s["bias"], e).to(DTYPES[case["dtype"]])


# ---------------------------------------------------------------------------
# what a pass cannot do without, and its values in 64 bits
# ---------------------------------------------------------------------------


def work(case):
    size = SIZES[case["dtype"]]
    if case["op"] == "route":
        T, E, k = case["tokens"], case["experts"], case["top"]
        return {"bytes": T * E * size + 16 * T * k + 4 * (E + 1), "flops": 4 * T * E}
    if case["op"] == "combine":
        T, k, n = case["tokens"], case["top"], case["n"]
        rows = T * k if not case["dropped"] else T * k * (1 - 1 / case["dropped"])
        return {"bytes": (rows + T * (2 if case["residual"] else 1)) * n * size + 8 * T * k, "flops": 2 * rows * n}
    rows, n, k, E = case["rows"], case["n"], case["k"], case["experts"]
    total = rows + case["spare"]
    sources = max(1, total // 2) if case["gather"] else total
    active = sum(c > 0 for c in _counts(rows, E)) if E else 1
    out = total * n * size + (active * n * size if case["bias"] else 0) + (4 * total if case["gather"] else 0)
    if case["op"] == "grouped":
        return {"bytes": sources * (k + 4) + active * n * (k + 4) + 4 * (E + 1) + out, "flops": 2 * rows * n * k}
    scales = k // GROUP if case["groups"] else 1
    return {"bytes": sources * k * size + active * n * (k // 2 + 4 * scales) + out, "flops": 2 * rows * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "route":
        v, k = s["logits"].double(), case["top"]
        gates = torch.softmax(v, -1).nan_to_num(0.0) if case["scoring"] == "softmax" else torch.sigmoid(v)
        weights = gates.topk(k, -1).values
        if case["renorm"]:
            weights = (weights / weights.sum(-1, keepdim=True)).nan_to_num(0.0)
        return None, weights, None, None, None
    if case["op"] == "combine":
        T, n = case["tokens"], case["n"]
        out = s["residual"].double() if s["residual"] is not None else torch.zeros(T, n, dtype=torch.float64, device="cuda")
        for j in range(case["top"]):
            at = s["pos"][:, j].long()
            out += (s["weights"][:, j].double() * (at >= 0))[:, None] * s["y"][at.clamp(min=0)].double()
        return out
    x = s["a"].double() * s["a_scale"].double() if case["op"] == "grouped" else s["x"].double()
    x = x if s["a_rows"] is None else x[s["a_rows"].long()]
    bounds = [0, x.shape[0]] if s["offsets"] is None else s["offsets"].tolist()
    y = torch.zeros(x.shape[0], case["n"], dtype=torch.float64, device="cuda")
    for e in range(len(bounds) - 1):
        begin, end = bounds[e], bounds[e + 1]
        if begin == end:
            continue
        one = (lambda t: t) if s["offsets"] is None else (lambda t: t[e])  # noqa: B023 (used in this turn only)
        w, scale = one(s["w"]), one(s["w_scale"]).double()
        if case["op"] == "matvec":
            codes = w.int() & 255
            w = torch.empty(case["n"], case["k"], dtype=torch.float64, device="cuda")
            w[:, 0::2], w[:, 1::2] = (codes % 16 + 8) % 16 - 8, (codes // 16 + 8) % 16 - 8
            if case["groups"]:
                scale = scale.repeat_interleave(GROUP, -1)
        w = w.double() * (scale if scale.dim() == 2 else scale[:, None])
        y[begin:end] = x[begin:end] @ w.T
        if s["bias"] is not None:
            y[begin:end] += one(s["bias"]).double()
    return y
