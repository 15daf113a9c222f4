"""The cases on which the routing and 8-bit integer operators are timed and compared with their plain forms.

Three operators:

* ``route``   - router logits to expert ids and weights: softmax or sigmoid scores, a balance bias that counts for the
  choice only, groups of experts, top-k, renormalised weights, a scale.
* ``linear``  - one matrix product in 8-bit integers: rows of x are quantised with a scale each (the largest magnitude
  becomes 127), the weight has a scale per output channel, the sums are integers.
* ``layer``   - the experts of a mixture-of-experts layer on given routes with such products: quantised x, gate and up
  product, SwiGLU, quantised again row by row, down product, weighted sum over a token's routes.

``own`` says which side ``run`` takes: the plain form below (elementary torch operations in 32 bits; the choice of
experts in 64 bits, where two scores may be next to each other) or the framework's operators.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def _route(tokens, experts, topk, score, dtype, *, bias=False, groups=1, kept=1, group_score="max", renormalize=True,
           scale=1.0, masked=0.0, name=None):
    case = {"op": "route", "tokens": tokens, "experts": experts, "topk": topk, "score": score, "dtype": dtype,
            "bias": bias, "groups": groups, "kept": kept, "group_score": group_score, "renormalize": renormalize,
            "scale": scale, "masked": masked}
    return case if name is None else dict(case, name=name)


def _linear(tokens, k, n, dtype, name=None):
    case = {"op": "linear", "tokens": tokens, "k": k, "n": n, "dtype": dtype}
    return case if name is None else dict(case, name=name)


def _layer(tokens, experts, topk, hidden, inter, routes, name=None):
    case = {"op": "layer", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "inter": inter,
            "routes": routes}
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # one token of a decode step, 256 experts in groups: launch latency is all of it
        _route(1, 256, 8, "sigmoid", "fp32", bias=True, groups=8, kept=4, group_score="top2", scale=2.5,
               name="route one token"),
        # a serving batch at the layer's headline size, plain softmax scores
        _route(1024, 128, 8, "softmax", "bf16", name="route batch"),
        # an odd batch with experts masked out (lost ranks, a row that may use none), groups of 20, raw weights
        _route(4099, 160, 6, "softmax", "fp16", bias=True, groups=8, kept=3, renormalize=False, scale=16.0, masked=0.05,
               name="route masked groups"),
        # a long prompt
        _route(32768, 256, 8, "sigmoid", "fp32", bias=True, groups=8, kept=4, group_score="top2", scale=2.5,
               name="route prompt"),
        # one token through a gate/up projection of the 2048 x 768 expert
        _linear(1, 2048, 1536, "bf16", name="linear one token"),
        # a serving batch: between streaming the weight and feeding the tensor cores
        _linear(193, 4096, 4096, "bf16", name="linear batch"),
        # nothing is a multiple of anything
        _linear(1021, 1999, 5003, "fp16", name="linear ragged"),
        # a prompt through a wide projection: the tensor cores bound it
        _linear(8192, 4096, 14336, "bf16", name="linear prompt"),
        # one decode step of the layer's headline shape: eight experts of 128 are read
        _layer(1, 128, 8, 2048, 768, "random", name="layer one token"),
        # an uneven batch over experts whose sizes are no multiple of a tile
        _layer(193, 60, 4, 2040, 1400, "skewed", name="layer ragged"),
        # the headline batch: every expert's weights are read once
        _layer(1024, 128, 8, 2048, 768, "random", name="layer batch"),
        # few large experts with many rows each
        _layer(2048, 8, 2, 4096, 14336, "random", name="layer large experts"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("route", "linear", "layer"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 3, 4, 8))
        experts = groups * _log(rng, max(2, 8 // groups), 256 // groups)
        kept = rng.randint(1, groups)
        topk = rng.randint(1, min(16, kept * (experts // groups)))
        return _route(_log(rng, 1, 32768), experts, topk, rng.choice(("softmax", "sigmoid")),
                      rng.choice(("bf16", "fp16", "fp32")), bias=rng.random() < 0.5, groups=groups, kept=kept,
                      group_score=rng.choice(("max", "top2")), renormalize=rng.random() < 0.7,
                      scale=rng.choice((1.0, 2.5, 16.0)), masked=rng.choice((0.0, 0.0, 0.05, 0.5)))
    if op == "linear":
        tokens, k = _log(rng, 1, 8192), _log(rng, 64, 8192)
        return _linear(tokens, k, _log(rng, 64, min(16384, 8192 * 4096 * 14336 // (tokens * k))),
                       rng.choice(("bf16", "fp16")))
    experts, hidden = _log(rng, 2, 128), _log(rng, 128, 4096)
    inter = _log(rng, 64, min(4096, 8 * 14336 * 4096 // (experts * hidden)))
    topk = rng.randint(1, min(8, experts))
    return _layer(_log(rng, 1, 4096 // topk), experts, topk, hidden, inter, rng.choice(("random", "skewed", "one")))


def work(case):
    t = case["tokens"]
    if case["op"] == "route":
        size = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": t * case["experts"] * size + (4 * case["experts"] if case["bias"] else 0) + t * case["topk"] * 8,
                "flops": 8 * t * case["experts"]}
    if case["op"] == "linear":
        k, n = case["k"], case["n"]
        return {"bytes": 2 * t * k + n * k + 4 * n + 2 * t * n, "flops": 2 * t * n * k}
    h, i, r = case["hidden"], case["inter"], t * case["topk"]
    # experts that a route reaches, from the distribution the routes are drawn from
    share = _popularity(case["experts"], case["routes"])
    used = sum(1.0 - (1.0 - min(1.0, p * case["topk"])) ** t for p in share)
    return {"bytes": used * (3 * h * i + 8 * i + 4 * h) + 4 * t * h + 8 * r, "flops": 6 * r * h * i}


def _popularity(experts, routes):
    if routes == "random":
        weight = [1.0] * experts
    elif routes == "skewed":
        weight = [1.0 / (e + 1) ** 1.2 for e in range(experts)]
    else:
        weight = [1.0] + [1e-9] * (experts - 1)
    total = sum(weight)
    return [w / total for w in weight]


# ------------------------------------------------------------------------------------------------ inputs
def _weight(g, experts, n, k, std):
    """Normal weights, quantised with one scale per output channel: int8 [experts, n, k] and float32 [experts, n]."""
    values = torch.empty(experts, n, k, dtype=torch.int8, device="cuda")
    scales = torch.empty(experts, n, dtype=torch.float32, device="cuda")
    for e in range(experts):
        w = torch.randn(n, k, generator=g, device="cuda").mul_(std)
        top = w.abs().amax(1, keepdim=True)
        scales[e] = top[:, 0] / 127
        values[e] = torch.round(w * 127 / top).to(torch.int8)
    return values, scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = {"case": case}
    t = case["tokens"]
    if case["op"] == "route":
        e = case["experts"]
        logits = torch.randn(t, e, generator=g, device="cuda") * 1.5
        if case["masked"]:
            u = torch.rand(t, e, generator=g, device="cuda")
            rows = torch.rand(t, 1, generator=g, device="cuda") < 1 / 64
            logits[(u < case["masked"]) | rows] = -math.inf
            logits[u < case["masked"] / 8] = math.nan
        state["logits"] = logits.to(DTYPES[case["dtype"]])
        state["bias"] = 0.1 * torch.randn(e, generator=g, device="cuda") if case["bias"] else None
        if own:
            from llm_gpu_kernels_b200.moe_router import RouterConfig, prepare_routing
            config = RouterConfig(score=case["score"], groups=case["groups"], kept_groups=case["kept"],
                                  group_score=case["group_score"], renormalize=case["renormalize"], scale=case["scale"])
            state["plan"] = prepare_routing(state["logits"], case["topk"], config=config, bias=state["bias"])
        return state
    if case["op"] == "linear":
        state["x"] = torch.randn(t, case["k"], generator=g, device="cuda").to(DTYPES[case["dtype"]])
        values, scales = _weight(g, 1, case["n"], case["k"], 0.02)
        state["values"], state["scales"] = values[0], scales[0]
        if own:
            from llm_gpu_kernels_b200.int8_linear import prepare_int8_linear
            from llm_gpu_kernels_b200.int8_weights import Int8Weight
            state["plan"] = prepare_int8_linear(state["x"], Int8Weight(state["values"], state["scales"]))
        return state
    e, k, h, i = case["experts"], case["topk"], case["hidden"], case["inter"]
    state["x"] = torch.randn(t, h, generator=g, device="cuda").to(torch.bfloat16)
    state["gate_up"] = _weight(g, e, 2 * i, h, 0.02)
    state["down"] = _weight(g, e, h, i, 0.02)
    popularity = torch.tensor(_popularity(e, case["routes"]), device="cuda")
    noise = -torch.log(-torch.log(torch.rand(t, e, generator=g, device="cuda").clamp(1e-9, 1 - 1e-6)))
    state["ids"] = torch.topk(torch.log(popularity) + noise, k, dim=1).indices.to(torch.int32)
    weights = torch.rand(t, k, generator=g, device="cuda") + 0.1
    state["weights"] = weights / weights.sum(1, keepdim=True)
    state["most"] = int(torch.bincount(state["ids"].flatten().long(), minlength=e).max())
    if own:
        from llm_gpu_kernels_b200.int8_weights import Int8Weight
        from llm_gpu_kernels_b200.moe_int8_cuda import prepare_int8_moe
        state["plan"] = prepare_int8_moe(state["x"], Int8Weight(*state["gate_up"]), Int8Weight(*state["down"]),
                                         state["ids"], state["weights"])
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return state["plan"].run()
    return {"route": _plain_route, "linear": _plain_linear, "layer": _plain_layer}[state["case"]["op"]](state)


def _plain_route(state):
    case = state["case"]
    l = state["logits"].double()
    out = torch.isnan(l) | (l == -math.inf)          # masked: never chosen while an unmasked expert is left
    l = torch.where(out, -math.inf, l)
    if case["score"] == "softmax":
        top = l.amax(1, keepdim=True)
        s = torch.exp(torch.where(out, -math.inf, l - torch.where(top == -math.inf, 0.0, top)))
        s = s / s.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        s = torch.where(out, 0.0, 1 / (1 + torch.exp(-l)))
    biased = state["bias"] is not None
    key = torch.where(out, -math.inf, s + state["bias"].double()) if biased else l   # scores grow with the logits
    if case["groups"] > 1:
        t, e, n = case["tokens"], case["experts"], case["groups"]
        if case["group_score"] == "max" or e == n:
            best = key.view(t, n, e // n).amax(2)
        else:
            ranked = torch.where(out, -math.inf, key if biased else s).view(t, n, e // n).sort(dim=2, descending=True).values
            best = ranked[:, :, 0] + torch.where(ranked[:, :, 1] == -math.inf, 0.0, ranked[:, :, 1])
        chosen = best.sort(dim=1, descending=True, stable=True).indices[:, :case["kept"]]
        kept = torch.zeros(t, n, dtype=torch.bool, device=l.device).scatter_(1, chosen, True)
        out = out | ~kept.repeat_interleave(e // n, 1)
        key = torch.where(out, -math.inf, key)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :case["topk"]]
    w = torch.where(out, 0.0, s).gather(1, ids)
    if case["renormalize"]:
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, 0.0)
    return ids.to(torch.int32), (w * case["scale"]).float()


def _quantised(x):
    """Rows as whole numbers in [-127, 127] (held in 32-bit floats) and their scales."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    q = torch.round(torch.where(top > 0, x * 127 / top, 0.0))
    return q, top / 127


def _plain_linear(state):
    q, scale = _quantised(state["x"])
    y = (q @ state["values"].float().T) * scale * state["scales"]
    return y.to(state["x"].dtype)


def _plain_layer(state):
    case = state["case"]
    e, k, i = case["experts"], case["topk"], case["inter"]
    q, scale = _quantised(state["x"])
    ids = state["ids"].flatten().long()
    (gate_up, gate_up_scale), (down, down_scale) = state["gate_up"], state["down"]
    if ids.numel() <= e:      # few routes: the weights of each route's expert
        rows, row_scale = q.repeat_interleave(k, 0)[:, None], scale.repeat_interleave(k, 0)[:, None]
        gate_up, gate_up_scale, down, down_scale = gate_up[ids], gate_up_scale[ids], down[ids], down_scale[ids]
        place = torch.arange(ids.numel(), device=ids.device)
    else:                     # the routes of each expert side by side, as many places as the busiest expert needs
        order = ids.argsort(stable=True)
        rank = torch.empty_like(ids)
        first = torch.searchsorted(ids[order], torch.arange(e, device=ids.device))
        rank[order] = torch.arange(ids.numel(), device=ids.device) - first[ids[order]]
        place = ids * state["most"] + rank
        rows = torch.zeros(e * state["most"], q.shape[1], device=q.device)
        rows[place] = q.repeat_interleave(k, 0)
        row_scale = torch.zeros(e * state["most"], 1, device=q.device)
        row_scale[place] = scale.repeat_interleave(k, 0)
        rows, row_scale = rows.view(e, -1, q.shape[1]), row_scale.view(e, -1, 1)
    both = torch.bmm(rows, gate_up.float().transpose(1, 2)) * row_scale * gate_up_scale[:, None]
    gate, up = both[..., :i], both[..., i:]
    a, a_scale = _quantised(gate / (1 + torch.exp(-gate)) * up)
    y = torch.bmm(a, down.float().transpose(1, 2)) * a_scale * down_scale[:, None]
    y = y.reshape(-1, y.shape[-1])[place].view(-1, k, y.shape[-1])
    return (y * state["weights"][..., None]).sum(1).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _exact_rows(x):
    x = x.to(torch.float64)
    top = x.abs().max(dim=-1).values
    q = (127.0 * x / top.clamp_min(1e-300).unsqueeze(-1)).round()
    return q, top / 127.0


def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "route":
        return _exact_route(case, state)
    if case["op"] == "linear":
        q, scale = _exact_rows(state["x"])
        return scale[:, None] * (q @ state["values"].to(torch.float64).t()) * state["scales"].to(torch.float64)
    q, scale = _exact_rows(state["x"])
    result = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
    i = case["inter"]
    for expert in range(case["experts"]):
        token, slot = torch.where(state["ids"] == expert)
        if token.numel() == 0:
            continue
        w1, s1 = (v[expert].to(torch.float64) for v in state["gate_up"])
        w2, s2 = (v[expert].to(torch.float64) for v in state["down"])
        gate = scale[token, None] * (q[token] @ w1[:i].t()) * s1[:i]
        up = scale[token, None] * (q[token] @ w1[i:].t()) * s1[i:]
        a, a_scale = _exact_rows(gate * torch.sigmoid(gate) * up)
        y = a_scale[:, None] * (a @ w2.t()) * s2
        result.index_add_(0, token, state["weights"][token, slot].to(torch.float64)[:, None] * y)
    return result


def _exact_route(case, state):
    x = state["logits"].to(torch.float64)
    usable = torch.isfinite(x)
    if case["score"] == "softmax":
        score = torch.softmax(x.masked_fill(~usable, -math.inf), 1).nan_to_num(0.0)
    else:
        score = torch.sigmoid(x.nan_to_num(0.0)) * usable
    bias = state["bias"]
    wanted = score + bias.to(torch.float64) if bias is not None else x
    wanted = wanted.masked_fill(~usable, -math.inf)
    if case["groups"] > 1:
        size = case["experts"] // case["groups"]
        in_group = wanted if bias is not None or case["group_score"] == "max" else score.masked_fill(~usable, -math.inf)
        take = 1 if case["group_score"] == "max" else min(2, size)
        most = in_group.unflatten(1, (case["groups"], size)).topk(take, dim=2).values
        value = most[..., 0] + most[..., 1:].masked_fill(most[..., 1:].isinf(), 0.0).sum(2)
        # the place of each group when they are ordered by value, the lower index first among equals
        before = (value[:, None, :] > value[:, :, None]) | ((value[:, None, :] == value[:, :, None]) & torch.ones(
            case["groups"], case["groups"], dtype=torch.bool, device=x.device).tril(-1))
        usable = usable & (before.sum(2) < case["kept"]).repeat_interleave(size, 1)
        wanted = wanted.masked_fill(~usable, -math.inf)
    ids = torch.argsort(wanted, dim=1, descending=True, stable=True)[:, :case["topk"]]
    weight = (score * usable).gather(1, ids)
    if case["renormalize"]:
        weight = (weight / weight.sum(1, keepdim=True)).nan_to_num(0.0)
    return ids, weight * case["scale"]
