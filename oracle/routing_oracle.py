"""Routing to experts in 64 bits, one row at a time in plain Python: the definition the routing operator is held to."""
import math


def route_row(logits, topk, *, score="softmax", bias=None, groups=1, kept_groups=None, group_score="max",
              renormalize=True, scale=1.0):
    """(ids, weights) of one row of Python floats."""
    experts = len(logits)
    kept_groups = groups if kept_groups is None else kept_groups
    seen = [e for e in range(experts) if logits[e] > -math.inf]               # false for NaN
    s = [0.0] * experts
    if score == "softmax" and seen:
        top = max(logits[e] for e in seen)
        part = {e: 1.0 if logits[e] == top else math.exp(logits[e] - top) for e in seen}
        for e in seen:
            s[e] = part[e] / math.fsum(part.values())
    elif score == "sigmoid":
        for e in seen:
            s[e] = 1 / (1 + math.exp(-logits[e])) if logits[e] > -700 else math.exp(logits[e])
    usable = [e for e in seen if bias is None or bias[e] > -math.inf]
    choice = {e: logits[e] if bias is None else s[e] + bias[e] for e in usable}
    if groups > 1:
        size = experts // groups
        worth = []
        for g in range(groups):
            inside = [s[e] if bias is None and group_score == "top2" else choice[e]
                      for e in usable if e // size == g]
            inside.sort(reverse=True)
            worth.append(-math.inf if not inside else inside[0] if group_score == "max" else sum(inside[:2]))
        order = sorted(range(groups), key=lambda g: (-worth[g], g))[:kept_groups]
        choice = {e: c for e, c in choice.items() if e // size in order}
    ids = sorted(choice, key=lambda e: (-choice[e], e))[:topk]
    weights = [s[e] for e in ids]
    rest = [e for e in range(experts) if e not in ids]
    while len(ids) < topk:
        ids.append(rest.pop(0))
        weights.append(0.0)
    total = math.fsum(weights)
    if renormalize:
        weights = [w / total if total > 0 else 0.0 for w in weights]
    return ids, [w * scale for w in weights]


def route(logits, topk, *, bias=None, **config):
    """Rows of a tensor [T, E]; returns lists of ids and weights."""
    bias = bias.double().tolist() if bias is not None else None
    rows = [route_row(row, topk, bias=bias, **config) for row in logits.double().tolist()]
    return [r[0] for r in rows], [r[1] for r in rows]
