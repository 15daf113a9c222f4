"""Routing to experts (``moe_router``): refusals and the oracle on the CPU, the kernels on a B200.

Ids have to equal those of the 64-bit oracle: the operator promises the choice of exact arithmetic. Weights are FP32
results of exp, a sum and a division or two. Their error is at most: expf 2 ulp (2^-22) in each score; the argument
l - max is rounded by 2^-24 |l - max|, at most 2^-24 * 32 = 2^-19 for the logits here (|l| < 16, less than 32 apart);
a sum of up to 256 scores 13 half-ulps, again 2^-20; two divisions and the scale 3 half-ulps. Together below
2^-18.3; RELATIVE is 2^-18.
"""
import ctypes
import math

import pytest
import torch

from llm_gpu_kernels_b200 import _native
from llm_gpu_kernels_b200.moe_router import RouterConfig, prepare_routing
from oracle import routing_oracle as R

RELATIVE = 2.0 ** -18
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("kw", [dict(score="relu"), dict(group_score="sum"), dict(groups=0), dict(groups=33),
                                dict(groups=4, kept_groups=5), dict(groups=4, kept_groups=0), dict(scale=0.0),
                                dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan)])
def test_config_refuses(kw):
    with pytest.raises(ValueError):
        RouterConfig(**kw)


@pytest.mark.parametrize("experts,topk,kw", [(10, 2, dict(groups=4)), (16, 0, {}), (16, 17, {}), (64, 33, {}),
                                             (16, 5, dict(groups=4, kept_groups=1))])
def test_config_refuses_choice(experts, topk, kw):
    with pytest.raises(ValueError):
        RouterConfig(**kw).check(experts, topk)


def test_prepare_refuses_host_tensors():
    with pytest.raises(ValueError, match="CUDA BF16/FP16/FP32 logits"):
        prepare_routing(torch.zeros(4, 8), 2)


def native_args(**kw):
    fields = dict(tokens=4, experts=16, topk=2, dtype=_native.FP32, pitch=16, logits=0x10000, ids=0x20000,
                  weights=0x30000)
    config = dict(score=0, groups=1, kept_groups=1, group_score=0, renormalize=1, scale=1.0)
    for name, value in kw.items():
        (config if name in config else fields)[name] = value
    return _native.RouteArgs(config=_native.RouterConfig(**config), **fields)


@pytest.mark.parametrize("kw", [
    dict(tokens=-1), dict(experts=0), dict(experts=257, pitch=257), dict(topk=0), dict(topk=17), dict(dtype=3),
    dict(pitch=15), dict(logits=None), dict(ids=None), dict(weights=None), dict(logits=0x10002), dict(ids=0x20002),
    dict(ids=0x20004, ids_are_int64=1), dict(weights=0x30001), dict(bias=0x40002), dict(score=2), dict(groups=3),
    dict(groups=0), dict(groups=4, kept_groups=5), dict(group_score=2), dict(scale=0.0), dict(scale=math.inf),
    dict(scale=math.nan), dict(groups=4, kept_groups=1, topk=5), dict(tokens=2 ** 31 - 1, topk=2)])
def test_library_refuses_before_any_launch(kw):
    assert _native.load().b200moe_route(ctypes.byref(native_args(**kw)), None) == _native.ERR_INVALID
    assert _native.last_error()


def test_library_accepts_no_tokens():
    assert _native.load().b200moe_route(ctypes.byref(native_args(tokens=0, logits=None)), None) == 0


def plan_code(**router):
    config = dict(score=0, groups=1, kept_groups=1, group_score=0, renormalize=1, scale=1.0)
    config.update(router)
    shape = _native.Shape(tokens=17, experts=128, topk=8, hidden=2048, intermediate=768, use_router=2,
                          router=_native.RouterConfig(**config))
    handle = ctypes.c_void_p()
    lib = _native.load()
    code = lib.b200moe_plan_create(ctypes.byref(shape), ctypes.byref(handle))
    if code == 0:
        lib.b200moe_plan_destroy(handle)
    return code


def test_plan_takes_a_configured_router():
    assert plan_code() == 0 and plan_code(score=1, groups=8, kept_groups=4, group_score=1, scale=2.5) == 0
    for bad in (dict(score=5), dict(groups=3), dict(groups=64, kept_groups=1), dict(groups=32, kept_groups=1),
                dict(scale=0.0)):
        assert plan_code(**bad) == _native.ERR_INVALID, bad


def test_oracle_by_hand():
    ids, w = R.route_row([0.0, 2.0, 1.0, 2.0], 2, renormalize=True)
    assert ids == [1, 3] and w == [0.5, 0.5]
    ids, w = R.route_row([0.0, 2.0, 1.0, 2.0], 3, score="sigmoid", bias=[1.0, 0.0, 0.0, 0.0], renormalize=False)
    assert ids == [0, 1, 3] and w[0] == 0.5                                 # the bias chooses, the score weighs
    ids, w = R.route_row([3.0, 0.0, 1.0, 1.0], 2, groups=2, kept_groups=1, group_score="top2", score="sigmoid")
    assert ids == [2, 3] and w == [0.5, 0.5]                                # 0.95 + 0.5 < 2 * 0.73
    ids, w = R.route_row([-math.inf, math.nan, 1.0, -math.inf], 3)
    assert ids == [2, 0, 1] and w == [1.0, 0.0, 0.0]
    assert R.route_row([-math.inf] * 4, 2) == ([0, 1], [0.0, 0.0])


# ------------------------------------------------------------------------------------------------ GPU
def agree(ids, weights, logits, topk, bias=None, **config):
    want_ids, want = R.route(logits.cpu(), topk, bias=bias.cpu() if bias is not None else None, **config)
    assert ids.cpu().tolist() == want_ids
    want = torch.tensor(want, dtype=torch.float64).reshape(weights.shape)
    got = weights.cpu().double()
    # subnormal results lose bits that a relative bound does not see
    assert torch.all((got - want).abs() <= RELATIVE * want.abs() + 2.0 ** -126), (got - want).abs().max()


def make_logits(tokens, experts, dtype, seed, dev, masked=0.0):
    g = torch.Generator().manual_seed(seed)
    logits = (1.5 * torch.randn(tokens, experts, generator=g)).clamp(-15.9, 15.9)
    if masked:
        u = torch.rand(tokens, experts, generator=g)
        logits[u < masked] = -math.inf
        logits[u < masked / 3] = math.nan
        logits[tokens // 2] = -math.inf            # a row whose mask leaves nothing
        logits[tokens // 3] = math.nan
    return logits.to(dtype).to(dev)


CASES = [
    # tokens, experts, topk, dtype, masked, bias, config
    (1, 1, 1, torch.float32, 0, False, {}),
    (5, 3, 2, torch.float32, 0, False, dict(score="sigmoid")),
    (33, 8, 2, torch.bfloat16, 0, False, {}),
    (70, 32, 32, torch.float16, 0, True, {}),
    (31, 33, 5, torch.float32, 0.3, True, dict(score="sigmoid", renormalize=False, scale=2.5)),
    (129, 64, 6, torch.bfloat16, 0, True, dict(score="sigmoid")),
    (40, 65, 8, torch.float32, 0, False, dict(renormalize=False)),
    (257, 128, 8, torch.bfloat16, 0, False, {}),
    (64, 128, 8, torch.float32, 0.9, True, {}),
    (50, 255, 12, torch.float16, 0.1, False, dict(score="sigmoid", scale=16.0)),
    (200, 256, 8, torch.float32, 0, True, dict(score="sigmoid", groups=8, kept_groups=4, group_score="top2", scale=2.5)),
    (90, 256, 8, torch.bfloat16, 0, False, dict(score="sigmoid", groups=8, kept_groups=4, group_score="top2")),
    (77, 160, 6, torch.float16, 0.05, True, dict(groups=8, kept_groups=3, renormalize=False, scale=16.0)),
    (60, 160, 6, torch.float32, 0.5, False, dict(groups=8, kept_groups=2, group_score="top2")),
    (48, 24, 3, torch.float32, 0, True, dict(groups=3, kept_groups=2, group_score="top2")),
    (48, 32, 4, torch.float32, 0.2, True, dict(groups=32, kept_groups=7, group_score="top2", score="sigmoid")),
    (48, 96, 4, torch.bfloat16, 0, False, dict(groups=2, kept_groups=1)),
    (30, 252, 9, torch.float32, 0, True, dict(groups=28, kept_groups=5, score="sigmoid")),
    (20, 250, 32, torch.float32, 0.4, True, dict(groups=10, kept_groups=2, group_score="top2")),
]


@gpu
@pytest.mark.parametrize("tokens,experts,topk,dtype,masked,biased,config", CASES)
def test_route_matches_64_bits(dev, tokens, experts, topk, dtype, masked, biased, config):
    logits = make_logits(tokens, experts, dtype, 3 * tokens + experts, dev, masked)
    bias = (0.1 * torch.randn(experts, generator=torch.Generator().manual_seed(7))).to(dev) if biased else None
    p = prepare_routing(logits, topk, config=RouterConfig(**config), bias=bias,
                        id_dtype=torch.int64 if tokens % 2 else torch.int32)
    p.ids.fill_(-7)
    p.routing_weights.fill_(math.nan)
    ids, weights = p.run()
    agree(ids, weights, logits, topk, bias, **config)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_closer_than_fp32(dev, score):
    """Selection scores 1e-8 and less apart: FP32 scores would tie or swap; the choice has to be the exact one."""
    g = torch.Generator().manual_seed(11)
    base = torch.randn(64, 1, generator=g)
    logits = (base + 1e-7 * torch.randn(64, 96, generator=g)).to(dev)
    bias = (1e-8 * torch.randn(96, generator=g)).to(dev)
    p = prepare_routing(logits, 8, config=RouterConfig(score=score), bias=bias)
    agree(p.ids, p.routing_weights, logits, 8, bias, score=score)
    config = dict(score=score, groups=8, kept_groups=3, group_score="top2")
    for b in (bias, None):
        p = prepare_routing(logits, 8, config=RouterConfig(**config), bias=b)
        agree(p.ids, p.routing_weights, logits, 8, b, **config)


@gpu
@pytest.mark.parametrize("experts,topk,config", [
    (128, 8, dict(groups=4, kept_groups=1)), (256, 32, dict(score="sigmoid")), (64, 8, {}), (16, 4, {}), (32, 32, {}),
    (160, 6, dict(groups=8, kept_groups=2, group_score="top2", renormalize=False)), (57, 16, dict(score="sigmoid"))])
@pytest.mark.parametrize("dtype,biased", [(torch.float32, True), (torch.bfloat16, False)])
def test_rows_with_fewer_experts_than_slots(dev, experts, topk, config, dtype, biased):
    g = torch.Generator().manual_seed(experts * topk)
    logits = make_logits(200, experts, torch.float32, 17, torch.device("cpu"))
    left = torch.randint(0, topk + 3, (200, 1), generator=g)      # experts that the mask leaves
    logits[torch.rand(200, experts, generator=g).argsort(-1).argsort(-1) >= left] = -math.inf
    logits = logits.to(dtype).to(dev)
    bias = (0.1 * torch.randn(experts, generator=g)).to(dev) if biased else None
    p = prepare_routing(logits, topk, config=RouterConfig(**config), bias=bias)
    agree(p.ids, p.routing_weights, logits, topk, bias, **config)


@gpu
@pytest.mark.parametrize("groups,size,topk,kept", [(4, 57, 8, 2), (3, 13, 4, 1), (8, 19, 8, 4), (2, 45, 16, 1), (3, 70, 6, 2),
                                                   (5, 31, 7, 3), (7, 9, 5, 2), (3, 40, 12, 2), (16, 5, 4, 3), (2, 1, 1, 1),
                                                   (32, 3, 2, 9), (3, 85, 32, 2), (6, 21, 10, 5), (2, 127, 9, 1)])
@pytest.mark.parametrize("masked,biased,score,group_score,dtype", [
    (0, True, "sigmoid", "top2", torch.float32), (0.5, False, "softmax", "top2", torch.bfloat16),
    (0.2, True, "softmax", "max", torch.float16), (0, False, "sigmoid", "max", torch.float32)])
def test_groups_of_any_size(dev, groups, size, topk, kept, masked, biased, score, group_score, dtype):
    experts = groups * size
    logits = make_logits(70, experts, dtype, 5 * experts + topk, dev, masked)
    bias = (0.1 * torch.randn(experts, generator=torch.Generator().manual_seed(3))).to(dev) if biased else None
    config = dict(score=score, groups=groups, kept_groups=kept, group_score=group_score)
    p = prepare_routing(logits, topk, config=RouterConfig(**config), bias=bias)
    agree(p.ids, p.routing_weights, logits, topk, bias, **config)
    wide = torch.zeros(70, experts + 5, dtype=dtype, device=dev)   # rows at any address
    wide[:, 3:3 + experts] = logits
    q = prepare_routing(wide[:, 3:3 + experts], topk, config=RouterConfig(**config), bias=bias)
    assert torch.equal(q.ids, p.ids) and torch.equal(q.routing_weights, p.routing_weights)


@gpu
@pytest.mark.parametrize("experts,topk,biased,config", [
    (256, 8, True, dict(score="sigmoid", groups=8, kept_groups=4, group_score="top2")),
    (256, 8, True, dict(score="sigmoid", groups=8, kept_groups=3)),
    (256, 8, False, dict(score="sigmoid", groups=8, kept_groups=4, group_score="top2")),
    (160, 6, True, dict(groups=8, kept_groups=3, renormalize=False)),
    (160, 6, False, dict(groups=8, kept_groups=2, group_score="top2")),
    (128, 8, True, dict(groups=4, kept_groups=2, group_score="top2")),
    (256, 8, True, {}), (128, 16, True, dict(score="sigmoid")), (64, 6, True, {}), (32, 4, True, dict(score="sigmoid")),
    (64, 8, False, {}), (200, 7, False, dict(score="sigmoid")), (16, 15, True, {}), (8, 8, True, dict(score="sigmoid")),
])
def test_a_few_close_choices(dev, experts, topk, biased, config):
    """Rows in which two or three experts, or two groups, are closer than FP32 can tell and the others are not."""
    g = torch.Generator().manual_seed(experts + topk)
    rows, groups = 240, config.get("groups", 1)
    size = experts // groups
    logits = (1.5 * torch.randn(rows, experts, generator=g)).double()
    bias = 0.1 * torch.randn(size, generator=g).repeat(groups) if biased else None
    score = torch.sigmoid if config.get("score") == "sigmoid" else lambda x: torch.softmax(x, -1)
    nudge = lambda: float(torch.randint(-2, 3, (1,), generator=g)) * 2.0 ** -24
    for r in range(rows):
        if r % 3 == 0 and groups > 1:            # two groups alike but for the last bits
            a, b = torch.randperm(groups, generator=g)[:2].tolist()
            logits[r, b * size:(b + 1) * size] = logits[r, a * size:(a + 1) * size]
            top = b * size + int(logits[r, b * size:(b + 1) * size].argmax())
            logits[r, top] += nudge() * abs(logits[r, top])
        if r % 3 != 1:
            continue
        c = score(logits[r]) + bias if biased else logits[r]
        order = c.argsort(descending=True)
        at = int(torch.randint(0, min(topk + 1, experts - 1), (1,), generator=g))
        for other in order[at + 1:at + 2 + r % 2].tolist():   # raised until it is level with the one at place `at`
            first = int(order[at])
            if not biased:
                logits[r, other] = logits[r, first] * (1 + nudge())
                continue
            low, high = -30.0, 30.0
            for _ in range(60):
                middle = (low + high) / 2
                trial = logits[r].clone()
                trial[other] = middle
                s = score(trial)
                if s[other] + bias[other] < s[first] + bias[first]:
                    low = middle
                else:
                    high = middle
            if -20 < low < 20:
                logits[r, other] = low * (1 + nudge())
    logits = logits.float().to(dev)
    bias = bias.to(dev) if biased else None
    p = prepare_routing(logits, topk, config=RouterConfig(**config), bias=bias)
    agree(p.ids, p.routing_weights, logits, topk, bias, **config)


@gpu
def test_ties_go_to_the_lower_index(dev):
    logits = torch.zeros(3, 64, device=dev)
    for bias in (None, torch.zeros(64, device=dev)):
        for groups in (1, 4):
            p = prepare_routing(logits, 5, config=RouterConfig(groups=groups, kept_groups=1), bias=bias)
            assert p.ids.tolist() == [[0, 1, 2, 3, 4]] * 3
            assert torch.allclose(p.routing_weights, torch.full((3, 5), 0.2, device=dev), rtol=RELATIVE, atol=0)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("config", [{}, dict(score="sigmoid"), dict(groups=8, kept_groups=3),
                                    dict(groups=8, kept_groups=3, group_score="top2"), dict(groups=3, kept_groups=2)])
def test_zeros_of_both_signs_tie(dev, dtype, config):
    g = torch.Generator().manual_seed(13)
    experts = 96 if config.get("groups") == 3 else 64
    logits = torch.where(torch.rand(50, experts, generator=g) < 0.5, -0.0, 0.0)
    logits[25:] = torch.where(torch.rand(25, experts, generator=g) < 0.8, logits[25:], -1.0 - torch.rand(25, experts, generator=g))
    logits = logits.to(dtype).to(dev)
    p = prepare_routing(logits, 6, config=RouterConfig(**config))
    agree(p.ids, p.routing_weights, logits, 6, **config)


@gpu
def test_extreme_logits(dev):
    """Infinities, the type's lowest value as a mask, and scores that leave the range of FP32."""
    inf, low = math.inf, torch.finfo(torch.float32).min
    rows = [[inf, 1.0, inf, 0.0], [low, low, 1.0, 0.5], [low, low, low, low], [-100.0, -101.0, -102.0, -103.0],
            [-800.0, -801.0, -802.0, -803.0], [3e38, -3e38, 0.0, 1.0], [1e-45, 0.0, -1e-45, 2e-45]]
    logits = torch.tensor(rows, device=dev)
    for score in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            for bias in (None, torch.tensor([0.5, -0.5, 0.25, 1e30], device=dev)):
                config = dict(score=score, renormalize=renormalize)
                p = prepare_routing(logits, 2, config=RouterConfig(**config), bias=bias)
                agree(p.ids, p.routing_weights, logits, 2, bias, **config)
    # a masked bias takes an expert out of the choice, not out of the softmax
    bias = torch.tensor([0.0, -inf, math.nan, 0.0], device=dev)
    logits = torch.tensor([[0.0, 5.0, 5.0, 1.0]], device=dev)
    p = prepare_routing(logits, 3, config=RouterConfig(renormalize=False), bias=bias)
    agree(p.ids, p.routing_weights, logits, 3, bias, renormalize=False)
    assert p.ids.tolist() == [[3, 0, 1]]


@gpu
def test_strided_rows_and_given_outputs(dev):
    wide = torch.randn(37, 300, device=dev)
    guard = torch.full((40, 6), -5, dtype=torch.int32, device=dev)
    for first in (0, 1, 4):
        logits = wide[:, first:first + 130]
        ids = guard[1:38]
        weights = torch.full((37, 6), math.nan, device=dev)
        p = prepare_routing(logits, 6, ids=ids, routing_weights=weights)
        assert p.ids is ids and p.routing_weights is weights
        agree(ids, weights, logits, 6)
        assert (guard[0] == -5).all() and (guard[38:] == -5).all()
    for tokens in (0, 1):
        p = prepare_routing(wide[:tokens, :130], 6)
        assert tuple(p.ids.shape) == (tokens, 6)


@gpu
def test_prepare_refuses(dev):
    logits = torch.zeros(4, 16, device=dev)
    ids, w = torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.zeros(4, 2, device=dev)
    bad = [
        dict(logits=logits.double()), dict(logits=logits.t()), dict(logits=logits[0]), dict(logits=logits[:1].expand(4, 16)),
        dict(logits=torch.zeros(4, 257, device=dev)), dict(topk=17), dict(topk=0), dict(bias=torch.zeros(16)),
        dict(bias=torch.zeros(15, device=dev)), dict(bias=torch.zeros(16, device=dev, dtype=torch.bfloat16)),
        dict(ids=ids[:3]), dict(ids=ids.float()), dict(routing_weights=w.double()), dict(id_dtype=torch.int16),
        dict(routing_weights=logits.view(-1)[:8].view(4, 2)), dict(config=RouterConfig(groups=3)),
    ]
    for kw in bad:
        args = dict(logits=logits, topk=2)
        args.update(kw)
        with pytest.raises(ValueError):
            prepare_routing(**args)
    with pytest.raises(TypeError):
        prepare_routing(logits, 2, config={"score": "softmax"})


@gpu
def test_route_captured_replayed_and_on_another_stream(dev):
    logits = make_logits(300, 256, torch.float32, 5, dev)
    bias = torch.zeros(256, device=dev)
    config = dict(score="sigmoid", groups=8, kept_groups=4, group_score="top2")
    p = prepare_routing(logits, 8, config=RouterConfig(**config), bias=bias)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.run()
    for seed in (21, 22):
        logits.copy_(make_logits(300, 256, torch.float32, seed, dev))
        bias.copy_(0.1 * torch.randn(256, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        agree(p.ids, p.routing_weights, logits, 8, bias, **config)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        logits.copy_(make_logits(300, 256, torch.float32, 23, dev))
        p.run()
    side.synchronize()
    agree(p.ids, p.routing_weights, logits, 8, bias, **config)


@gpu
def test_route_traces(dev):
    logits = make_logits(40, 64, torch.bfloat16, 9, dev)
    p = prepare_routing(logits, 4, config=RouterConfig(score="sigmoid", renormalize=False, scale=2.0))
    want = (p.ids.clone(), p.routing_weights.clone())

    def layer(scale):
        ids, weights = p.run()
        return ids, weights * scale

    p.ids.zero_()
    ids, weights = torch.compile(layer, fullgraph=True, backend="aot_eager")(torch.tensor(2.0, device=dev))
    assert torch.equal(ids, want[0]) and torch.equal(weights, 2 * want[1])


# ---- the router inside a prepared layer
LAYERS = [
    # tokens, experts, topk, hidden, inter, schedule, bias, config
    (1, 16, 2, 128, 64, "tcgen05", True, dict(score="sigmoid", groups=4, kept_groups=2, group_score="top2", scale=2.5)),
    (150, 128, 8, 256, 64, "tcgen05", True, dict(score="sigmoid")),
    (130, 256, 8, 512, 64, "tcgen05", True, dict(score="sigmoid", groups=8, kept_groups=4, group_score="top2")),
    (300, 60, 4, 256, 64, "tcgen05", False, dict(renormalize=False)),
    (40, 40, 3, 67, 33, "generic", True, dict(score="sigmoid", groups=5, kept_groups=2, scale=0.5)),
    (9, 7, 2, 67, 33, "generic", False, dict(score="sigmoid")),
    (2500, 32, 2, 128, 64, "tcgen05", True, dict(groups=4, kept_groups=2)),
    (64, 152, 8, 128, 64, "tcgen05", True, dict(score="sigmoid", groups=8, kept_groups=3, group_score="top2")),
    (40, 225, 6, 128, 64, "tcgen05", True, dict(groups=3, kept_groups=2)),
    (33, 39, 3, 67, 33, "generic", False, dict(groups=3, kept_groups=2)),
]


def exact_layer_logits(tokens, experts, hidden, seed):
    """x and router weight whose logits are exact in FP32 whatever the order of the sum (small multiples of 1/64), and
    distinct enough that the choice does not hang on rounding."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-8, 9, (tokens, hidden), generator=g).float() / 8
    wr = torch.randint(-8, 9, (experts, hidden), generator=g).float() / 32
    return x.bfloat16(), wr.bfloat16()


@gpu
@pytest.mark.parametrize("t,e,k,h,i,schedule,biased,config", LAYERS)
def test_configured_router_in_a_layer(dev, t, e, k, h, i, schedule, biased, config):
    from llm_gpu_kernels_b200.moe import prepare_moe
    from oracle import moe_oracle as O
    x, wr = exact_layer_logits(t, e, h, 3 * t + e)
    g = torch.Generator().manual_seed(1)
    gate_up = (0.05 * torch.randn(e, 2 * i, h, generator=g)).bfloat16()
    down = (0.05 * torch.randn(e, h, i, generator=g)).bfloat16()
    bias = 0.1 * torch.randn(e, generator=g) if biased else None
    ids = torch.zeros(t, k, dtype=torch.int64 if t % 2 else torch.int32, device=dev)
    rw = torch.zeros(t, k, device=dev)
    p = prepare_moe(x.to(dev), gate_up.to(dev), down.to(dev), ids, rw, router_weight=wr.to(dev), schedule=schedule,
                    router=RouterConfig(**config), router_bias=bias.to(dev) if biased else None)
    out = p.run()
    p.check_inputs()
    logits = x.double() @ wr.double().T
    want_ids, want = R.route(logits, k, bias=bias, **config)
    assert ids.cpu().tolist() == want_ids
    want = torch.tensor(want, dtype=torch.float64)
    assert torch.all((rw.cpu().double() - want).abs() <= RELATIVE * want.abs() + 2.0 ** -126)
    m = O.error_metrics(out.float().cpu(), O.moe_oracle(x, gate_up, down, ids.cpu(), rw.cpu()))
    assert m["finite"] and m["relative_rms"] <= 5e-3, m


@gpu
def test_layer_refuses_router_without_weight(dev):
    from llm_gpu_kernels_b200.moe import prepare_moe
    x, wr = exact_layer_logits(4, 8, 128, 1)
    gate_up, down = torch.zeros(8, 128, 128, device=dev).bfloat16(), torch.zeros(8, 128, 64, device=dev).bfloat16()
    ids, rw = torch.zeros(4, 2, dtype=torch.int32, device=dev), torch.zeros(4, 2, device=dev)
    x, wr = x.to(dev), wr.to(dev)
    for kw in (dict(router=RouterConfig()), dict(router_bias=torch.zeros(8, device=dev)),
               dict(router_weight=wr, router=RouterConfig(groups=3)),
               dict(router_weight=wr, router=RouterConfig(groups=8, kept_groups=1)),
               dict(router_weight=wr, router_bias=torch.zeros(7, device=dev))):
        with pytest.raises(ValueError):
            prepare_moe(x, gate_up, down, ids, rw, **kw)
    with pytest.raises(TypeError):
        prepare_moe(x, gate_up, down, ids, rw, router_weight=wr, router="sigmoid")


@gpu
def test_routing_feeds_a_layer(dev):
    """Logits a program has already: the routing writes the tensors that the prepared layer takes as its routes."""
    from llm_gpu_kernels_b200.moe import prepare_moe
    t, e, k, h, i = 50, 16, 3, 128, 64
    x, wr = exact_layer_logits(t, e, h, 4)
    g = torch.Generator().manual_seed(1)
    gate_up = (0.05 * torch.randn(e, 2 * i, h, generator=g)).bfloat16().to(dev)
    down = (0.05 * torch.randn(e, h, i, generator=g)).bfloat16().to(dev)
    x, wr = x.to(dev), wr.to(dev)
    config = RouterConfig(score="sigmoid", groups=4, kept_groups=2)
    routing = prepare_routing((x.float() @ wr.float().T), k, config=config)
    layer = prepare_moe(x, gate_up, down, routing.ids, routing.routing_weights)
    ids, rw = torch.zeros(t, k, dtype=torch.int32, device=dev), torch.zeros(t, k, device=dev)
    whole = prepare_moe(x, gate_up, down, ids, rw, router_weight=wr, router=config)
    routing.ids.zero_()
    routing.run()
    assert torch.equal(layer.run(), whole.run())
    assert torch.equal(routing.ids, ids) and torch.equal(routing.routing_weights, rw)


def _one_rank(rank, port, score):
    """A configured router in both expert-parallel layers on one rank, against the layer on one GPU."""
    import os
    import torch.distributed as dist
    from llm_gpu_kernels_b200.moe_ep import prepare_ep_moe, prepare_peer_ep_moe
    from llm_gpu_kernels_b200.moe_ranked import prepare_ranked_moe_launcher
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), NCCL_NVLS_ENABLE="0")
    torch.cuda.set_device(0)
    dev = torch.device("cuda", 0)
    dist.init_process_group("nccl", rank=0, world_size=1, device_id=dev)
    try:
        t, e, k, h, i = 50, 16, 4, 128, 64
        g = torch.Generator().manual_seed(5)
        draw = lambda *shape: (torch.randn(*shape, generator=g) * 0.1).bfloat16().to(dev)
        x, wr, gate_up, down = draw(t, h), draw(e, h), draw(e, 2 * i, h), draw(e, h, i)
        how = dict(router_weight=wr, router=RouterConfig(score=score, groups=4, kept_groups=2, scale=2.5),
                   router_bias=torch.linspace(-0.2, 0.2, e, device=dev))
        routes = lambda: (torch.zeros(t, k, dtype=torch.int32, device=dev), torch.zeros(t, k, device=dev))
        ids, weights = routes()
        ep = prepare_ep_moe(x, gate_up, down, ids, weights, experts=e, **how)
        tile = ep.backend.expert_plan
        ids1, weights1 = routes()
        single = prepare_ranked_moe_launcher(x, gate_up, down, ids1, weights1, token_tile=tile.token_tile,
                                             down_tiles=tile.down_tiles, **how)
        expected = single.run()
        out = ep.run()
        assert torch.equal(ids, ids1) and torch.equal(weights, weights1) and torch.equal(out, expected)
        ids2, weights2 = routes()
        peer = prepare_peer_ep_moe(x, gate_up, down, ids2, weights2, experts=e, **how)
        try:
            out = peer.run()
            torch.cuda.synchronize()
            peer.check_inputs()
            assert torch.equal(ids2, ids1) and torch.equal(weights2, weights1) and torch.equal(out, expected)
        finally:
            peer.close()
    finally:
        dist.destroy_process_group()


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_configured_router_expert_parallel(score):
    torch.multiprocessing.spawn(_one_rank, args=(29747, score), nprocs=1, join=True)


def test_expert_side_has_no_router(monkeypatch):
    """Only the plan that owns the tokens routes: the plan of the local experts gets no router arguments."""
    from types import SimpleNamespace
    from llm_gpu_kernels_b200 import moe_ep
    calls = []
    monkeypatch.setattr(moe_ep, "_prepare", lambda *args, **kw: calls.append(kw) or SimpleNamespace())
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    how = dict(router_weight=torch.zeros(8, 64), router=RouterConfig(score="sigmoid"), router_bias=torch.zeros(8))
    moe_ep.CudaBackend(x, torch.zeros(8, 128, 64), torch.zeros(8, 64, 64), torch.zeros(4, 2), torch.zeros(4, 2),
                       experts=8, capacity=8, global_routes=8, **how)
    token, expert = calls
    assert all(token[name] is value for name, value in how.items())
    assert not any(name in expert and expert[name] is not None for name in how)


# ---- finite masks: the lowest value of a type and others that stand for "not this one"
FINITE_MASKS = [torch.finfo(torch.float32).min, -1e31, -1.0000001e30, -1e30, -1e29, -1e9]
MASKED_GROUPS = [
    # groups, size, kept, topk
    (2, 4, 1, 2), (8, 4, 3, 6), (8, 32, 4, 8), (4, 57, 2, 8), (3, 13, 1, 4), (16, 5, 4, 3), (32, 2, 9, 4), (3, 70, 2, 6)]


def few_left(rows, groups, size, mask, g):
    """[rows, groups * size] factors of a mask: each group keeps none, one, two or all of its experts."""
    left = torch.tensor([0, 1, 1, 2, size])[torch.randint(0, 5, (rows, groups, 1), generator=g)]
    out = torch.rand(rows, groups, size, generator=g).argsort(-1).argsort(-1) >= left
    return out.view(rows, groups * size)


@gpu
@pytest.mark.parametrize("groups,size,kept,topk", MASKED_GROUPS)
@pytest.mark.parametrize("mask", FINITE_MASKS)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_finite_masks_in_groups(dev, groups, size, kept, topk, mask, score):
    """A masked expert counts with the value it has, not with that of the worst one that is left."""
    g = torch.Generator().manual_seed(groups * size + kept)
    experts = groups * size
    logits = make_logits(90, experts, torch.float32, experts + kept, torch.device("cpu"))
    out = few_left(90, groups, size, mask, g)
    logits[:60][out[:60]] = mask
    logits[50:60] = torch.where(out[50:60], mask, 0.1)            # all that is left is alike
    logits[40:50] = torch.where(out[40:50], 2 * torch.tensor(mask), logits[40:50])   # -inf for the lowest value
    logits = logits.to(dev)
    bias = 0.1 * torch.randn(experts, generator=g)
    for b in (None, bias, torch.where(out[0], mask, bias), torch.where(out[1], mask, bias)):
        b = b.to(dev) if b is not None else None
        for group_score in ("top2", "max"):
            config = dict(score=score, groups=groups, kept_groups=kept, group_score=group_score)
            p = prepare_routing(logits, topk, config=RouterConfig(**config), bias=b)
            agree(p.ids, p.routing_weights, logits, topk, b, **config)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["top2", "max"])
def test_values_as_low_as_masks_in_groups(dev, score, group_score):
    """Ordinary values among which some lie near -1e30: two of them add up to less than one and a mask."""
    g = torch.Generator().manual_seed(19)
    values = torch.tensor([0.5, -9e29, -6e29, -4e29, -1e29, -1e30, -1.2e30, -1.9e30, -3e38, -1e38, 1e30, 2.5])
    logits = values[torch.randint(0, 12, (400, 32), generator=g)]
    bias = values[torch.randint(0, 11, (32,), generator=g)]
    for groups, kept in ((8, 3), (16, 5), (4, 2)):
        config = dict(score=score, groups=groups, kept_groups=kept, group_score=group_score)
        for l, b in ((logits, None), (logits, bias), (torch.randn(400, 32, generator=g), bias)):
            l, b = l.to(dev), b.to(dev) if b is not None else None
            p = prepare_routing(l, 4, config=RouterConfig(**config), bias=b)
            agree(p.ids, p.routing_weights, l, 4, b, **config)


@gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("pairs", [1, 4])
def test_groups_next_to_each_other(dev, score, dtype, pairs):
    """Two groups of two experts whose sums of scores differ by a few millionths, logits of both signs."""
    g = torch.Generator().manual_seed(31 + pairs)
    two = (1.5 * torch.randn(200000, 2, generator=g)).to(dtype)
    worth = (torch.exp(two.double()) if score == "softmax" else torch.sigmoid(two.double())).sum(1)
    two = two[worth.argsort()[2000:198000]]
    at = torch.randint(0, two.shape[0] - 1, (6000,), generator=g)
    groups = torch.stack([two[at], two[at + 1]], 1)                                  # [rows, group, expert]
    groups = torch.where(torch.rand(6000, 1, 1, generator=g) < 0.5, groups, groups.flip(1))
    if pairs > 1:                                                                    # among groups that are far below
        rest = torch.full((6000, 2 * pairs - 2, 2), -9.0, dtype=dtype)
        groups = torch.cat([rest[:, :pairs], groups, rest[:, pairs:]], 1)
    logits = groups.reshape(6000, -1).to(dev)
    config = dict(score=score, groups=2 * pairs, kept_groups=1, group_score="top2")
    p = prepare_routing(logits, 2, config=RouterConfig(**config))
    agree(p.ids, p.routing_weights, logits, 2, **config)


@gpu
@pytest.mark.parametrize("config", [{}, dict(score="sigmoid", groups=4, kept_groups=2, scale=2.5), dict(renormalize=False)])
def test_library_rounds_weights_to_bf16(dev, config):
    """A form that only the C entry has; inside a layer it is ``router_bf16_weights``."""
    logits = make_logits(60, 64, torch.float32, 29, dev)
    p = prepare_routing(logits, 6, config=RouterConfig(**config))
    ids, weights = torch.zeros_like(p.ids), torch.zeros_like(p.routing_weights)
    args = _native.RouteArgs.from_buffer_copy(p._args)
    args.config.bf16_weights, args.ids, args.weights = 1, ids.data_ptr(), weights.data_ptr()
    assert _native.load().b200moe_route(ctypes.byref(args), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(ids, p.ids) and torch.equal(weights, p.routing_weights.bfloat16().float())
