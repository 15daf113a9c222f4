"""Products in 8-bit integers (``int8_linear``, ``moe_int8_cuda``): refusals on the CPU, the kernels on a B200.

Bounds. Quantised values have to equal the 64-bit oracle's. A product's sum is exact; float(sum), the row scale, the
product of the two scales and the last multiplication are four roundings of 2^-24, then one to the output type
(HALF[dtype], half a step): STEP(dtype) = HALF + 2^-21 relative, and half the smallest subnormal of FP16.
SwiGLU: gate and up carry four roundings each; silu passes an error of the gate on times at most 1 + |gate|; __expf is
within 2^-22 + |gate| 2^-23; an addition, a division and a product follow: (16 + 6 |gate|) 2^-24 in all.
"""
import ctypes
import math

import pytest
import torch

from llm_gpu_kernels_b200 import _native
from llm_gpu_kernels_b200.int8_linear import prepare_int8_linear
from llm_gpu_kernels_b200.int8_weights import MAX_K, Int8Weight, quantize_int8, row_pitch
from llm_gpu_kernels_b200.moe_int8_cuda import prepare_int8_moe
from llm_gpu_kernels_b200.moe_router import RouterConfig
from oracle import int8_oracle as Q
from oracle import moe_oracle as O
from oracle import routing_oracle as R
from tests.util import make_ids

gpu = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half the smallest subnormal


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def near(got, want, dtype):
    """got (rounded to dtype) against want in float64; NaN where NaN is due."""
    got, want = got.cpu().double(), want.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    limit = (HALF[dtype] + 2.0 ** -21) * want.abs() + TINY[dtype]
    bad = ok & ((got - want).abs() > limit)
    assert not bad.any(), (int(bad.sum()), got[bad][:4], want[bad][:4])


# ------------------------------------------------------------------------------------------------ CPU
def linear_code(**kw):
    fields = dict(tokens=4, k=64, n=32, dtype=_native.BF16)
    fields.update(kw)
    lib, handle = _native.load(), ctypes.c_void_p()
    code = lib.b200moe_linear_create(ctypes.byref(_native.LinearShape(**fields)), ctypes.byref(handle))
    return lib, code, handle


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(k=0), dict(k=MAX_K + 1), dict(n=0), dict(dtype=_native.FP32),
                                dict(dtype=7), dict(tokens=2 ** 31 - 1), dict(n=2 ** 31 - 1),
                                dict(tokens=2 ** 30, n=2 ** 30)])
def test_linear_create_refuses(kw):
    _, code, _ = linear_code(**kw)
    assert code == _native.ERR_INVALID and _native.last_error()


def test_linear_workspace_and_state():
    lib, code, handle = linear_code(tokens=5, k=67)
    assert code == 0
    w = _native.LinearWorkspace()
    assert lib.b200moe_linear_workspace(handle, ctypes.byref(w)) == 0
    assert (w.x_q, w.x_scale, w.status) == (5 * 80, 20, 4) and w.launches >= 1
    assert lib.b200moe_linear_forward(handle, None) == _native.ERR_STATE
    good = dict(x=0x10000, x_pitch=67, weight=0x20000, weight_scale=0x30000, output=0x40000, x_q=0x50000,
                x_scale=0x60000, status=0x70000)
    for bad in (dict(x=None), dict(weight=None), dict(output=None), dict(x_q=None), dict(status=None), dict(x_pitch=66),
                dict(weight=0x20008), dict(x_q=0x50008), dict(x=0x10001), dict(output=0x40001), dict(x_scale=0x60002),
                dict(weight_scale=0x30001), dict(status=0x70002), dict(output=0x10000), dict(x_q=0x20000)):
        assert lib.b200moe_linear_bind(handle, ctypes.byref(_native.LinearBuffers(**{**good, **bad}))) == _native.ERR_INVALID
    assert lib.b200moe_linear_forward(handle, None) == _native.ERR_STATE
    lib.b200moe_linear_destroy(handle)
    for name in ("create", "workspace", "bind", "forward"):
        args = (None, None)
        assert getattr(lib, f"b200moe_linear_{name}")(*args) == _native.ERR_INVALID


def plan_code(**kw):
    fields = dict(tokens=17, experts=128, topk=8, hidden=2048, intermediate=768, gate_up_format=_native.WEIGHTS_INT8,
                  down_format=_native.WEIGHTS_INT8)
    fields.update(kw)
    lib, handle = _native.load(), ctypes.c_void_p()
    code = lib.b200moe_plan_create(ctypes.byref(_native.Shape(**fields)), ctypes.byref(handle))
    ws = _native.Workspace()
    if code == 0:
        lib.b200moe_plan_workspace(handle, ctypes.byref(ws))
        lib.b200moe_plan_destroy(handle)
    return code, ws


def test_plan_formats():
    code, ws = plan_code()
    r = 17 * 8
    assert code == 0 and ws.gathers == 0 and ws.grouped_input == 0 and ws.source_rows == 0
    assert ws.activated == r * 768 * 4 and ws.x_q == r * 2048 and ws.x_scale == r * 4
    assert ws.activated_q == r * 768 and ws.activated_scale == r * 4 and ws.schedule == _native.SCHEDULE_TCGEN05
    code, ws = plan_code(hidden=67, intermediate=33)
    assert code == 0 and ws.x_q == r * 80 and ws.activated_q == r * 48
    assert plan_code(tokens=0)[0] == 0
    assert plan_code(down_format=_native.WEIGHTS_BF16)[0] == _native.ERR_INVALID
    assert plan_code(gate_up_format=_native.WEIGHTS_W4G128)[0] == _native.ERR_INVALID
    assert plan_code(gate_up_format=3, down_format=3)[0] == _native.ERR_INVALID
    assert plan_code(hidden=MAX_K + 1, tokens=1)[0] == _native.ERR_INVALID
    for kw in (dict(schedule=_native.SCHEDULE_GENERIC), dict(route_only=1), dict(external_dispatch=2)):
        assert plan_code(**kw)[0] == _native.ERR_UNSUPPORTED
    plain = plan_code(gate_up_format=0, down_format=0)[1]
    assert (plain.x_q, plain.x_scale, plain.activated_q, plain.activated_scale) == (0, 0, 0, 0)


def test_quantize_int8_weight():
    g = torch.Generator().manual_seed(0)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        w = torch.randn(3, 20, 67, generator=g).to(dtype)
        w[1, 4] = 0
        q = quantize_int8(w)
        want, scale = Q.quantize_rows(w)
        assert torch.equal(q.values.double(), want) and torch.equal(q.scales, scale.float())
        assert q.storage.shape == (3, 20, 80) and (q.storage[..., 67:] == 0).all()
        assert torch.equal(q.storage[..., :67], q.values)
        assert torch.equal(q.dequantize(), q.values.float() * q.scales[..., None])
        one = quantize_int8(w[0])
        assert torch.equal(one.values, q.values[0]) and torch.equal(one.scales, q.scales[0])
    aligned = quantize_int8(torch.randn(4, 64, generator=g))
    assert aligned.storage is aligned.values and row_pitch(64) == 64
    for value in (math.inf, math.nan):
        w = torch.zeros(2, 16)
        w[1, 3] = value
        with pytest.raises(ValueError):
            quantize_int8(w)


@pytest.mark.parametrize("values,scales", [
    (torch.zeros(4, 16), torch.zeros(4)), (torch.zeros(4, 16, dtype=torch.int8), torch.zeros(5)),
    (torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4).double()), (torch.zeros(4, dtype=torch.int8), torch.zeros(())),
    (torch.zeros(4, 0, dtype=torch.int8), torch.zeros(4)),
    (torch.zeros(1, MAX_K + 1, dtype=torch.int8), torch.zeros(1)),
    (torch.zeros(4, 16, dtype=torch.int8), torch.zeros(8)[::2])])
def test_int8_weight_refuses(values, scales):
    with pytest.raises(ValueError):
        Int8Weight(values, scales)


def test_prepare_refuses_host_tensors():
    w = quantize_int8(torch.ones(4, 64))
    with pytest.raises(ValueError, match="CUDA BF16/FP16"):
        prepare_int8_linear(torch.zeros(2, 64).bfloat16(), w)
    with pytest.raises(ValueError, match="CUDA device"):
        prepare_int8_moe(torch.zeros(2, 64).bfloat16(), quantize_int8(torch.ones(2, 128, 64)),
                         quantize_int8(torch.ones(2, 64, 64)), torch.zeros(2, 1), torch.zeros(2, 1))
    with pytest.raises(TypeError):
        prepare_int8_moe(torch.zeros(2, 64).bfloat16(), torch.ones(2, 128, 64), torch.ones(2, 64, 64), None, None)


# ------------------------------------------------------------------------------------------------ GPU: dense product
LINEAR = [
    (1, 1, 1, torch.bfloat16), (1, 64, 32, torch.float16), (2, 16, 257, torch.bfloat16), (3, 67, 5, torch.float16),
    (5, 2048, 1536, torch.bfloat16), (8, 100, 128, torch.bfloat16), (9, 129, 127, torch.float16),
    (16, 128, 256, torch.bfloat16), (17, 127, 255, torch.bfloat16), (31, 1000, 33, torch.float16),
    (64, 4096, 64, torch.bfloat16), (65, 1040, 511, torch.bfloat16), (128, 72, 1024, torch.bfloat16),
    (129, 15, 600, torch.float16), (300, 513, 700, torch.bfloat16), (1021, 640, 257, torch.float16),
    (2, 10000, 40, torch.bfloat16), (140, 8200, 300, torch.bfloat16), (700, 256, 2048, torch.bfloat16),
    (2049, 384, 520, torch.bfloat16),
]


def linear_inputs(t, k, n, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * t + k + n)
    x = torch.randn(t, k, generator=g).to(dtype)
    return x.to(dev), quantize_int8(0.05 * torch.randn(n, k, generator=g)).to(dev)


@gpu
@pytest.mark.parametrize("t,k,n,dtype", LINEAR)
def test_linear_matches_64_bits(dev, t, k, n, dtype):
    x, w = linear_inputs(t, k, n, dtype, dev)
    p = prepare_int8_linear(x, w)
    p.output.fill_(math.nan)
    p.x_q.fill_(77)
    out = p.run()
    p.check()
    near(out, Q.linear(x.cpu(), w.values.cpu(), w.scales.cpu()), dtype)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k", [(40, 72), (33, 1000), (7, 2048), (200, 6000), (3, 9001)])
def test_quantised_rows_are_exact(dev, dtype, t, k):
    """Quotients that are exactly a half (rows whose largest magnitude is 127 times a power of two, or 254), rows of tiny
    and of huge values, zeros, one value only."""
    g = torch.Generator().manual_seed(t + k)
    x = torch.randn(t, k, generator=g)
    x[1] = torch.randint(-254, 255, (k,), generator=g) / 2.0
    x[1, 0] = 127.0
    x[2] = torch.randint(-127, 128, (k,), generator=g).float()
    x[2, k - 1] = -254.0
    if t > 6:
        x[3] = 0
        x[4] = 0
        x[4, k // 2] = -3e-5
        x[5] *= torch.finfo(dtype).max / 8
        x[6] *= torch.finfo(dtype).smallest_normal
    if t > 30:
        x[7] = x[7].sign() * torch.finfo(dtype).tiny * 2.0 ** -6   # subnormals
        x[8] = -torch.finfo(dtype).max
        x[9] = torch.rand(k, generator=g) * 2.0 ** -7
    x = x.to(dtype).to(dev)
    w = quantize_int8(torch.ones(4, k)).to(dev)
    p = prepare_int8_linear(x, w)
    if p.kernel_launches == 1:   # one token: quantised inside the product
        pytest.skip("no quantised rows in memory")
    q, scale = Q.quantize_rows(x.cpu())
    assert torch.equal(p.x_q[:, :k].cpu().double(), q)
    assert (p.x_q[:, k:] == 0).all()
    assert torch.equal(p.x_scale.cpu(), (x.cpu().float().abs().amax(-1) / 127))


@gpu
@pytest.mark.parametrize("t", [1, 6, 40])
def test_rows_that_are_not_finite(dev, t):
    x, w = linear_inputs(t, 200, 70, torch.bfloat16, dev)
    x[t - 1, 199] = math.nan
    if t > 2:
        x[0, 0] = math.inf
        x[2, 50] = -math.inf
        x[2, 51] = math.nan
    out = prepare_int8_linear(x, w).output
    near(out, Q.linear(x.cpu(), w.values.cpu(), w.scales.cpu()), torch.bfloat16)
    assert torch.isnan(out[t - 1]).all()


@gpu
@pytest.mark.parametrize("t", [1, 20])
def test_largest_sum(dev, t):
    """K = 131072 with every product 127 * 127: the sum is just below 2^31."""
    x = torch.ones(t, MAX_K, dtype=torch.bfloat16, device=dev)
    x[t - 1] = -1
    values = torch.full((3, MAX_K), 127, dtype=torch.int8, device=dev)
    values[1] = -127
    w = Int8Weight(values, torch.full((3,), 2.0 ** -20, device=dev))
    near(prepare_int8_linear(x, w).output, Q.linear(x.cpu(), values.cpu(), w.scales.cpu()), torch.bfloat16)


@gpu
def test_linear_strides_and_guards(dev):
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(50, 300, generator=g).bfloat16().to(dev)
    w = quantize_int8(torch.randn(90, 130, generator=g)).to(dev)
    for t in (1, 4, 50):
        for first in (0, 1, 8):
            x = wide[:t, first:first + 130]
            guard = torch.full((t + 2, 90), 7.0, dtype=torch.bfloat16, device=dev)
            p = prepare_int8_linear(x, w, output=guard[1:t + 1])
            near(p.output, Q.linear(x.cpu(), w.values.cpu(), w.scales.cpu()), torch.bfloat16)
            assert (guard[0] == 7).all() and (guard[t + 1] == 7).all()
    assert prepare_int8_linear(wide[:0, :130], w).run().shape == (0, 90)
    # int8 values that are a slice of something wider
    values = torch.randint(-127, 128, (90, 200), dtype=torch.int8, device=dev)[:, 3:131]
    part = Int8Weight(values, w.scales)
    near(prepare_int8_linear(wide[:20, :128], part).output, Q.linear(wide[:20, :128].cpu(), values.cpu(), w.scales.cpu()),
         torch.bfloat16)


@gpu
def test_linear_refuses(dev):
    x, w = linear_inputs(6, 64, 32, torch.bfloat16, dev)
    out = torch.empty(6, 32, dtype=torch.bfloat16, device=dev)
    for args, kw in (((x.float(), w), {}), ((x[0], w), {}), ((x.t(), w), {}), ((x[:1].expand(6, 64), w), {}),
                     ((x[:, :63], w), {}), ((x, w.to("cpu")), {}), ((x, quantize_int8(torch.ones(1, 32, 64)).to(dev)), {}),
                     ((x, w), dict(output=out[:5])), ((x, w), dict(output=out.half())), ((x, w), dict(output=out.cpu())),
                     ((x, w), dict(output=x[:, :32])), ((x, w), dict(output=x.view(-1)[:192].view(6, 32)))):
        with pytest.raises(ValueError):
            prepare_int8_linear(*args, **kw)
    with pytest.raises(TypeError):
        prepare_int8_linear(x, torch.ones(32, 64, device=dev))


@gpu
@pytest.mark.parametrize("t", [1, 3, 200])
def test_linear_captured_streams_and_traced(dev, t):
    x, w = linear_inputs(t, 512, 300, torch.bfloat16, dev)
    p = prepare_int8_linear(x, w)
    other = prepare_int8_linear(x.clone(), w)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        p.run()
    for seed in (1, 2):
        x.copy_(torch.randn(t, 512, generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        near(p.output, Q.linear(x.cpu(), w.values.cpu(), w.scales.cpu()), torch.bfloat16)
    # two prepared products at the same time on two streams
    want = p.output.clone()
    other.x.copy_(x)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(a):
            p.run()
        with torch.cuda.stream(b):
            other.run()
    torch.cuda.synchronize()
    assert torch.equal(p.output, want) and torch.equal(other.output, want)
    p.output.zero_()
    got = torch.compile(lambda s: p.run() * s, fullgraph=True, backend="aot_eager")(torch.tensor(2.0, device=dev))
    assert torch.equal(got, want * 2)


# ------------------------------------------------------------------------------------------------ GPU: the layer
def layer_inputs(t, e, k, h, i, pattern, dev, seed=0, id_dtype=torch.int32):
    g = torch.Generator().manual_seed(seed + 3 * t + e + h)
    x = torch.randn(t, h, generator=g).bfloat16()
    gate_up = quantize_int8(0.05 * torch.randn(e, 2 * i, h, generator=g))
    down = quantize_int8(0.05 * torch.randn(e, h, i, generator=g))
    ids = make_ids(t, e, k, pattern, g).to(id_dtype)
    rw = torch.rand(t, k, generator=g)
    return x.to(dev), gate_up.to(dev), down.to(dev), ids.to(dev), rw.to(dev)


def check_layer(p, x, gate_up, down, ids, rw):
    """Each stage against 64 bits on what the stage before it wrote, then the whole against the definition."""
    base = p.base
    p.check_inputs()
    x, ids, rw = x.cpu(), ids.cpu().long(), rw.cpu()
    t, k = ids.shape
    e, h, inter = down.shape
    q, scale = Q.quantize_rows(x)
    counts, offsets, ranks, mapping = O.dispatch_oracle(ids, e)
    x_q = base.x_q[:, :x.shape[1]].cpu().double()
    valid = mapping >= 0      # the routes' rows in grouped order
    assert torch.equal(x_q[mapping[valid].long()], q.repeat_interleave(k, 0)[valid])
    assert torch.equal(base.mapping.cpu(), mapping) and torch.equal(base.counts.cpu(), counts)
    values, scales = gate_up.values.cpu().double(), gate_up.scales.cpu().double()
    dvalues, dscales = down.values.cpu().double(), down.scales.cpu().double()
    activated, a_q = base.activated.cpu().double(), base.activated_q.cpu()[:, :inter].double()
    a_scale, y = base.activated_scale.cpu().double(), base.down_output.cpu()
    for expert in range(e):
        lo, hi = int(offsets[expert]), int(offsets[expert] + counts[expert])
        if lo == hi:
            continue
        rows = torch.empty(hi - lo, dtype=torch.long)
        flat = torch.where(ids.flatten() == expert)[0]
        rows[mapping[flat].long() - lo] = flat // k
        both = (q[rows] @ values[expert].T) * scale[rows, None] * scales[expert]
        gate, up = both[:, :inter], both[:, inter:]
        want = Q.swiglu(gate, up)
        limit = (16 + 6 * gate.abs()) * 2.0 ** -24 * want.abs() + 2.0 ** -140
        assert torch.equal(torch.isnan(activated[lo:hi]), torch.isnan(want))
        assert not ((activated[lo:hi] - want).abs() > limit).any()
        want_q, want_s = Q.quantize_rows(activated[lo:hi])
        assert torch.equal(a_q[lo:hi], want_q)
        near(y[lo:hi], (a_q[lo:hi] @ dvalues[expert].T) * a_scale[lo:hi, None] * dscales[expert], torch.bfloat16)
        got_s = a_scale[lo:hi]
        assert torch.equal(torch.isnan(got_s), torch.isnan(want_s))
        assert not ((got_s - want_s).abs() > 2.0 ** -24 * want_s + 2.0 ** -149).any()
    # the combine: K products and sums in FP32, one rounding
    out = base.output.cpu().double()
    take = mapping.view(t, k).long()
    terms = torch.where((take >= 0)[..., None], y.double()[take.clamp_min(0)] * rw.double()[..., None], 0.0)
    want = terms.sum(1)
    limit = HALF[torch.bfloat16] * want.abs() + (2 * k + 1) * 2.0 ** -24 * terms.abs().sum(1) + TINY[torch.bfloat16]
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert not ((out - want).abs() > limit).any()
    # whole: two BF16 roundings (2^-8 each), and activated values that FP32 moves across a border of the 8-bit grid:
    # 2^-20 of a value is off, so at most one in 127 * 2^-20 / 0.01 moves by one of >= 0.01 of the row: below 1e-3
    exact = Q.layer(x, gate_up.values.cpu(), gate_up.scales.cpu(), down.values.cpu(), down.scales.cpu(), ids, rw)
    fine = ~torch.isnan(exact)
    off = torch.linalg.norm((out - exact)[fine]) / torch.linalg.norm(exact[fine]).clamp_min(1e-300)
    assert off <= 2 * 2.0 ** -8 + 1e-3, off


LAYER = [
    # tokens, experts, topk, hidden, inter, pattern, token tile
    (1, 1, 1, 16, 16, "random", 0), (1, 8, 2, 256, 128, "random", 0), (2, 3, 2, 67, 33, "random", 0),
    # one token of up to 8 routes and two of up to 2 without tensor cores, and the same with a pinned tile, which is with
    # them
    (1, 8, 2, 256, 128, "random", 16), (2, 3, 2, 67, 33, "random", 16), (1, 9, 9, 72, 40, "random", 0), (2, 9, 3, 72, 40, "random", 0),
    (1, 8, 8, 2100, 1030, "random", 0),
    (4, 4, 4, 520, 2050, "random", 0), (16, 16, 2, 24, 1, "random", 0), (31, 2, 1, 1, 40, "random", 0), (32, 4, 1, 40, 17, "all_hot", 0),
    (33, 4, 1, 40, 17, "all_hot", 0),
    (17, 16, 4, 128, 96, "random", 0), (40, 8, 2, 256, 128, "random", 16), (40, 8, 2, 256, 128, "all_hot", 0),
    (33, 5, 3, 200, 130, "last_hot", 32), (64, 4, 2, 520, 264, "random", 64), (130, 4, 4, 128, 384, "random", 128),
    (300, 2, 1, 384, 256, "random", 256), (97, 32, 4, 1000, 72, "hot", 0), (50, 64, 8, 72, 40, "duplicate", 0),
    (600, 6, 3, 136, 200, "random", 0), (900, 2, 2, 131, 72, "random", 0), (500, 1, 1, 264, 256, "random", 0), (500, 1, 1, 2048, 64, "random", 0),
    (400, 1, 1, 4100, 40, "random", 16), (1, 1, 1, 5000, 700, "random", 0), (5, 32, 4, 2048, 768, "random", 0), (1100, 3, 2, 256, 1100, "random", 0),
]


@gpu
@pytest.mark.parametrize("t,e,k,h,i,pattern,tile", LAYER)
def test_layer_matches_64_bits(dev, t, e, k, h, i, pattern, tile):
    args = layer_inputs(t, e, k, h, i, pattern, dev, id_dtype=torch.int64 if t % 2 else torch.int32)
    p = prepare_int8_moe(*args, token_tile=tile)
    p.base.output.fill_(math.nan)
    p.run()
    check_layer(p, *args)
    again = p.base.output.clone()
    assert torch.equal(p.run(), again)


@gpu
def test_layer_bad_rows_ids_and_weights(dev):
    x, gate_up, down, ids, rw = layer_inputs(24, 6, 2, 96, 80, "random", dev)
    x[3, 5] = math.nan
    x[7] = 0
    x[9, 0] = math.inf
    p = prepare_int8_moe(x, gate_up, down, ids, rw)
    check_layer(p, x, gate_up, down, ids, rw)
    out = p.run()
    assert torch.isnan(out[3]).all() and torch.isnan(out[9]).all() and (out[7] == 0).all()
    assert not torch.isnan(out[[0, 1, 2, 4, 5, 6, 8]]).any()
    ids[1, 0], ids[2, 1] = 6, -1
    out = p.run()
    with pytest.raises(ValueError, match="status=1"):
        p.check_inputs()
    one = rw.clone()
    one[1, 0] = one[2, 1] = 0
    exact = Q.layer(x[:3].cpu(), gate_up.values.cpu(), gate_up.scales.cpu(), down.values.cpu(), down.scales.cpu(),
                    ids[:3].cpu().long(), one[:3].cpu())
    assert torch.linalg.norm(out[:3].cpu().double() - exact) <= (2 * 2.0 ** -8 + 1e-3) * torch.linalg.norm(exact)
    assert prepare_int8_moe(x[:0], gate_up, down, ids[:0], rw[:0]).run().shape == (0, 96)


@gpu
def test_layer_residual_graph_stream(dev):
    x, gate_up, down, ids, rw = layer_inputs(90, 16, 4, 256, 192, "random", dev)
    residual = torch.randn(90, 256, device=dev).bfloat16()
    plain = prepare_int8_moe(x, gate_up, down, ids, rw)
    p = prepare_int8_moe(x, gate_up, down, ids, rw, residual=residual)
    assert torch.equal(p.run(), residual + plain.run())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        p.run()
    other = layer_inputs(90, 16, 4, 256, 192, "hot", dev, seed=5)
    for mine, new in ((x, other[0]), (ids, other[3]), (rw, other[4])):
        mine.copy_(new)
    graph.replay()
    torch.cuda.synchronize()
    got = p.base.output.clone()
    assert torch.equal(got, residual + plain.run())
    side = torch.cuda.Stream()
    p.base.output.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        p.run()
    side.synchronize()
    assert torch.equal(p.base.output, got)
    for launch in p.launches:   # the stages one by one
        launch.run()
    assert torch.equal(p.base.output, got)


@gpu
def test_layer_traces(dev):
    args = layer_inputs(20, 8, 2, 128, 64, "random", dev)
    p = prepare_int8_moe(*args)
    want = p.run().clone()
    p.base.output.zero_()
    got = torch.compile(lambda s: p.run() * s, fullgraph=True, backend="aot_eager")(torch.tensor(2.0, device=dev))
    assert torch.equal(got, want * 2)


@gpu
def test_layer_refuses(dev):
    x, gate_up, down, ids, rw = layer_inputs(4, 4, 2, 64, 32, "random", dev)
    for args in ((x, down, gate_up, ids, rw), (x[:, :48].contiguous(), gate_up, down, ids, rw), (x.half(), gate_up, down, ids, rw),
                 (x, gate_up, down, ids[:3], rw), (x, gate_up.to("cpu"), down, ids, rw), (x, gate_up, down, ids, rw.double())):
        with pytest.raises(ValueError):
            prepare_int8_moe(*args)
    for args in ((x, gate_up.values, down, ids, rw), (x, gate_up, down.values, ids, rw)):
        with pytest.raises(TypeError):
            prepare_int8_moe(*args)
    with pytest.raises(ValueError):
        prepare_int8_moe(x, gate_up, down, ids, rw, token_tile=48)
    from llm_gpu_kernels_b200.moe_ranked import prepare_ranked_moe_launcher
    plain = lambda w: w.dequantize().bfloat16()
    for args in ((x, gate_up, plain(down), ids, rw), (x, plain(gate_up), down, ids, rw)):
        with pytest.raises(TypeError, match="both be Int8Weight"):
            prepare_ranked_moe_launcher(*args)


@gpu
@pytest.mark.parametrize("t,h", [(1, 256), (60, 256), (300, 136), (20, 67)])
def test_router_experts_and_shared_product_together(dev, t, h):
    """A whole layer: sigmoid router with a bias and groups, experts in 8 bits, and a shared product of the same x added
    as the residual."""
    e, k, i = 32, 4, 96
    g = torch.Generator().manual_seed(t)
    x = (torch.randint(-8, 9, (t, h), generator=g).float() / 8).bfloat16()      # exact logits, as in the routing tests
    wr = (torch.randint(-8, 9, (e, h), generator=g).float() / 32).bfloat16()
    bias = 0.1 * torch.randn(e, generator=g)
    gate_up = quantize_int8(0.05 * torch.randn(e, 2 * i, h, generator=g))
    down = quantize_int8(0.05 * torch.randn(e, h, i, generator=g))
    shared = quantize_int8(0.05 * torch.randn(h, h, generator=g))
    config = dict(score="sigmoid", groups=8, kept_groups=3, group_score="top2", scale=2.5)
    ids, rw = torch.zeros(t, k, dtype=torch.int32, device=dev), torch.zeros(t, k, device=dev)
    xd = x.to(dev)
    side = prepare_int8_linear(xd, shared.to(dev))
    layer = prepare_int8_moe(xd, gate_up.to(dev), down.to(dev), ids, rw, router_weight=wr.to(dev),
                             router=RouterConfig(**config), router_bias=bias.to(dev), residual=side.output)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        side.run()
        layer.run()
    ids.zero_()
    graph.replay()
    torch.cuda.synchronize()
    layer.check_inputs()
    want_ids, want_w = R.route(x.double() @ wr.double().T, k, bias=bias, **config)
    assert ids.cpu().tolist() == want_ids
    exact = Q.linear(x, shared.values, shared.scales) + Q.layer(
        x, gate_up.values, gate_up.scales, down.values, down.scales, torch.tensor(want_ids),
        torch.tensor(want_w, dtype=torch.float64))
    # one more BF16 rounding than the layer alone: that of the shared product
    off = torch.linalg.norm(layer.base.output.cpu().double() - exact) / torch.linalg.norm(exact)
    assert off <= 4 * 2.0 ** -8 + 1e-3, off


# ---- what PyTorch learns of a run
def prepared_of_each_kind(dev):
    from llm_gpu_kernels_b200.moe_router import prepare_routing
    from llm_gpu_kernels_b200.moe_ranked import prepare_ranked_moe_launcher
    x, gate_up, down, ids, rw = layer_inputs(20, 8, 2, 128, 64, "random", dev)
    layer = prepare_int8_moe(x, gate_up, down, ids, rw)
    plain = prepare_ranked_moe_launcher(x, gate_up.dequantize().bfloat16(), down.dequantize().bfloat16(), ids, rw)
    linear = prepare_int8_linear(x, Int8Weight(gate_up.values[0], gate_up.scales[0]))
    routing = prepare_routing(torch.randn(20, 8, device=dev), 2)
    return [("forward", layer.run, layer.base.output), ("forward", plain.run, plain.base.output),
            ("int8_linear", linear.run, linear.output), ("route", routing.run, routing.routing_weights)]


@gpu
def test_run_counts_as_a_change_in_place(dev):
    """A result that autograd saved and a later run overwrote may not give a gradient in silence."""
    for name, run, result in prepared_of_each_kind(dev):
        run()
        factor = torch.ones(result.shape, device=dev, requires_grad=True, dtype=result.dtype)
        (result * factor).sum().backward()
        assert torch.equal(factor.grad, result), name
        loss = (result * factor).sum()
        run()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@gpu
def test_dispatch_modes_see_the_operators(dev):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    for name, run, result in prepared_of_each_kind(dev):
        want = result.clone()
        seen = []
        result.zero_()
        with Names():
            run()
        assert f"b200moe::{name}" in seen and torch.equal(result, want)


def test_expert_parallelism_refuses():
    from llm_gpu_kernels_b200.moe_ep import prepare_ep_moe, prepare_peer_ep_moe
    gate_up, down = quantize_int8(torch.ones(4, 64, 32)), quantize_int8(torch.ones(4, 32, 32))
    x, ids, rw = torch.ones(2, 32).bfloat16(), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, 2)
    for prepare in (prepare_ep_moe, prepare_peer_ep_moe):
        for weights in ((gate_up, down), (gate_up, torch.ones(4, 32, 32)), (torch.ones(4, 64, 32), down)):
            with pytest.raises(TypeError, match="not Int8Weight"):
                prepare(x, *weights, ids, rw, experts=4)


@pytest.mark.parametrize("shape", [(0, 4), (4, 0), (2, 0, 4), (2, 4, 0), (0, 4, 4)])
def test_quantize_int8_refuses_empty(shape):
    with pytest.raises(ValueError):
        quantize_int8(torch.zeros(shape))


# ---- precision and length of the layer
@gpu
@pytest.mark.parametrize("t,e,k,h,i,tile", [(1, 8, 8, 256, 128, 0), (1, 8, 2, 67, 33, 16), (2, 4, 2, 264, 70, 0), (40, 8, 2, 256, 128, 0),
                                            (33, 5, 3, 200, 130, 0), (300, 4, 4, 1030, 72, 0), (900, 2, 2, 384, 256, 256)])
def test_rows_are_rounded_once(dev, t, e, k, h, i, tile):
    """Down rows and their weighted sum stay in FP32; BF16 comes with the result. y: two scales and the sum, four
    roundings of 2^-24; the combine: K products and additions."""
    x, gate_up, down, ids, rw = layer_inputs(t, e, k, h, i, "random", dev, seed=4)
    p = prepare_int8_moe(x, gate_up, down, ids, rw, token_tile=tile)
    base = p.base
    assert base.down_output.dtype == torch.float32
    mapping = base.mapping.cpu().long().view(t, k)
    a = base.activated_q[:, :i].cpu().double()[mapping]            # [t, k, i]
    dvalues, dscales = down.values.cpu().double(), down.scales.cpu().double()
    ids = ids.cpu().long()
    y = torch.empty(t, k, h, dtype=torch.float64)
    for expert in range(e):
        at = ids == expert
        y[at] = (a[at] @ dvalues[expert].T) * dscales[expert]
    y *= base.activated_scale.cpu().double()[mapping][..., None]
    got = base.down_output.cpu().double()[mapping]
    assert not ((got - y).abs() > 2.0 ** -21 * y.abs()).any()
    terms = y * rw.cpu().double()[..., None]
    want, out = terms.sum(1), base.output.cpu().double()
    limit = HALF[torch.bfloat16] * want.abs() + (2.0 ** -21 + (k + 1) * 2.0 ** -24) * terms.abs().sum(1)
    assert not ((out - want).abs() > limit).any()


# ---- scales whose product leaves the range of FP32 though the result does not
def far_scales(t, k, n, dtype, g, exponents):
    """x whose row maxima are near 2^exponents[0], a weight whose channel scales are near 2^exponents[1], in pairs such
    that the results stay in the range of the type; and every third channel with a sum of zero."""
    x = torch.randn(t, k, generator=g).clamp(-4, 4)
    values = torch.randint(-127, 128, (n, k), dtype=torch.int8, generator=g)
    values[::3] = 0
    x, scales = x * 2.0 ** exponents[0], (1 + torch.rand(n, generator=g)) * 2.0 ** exponents[1]
    return x.to(dtype), values, scales


FAR = [   # BF16 rows (2^row) and channel scales (2^channel): products of the scales subnormal, zero or infinite in FP32
    (-115, -25), (-118, -18), (-100, -42), (-60, -85), (-110, -45), (118, 30), (120, 126), (100, 60), (-90, -36)]


@gpu
@pytest.mark.parametrize("row,channel", FAR)
@pytest.mark.parametrize("t,k,n", [(1, 600, 70), (2, 600, 70), (20, 600, 70), (20, 8192, 260), (130, 2048, 512), (300, 160, 129)])
def test_scales_far_apart(dev, t, k, n, row, channel):
    g = torch.Generator().manual_seed(t + k)
    x, values, scales = far_scales(t, k, n, torch.bfloat16, g, (row, channel))
    if row + channel > 100:
        values[:] = 0            # any other sum leaves BF16
        values[1, 0], values[1, 1] = 64, -64
        x[:, 1] = x[:, 0]        # ... and two that cancel
    if t > 2:
        x[t // 2] = 0
    want = Q.linear(x, values, scales)
    p = prepare_int8_linear(x.to(dev), Int8Weight(values.to(dev), scales.to(dev)))
    near(p.output, want, torch.bfloat16)
    assert row + channel > 100 or (want != 0).any()


@gpu
@pytest.mark.parametrize("t,e,k", [(1, 4, 2), (40, 4, 2), (300, 3, 1)])
@pytest.mark.parametrize("row,gate,up,down", [(-110, 117, -20, 30), (-110, 117, -14, -10), (110, -103, 30, 0)])
def test_layer_scales_far_apart(dev, t, e, k, row, gate, up, down):
    g = torch.Generator().manual_seed(t)
    h, i = 256, 128
    x = (torch.randn(t, h, generator=g).clamp(-4, 4) * 2.0 ** row).bfloat16()
    values = torch.randint(-127, 128, (e, 2 * i, h), dtype=torch.int8, generator=g)
    values[:, i + 5] = 0
    if up > 0:
        values[:, i:] = 0                        # any other sum leaves FP32
    scales = (1 + torch.rand(e, 2 * i, generator=g))
    scales[:, :i] *= 2.0 ** (gate - 17)          # sums of 256 products of two numbers up to 127 are some 2^17
    scales[:, i:] *= 2.0 ** up
    dvalues = torch.randint(-127, 128, (e, h, i), dtype=torch.int8, generator=g)
    dscales = (1 + torch.rand(e, h, generator=g)) * 2.0 ** down
    ids, rw = make_ids(t, e, k, "random", g).to(torch.int32), torch.rand(t, k, generator=g)
    args = (x.to(dev), Int8Weight(values.to(dev), scales.to(dev)), Int8Weight(dvalues.to(dev), dscales.to(dev)),
            ids.to(dev), rw.to(dev))
    check_layer(prepare_int8_moe(*args), *args)


# ---- the quantised rows of one or two tokens, which the product without tensor cores makes itself
@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,k", [(1, 72), (1, 1000), (1, 2048), (1, 9001), (1, 5), (2, 72), (2, 1000), (2, 2048), (2, 6000)])
def test_quantised_rows_of_a_few_tokens(dev, dtype, t, k):
    """Row by row the cases of test_quantised_rows_are_exact, in memory after a run and bit for bit what a batch gives."""
    g = torch.Generator().manual_seed(t + k)
    rows = torch.randn(10, k, generator=g)
    rows[1] = torch.randint(-254, 255, (k,), generator=g) / 2.0
    rows[1, 0] = 127.0
    rows[2] = torch.randint(-127, 128, (k,), generator=g).float()
    rows[2, k - 1] = -254.0
    rows[3] = 0
    rows[4] = 0
    rows[4, k // 2] = -3e-5
    rows[5] *= torch.finfo(dtype).max / 8
    rows[6] *= torch.finfo(dtype).smallest_normal
    rows[7] = rows[7].sign() * torch.finfo(dtype).tiny * 2.0 ** -6
    rows[8] = -torch.finfo(dtype).max
    rows[9] = torch.rand(k, generator=g) * 2.0 ** -7
    rows = rows.to(dtype).to(dev)
    w = quantize_int8(0.05 * torch.randn(70, k, generator=g)).to(dev)
    x = rows[:t].clone()
    p = prepare_int8_linear(x, w)
    assert p.kernel_launches == 1
    batch = prepare_int8_linear(rows, w)
    for first in range(0, 10, t):
        x.copy_(rows[first:first + t])
        p.x_q.fill_(77)
        p.x_scale.fill_(math.nan)
        out = p.run()
        q, _ = Q.quantize_rows(x.cpu())
        assert torch.equal(p.x_q[:, :k].cpu().double(), q) and (p.x_q[:, k:] == 0).all()
        assert torch.equal(p.x_scale.cpu(), x.cpu().float().abs().amax(-1) / 127)
        assert torch.equal(out, batch.output[first:first + t])
    x[t - 1, k // 2] = math.inf
    p.run()
    assert torch.isnan(p.x_scale[t - 1]) and (p.x_q[t - 1] == 0).all()


@gpu
@pytest.mark.parametrize("t,e,k,h,i,pattern", [(2100, 128, 8, 72, 40, "random"), (5000, 16, 4, 96, 33, "hot"), (17000, 3, 1, 40, 24, "random"),
                                               (2049, 256, 8, 48, 16, "duplicate")])
def test_layer_with_many_routes(dev, t, e, k, h, i, pattern):
    """More routes than one launch of the dispatch ranks (16384): it takes three kernels and writes no rows."""
    args = layer_inputs(t, e, k, h, i, pattern, dev, id_dtype=torch.int64 if t % 2 else torch.int32)
    p = prepare_int8_moe(*args)
    p.base.output.fill_(math.nan)
    p.run()
    check_layer(p, *args)
