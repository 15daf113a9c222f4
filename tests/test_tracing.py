"""Whatever records or replaces PyTorch operators has to see a prepared object's ``run()`` as its operator: a recording
without it would give the results of the day it was made, whatever the inputs are by then."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from llm_gpu_kernels_b200 import _native
from tests.test_int8 import prepared_of_each_kind

gpu = pytest.mark.gpu


class FunctionMode(TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.seen.append(str(func))
        return func(*args, **(kwargs or {}))


class DispatchMode(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def answers(how):
    """What ``tracing()`` says while ``how`` runs a function of one tensor."""
    said = []

    def function(x):
        said.append(_native.tracing())
        return x * 2

    how(function, torch.ones(3))
    return said[0]


def under(mode):
    def how(f, x):
        with mode():
            f(x)
    return how


def test_recorders_are_noticed():
    assert answers(lambda f, x: torch.jit.trace(f, (x,), check_trace=False))
    for pre_dispatch in (False, True):
        assert answers(lambda f, x: make_fx(f, pre_dispatch=pre_dispatch)(x))
    assert answers(lambda f, x: make_fx(torch.func.functionalize(f))(x))
    assert answers(under(FunctionMode)) and answers(under(DispatchMode))
    assert answers(under(lambda: torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU])))


def test_nothing_else_is_taken_for_a_recorder():
    """Ordinary calls, for which the operator's dispatch would cost more than a small forward takes."""
    assert not answers(lambda f, x: f(x))
    for mode in (torch.no_grad, torch.inference_mode, torch.enable_grad, lambda: torch.autocast("cpu"),
                 lambda: torch.device("cpu"), lambda: torch.random.fork_rng(devices=[])):
        assert not answers(under(mode))


def change_inputs(dev):
    """(operator's name, run, result, change): ``change()`` puts other values into an input of that prepared object."""
    for name, run, result in prepared_of_each_kind(dev):
        owner = run.__self__
        base = getattr(owner, "base", owner)
        tensor = base.logits if name == "route" else base.x
        yield name, run, result, lambda tensor=tensor: tensor.neg_()


@gpu
@pytest.mark.parametrize("how", ["jit", "make_fx", "pre_dispatch"])
def test_a_recording_runs_the_kernels_again(how):
    dev = torch.device("cuda:0")
    one = torch.ones((), device=dev)
    for name, run, result, change in change_inputs(dev):
        def step(factor):
            run()
            return result * factor

        if how == "jit":
            recorded = torch.jit.trace(step, (one,), check_trace=False)
        else:
            recorded = make_fx(step, pre_dispatch=how == "pre_dispatch")(one)
        change()
        got = recorded(one).clone()
        result.zero_()
        run()
        assert torch.equal(got, result) and result.any(), name


@gpu
def test_function_modes_see_the_operators():
    dev = torch.device("cuda:0")
    for name, run, result in prepared_of_each_kind(dev):
        want = result.clone()
        result.zero_()
        mode = FunctionMode()
        with mode:
            run()
        assert any(f"b200moe.{name}" in seen for seen in mode.seen), (name, mode.seen)
        assert torch.equal(result, want)


@gpu
def test_profiles_name_the_operators():
    dev = torch.device("cuda:0")
    for name, run, _ in prepared_of_each_kind(dev):
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as profile:
            run()
        assert f"b200moe::{name}" in [event.key for event in profile.key_averages()]


@gpu
@pytest.mark.parametrize("what", ["x", "ids", "residual", "router_bias", "router_weight", "logits", "bias", "linear"])
def test_a_compiled_region_that_changes_an_input_runs_on_the_new_values(what):
    """Under a functionalising compiler the change is a new tensor, which reaches the bound one only after the region."""
    from llm_gpu_kernels_b200.int8_linear import prepare_int8_linear
    from llm_gpu_kernels_b200.moe import prepare_moe
    from llm_gpu_kernels_b200.moe_router import RouterConfig, prepare_routing
    from tests.test_int8 import layer_inputs
    dev = torch.device("cuda:0")
    x, gate_up, down, ids, rw = layer_inputs(20, 8, 2, 128, 64, "random", dev)
    plain = lambda w: w.dequantize().bfloat16()
    g = torch.Generator().manual_seed(3)
    if what in ("x", "ids", "residual"):
        residual = torch.randn(20, 128, generator=g).bfloat16().to(dev)
        prepared = prepare_moe(x, plain(gate_up), plain(down), ids, rw, residual=residual)
        changed = {"x": x, "ids": ids, "residual": residual}[what]
    elif what in ("router_bias", "router_weight"):
        weight = torch.randn(8, 128, generator=g).bfloat16().to(dev)
        bias = torch.zeros(8, device=dev)
        prepared = prepare_moe(x, plain(gate_up), plain(down), ids, rw, router_weight=weight, router_bias=bias,
                               router=RouterConfig(score="sigmoid"))
        changed = bias if what == "router_bias" else weight
    elif what in ("logits", "bias"):
        logits, bias = torch.randn(20, 8, generator=g).to(dev), torch.zeros(8, device=dev)
        prepared = prepare_routing(logits, 2, bias=bias)
        changed = logits if what == "logits" else bias
    else:
        from llm_gpu_kernels_b200.int8_weights import Int8Weight
        prepared = prepare_int8_linear(x, Int8Weight(gate_up.values[0], gate_up.scales[0]))
        changed = x
    first = lambda out: out[1] if isinstance(out, tuple) else out
    other = (torch.flip(changed, [0]) + 1) % 8 if what == "ids" else torch.linspace(
        -2, 2, changed.numel(), device=dev).view(changed.shape).to(changed.dtype)

    def step(new):
        changed.copy_(new)
        return first(prepared.run()) * 1

    before = first(prepared.run()).clone()
    got = torch.compile(step, fullgraph=True, backend="aot_eager")(other)
    assert torch.equal(changed, other)
    want = first(prepared.run())
    assert torch.equal(got, want) and not torch.equal(want, before)
