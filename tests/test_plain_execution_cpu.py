"""What makes a call go through the registered operators instead of past them (CPU)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

from dist_moe_b200._bf16 import _plain_execution
from dist_moe_b200._call import traced


def _seen(run):
    found = []
    run(lambda a: found.append(_plain_execution(a)) or a * 2, torch.ones(3))
    assert _plain_execution(torch.ones(3)) and found  # and nothing is left behind
    return not any(found)


class _Functions(TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class _Operators(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _under(mode):
    def run(f, x):
        with mode():
            f(x)

    return run


@pytest.mark.parametrize("run", [
    lambda f, x: make_fx(f)(x), lambda f, x: make_fx(f, tracing_mode="fake")(x), lambda f, x: make_fx(f, pre_dispatch=True)(x),
    lambda f, x: torch.jit.trace(f, (x,), check_trace=False), lambda f, x: torch.func.vmap(f)(x), lambda f, x: torch.func.jvp(f, (x,), (x,)),
    lambda f, x: f(FakeTensorMode().from_tensor(x)), _under(_Operators), _under(_Functions)])
def test_noticed(run):
    assert _seen(run)


@pytest.mark.parametrize("run", [_under(torch.no_grad), _under(torch.inference_mode), lambda f, x: f(torch.nn.Parameter(x)),
                                 _under(lambda: torch.device("cpu")),
                                 _under(lambda: torch.autocast("cpu", dtype=torch.bfloat16))])
def test_left_alone(run):
    assert not _seen(run)


def test_a_default_device_does_not_hide_another_mode():
    with torch.device("cpu"), _Functions():
        assert not _plain_execution(torch.ones(3))
    with _Functions(), torch.device("cpu"):
        assert not _plain_execution(torch.ones(3))
    torch.set_default_device("cpu")
    try:
        assert _plain_execution(torch.ones(3))
    finally:
        torch.set_default_device(None)


def test_tracers_are_told_from_other_modes():
    found = {}
    make_fx(lambda a: found.update(make_fx=traced()) or a * 2)(torch.ones(3))
    torch.jit.trace(lambda a: found.update(jit=traced()) or a * 2, (torch.ones(3),), check_trace=False)
    with _Operators(), _Functions():
        found["modes"] = traced()
    found["nothing"] = traced()
    assert found == {"make_fx": True, "jit": True, "modes": False, "nothing": False}
