"""Attention, rotary positions and layer norm run on tensors in memory: what traces a call or stands for a tensor is
refused before anything is allocated or launched (on the CPU; no case reaches a device)."""
import warnings

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from crack_detection_federatedlearning_grpc_amd import ops

BF = torch.bfloat16
POS = torch.zeros(1, 5, dtype=torch.int32)
CALLS = {
    "attention": (lambda t: ops.attention(t, t, t), (2, 5, 2, 32)),
    "attention_qkv": (lambda t: ops.attention_qkv(t, 2), (2, 5, 6, 32)),
    "layer_norm": (lambda t: ops.layer_norm(t), (6, 32)),
    "rotary": (lambda t: ops.rotary(t, POS, (32,)), (2, 5, 2, 32)),
}
TRACED = "cannot be traced"


@pytest.fixture(params=list(CALLS))
def call(request):
    f, shape = CALLS[request.param]
    return f, torch.zeros(shape, dtype=BF)


@pytest.mark.parametrize("grad", [False, True])
def test_jit_trace_is_refused(call, grad):
    f, x = call
    with warnings.catch_warnings(), pytest.raises(NotImplementedError, match=TRACED):
        warnings.simplefilter("ignore")
        torch.jit.trace(f, (x.requires_grad_(grad),))


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_make_fx_is_refused(call, mode):
    f, x = call
    with pytest.raises(NotImplementedError, match=TRACED):
        make_fx(f, tracing_mode=mode)(x)


def test_functional_tensors_are_refused(call):
    f, x = call
    with pytest.raises(NotImplementedError, match=TRACED):
        torch.func.functionalize(f)(x)


def test_fake_device_tensors_are_refused(call):
    """They pass for device tensors and have no address: inside their mode, and outside of it."""
    f, x = call
    with FakeTensorMode():
        fake = torch.empty(x.shape, dtype=BF, device="cuda")
        assert fake.is_cuda
        with pytest.raises(NotImplementedError, match=TRACED):
            f(fake)
        with pytest.raises(NotImplementedError, match=TRACED):
            f(x)
    with pytest.raises(NotImplementedError, match=TRACED):
        f(fake)


def test_other_arguments_that_are_fake_are_refused():
    with FakeTensorMode():
        mask = torch.ones(5, 5, dtype=torch.bool, device="cuda")
        lengths = torch.ones(2, dtype=torch.int32, device="cuda")
        w = torch.ones(32, device="cuda")
        pos = torch.ones(1, 5, device="cuda")
    q = torch.zeros(2, 5, 2, 32, dtype=BF)
    for f in (lambda: ops.attention(q, q, q, mask=mask), lambda: ops.attention(q, q, q, lengths=lengths),
              lambda: ops.layer_norm(q, w), lambda: ops.layer_norm(q, bias=w), lambda: ops.rotary(q, pos, (32,))):
        with pytest.raises(NotImplementedError, match=TRACED):
            f()


def test_zero_tensors_are_refused(call):
    f, x = call
    with pytest.raises(NotImplementedError, match=TRACED):
        f(torch._efficientzerotensor(x.shape, dtype=BF))


def test_modes_that_only_watch_are_no_tracing(call):
    """A dispatch mode that counts or saves calls lets the call through to its other checks."""
    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    f, x = call
    with Watch(), pytest.raises(RuntimeError, match="device tensor"):
        f(x)


def test_tangents_of_positions_are_refused():
    """A forward-mode derivative along the positions would be lost."""
    import torch.autograd.forward_ad as fwd
    x, pos = torch.zeros(2, 5, 4, 32, dtype=BF), torch.zeros(2, 5)
    with fwd.dual_level():
        dual = fwd.make_dual(pos, torch.ones_like(pos))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="positions have no gradient"):
                ops.rotary(x, dual, (16, 16))
