"""8-bit operators under what records or transforms calls: torch.compile runs them as they are; traces, which would be run again without the launches, and values that memory does not hold are refused."""
import pytest
import torch

from .test_fp8 import F32, gen, gpu


def inputs():
    from jacobiforcing_amd import layer_ops as LO
    x, w = torch.randn(5, 512, generator=gen(1)).cuda(), torch.randn(512, 512, generator=gen(2)).cuda()
    return x, w, LO.fp8_weight(w)


def layer(LO, x, w8):
    half = LO.Fp8Weight(w8.data[:, :256], w8.scale[:, :2])
    h = LO.add_rmsnorm_fp8(x, x * 0.5, None, 1e-6)
    return LO.linear_fp8(LO.linear_gated_fp8(h, w8, 2), half) + LO.linear_fp8(LO.gated_act_fp8(x, 0, 256, 256, 2), half, x[0]) * 2 + LO.linear_fp8(LO.quantize_fp8(x), w8, None, F32).bfloat16()


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_compiled(native, monkeypatch):
    from jacobiforcing_amd import _native as N, layer_ops as LO
    x, w, w8 = inputs()
    if not native:
        monkeypatch.setattr(LO, "_H", N._NoHost())
    torch._dynamo.reset()
    with torch.no_grad():
        # (the backend that leaves the products and sums between the calls as they are: a fused one rounds them otherwise)
        want, got = layer(LO, x.clone(), w8), torch.compile(lambda x: layer(LO, x, w8), backend="eager")(x.clone())
        assert torch.equal(got, want)
        assert torch.equal(torch.compile(lambda w: LO.fp8_weight(w * 2).data.float(), backend="eager")(w), LO.fp8_weight(w * 2).data.float())
    torch._dynamo.reset()


def calls(LO, x, w8):
    x8 = LO.quantize_fp8(x)
    return (lambda t: LO.quantize_fp8(t).data.float(), lambda t: LO.add_rmsnorm_fp8(t, None, None, 1e-6).data.float(), lambda t: LO.add_rmsnorm_fp8(x.clone(), t, None, 1e-6).data.float(),
            lambda t: LO.add_rmsnorm_fp8(x.clone(), None, t[0], 1e-6).data.float(), lambda t: LO.gated_act_fp8(t, 0, 256, 256, 2).data.float(), lambda t: LO.fp8_weight(t).data.float(),
            lambda t: LO.linear_fp8(x8, w8, t[0]))


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_values_that_memory_does_not_hold(native, monkeypatch):
    from jacobiforcing_amd import _native as N, layer_ops as LO
    x, _, w8 = inputs()
    if not native:
        monkeypatch.setattr(LO, "_H", N._NoHost())
    for call in calls(LO, x, w8):
        lazy = torch._neg_view(x.clone())
        with torch.no_grad():
            with pytest.raises(ValueError, match="resolve_neg"):
                call(lazy)
            call(lazy.resolve_neg())
    a = torch.complex(x, x).conj().imag                 # every other float, besides
    with pytest.raises(ValueError):
        LO.quantize_fp8(a)
    with pytest.raises(ValueError, match="resolve_neg"):
        LO.linear_fp8(LO.Fp8Rows(LO.quantize_fp8(x, F32).data, torch._neg_view(LO.quantize_fp8(x, F32).scale)), LO.fp8_weight(torch.ones(128, 512, device="cuda"), F32))


@gpu
def test_traces():
    from torch.fx.experimental.proxy_tensor import make_fx
    from jacobiforcing_amd import layer_ops as LO
    x, _, w8 = inputs()
    x8 = LO.quantize_fp8(x)
    with torch.no_grad():
        for call in (*calls(LO, x, w8), lambda t: LO.linear_fp8(x8, w8) + t[0], lambda t: LO.linear_gated_fp8(x8, w8, 2).data.float() + t[0, 0]):
            with pytest.raises(ValueError, match="trace"):
                torch.jit.trace(call, (x.clone(),), check_trace=False)
            with pytest.raises(ValueError, match="trace"):
                make_fx(call)(x.clone())


@gpu
def test_modes_that_only_look_on():
    """Calls under a mode that neither records nor replaces tensors give what they give without."""
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode
    from jacobiforcing_amd import layer_ops as LO

    class Function(TorchFunctionMode):
        def __torch_function__(self, fn, types, args=(), kwargs=None):
            return fn(*args, **(kwargs or {}))

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, fn, types, args=(), kwargs=None):
            return fn(*args, **(kwargs or {}))

    x, _, w8 = inputs()
    with torch.no_grad():
        want = layer(LO, x.clone(), w8)
        for mode in (Function, Dispatch):
            with mode():
                got = layer(LO, x.clone(), w8)
            assert torch.equal(got, want), mode
