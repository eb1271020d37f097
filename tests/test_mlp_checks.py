"""What linear_act, layer_norm, the gradient norm and the clipped update check on the host, without a GPU."""
import pytest
import torch


def traced(call, x):
    """`call` under each tracer"""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    yield lambda: torch.jit.trace(call, x, check_trace=False)
    yield lambda: make_fx(call)(x)
    yield lambda: make_fx(call, tracing_mode="fake")(x)

    def fake():
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            call(mode.from_tensor(x))
    yield fake


def test_tracing_is_refused():
    """a trace would hold the result's allocation and not the launch that fills it"""
    from cinema_amd.models.inr_decoder import LatentRegressor
    from cinema_amd.models.mlp import LayerNorm, LinearAct, layer_norm, linear_act
    from cinema_amd.optim import grad_norm
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)

    def norm(x):
        p = torch.nn.Parameter(torch.zeros(4, 8))
        p.grad = x
        return grad_norm([p])
    for call in (lambda x: linear_act(x, w), lambda x: layer_norm(x), norm):
        for run in traced(call, x):
            with pytest.raises(NotImplementedError, match="traced"):
                run()
    for module in (LinearAct(8, 6), LayerNorm(8), LatentRegressor([8], precision="fp32")):
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(module, x, check_trace=False)
    with pytest.raises(RuntimeError, match="must live on the GPU"):            # outside a tracer: the check after it
        linear_act(x, w)
