"""What linear_act, layer_norm, the gradient norm and the clipped update check on the host, without a GPU."""
import ctypes

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


def test_clipping_tells_shared_memory_from_interleaved():
    """gradients that share a value are refused, however they are strided; neighbours in one table are not (they are refused one
    check later here, for being on the CPU)"""
    from cinema_amd import _lib
    from cinema_amd.optim import clip_grad_norm_, grad_norm
    t = torch.ones(8, 12)
    line = torch.ones(100)
    cube = torch.ones(4, 6, 5)
    for a, b in [(t, t.t()), (t[:, :6], t[:, 5:]), (t[:, :6].t(), t[:, 3:9].t()), (t[::2], t[2]), (t[:, 3], t[4]), (line[::2], line[4:9]),
                 (line[:50], line[::7]), (line[::2], line[::3]), (cube[:, :3, :4], cube[:, 2:, 1:]), (t[2:4], t[:, 1:5].t()), (line[3:4], line),
                 (t[:, 2], t[:, 2]), (t[:0], t), (t[1:1], t[1:2].t())]:
        ps = [torch.nn.Parameter(torch.zeros(g.shape)) for g in (a, torch.ones(3), b)]
        for p, g in zip(ps, (a, torch.ones(3), b)):
            p.grad = g
        shared = bool(set(addresses(a)) & set(addresses(b)))
        for order in (ps, ps[::-1]):
            with pytest.raises(ValueError if shared else _lib.CinemaHipError, match="overlaps" if shared else "must live on the GPU"):
                clip_grad_norm_(order, 1.0)
        with pytest.raises(_lib.CinemaHipError, match="must live on the GPU"):       # reading twice is no clash
            grad_norm(ps)
    for parts in ([t[:, :6].t(), t[:, 6:].t()], [t[::2], t[1::2]], [line[::3], line[1::3], line[2::3]], [cube[:, :3, :4], cube[:, 3:, 2:], cube[:, :3, 4]],
                  [t[:4], t[4:, :7], t[4:, 7:]]):
        ps = [torch.nn.Parameter(torch.zeros(g.shape)) for g in parts]
        for p, g in zip(ps, parts):
            p.grad = g
        for order in (ps, ps[::-1]):
            with pytest.raises(_lib.CinemaHipError, match="must live on the GPU"):
                clip_grad_norm_(order, 1.0)


def addresses(t):
    """where the values of `t` lie, one by one"""
    at = torch.full(t.shape, t.storage_offset())
    for k, (size, stride) in enumerate(zip(t.shape, t.stride())):
        at = at + (torch.arange(size) * stride).view([-1 if j == k else 1 for j in range(t.dim())])
    return (t.untyped_storage().data_ptr() + t.element_size() * at).flatten().tolist()


def test_64_bit_norm_entry_points_check_their_arguments():
    from cinema_amd import _lib
    lib = _lib.load()
    t = (_lib.GradTensor * 1)()
    t[0].g, t[0].n, t[0].dtype = 256, 4, 0
    one = ctypes.c_void_p(256)
    for at, v in [(2, 3), (3, None), (4, None), (5, None)]:
        a = [t, 1, 2, one, one, one, None]
        a[at] = v
        assert lib.cinema_grad_norm_f64(*a) != 0 and b"cinema_grad_norm_f64" in lib.cinema_last_error()
    assert lib.cinema_adamw_step_clipped_f64((_lib.AdamWGroup * 1)(), 1, 0, None, 1.0, None) != 0


def test_c_entry_points_refuse_bounds_that_would_turn_gradients():
    """a negative or undefined bound is an error before anything is launched (a negative factor would turn every gradient)"""
    from cinema_amd import _lib
    lib = _lib.load()
    t = (_lib.GradTensor * 1)()
    t[0].g, t[0].n, t[0].dtype = 256, 4, 0
    one, group = ctypes.c_void_p(256), (_lib.AdamWGroup * 1)()
    for bad in (-1.0, -1e-30, float("nan"), -float("inf")):
        assert lib.cinema_grad_clip(t, 1, 2, bad, one, one, None) != 0
        assert b"max_norm" in lib.cinema_last_error()
        for step in (lib.cinema_adamw_step_clipped, lib.cinema_adamw_step_clipped_f64):
            assert step(group, 1, 0, one, bad, None) != 0
            assert b"max_norm" in lib.cinema_last_error()
        assert lib.cinema_layer_norm_forward(one, 8, None, None, 0, 4, 8, bad, _lib.DT_F32, one, None, None, None) != 0
        assert b"eps" in lib.cinema_last_error()
