"""What linear_act, layer_norm and the gradient norm refuse, without a GPU: arguments are checked before the device is."""
import math

import pytest
import torch


def test_linear_act_refusals():
    from cinema_amd.models.mlp import LinearAct, linear_act
    x, w, b = torch.zeros(4, 8), torch.zeros(6, 8), torch.zeros(6)
    for bad in [dict(activation="tanh"), dict(weight=torch.zeros(6, 7)), dict(weight=torch.zeros(8)), dict(weight=torch.zeros(0, 8)),
                dict(bias=torch.zeros(5)), dict(residual=torch.zeros(4, 7)), dict(residual=torch.zeros(6)), dict(x=torch.zeros(()))]:
        with pytest.raises(ValueError):
            linear_act(**{"x": x, "weight": w, "bias": b, **bad})
    for bad in [dict(x=x.double()), dict(weight=w.half()), dict(bias=b.bfloat16()), dict(residual=torch.zeros(4, 6).half()), dict(x=x.long())]:
        with pytest.raises(TypeError):
            linear_act(**{"x": x, "weight": w, "bias": b, **bad})
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        linear_act(x, w, b)
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        linear_act(x.bfloat16(), w.bfloat16(), b)            # a 32-bit bias beside 16-bit rows is allowed
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        linear_act(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), w, b)
    with pytest.raises(ValueError):
        LinearAct(4, 4, activation="sine")
    assert set(LinearAct(4, 6).state_dict()) == {"weight", "bias"}


def test_layer_norm_refusals():
    from cinema_amd.models.mlp import LayerNorm, layer_norm
    x = torch.zeros(4, 8)
    for bad in [dict(weight=torch.zeros(7)), dict(bias=torch.zeros(1, 8)), dict(eps=-1.0), dict(eps=float("nan")), dict(x=torch.zeros(4, 0)),
                dict(x=torch.zeros(()))]:
        with pytest.raises(ValueError):
            layer_norm(**{"x": x, **bad})
    for bad in [dict(x=x.double()), dict(weight=torch.zeros(8).half()), dict(x=x.half(), weight=torch.zeros(8), bias=torch.zeros(8).half())]:
        with pytest.raises(TypeError):
            layer_norm(**{"x": x, **bad})
    with pytest.raises(RuntimeError, match="must live on the GPU"):
        layer_norm(x)
    with pytest.raises(NotImplementedError):
        LayerNorm((4, 8))
    with pytest.raises(ValueError):
        LayerNorm(8)(torch.zeros(4, 6))
    assert set(LayerNorm(8).state_dict()) == {"weight", "bias"}


def test_gradient_norm_refusals():
    from cinema_amd import _lib
    from cinema_amd.optim import HipAdamW, clip_grad_norm_, grad_norm
    p = torch.nn.Parameter(torch.zeros(4))
    assert float(grad_norm([p])) == 0.0 and float(clip_grad_norm_(p, 1.0)) == 0.0      # no gradient
    p.grad = torch.ones(4)
    for bad in (3.0, 0.0, -math.inf):
        with pytest.raises(ValueError):
            grad_norm([p], bad)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            clip_grad_norm_([p], bad)
        with pytest.raises(ValueError):
            HipAdamW([p], max_grad_norm=bad)
    with pytest.raises(ValueError, match="twice"):
        clip_grad_norm_([p, p], 1.0)
    with pytest.raises(_lib.CinemaHipError, match="must live on the GPU"):
        clip_grad_norm_([p], 1.0)
    q = torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))
    q.grad = torch.ones(4, dtype=torch.float64)
    with pytest.raises(TypeError):
        grad_norm([p, q])


def test_c_entry_points_check_their_arguments():
    """size queries are host arithmetic; bad sizes, types and null operands come back as errors before anything is launched"""
    import ctypes as C
    from cinema_amd import _lib
    lib = _lib.load()
    dt = _lib.DT_BF16
    x = C.c_void_p(1 << 20)
    assert lib.cinema_linear_work_bytes(x, 512, x, 25000, 512, 512, 2, dt, 0) == 0
    assert lib.cinema_linear_work_bytes(x, 512, x, 25000, 512, 512, 2, dt, 1) >= 25000 * 512 * 2
    assert lib.cinema_linear_work_bytes(x, 511, x, 25000, 511, 512, 2, dt, 0) >= 25000 * 512 * 2        # packed rows
    assert lib.cinema_linear_work_bytes(C.c_void_p((1 << 20) + 2), 512, x, 25000, 512, 512, 2, dt, 0) >= 25000 * 512 * 2
    for bad in [(0, 8, 8, dt), (8, 0, 8, dt), (8, 8, -1, dt), (8, 8, 8, 3), (1 << 31, 8, 8, dt), (8, 1 << 20, 8, dt), (1 << 30, 8, 1 << 19, dt)]:
        for back in (0, 1):
            assert lib.cinema_linear_work_bytes(x, 8, x, *bad[:3], 2, bad[3], back) == -1
        assert b"cinema_linear" in lib.cinema_last_error()
    one = C.c_void_p(256)
    ok = [one, 8, one, None, 0, None, 0, 16, 8, 8, 0, dt, None, 0, one, None, None]
    for at, v in [(0, None), (1, 7), (2, None), (10, 5), (10, -1), (11, 9), (14, None), (7, 0)]:
        a = list(ok)
        a[at] = v
        assert lib.cinema_linear_forward(*a) != 0
    a = list(ok)
    a[5], a[6] = one, 7
    assert lib.cinema_linear_forward(*a) != 0                                    # residual rows closer than a row
    ok = [one, one, 0, one, 8, one, 5000, 8, 8, 1, dt, 0, one, one, one, one, None]
    for at, v in [(0, None), (1, None), (3, None), (4, 7), (5, None), (9, 5), (10, 4), (15, None), (6, 0)]:
        a = list(ok)
        a[at] = v
        assert lib.cinema_linear_backward(*a) != 0
    assert lib.cinema_layer_norm_work_bytes(100, 512, dt) > 0
    for bad in [(0, 8, dt), (8, 0, dt), (8, 8, 5), (1 << 31, 8, dt), (1 << 22, 1 << 20, dt), (8, (1 << 24) + 1, dt)]:
        assert lib.cinema_layer_norm_work_bytes(*bad) == -1
    assert lib.cinema_layer_norm_forward(None, 8, None, None, 0, 4, 8, 1e-5, dt, one, None, None, None) != 0
    assert lib.cinema_layer_norm_forward(one, 7, None, None, 0, 4, 8, 1e-5, dt, one, None, None, None) != 0
    assert lib.cinema_layer_norm_forward(one, 8, None, None, 0, 4, 8, 1e-5, dt, one, one, None, None) != 0
    assert lib.cinema_layer_norm_backward(one, one, 8, None, 0, one, one, 4, 8, dt, None, one, None, None, None) != 0
    assert lib.cinema_grad_norm_work_bytes(-1) == -1
    t = (_lib.GradTensor * 1)()
    t[0].g, t[0].n, t[0].dtype = 256, 4, 7
    assert lib.cinema_grad_norm(t, 1, 2, one, one, None) != 0
    t[0].dtype, t[0].n = 0, -1
    assert lib.cinema_grad_norm(t, 1, 2, one, one, None) != 0
    t[0].n = 4
    assert lib.cinema_grad_norm(t, 1, 3, one, one, None) != 0
    assert lib.cinema_grad_clip(t, 1, 2, 1.0, None, one, None) != 0
    assert lib.cinema_adamw_step_clipped((_lib.AdamWGroup * 1)(), 1, 0, None, 1.0, None) != 0
    # struct layout of the table
    assert C.sizeof(_lib.GradTensor) == 24


def test_clipped_step_refuses_a_norm_it_cannot_use():
    from cinema_amd._lib import CinemaHipError
    from cinema_amd.optim import HipAdamW
    p = torch.nn.Parameter(torch.zeros(4))
    p.grad = torch.ones(4)
    with pytest.raises(ValueError, match="max_grad_norm"):
        HipAdamW([p]).step(grad_norm=torch.ones(()))
    opt = HipAdamW([p], max_grad_norm=1.0)
    for bad in [torch.ones((), dtype=torch.float64), torch.ones(2), torch.ones((), device="meta")]:
        with pytest.raises(CinemaHipError, match="grad_norm"):
            opt.step(grad_norm=bad)
    assert not opt.state
