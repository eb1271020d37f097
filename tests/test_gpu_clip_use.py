"""clip_grad_norm_, grad_norm and HipAdamW(max_grad_norm=) beside what else a program does with its gradients."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def params(*grads):
    out = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, device=g.device, dtype=g.dtype))
        p.grad = g
        out.append(p)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_clipping_counts_as_a_write(dtype):
    """a graph that saved a gradient notices that it was clipped since, strided gradients as well as contiguous ones"""
    from cinema_amd.optim import clip_grad_norm_
    base = torch.randn(50, 12, device="cuda").to(dtype)
    for g in (base[:, :6].t(), torch.randn(30, device="cuda").to(dtype)):
        (p,) = params(g)
        before = p.grad._version
        s = torch.ones((), device="cuda", dtype=dtype, requires_grad=True)
        y = s * p.grad                          # saves the gradient
        clip_grad_norm_([p], 0.1)
        assert p.grad._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()
    with torch.inference_mode():
        (p,) = params(torch.ones(6, 4, device="cuda", dtype=dtype).t())
        assert abs(float(clip_grad_norm_([p], 1e-3)) - 24 ** 0.5) < 1e-5
        assert float(p.grad.double().norm()) < 1.1e-3


def test_neighbours_in_one_table_are_clipped_each():
    """columns of one table as gradients of several parameters; a table beside a transposed view of it is refused untouched"""
    from cinema_amd.optim import clip_grad_norm_
    base = torch.randn(50, 12, device="cuda")
    was = base.double()
    ps = params(base[:, :5].t(), base[:, 5:7], base[:, 7:].t())
    norm = float(was.norm())
    assert abs(float(clip_grad_norm_(ps, norm / 4)) - norm) <= norm * 2.0 ** -23
    assert bool(((base.double() - was * (norm / 4 / (norm + 1e-6))).abs() <= was.abs() * 2.0 ** -22).all())
    square = torch.randn(8, 8, device="cuda")
    was = square.clone()
    with pytest.raises(ValueError, match="overlaps"):
        clip_grad_norm_(params(square, square.t()), 0.1)
    assert torch.equal(square, was)


@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("bad", ["strided", "other device", "type"])
def test_a_refused_update_changes_nothing(bad, clip):
    """a parameter that cannot be updated is found before any other's step count, moments or values change"""
    from cinema_amd import _lib
    from cinema_amd.optim import HipAdamW
    other = {"strided": lambda: torch.ones(16, device="cuda")[::2], "other device": lambda: torch.ones(8),
             "type": lambda: torch.ones(8, device="cuda", dtype=torch.bfloat16)}[bad]()
    p, q = params(torch.ones(8, device="cuda"), other)
    opt = HipAdamW([p, q], lr=0.1, max_grad_norm=clip)
    for _ in range(2):
        with pytest.raises((_lib.CinemaHipError, ValueError)):
            opt.step()
    assert not opt.state and opt.grad_norm is None and not p.any() and bool((p.grad == 1).all())
    q.grad = None                               # without it: the first step, as if none had been tried
    opt.step()
    assert opt.state[p]["step"] == 1
    r = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    r.grad = p.grad.clone()
    fresh = HipAdamW([r], lr=0.1, max_grad_norm=clip)
    fresh.step()
    assert torch.equal(p, r)


@pytest.mark.parametrize("n", [1, 1000])
def test_clipped_update_where_the_norm_leaves_fp32(n):
    """gradients of 3e38: their norm is beyond fp32 for n = 1000, and clipping has to leave them 0.5 / sqrt(n) each, in the update as
    in clip_grad_norm_ before it.  The factor has fp32's least step, 2^-149: half of that is its error.  The first update is
    lr * g / (|g| + eps / sqrt(bias correction)), within 2^-20 of lr"""
    from cinema_amd.optim import HipAdamW, clip_grad_norm_
    got = []
    for fused in (False, True):
        (p,) = params(torch.full((n,), 3e38, device="cuda"))
        opt = HipAdamW([p], lr=0.125, weight_decay=0.0, max_grad_norm=0.5 if fused else None)
        if not fused:
            clip_grad_norm_([p], 0.5)
            want = 0.5 / n ** 0.5
            assert abs(float(p.grad[0]) - want) <= want * 2.0 ** -22 + 3e38 * 2.0 ** -150
        opt.step()
        got.append(p.detach().clone())
        assert torch.equal(opt.state[p]["exp_avg"] > 0.09 * want, torch.ones_like(p, dtype=torch.bool))
    assert bool((got[1] + 0.125).abs().max() <= 0.125 * 2.0 ** -19)
    assert float((got[1] - got[0]).abs().max()) <= 0.125 * 2.0 ** -19


def test_a_given_norm_in_either_type():
    """fp32 and fp64 values clip, also the union norm as it comes; anything else is refused and changes nothing"""
    from cinema_amd import _lib
    from cinema_amd import parallel as par
    from cinema_amd.optim import HipAdamW
    outs = []
    for given in (lambda n: None, lambda n: n.float(), lambda n: n, lambda n: par.union_grad_norm(n.float(), None)):
        (p,) = params(torch.linspace(-1, 1, 77, device="cuda"))
        opt = HipAdamW([p], lr=0.1, max_grad_norm=0.25)
        n = p.grad.double().norm()
        opt.step(grad_norm=given(n))
        assert opt.grad_norm.dtype == torch.float32 and opt.grad_norm.dim() == 0 and abs(float(opt.grad_norm) - float(n)) <= float(n) * 2.0 ** -22
        outs.append(p.detach().clone())
    assert all(float((o - outs[0]).abs().max()) <= 0.1 * 2.0 ** -18 for o in outs)
    one, kept = torch.ones((), device="cuda"), opt.grad_norm
    for bad in [one.half(), one.long(), one.cpu(), one.double().cpu(), torch.ones(2, device="cuda"), torch.ones(2, device="cuda").double()]:
        with pytest.raises(_lib.CinemaHipError, match="grad_norm"):
            opt.step(grad_norm=bad)
    assert opt.grad_norm is kept and opt.state[p]["step"] == 1


def test_no_gradients_have_the_norm_0_where_the_parameters_are():
    from cinema_amd.optim import clip_grad_norm_, grad_norm
    p = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    q = torch.nn.Parameter(torch.zeros(3))
    for call in (grad_norm, lambda ps: clip_grad_norm_(ps, 1.0), lambda ps: clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)):
        for ps, device in ((p, "cuda"), ([p], "cuda"), (iter([p, q]), "cuda"), ([q], "cpu"), ([], "cpu")):
            n = call(ps)
            assert n.device.type == device and n.dtype == torch.float32 and n.dim() == 0 and float(n) == 0.0
    p.grad = torch.full((3,), 2.0, device="cuda")
    assert grad_norm([q, p], 1.0).device.type == "cuda" and float(grad_norm(iter([q, p]), 1.0)) == 6.0
    assert float(clip_grad_norm_(iter([q, p]), 3.0, 1.0, error_if_nonfinite=True)) == 6.0 and abs(float(p.grad[0]) - 1.0) < 1e-6
    with pytest.raises(ValueError):
        grad_norm([q], 3.0)
