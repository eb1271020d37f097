"""linear_act and layer_norm at long reductions, far offsets and many tiles, where a bound on the worst order of the sums would pass
a result of zeros.  Three kinds of check that do not:

* whole numbers small enough that every sum is exact in any order (all partial sums below 2^24): each output equals the exact
  one rounded once, so a missing term, tile or split shows in a single bit;
* smooth activations, as whole matrices: relative to the 2-norm, with sums that grow like the root of their length;
* differences of the kernel's own output along the gradient, whose truncation is known from the formula in 64 bits."""
import math

import pytest
import torch

from test_gpu_mlp import ACTS, DTYPES, U, act64, slope64

pytestmark = pytest.mark.gpu


def ints(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda", dtype=torch.int8)


def same(got, want, what):
    """`got` against the exact whole numbers, rounded once; they are not nearly all zero (least for dx of one feature behind relu:
    2 / 3 of dy, 4 / 5 of w and about 0.45 of the gates are not)"""
    assert float((want != 0).double().mean()) > 0.1 or want.numel() < 8, what
    assert float(want.abs().max()) < 2.0 ** 24
    want = want.to(got.dtype)
    if not torch.equal(got, want):
        bad = (got != want).flatten()
        i = int(bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} differ, first at {i}: {float(got.flatten()[i])} for {float(want.flatten()[i])}")


def check_exact(m, k, n, dtype, act, rows=1 << 12):
    """x, w in -2 .. 2 and dy in -1 .. 1: |terms| of a sum are at most 4 and 2, so 2^22 and 2^23 of them stay exact"""
    from cinema_amd.models.mlp import linear_act
    assert max(k, n, m) <= 1 << 21
    g = torch.Generator(device="cuda").manual_seed(m + 3 * k + 7 * n)
    x, w, b, r, dy = ints(g, -2, 2, m, k), ints(g, -2, 2, n, k), ints(g, -3, 3, n), ints(g, -4, 4, m, n), ints(g, -1, 1, m, n)
    leaves = [t.to(dtype).requires_grad_(True) for t in (x, w, b, r)]
    y = linear_act(*leaves, act)
    grads = torch.autograd.grad(y, leaves, dy.to(dtype))
    what = f"{m}x{k}x{n} {dtype} {act}"
    wd, dw, db = w.double(), torch.zeros(n, k, device="cuda", dtype=torch.float64), torch.zeros(n, device="cuda", dtype=torch.float64)
    for i in range(0, m, rows):                                     # a block of rows at a time: 64 bits of everything do not fit
        s = slice(i, i + rows)
        xd, z = x[s].double(), x[s].double() @ wd.t() + b.double()
        same(y[s].detach(), act64(z, act) + r[s].double(), f"y of {what}, rows from {i}")
        dz = dy[s].double() * (z > 0 if act == "relu" else 1.0)
        same(grads[0][s], dz @ wd, f"dx of {what}, rows from {i}")
        dw += dz.t() @ xd
        db += dz.sum(0)
    same(grads[1], dw, f"dw of {what}")
    same(grads[2], db, f"db of {what}")
    assert torch.equal(grads[3], dy.to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (16, (1 << 20) - 1, 4), (3, (1 << 20) - 1, 2), (8, 5, 100003), (300001, 5, 1), (33001, 33, 4), (4099, 257, 3),
                                   (20000, 3, 2), (971, 1, 3), (5000, 72, 136), (4097, 257, 130), (2048, 4096, 8), (40, 6000, 24), (3000, 1032, 520),
                                   (25000, 512, 512), (12500, 264, 520), (1000, 1288, 1001), (2040, 4104, 2040), (200, 300, 257), (64, 256, 64)])
def test_linear_sums_are_whole(m, k, n, act, dtype):
    check_exact(m, k, n, dtype, act)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_sums_are_whole_on_the_largest_tiles(dtype):
    check_exact(33001, 1031, 4103, dtype, "relu", 1 << 14)
    if dtype != torch.float32:
        check_exact(33000, 1032, 4104, dtype, "none", 1 << 14)


def test_linear_sums_are_whole_beyond_32_bit_offsets():
    check_exact(70000, 8, 32768, torch.bfloat16, "relu", 1 << 13)


def near(got, want, allowed, what):
    e, size = float((got.double() - want).norm()), float(want.norm())
    assert size > 0 and e <= allowed * size, f"{what}: off by {e / size:.3e} of its norm, allowed {allowed:.3e}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,k,n", [(16, (1 << 20) - 1, 4), (300001, 5, 1), (20000, 3, 2), (4097, 257, 130), (2048, 4096, 8), (25000, 512, 512), (33001, 1031, 517)])
def test_linear_smooth_activations_by_the_norm(m, k, n, act, dtype):
    """roundings of single values (output U, dz U, a kept z 2^-11) count once each against the norm of what they are summed into, the
    terms' signs being independent; a sum of L fp32 terms walks sqrt(L) steps of 2^-23; the activation's 2^-21 of |z| + 4 squared is
    below 2^-15 of a value of size 1.  A sum that loses one 64th of its terms is off by 1 / 8."""
    from cinema_amd.models.mlp import linear_act
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    rn = lambda *s, c=1.0: (torch.randn(*s, generator=g, device="cuda") * c).to(dtype)
    x, w, b, dy = rn(m, k), rn(n, k, c=1 / math.sqrt(k)), rn(n, c=0.2), rn(m, n, c=0.1)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = linear_act(*leaves, None, act)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    z = x.double() @ w.double().t() + b.double()
    dz = dy.double() * slope64(z, act)
    kept = 0.0 if dtype == torch.float32 else 2.0 ** -10
    for got, want, length in ((y.detach(), act64(z, act), k), (dx, dz @ w.double(), n), (dw, dz.t() @ x.double(), m), (db, dz.sum(0), m)):
        allowed = 2 * U[dtype] + kept + 2.0 ** -15 + (8 + math.sqrt(length) + math.sqrt(k)) * 2.0 ** -22
        assert allowed < 0.02
        near(got, want, allowed, f"{tuple(got.shape)} of {m}x{k}x{n} {act}")


def along_gradients(call, formula, leaves, dy):
    """central differences along each gradient's own direction, whose derivative is the gradient's norm.  The same difference of the
    formula in 64 bits tells the truncation; the outputs' rounding (2^-19 of their magnitude for these short sums) counts at its
    worst.  What is allowed stays below a twentieth of the derivative, so a zero, a wrong sign or a wrong factor does not pass."""
    own = [t.clone().requires_grad_(True) for t in leaves]
    wide = [t.double().requires_grad_(True) for t in leaves]
    y, y64 = call(*own), formula(*wide)
    grads, grads64 = torch.autograd.grad(y, own, dy), torch.autograd.grad(y64, wide, dy.double())
    h = 2.0 ** -4
    for i, (g, g64) in enumerate(zip(grads, grads64)):
        d = (g64 / g64.norm()).float()
        moved = lambda f, s, ts: (f(*[t + s * h * d.to(t.dtype) if j == i else t for j, t in enumerate(ts)]).double() * dy.double()).sum()
        with torch.no_grad():
            got = float(moved(call, 1, leaves) - moved(call, -1, leaves)) / (2 * h)
            exact = [t.double() for t in leaves]
            true = float(moved(formula, 1, exact) - moved(formula, -1, exact)) / (2 * h)
        slope = float((g64 * d.double()).sum())
        allowed = abs(true - slope) + 2.0 ** -19 * float(((y.detach().abs() + 1) * dy.abs()).sum()) / h
        assert allowed < 0.05 * slope, (i, allowed, slope)
        assert abs(float((g.double() * d.double()).sum()) - got) <= allowed, i


@pytest.mark.parametrize("act", [a for a in ACTS if a != "relu"])
def test_linear_gradients_match_differences_along_themselves(act):
    from cinema_amd.models.mlp import linear_act
    g = torch.Generator(device="cuda").manual_seed(2)
    r = lambda *s, c=1.0: torch.randn(*s, generator=g, device="cuda") * c
    leaves = [r(24, 20), r(28, 20, c=0.2), r(28, c=0.2), r(24, 28)]
    along_gradients(lambda *t: linear_act(*t, act), lambda x, w, b, q: act64(x @ w.t() + b, act) + q, leaves, r(24, 28, c=0.1))


def test_layer_norm_gradients_match_differences_along_themselves():
    from cinema_amd.models.mlp import layer_norm
    g = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")

    def formula(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * w + b
    along_gradients(layer_norm, formula, [r(12, 40), 1 + 0.1 * r(40), 0.1 * r(40)], r(12, 40))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", [(530000, 4), (70001, 257), (4500, 520), (600, 5000), (70, 33000), (3, 300007)])
def test_layer_norm_by_the_norm(m, d, dtype):
    """roundings as above; a row's statistics are sums of d terms, dw and db of m"""
    from cinema_amd.models.mlp import layer_norm
    g = torch.Generator(device="cuda").manual_seed(m + d)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w, b, dy = (0.3 + 1.5 * r(m, d)).to(dtype), 1 + 0.2 * r(d), 0.2 * r(d), (0.1 * r(m, d)).to(dtype)
    if dtype == torch.float32 or d % 2:
        w, b = w.to(dtype), b.to(dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    c = x - x.mean(1, keepdim=True)
    rs = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5)
    h, gw = c * rs, dy * w
    want = {"y": h * w + b, "dx": rs * (gw - gw.mean(1, keepdim=True) - h * (gw * h).mean(1, keepdim=True)), "dw": (dy * h).sum(0), "db": dy.sum(0)}
    for name, got in (("y", y.detach()), ("dx", dx), ("dw", dw), ("db", db)):
        # rows of four values may lie close together, and 1 / s magnifies what the mean lost
        allowed = U[got.dtype] + (64 + math.sqrt(m) + math.sqrt(d)) * 2.0 ** -22 * (64 if d < 16 else 1)
        assert allowed < 0.05
        near(got, want[name], allowed, f"{name} of {m}x{d} {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(4000, 264, 1001), (12001, 200, 777), (16384, 512, 1023), (16400, 512, 1023), (12000, 513, 1001), (30001, 72, 1003),
                                   (4100, 1024, 1022), (4100, 1032, 1022), (4110, 1024, 1022)])
def test_linear_sums_are_whole_where_odd_rows_change_tiles(m, k, n, dtype):
    """either side of where a residual or a kept z on odd rows takes smaller tiles: 2^24 outputs and 512 values of r, 2^22 and 1024"""
    check_exact(m, k, n, dtype, "relu", 1 << 14)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,k,n", [(1, 1, 10000), (3, 1, 4000), (9, 2, 4096), (2, 30, 8000), (1, 200, 9000), (64, 1, 4099), (256, 1, 2100), (1, 8, 300000),
                                   (971, 1, 3), (20000, 3, 2)])
def test_linear_gradients_of_few_values_by_the_norm(m, k, n, act, dtype):
    """dx of few values from many features, as dW of few from many rows: dz stays in 32 bits, so a gradient is off by its own rounding,
    U of each value at most, and by the fp32 sums, relative to the norm of what is summed.  Ten inputs, as a single one may be lucky"""
    from cinema_amd.models.mlp import linear_act
    for seed in range(10):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rn = lambda *s, c=1.0: (torch.randn(*s, generator=g, device="cuda") * c).to(dtype)
        x, w, b, dy = rn(m, k), rn(n, k, c=1 / math.sqrt(k)), rn(n, c=0.2), rn(m, n, c=0.1)
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        dx, dw, db = torch.autograd.grad(linear_act(*leaves, None, act), leaves, dy)
        z = x.double() @ w.double().t() + b.double()
        dz = dy.double() * slope64(z, act)
        W, X, one = w.double(), x.double(), torch.ones(1, m, device="cuda", dtype=torch.float64)
        for got, a, c in ((dx, dz, W), (dw, dz.t(), X), (db, one, dz)):
            want = (a @ c).view_as(got)
            # a term's own error, of the activation and of z: (|z| + 4)^2 2^-21 of it, far below 2^-16; they add like their signs
            terms = float(((a * a) @ (c * c)).sum().sqrt())
            allowed = U[dtype] * float(want.norm()) + terms * (2.0 ** -15 + (8 + math.sqrt(max(m, n)) + math.sqrt(k)) * 2.0 ** -22)
            assert float((got.double() - want).norm()) <= allowed, (seed, float((got.double() - want).norm()) / float(want.norm()), allowed / float(want.norm()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [8, 4000])
def test_gelu_keeps_its_relative_accuracy_far_below_zero(rows, dtype):
    """z Phi(z) and its slope at z from -0.02 to -12, where they fall to 1e-31: relative to the value, half a step of the type (the slope
    leaves its root at -0.75 out), 2^-17 for the 16-bit types' polynomial, and for every type what the exponent makes of its own
    rounding: z^2 2^-24 for the square and its factor, z^2 2^-24 more for z / sqrt 2 inside the fp32 library function, 16 * 2^-24 for
    the products"""
    from cinema_amd.models.mlp import linear_act
    z = -torch.linspace(0.02, 12.0, rows, device="cuda").to(dtype)
    x = z.view(-1, 1).clone().requires_grad_(True)
    w = torch.ones(1, 1, device="cuda", dtype=dtype)
    y = linear_act(x, w, None, None, "gelu")
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    zd = z.double()
    cdf = 0.5 * torch.special.erfc(-zd / math.sqrt(2))
    slope = cdf + zd * torch.exp(-0.5 * zd * zd) / math.sqrt(2 * math.pi)
    smallest = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[dtype]
    rel = U[dtype] + (0 if dtype == torch.float32 else 2.0 ** -17) + 2 * zd * zd * 2.0 ** -24 + 16 * 2.0 ** -24
    for got, want, keep in ((y.detach().flatten(), zd * cdf, zd < 0), (dx.flatten(), slope, (zd + 0.75).abs() > 0.2)):
        # the slope is the difference of two terms: its error counts against their sum of magnitudes
        size = want.abs() if want is not slope else cdf + (slope - cdf).abs()
        bad = ((got.double() - want).abs() > rel * size + smallest)[keep]
        assert not bad.any(), (float(zd[keep][bad][0]), float(got.double()[keep][bad][0]), float(want[keep][bad][0]))
