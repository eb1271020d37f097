"""linear_act, layer_norm and the gradient norm (cinema_amd/models/mlp.py, cinema_amd/optim.py) against their formulas in 64
bits.  Every tolerance is a bound by arithmetic, elementwise: half a step of the output's type (U), the fp32 sums' error
(number of additions * 2^-24 * sum of magnitudes, 2^-23 for the matrix unit, whose additions may truncate), and what the
activation's own evaluation and the kept pre-activation add."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step, relative
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}           # half of the least step, absolute
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LIP = 1.13          # |act'| at most (gelu: 1.129)
CURV = 0.8          # |act''| at most (gelu: 0.798)


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z * torch.sigmoid(z) if act == "silu" else z * 1.0


def slope64(z, act):
    z = z.detach().requires_grad_(True)
    return torch.autograd.grad(act64(z, act).sum(), z)[0]


def within(got, want, bound, what):
    d = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all()), what
    bad = d > bound
    if bad.any():
        i = int((d / bound).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {i}: got {float(got.flatten()[i])!r}, "
                             f"want {float(want.flatten()[i])!r}, off {float(d.flatten()[i]):.3e}, allowed {float(bound.flatten()[i]):.3e}")


def linear_data(m, k, n, dtype, seed=0, res=True, bias_dtype=None):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    r = lambda *s, c=1.0: torch.randn(*s, generator=g, device="cuda") * c
    return (r(m, k).to(dtype), r(n, k, c=1 / math.sqrt(k)).to(dtype), r(n, c=0.2).to(bias_dtype or dtype), r(m, n).to(dtype) if res else None,
            r(m, n, c=0.1).to(dtype))


def linear_bounds(x, w, b, r, dy, act):
    """{name: (value, bound)} of y, dx, dw, db for data of one type."""
    t = x.dtype
    m, k = x.shape
    n = w.shape[0]
    X, W, DY = x.double(), w.double(), dy.double()
    z = X @ W.t() + (0 if b is None else b.double())
    s = X.abs() @ W.abs().t() + (0 if b is None else b.double().abs())
    ez = (k + 2) * 2.0 ** -23 * s
    ea = (z.abs() + 4) ** 2 * 2.0 ** -21                                   # the activation's own evaluation
    if act == "none":
        ea = torch.zeros_like(z)
    y = act64(z, act) + (0 if r is None else r.double())
    ey = LIP * ez + ea + y.abs() * (U[t] + 2.0 ** -23) + 2.0 ** -23 * (0 if r is None else r.double().abs()) + TINY[t]
    sl = slope64(z, act)
    dz = DY * sl
    kept = 0 if act == "none" or t == torch.float32 else z.abs() * 2.0 ** -11 + 2.0 ** -25
    es = torch.zeros_like(z) if act == "none" else CURV * (ez + kept) + ea
    if act == "relu":
        es = (z.abs() <= ez).double()                                      # either side of the kink
    e_raw = DY.abs() * es + dz.abs() * 2.0 ** -23
    e_dz = e_raw + (0 if act == "none" else (dz.abs() + e_raw) * U[t] + TINY[t])
    adz = dz.abs() + e_dz
    dx, dw, db = dz @ W, dz.t() @ X, dz.sum(0)
    e = {"dx": e_dz @ W.abs() + (n + 2) * 2.0 ** -23 * (adz @ W.abs()), "dw": e_dz.t() @ X.abs() + (m + 2) * 2.0 ** -23 * (adz.t() @ X.abs()),
         "db": e_raw.sum(0) + (m + 2) * 2.0 ** -24 * adz.sum(0)}
    out = {"y": (y, ey)}
    for name, v in (("dx", dx), ("dw", dw), ("db", db)):
        u = U[b.dtype] if name == "db" and b is not None else U[t]
        ty = TINY[b.dtype] if name == "db" and b is not None else TINY[t]
        out[name] = (v, e[name] + (v.abs() + e[name]) * u + ty)
    return out


def check_linear(m, k, n, dtype, act, res=True, bias=True, bias_dtype=None, x=None):
    from cinema_amd.models.mlp import linear_act
    x0, w, b, r, dy = linear_data(m, k, n, dtype, seed=m + 3 * k + 7 * n, res=res, bias_dtype=bias_dtype)
    if x is not None:
        x0 = x(x0)
    b = b if bias else None
    want = linear_bounds(x0, w, b, r, dy, act)
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x0, w, b, r)]
    y = linear_act(leaves[0], leaves[1], leaves[2], leaves[3], act)
    with torch.no_grad():
        y_eval = linear_act(x0, w, b, r, act)
    assert torch.equal(y, y_eval)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dy)
    names = [nm for nm, t in zip(("dx", "dw", "db", "dr"), leaves) if t is not None]
    got = dict(zip(names, grads), y=y.detach())
    for nm in got:
        if nm == "dr":
            assert torch.equal(got[nm], dy)
        else:
            within(got[nm], *want[nm], f"{nm} of {m}x{k}x{n} {dtype} {act}")


SHAPES = [(1, 1, 1), (1, 256, 64), (2, 33, 5), (8, 64, 130), (9, 64, 32), (64, 256, 64), (17, 1, 40), (65, 257, 1), (129, 40, 131),
          (300, 512, 72), (130, 136, 264)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_matches_its_formula(m, k, n, dtype):
    check_linear(m, k, n, dtype, "gelu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("res,bias", [(True, True), (False, True), (False, False)])
def test_linear_activations(act, res, bias, dtype):
    check_linear(70, 96, 80, dtype, act, res, bias)
    check_linear(3, 96, 80, dtype, act, res, bias)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(5000, 72, 136), (4097, 257, 130), (2048, 4096, 8), (40, 6000, 24), (3000, 1032, 520)])
def test_linear_long_reductions_and_many_tiles(m, k, n, dtype):
    """split reductions (weight gradients over many rows, few outputs over a long k) and more tiles than one pass"""
    check_linear(m, k, n, dtype, "silu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_fp32_bias(dtype):
    check_linear(100, 64, 72, dtype, "gelu_tanh", bias_dtype=torch.float32)
    check_linear(1, 64, 72, dtype, "gelu_tanh", bias_dtype=torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("view", ["rows_of_wider", "offset", "transposed", "expanded", "three_dims"])
def test_linear_strides(view, dtype):
    """rows of a wider table, an offset that breaks 16-byte alignment, a transposed and an expanded input"""
    def make(x):
        m, k = x.shape
        if view == "rows_of_wider":
            wide = torch.full((m, k + 24), float("nan"), device="cuda", dtype=dtype)
            wide[:, 8:8 + k] = x
            return wide[:, 8:8 + k]
        if view == "offset":
            wide = torch.full((m * (k + 1) + 1,), float("nan"), device="cuda", dtype=dtype)
            v = wide[1:].view(m, k + 1)[:, :k]
            v.copy_(x)
            return v
        if view == "transposed":
            return x.t().contiguous().t()
        if view == "expanded":
            return x[:1].expand(m, k)
        return x
    if view != "three_dims":
        check_linear(133, 64, 72, dtype, "silu", x=make)
        return
    from cinema_amd.models.mlp import linear_act
    x, w, b, r, _ = linear_data(4 * 35, 64, 72, dtype)
    want = linear_act(x, w, b, r, "relu")
    got = linear_act(x.view(4, 35, 64), w, b, r.view(4, 35, 72), "relu")
    assert got.shape == (4, 35, 72) and torch.equal(got.view(-1, 72), want)
    assert torch.equal(linear_act(x[0], w, b, r[0], "relu"), linear_act(x[:1], w, b, r[:1], "relu")[0])


@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_linear_reads_no_row_or_column_that_is_not_its_own(m):
    """NaN behind the rows, in the padding of strided rows and around the output: none of it arrives"""
    from cinema_amd.models.mlp import linear_act
    for k, n in ((64, 72), (65, 71)):
        x, w, b, r, dy = linear_data(m, k, n, torch.bfloat16)
        want = linear_act(x, w, b, r, "gelu")
        xt = torch.full((m + 3, k + 16), float("nan"), device="cuda", dtype=x.dtype)
        xt[:m, :k] = x
        rt = torch.full((m + 3, n + 8), float("nan"), device="cuda", dtype=x.dtype)
        rt[:m, :n] = r
        got = linear_act(xt[:m, :k], w, b, rt[:m, :n], "gelu")
        assert torch.equal(got, want)


def test_linear_non_finite_rows_stay_in_their_rows():
    from cinema_amd.models.mlp import linear_act
    for dtype in DTYPES:
        for m in (4, 200):
            x, w, b, r, dy = linear_data(m, 72, 80, dtype)
            x[1, 3] = float("nan")
            x[2, 5] = float("inf")
            y = linear_act(x, w, b, r, "none").double()
            z = x.double() @ w.double().t() + b.double() + r.double()
            assert torch.equal(torch.isnan(y), torch.isnan(z)) and torch.equal(torch.isinf(y), torch.isinf(z))
            yr = linear_act(x, w, b, None, "relu")
            assert torch.isnan(yr[1]).all() and torch.isfinite(yr[3:]).all()


@pytest.mark.parametrize("act", ACTS)
def test_linear_far_pre_activations(act):
    """pre-activations far out, where exponentials overflow: value and slope at their limits"""
    from cinema_amd.models.mlp import linear_act
    for dtype in DTYPES:
        mags = [0.0, 1e-3, 5.0, 12.0, 30.0, 90.0, 300.0, 3e4]
        x = torch.tensor([[s * v] for v in mags for s in (1, -1)], device="cuda").to(dtype).requires_grad_(True)
        w = torch.ones(1, 1, device="cuda", dtype=dtype)
        y = linear_act(x, w, None, None, act)
        z = x.detach().double()
        bound = act64(z, act).abs() * (U[dtype] + 2.0 ** -20) + z.abs() * 2.0 ** -21 + TINY[dtype]
        within(y.detach(), act64(z, act), bound, act)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        sl = torch.where(z > 0, 1.0, 0.0) if act == "relu" else slope64(z, act)
        kept = 0 if dtype == torch.float32 else z.abs().clamp_max(20) * 2.0 ** -11 * CURV
        within(dx, sl, 2 * U[dtype] * sl.abs() + (z.abs().clamp_max(20) + 4) ** 2 * 2.0 ** -21 + kept + 2 * TINY[dtype], act)


def test_linear_relu_slope_of_tiny_positive_values():
    """pre-activations that fp16 rounds to zero keep their sign for the slope"""
    from cinema_amd.models.mlp import linear_act
    x = torch.tensor([[1e-9], [-1e-9], [3e-8], [0.0]], device="cuda").to(torch.bfloat16).requires_grad_(True)
    for rows in (x, x.repeat(20, 1)):
        y = linear_act(rows, torch.ones(1, 1, device="cuda", dtype=torch.bfloat16), None, None, "relu")
        (g,) = torch.autograd.grad(y, rows, torch.ones_like(y))
        assert g.flatten()[:4].tolist() == [1.0, 0.0, 1.0, 0.0]


def test_linear_gradients_match_differences():
    """fp32 gradients against central differences of the kernel's own output along random directions.  step h = 2^-6:
    truncation at most h^2 / 6 * |third derivative along the direction|, rounding of the two outputs over 2 h."""
    from cinema_amd.models.mlp import linear_act
    x, w, b, r, dy = linear_data(24, 20, 28, torch.float32)
    for act in ("none", "gelu", "gelu_tanh", "silu"):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        y = linear_act(*leaves, act)
        grads = torch.autograd.grad(y, leaves, dy)
        for i, (t, g) in enumerate(zip((x, w, b, r), grads)):
            d = torch.randn_like(t)
            d /= d.norm()
            h = 2.0 ** -6
            f = lambda s: (linear_act(*[u + s * h * d if j == i else u for j, u in enumerate((x, w, b, r))], act).double() * dy.double()).sum()
            want = float((f(1) - f(-1)) / (2 * h))
            # z moves by at most h * |d| * max(|x|, |w|) row norms (< 8 here): |act'''| <= 2 bounds the third derivative
            zmax = 8.0
            trunc = h * h / 6 * 2 * zmax ** 3 * float(dy.abs().sum()) / math.sqrt(dy.numel())
            rounding = 2.0 ** -20 * float((y.detach().abs() * dy.abs()).sum()) / (2 * h)
            assert abs(float((g.double() * d.double()).sum()) - want) <= trunc + rounding, (act, i)


def test_linear_partial_gradients_and_empty_rows():
    from cinema_amd.models.mlp import linear_act
    x, w, b, r, dy = linear_data(40, 24, 32, torch.bfloat16)
    full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
    all_g = torch.autograd.grad(linear_act(*full, "silu"), full, dy)
    for i in range(4):
        part = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b, r))]
        (g,) = torch.autograd.grad(linear_act(*part, "silu"), [part[i]], dy)
        assert torch.equal(g, all_g[i])
    e = [t.clone().requires_grad_(True) for t in (x[:0], w, b, r[:0])]
    y = linear_act(*e, "silu")
    assert y.shape == (0, 32)
    g = torch.autograd.grad(y, e, torch.empty_like(y))
    assert g[0].shape == (0, 24) and all(not t.any() for t in g)
    y = linear_act(*full, "none")
    y.sum().backward()                              # an expanded gradient
    assert torch.equal(full[2].grad, torch.full_like(b, 40.0))
    with pytest.raises(RuntimeError, match="second derivative"):
        v = x.clone().requires_grad_(True)
        torch.autograd.grad(linear_act(v, w, b, None, "silu").sum(), v, create_graph=True)


def test_linear_autocast_casts_like_a_linear_layer():
    from cinema_amd.models.mlp import LinearAct
    layer = LinearAct(64, 48, activation="relu").cuda()
    x = torch.randn(50, 64, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = layer(x)
    assert y.dtype == torch.bfloat16
    z = x.bfloat16().double() @ layer.weight.bfloat16().double().t() + layer.bias.double()
    within(y.detach(), z.clamp_min(0).detach(), (z.abs() * U[torch.bfloat16] + 66 * 2.0 ** -23 * (x.double().abs() @ layer.weight.double().abs().t() * 1.02 + 1)).detach(), "autocast")
    y.float().sum().backward()
    assert layer.weight.grad.dtype == torch.float32 and layer.bias.grad.dtype == torch.float32


# ---- layer norm -------------------------------------------------------------------------------------------------------------
def norm_bounds(x, w, b, dy, eps):
    t, (m, d) = x.dtype, x.shape
    X, G = x.double(), dy.double()
    W = torch.ones(d, device="cuda", dtype=torch.float64) if w is None else w.double()
    B = 0 if b is None else b.double()
    steps = 80 + d // 128                                          # additions behind one another in a row sum, at most
    e24 = 2.0 ** -24
    mu = X.mean(1, keepdim=True)
    var = ((X - mu) ** 2).mean(1, keepdim=True)
    rs = 1 / torch.sqrt(var + eps)
    h = (X - mu) * rs
    emu = steps * e24 * X.abs().mean(1, keepdim=True) + 2 * e24 * mu.abs()
    e_rs = (steps + 10) * e24 + emu ** 2 / (var + eps)             # relative
    eh = rs * (emu + 2 * e24 * (X - mu).abs()) + h.abs() * e_rs
    y = h * W + B
    ey = W.abs() * eh + 3 * e24 * ((h * W).abs() + (B if isinstance(B, int) else B.abs())) + U[t] * y.abs() + TINY[t]
    gw = G * W
    c1, c2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    e1 = (steps + 3) * e24 * gw.abs().mean(1, keepdim=True)
    e2 = (gw.abs() * eh).mean(1, keepdim=True) + (steps + 4) * e24 * (gw * h).abs().mean(1, keepdim=True)
    dx = rs * (gw - c1 - h * c2)
    inner = gw.abs() + c1.abs() + (h * c2).abs()
    edx = rs * (e1 + h.abs() * e2 + eh * c2.abs() + eh * e2 + 5 * e24 * inner) + rs * inner * e_rs
    edx = edx + U[t] * (dx.abs() + edx) + TINY[t]
    wt = t if w is None and b is None else (w if w is not None else b).dtype
    dw, db = (G * h).sum(0), G.sum(0)
    edw = (G.abs() * eh).sum(0) + (m + 4) * e24 * (G * h).abs().sum(0)
    edb = (m + 4) * e24 * G.abs().sum(0)
    return {"y": (y, ey), "dx": (dx, edx), "dw": (dw, edw + U[wt] * (dw.abs() + edw) + TINY[wt]), "db": (db, edb + U[wt] * (db.abs() + edb) + TINY[wt])}


def check_norm(m, d, dtype, weights="same", bias=True, mean=0.3, scale=1.5, eps=1e-5, x=None):
    from cinema_amd.models.mlp import layer_norm
    g = torch.Generator(device="cuda").manual_seed(m * 31 + d)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x0 = (r(m, d) * scale + mean).to(dtype)
    if x is not None:
        x0 = x(x0)
    wt = torch.float32 if weights == "fp32" else dtype
    w = (1 + 0.2 * r(d)).to(wt) if weights != "none" else None
    b = (0.2 * r(d)).to(wt) if bias else None
    dy = (0.1 * r(m, d)).to(dtype)
    want = norm_bounds(x0, w, b, dy, eps)
    leaves = {k: t.detach().requires_grad_(True) for k, t in (("dx", x0), ("dw", w), ("db", b)) if t is not None}
    y = layer_norm(leaves["dx"], leaves.get("dw"), leaves.get("db"), eps)
    with torch.no_grad():
        assert torch.equal(y, layer_norm(x0, w, b, eps))
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)), y=y.detach())
    for k, v in got.items():
        within(v, *want[k], f"{k} of {m}x{d} {dtype} weights {weights}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [1, 2, 3, 7, 64, 256, 257, 512, 1000, 1024, 1500, 2048, 2049, 4096, 5001, 8192, 16384, 16392, 20011])
def test_layer_norm_matches_its_formula(d, dtype):
    for m in (1, 5, 37):
        check_norm(m, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,d", [(64, 256), (2100, 72), (4500, 520), (1200, 2056), (600, 5000), (70, 33000)])
def test_layer_norm_many_rows(m, d, dtype):
    check_norm(m, d, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weights,bias", [("fp32", True), ("none", False), ("fp32", False), ("none", True)])
def test_layer_norm_weights(weights, bias, dtype):
    for m, d in ((40, 96), (40, 6000), (3, 40000)):
        check_norm(m, d, dtype, weights, bias)


def test_layer_norm_rows_off_centre_and_constant():
    """a mean a thousand times the spread, and rows without any spread"""
    from cinema_amd.models.mlp import layer_norm
    check_norm(20, 512, torch.float32, mean=1000.0, scale=1.0)
    check_norm(20, 9000, torch.float32, mean=-300.0, scale=1.0)
    x = torch.full((9, 260), 3.0, device="cuda", requires_grad=True)
    b = torch.randn(260, device="cuda")
    y = layer_norm(x, None, b)
    assert torch.equal(y, b.expand(9, 260))
    (g,) = torch.autograd.grad(y, x, torch.randn(9, 260, device="cuda"))
    assert torch.isfinite(g).all()


@pytest.mark.parametrize("view", ["rows_of_wider", "offset", "transposed", "three_dims"])
def test_layer_norm_strides(view):
    from cinema_amd.models.mlp import layer_norm

    def make(x):
        m, k = x.shape
        if view == "transposed":
            return x.t().contiguous().t()
        wide = torch.full((m, k + 17), float("nan"), device="cuda", dtype=x.dtype)
        at = 8 if view == "rows_of_wider" else 1
        wide[:, at:at + k] = x
        return wide[:, at:at + k]
    if view == "three_dims":
        x = torch.randn(3, 5, 48, device="cuda")
        assert torch.equal(layer_norm(x).view(15, 48), layer_norm(x.view(15, 48)))
        assert torch.equal(layer_norm(x[0, 0]), layer_norm(x.view(15, 48))[0])
        return
    for dtype in DTYPES:
        for d in (96, 3000):
            check_norm(33, d, dtype, x=make)


def test_layer_norm_non_finite_rows_stay_in_their_rows_and_empty():
    from cinema_amd.models.mlp import layer_norm
    for d in (100, 5000, 40000):
        x = torch.randn(8, d, device="cuda")
        want = layer_norm(x)
        x[2, 3], x[5, 7] = float("nan"), float("inf")
        y = layer_norm(x)
        ok = torch.tensor([0, 1, 3, 4, 6, 7], device="cuda")
        assert torch.isnan(y[2]).all() and torch.isnan(y[5]).any() and torch.equal(y[ok], want[ok])
    w = torch.ones(16, device="cuda", requires_grad=True)
    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    y = layer_norm(x, w)
    g = torch.autograd.grad(y, [x, w], y)
    assert g[0].shape == (0, 16) and not g[1].any()


def test_layer_norm_gradients_match_differences():
    """central differences of the fp32 output in 64-bit sums; step 2^-5 of unit directions on rows of spread 1: the third
    derivative of the normalisation along a unit direction is below 15, the outputs' rounding is divided by 2 h"""
    from cinema_amd.models.mlp import layer_norm
    x, w, b = torch.randn(12, 40, device="cuda"), 1 + 0.1 * torch.randn(40, device="cuda"), 0.1 * torch.randn(40, device="cuda")
    dy = torch.randn(12, 40, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = layer_norm(*leaves)
    for i, (t, g) in enumerate(zip((x, w, b), torch.autograd.grad(y, leaves, dy))):
        d = torch.randn_like(t)
        d /= d.norm()
        h = 2.0 ** -5
        f = lambda s: (layer_norm(*[u + s * h * d if j == i else u for j, u in enumerate((x, w, b))]).double() * dy.double()).sum()
        want = float((f(1) - f(-1)) / (2 * h))
        allowed = h * h / 6 * 15 * float(dy.norm()) + 2.0 ** -20 * float((y.detach().abs() * dy.abs()).sum()) / (2 * h)
        assert abs(float((g.double() * d.double()).sum()) - want) <= allowed, i


# ---- gradient norm ------------------------------------------------------------------------------------------------------------
def make_params(sizes, dtypes, seed=0, scale=0.01):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ps = []
    for i, n in enumerate(sizes):
        t = dtypes[i % len(dtypes)]
        p = torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=t))
        p.grad = (torch.randn(n, generator=g, device="cuda") * scale * (1 + i % 3)).to(t)
        ps.append(p)
    return ps


def norm64(ps, p):
    flat = torch.cat([q.grad.double().flatten() for q in ps if q.grad is not None])
    return float(flat.abs().max() if p == math.inf else flat.abs().pow(p).sum().pow(1 / p))


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("sizes", [[1], [7, 1, 65536, 0, 33], [70001] * 3 + [5] * 100, [(1 << 22) + 3, 1000], [300] * 250])
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16, torch.float32, torch.float16]])
def test_clip_matches_its_formula(sizes, dtypes, p):
    from cinema_amd.optim import clip_grad_norm_, grad_norm
    ps = make_params(sizes, dtypes, seed=len(sizes))
    ps.append(torch.nn.Parameter(torch.zeros(3, device="cuda")))        # no gradient
    want = norm64(ps, p)
    before = [q.grad.clone() if q.grad is not None else None for q in ps]
    assert abs(float(grad_norm(ps, p)) - want) <= want * 2.0 ** -23
    n = clip_grad_norm_(ps, want * 1.01, p)                              # below the bound: untouched
    assert n.dim() == 0 and abs(float(n) - want) <= want * 2.0 ** -23
    assert all(q.grad is None or torch.equal(q.grad, g) for q, g in zip(ps, before))
    m = want / 3
    assert abs(float(clip_grad_norm_(ps, m, p)) - want) <= want * 2.0 ** -23
    c = m / (want + 1e-6)
    for q, g in zip(ps, before):
        if g is not None and g.numel():
            v = g.double() * c
            within(q.grad, v, v.abs() * (U[g.dtype] + 2.0 ** -21) + TINY[g.dtype], f"{g.numel()} {g.dtype}")


def test_clip_agrees_with_torch_on_special_values():
    from cinema_amd.optim import clip_grad_norm_
    for bad in (float("inf"), float("nan")):
        for p in (1.0, 2.0, math.inf):
            a, b = make_params([40, 3000], [torch.float32], 5), make_params([40, 3000], [torch.float32], 5)
            a[1].grad[2999] = b[1].grad[2999] = bad
            n, want = clip_grad_norm_(a, 0.5, p), torch.nn.utils.clip_grad_norm_(b, 0.5, p)
            assert str(float(n)) == str(float(want))
            for x, y in zip(a, b):
                assert torch.equal(torch.isnan(x.grad), torch.isnan(y.grad)) and torch.equal(torch.nan_to_num(x.grad), torch.nan_to_num(y.grad))
    ps = make_params([100], [torch.float32])
    ps[0].grad[5] = float("nan")
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_(ps, 1.0, error_if_nonfinite=True)
    assert torch.isfinite(ps[0].grad[:5]).all()
    big = make_params([1000], [torch.float32], scale=1e25)              # squares beyond fp32
    want = norm64(big, 2.0)
    assert abs(float(clip_grad_norm_(big, 1.0)) - want) <= want * 2.0 ** -23
    small = make_params([1000], [torch.float32], scale=1e-30)
    want = norm64(small, 2.0)
    assert abs(float(clip_grad_norm_(small, 1.0)) - want) <= want * 2.0 ** -23
    zero = make_params([64], [torch.float32], scale=0.0)
    assert float(clip_grad_norm_(zero, 0.0)) == 0.0 and not zero[0].grad.any()


def test_clip_strided_gradients_and_refusals():
    from cinema_amd import _lib
    from cinema_amd.optim import clip_grad_norm_, grad_norm
    p = torch.nn.Parameter(torch.zeros(6, 50, device="cuda"))
    base = torch.randn(50, 12, device="cuda")
    p.grad = base[:, :6].t()
    want, rest = float(p.grad.double().norm()), base[:, 6:].clone()
    g0 = p.grad.clone()
    assert abs(float(clip_grad_norm_(p, 1.0)) - want) <= want * 2.0 ** -23
    within(p.grad, g0.double() / (want + 1e-6), g0.double().abs() * 2.0 ** -21, "strided")
    assert torch.equal(base[:, 6:], rest)
    with pytest.raises(ValueError, match="twice"):
        clip_grad_norm_([p, p], 1.0)
    q = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    flat = torch.ones(12, device="cuda")
    q.grad = flat[:8]
    r = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    r.grad = flat[4:]
    with pytest.raises(ValueError, match="overlaps"):
        clip_grad_norm_([q, r], 1.0)
    assert float(grad_norm([q, r], 1.0)) == 16.0                          # reading twice is no clash
    e = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    e.grad = torch.ones(1, device="cuda").expand(8)
    with pytest.raises((ValueError, RuntimeError)):
        clip_grad_norm_(e, 1.0)
    c = torch.nn.Parameter(torch.zeros(8))
    c.grad = torch.ones(8)
    with pytest.raises(ValueError, match="devices"):
        grad_norm([q, c])
    assert float(grad_norm([])) == 0.0
    none = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    none.grad = torch.zeros(4, device="cuda")
    assert float(clip_grad_norm_([none], 1.0)) == 0.0
    assert _lib.load().cinema_grad_norm_work_bytes(3) > 0


def adam_steps(make_opt, clip, steps, n_tensors=11):
    torch.manual_seed(3)
    ps = [torch.nn.Parameter(torch.randn(37 + 100 * i, device="cuda")) for i in range(n_tensors)]
    opt = make_opt(ps)
    norms = []
    for s in range(steps):
        g = torch.Generator(device="cuda").manual_seed(s)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g, device="cuda") * (0.01 if s % 2 else 1.0)
        norms.append(clip(ps, opt))
        opt.step()
    return ps, norms, opt


def test_adamw_with_clipping_equals_clipping_then_adamw():
    """max_grad_norm in the update against clip_grad_norm_ before it: the same fp32 factor times the same gradient"""
    from cinema_amd.optim import HipAdamW, clip_grad_norm_
    a, na, _ = adam_steps(lambda ps: HipAdamW(ps, lr=1e-2), lambda ps, o: clip_grad_norm_(ps, 0.7), 4)
    for clear in (False, True):
        b, _, opt = adam_steps(lambda ps: HipAdamW(ps, lr=1e-2, max_grad_norm=0.7, clear_grads=clear), lambda ps, o: None, 4)
        # the factor: fp32 of max_norm / (norm + 1e-6), from the norm in 64 bits there, rounded to fp32 here: 2 * 2^-24 apart.
        # an update is lr * m / sqrt(v), at most 3.2 lr with these betas, so its parts moving by 2^-22 move it by 2^-19 lr
        for x, y in zip(a, b):
            assert float((x - y).abs().max()) <= 4 * 1e-2 * 2.0 ** -19 + 4 * 4 * 2.0 ** -24
            assert not clear or not y.grad.any()
        assert abs(float(opt.grad_norm) - float(na[-1])) <= float(na[-1]) * 2.0 ** -23
    c, _, _ = adam_steps(lambda ps: HipAdamW(ps, lr=1e-2, max_grad_norm=1e9), lambda ps, o: None, 3)
    d, _, _ = adam_steps(lambda ps: HipAdamW(ps, lr=1e-2), lambda ps, o: None, 3)
    assert all(torch.equal(x, y) for x, y in zip(c, d))                    # never clipped: the plain update bit for bit
    with pytest.raises(ValueError):
        HipAdamW(c, max_grad_norm=-1.0)


# ---- together -------------------------------------------------------------------------------------------------------------------
def test_operators_are_reproducible_and_replay_in_a_graph():
    """equal bits from equal inputs; a captured block (forward, backward, clip) replays with eager work in between"""
    from cinema_amd.models.mlp import layer_norm, linear_act
    from cinema_amd.optim import clip_grad_norm_
    x, w, b, r, dy = linear_data(3000, 264, 264, torch.bfloat16, res=False)
    nw, nb = torch.ones(264, device="cuda"), torch.zeros(264, device="cuda")
    leaves = [t.requires_grad_(True) for t in (x, w, b, nw, nb)]
    holders = [torch.nn.Parameter(torch.empty(t.shape, device="cuda", dtype=t.dtype)) for t in (w, b, nw, nb)]

    def block():
        y = linear_act(layer_norm(x, nw, nb), w, b, x, "gelu")
        gs = torch.autograd.grad(y, leaves, dy)
        for p, g in zip(holders, gs[1:]):
            p.grad = g
        n = clip_grad_norm_(holders, 0.05)
        return [y, gs[0], n] + [p.grad for p in holders]

    eager = [t.detach().clone() for t in block()]
    again = [t.detach().clone() for t in block()]
    assert all(torch.equal(p, q) for p, q in zip(eager, again))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        block()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        want = [t.detach().clone() for t in block()]
        assert all(torch.equal(p, q) for p, q in zip(got, want)), i


@pytest.mark.parametrize("op", ["linear_act", "layer_norm"])
def test_capture_beside_a_living_eager_graph_is_refused(op):
    """a leaf whose accumulator belongs to the default stream cannot be captured with its gradients; without them it can"""
    from cinema_amd.models.mlp import layer_norm, linear_act
    x = torch.randn(40, 64, device="cuda")
    w = torch.randn(64, 64, device="cuda") if op == "linear_act" else torch.randn(64, device="cuda")
    w.requires_grad_(True)
    call = linear_act if op == "linear_act" else layer_norm
    eager = call(x, w)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            call(x, w)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = call(x, w)
    graph.replay()
    assert torch.equal(y, eager)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = call(x, w)
        (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        v = call(x, w)
        assert torch.equal(y, v) and torch.equal(dw, torch.autograd.grad(v, w, torch.ones_like(v))[0])
        del v


@pytest.mark.parametrize("m,k,n", [(4099, 257, 3), (33001, 33, 4), (300001, 5, 1), (1030, 1024, 2)])
@pytest.mark.parametrize("act", ["none", "relu", "silu"])
def test_linear_few_features_of_many_rows(m, k, n, act):
    check_linear(m, k, n, torch.float32, act)


def test_two_streams_at_once():
    """calls on two streams share nothing"""
    from cinema_amd.models.mlp import linear_act
    data = [linear_data(2500, 136, 264, torch.bfloat16, seed=i) for i in range(2)]
    want = []
    for x, w, b, r, dy in data:
        x.requires_grad_(True), w.requires_grad_(True)
        want.append(torch.autograd.grad(linear_act(x, w, b, r, "silu"), [x, w], dy))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    for _ in range(3):
        got = []
        for s, (x, w, b, r, dy) in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(torch.autograd.grad(linear_act(x, w, b, r, "silu"), [x, w], dy))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for g, v in zip(got, want) for p, q in zip(g, v))


def test_negated_views_and_infinite_gradients():
    """lazily negated inputs count with their sign; relu's closed gates stop an infinite gradient"""
    from cinema_amd.models.mlp import layer_norm, linear_act
    x, w, b, r, dy = linear_data(40, 24, 32, torch.float32)
    assert torch.equal(linear_act(torch._neg_view(x), w, b, r, "none"), linear_act(-x, w, b, r, "none"))
    assert torch.equal(layer_norm(torch._neg_view(x)), layer_norm(-x))
    for rows in (4, 40):
        xg = x[:rows].clone().requires_grad_(True)
        y = linear_act(xg, w, None, None, "relu")
        g = torch.full_like(y, float("inf"))
        (dx,) = torch.autograd.grad(y, xg, torch.where(y > 0, torch.ones_like(g), g))
        assert torch.isfinite(dx).all()


# ---- the framework's own callers --------------------------------------------------------------------------------------------
def regressor_pair(precision, **kw):
    """the regressor on the HIP operators, and the same parameters in torch's layers in 64 bits"""
    from cinema_amd.models.inr_decoder import LatentRegressor
    torch.manual_seed(11)
    own = LatentRegressor([256, 3, 3, 3], precision=precision, **kw).cuda()
    ref = LatentRegressor([256, 3, 3, 3], **kw).cuda().double()
    ref.load_state_dict(own.state_dict())
    return own, ref


@pytest.mark.parametrize("kw", [{}, {"hidden": (64, 64, 32), "layer_norm": True, "residual": True}])
@pytest.mark.parametrize("precision,tol", [("fp32", 2e-6), ("bf16", 3e-2)])
@pytest.mark.parametrize("rows", [1, 64, 300])
def test_latent_regressor_runs_the_operators(rows, precision, tol, kw):
    """three or four layers deep: outputs and gradients in units of their largest value.  fp32: each layer's sums are within
    256 * 2^-24 of their magnitudes in the worst case, a tenth of that in practice for random signs -- 2e-6 allows 2^-19.  bf16:
    weights, rows and gradients are rounded by up to 2^-8 five times along the deepest path (5 * 2^-8 = 2e-2), plus the kinks"""
    own, ref = regressor_pair(precision, **kw)
    x = 0.5 + torch.randn(rows, 256, device="cuda")
    dy = torch.randn(rows, 1, device="cuda")
    xo, xr = x.clone().requires_grad_(True), x.double().requires_grad_(True)
    yo, yr = own(xo), ref(xr)
    assert yo.dtype == torch.float32 and yo.shape == (rows, 1)
    assert float((yo.detach().double() - yr.detach()).abs().max()) <= tol * max(float(yr.detach().abs().max()), 1.0)
    yo.backward(dy)
    yr.backward(dy.double())
    assert set(own.state_dict()) == set(ref.state_dict())
    if precision == "fp32":
        for (n, p), q in zip(own.named_parameters(), ref.parameters()):
            assert float((p.grad.double() - q.grad).abs().max()) <= 20 * tol * max(float(q.grad.abs().max()), 1e-3), n
    else:
        for (n, p), q in zip(own.named_parameters(), ref.parameters()):        # relu's kinks move single entries: the 2-norm
            assert float((p.grad.double() - q.grad).norm()) <= 0.1 * float(q.grad.norm()) + 1e-6, n


def test_latent_regressor_trains_with_clipping():
    """the set as it is used: norm, layers, residual, clipped AdamW -- gradients arrive, the norm is the gradients' own, and the
    parameters move as torch's clip + AdamW move them from the same gradients"""
    from cinema_amd.optim import HipAdamW
    own, _ = regressor_pair("fp32", hidden=(64, 64, 32), layer_norm=True, residual=True)
    opt = HipAdamW(own.parameters(), lr=1e-3, max_grad_norm=0.5)
    twin = [torch.nn.Parameter(p.detach().clone()) for p in own.parameters()]
    topt = torch.optim.AdamW(twin, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)
    x, t = torch.randn(64, 256, device="cuda"), 10 * torch.randn(64, 1, device="cuda")
    for _ in range(3):
        opt.zero_grad()
        ((own(x) - t) ** 2).mean().backward()
        for p, q in zip(own.parameters(), twin):
            q.grad = p.grad.clone()
        want = torch.nn.utils.clip_grad_norm_(twin, 0.5)
        opt.step()
        topt.step()
        assert float(want) > 0.5 and abs(float(opt.grad_norm) - float(want)) <= 1e-5 * float(want)
        for p, q in zip(own.parameters(), twin):
            # an update is at most about lr; the two factors and moments differ by a few 2^-24 relative
            assert float((p.detach() - q.detach()).abs().max()) <= 1e-3 * 1e-3 + float(q.detach().abs().max()) * 2.0 ** -22
            q.data.copy_(p.detach())


@pytest.mark.parametrize("split", ["train", "val"])
def test_trainer_clips_the_whole_step(split):
    """args['optimizer']['max_grad_norm']: the norm over all tables and the decoder, and the update of clipped gradients"""
    from cinema_amd.trainer import HotPathTrainer, SubjectStore
    from test_gpu_trainer import base_args
    outs = []
    for limit in (None, 1e-3):
        args = base_args([32, 3, 3, 3], 64, 2, [1], [1, 4], 1 if split == "val" else 0, "fp32")
        if limit is not None:
            args["optimizer"]["max_grad_norm"] = limit
        torch.manual_seed(0)
        store = SubjectStore.synthetic(3, (16, 16, 16), 155.0 / 16, [155, 155, 155], 1, 4, seed=3, device="cuda:0",
                                       cond_dims=1 if split == "val" else 0)
        store.shuffle(torch.Generator(device="cuda").manual_seed(1))
        tr = HotPathTrainer(args, store, "cuda:0", split=split, keep_grads=True)
        before = [p.detach().clone() for g in tr.opt_local.param_groups for p in g["params"]]
        tr.step(0, 500)
        params = [p for g in tr.opt_local.param_groups for p in g["params"]]
        outs.append((tr, before, params, [p.grad.clone() for p in params]))
    (tr0, _, _, g0), (tr, before, params, grads) = outs
    for a, b in zip(g0, grads):
        # the gradients stay as they were; the trainer's fp32 kernels add with atomics, two runs agree to their parity bound
        assert float((a - b).abs().max()) <= 1e-4 * float(a.abs().max())
    total = float(torch.cat([g.double().flatten() for g in grads]).norm())
    assert tr0.opt_local.grad_norm is None
    assert total > 1e-3 and abs(float(tr.opt_local.grad_norm) - total) <= total * 2.0 ** -22
    for p, b, g, grp in zip(params, before, grads, [gr for gr in tr.opt_local.param_groups for _ in gr["params"]]):
        q = torch.nn.Parameter(b.clone())
        q.grad = g * (1e-3 / (total + 1e-6))
        torch.optim.AdamW([q], lr=grp["lr"], weight_decay=grp["weight_decay"]).step()
        # first step: lr * g / (|g| + eps) with eps = 1e-8; where |g| is near eps the factor's 2^-22 moves it by as much
        assert float((p.detach() - q.detach()).abs().max()) <= grp["lr"] * 2e-5 + float(b.abs().max()) * 2.0 ** -22


# ---- far offsets --------------------------------------------------------------------------------------------------------------
def test_linear_beyond_32_bit_offsets():
    """y and dy of 70 000 x 32 768 values (2.3 G): the last rows and columns against the formula"""
    from cinema_amd.models.mlp import linear_act
    m, k, n = 70000, 8, 32768
    x, w, b, _, _ = linear_data(m, k, n, torch.bfloat16, res=False)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = linear_act(xg, wg, b, None, "silu")
    dy = torch.empty_like(y).normal_(0, 0.1)
    dx, dw = torch.autograd.grad(y, [xg, wg], dy)
    want = linear_bounds(x[-64:], w, b, None, dy[-64:], "silu")
    within(y.detach()[-64:], *want["y"], "y")
    within(dx[-64:], *want["dx"], "dx")
    cols = slice(n - 16, n)
    want = linear_bounds(x, w[cols], b[cols], None, dy[:, cols], "silu")
    within(dw[cols], *want["dw"], "dw")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_linear_longest_reduction(dtype):
    check_linear(16, (1 << 20) - 1, 4, dtype, "silu")
    check_linear(3, (1 << 20) - 1, 2, dtype, "none")


def test_layer_norm_and_clip_beyond_32_bit_offsets():
    from cinema_amd.models.mlp import layer_norm
    from cinema_amd.optim import clip_grad_norm_
    m, d = 530000, 4096
    x = torch.empty(m, d, device="cuda", dtype=torch.bfloat16).normal_(0.3, 1.5).requires_grad_(True)
    w, b = torch.ones(d, device="cuda"), torch.zeros(d, device="cuda")
    y = layer_norm(x, w, b)
    dy = torch.empty_like(y).normal_(0, 0.1)
    (dx,) = torch.autograd.grad(y, x, dy)
    want = norm_bounds(x.detach()[-50:], w, b, dy[-50:], 1e-5)
    within(y.detach()[-50:], *want["y"], "y")
    within(dx[-50:], *want["dx"], "dx")
    del x, y, dy
    g = dx.view(-1)
    p = torch.nn.Parameter(torch.empty(1, device="cuda", dtype=torch.bfloat16).expand(g.numel()))
    p.grad = g
    tail = g[-1000:].double()
    norm = math.sqrt(sum(float(c.double().square().sum()) for c in g.split(1 << 28)))
    assert abs(float(clip_grad_norm_(p, norm / 2)) - norm) <= norm * 2.0 ** -22
    within(g[-1000:], tail * ((norm / 2) / (norm + 1e-6)), tail.abs() * 2.0 ** -7.9, "clipped tail")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k,n", [(2040, 4104, 2040), (2040, 2040, 4104), (1000, 1288, 1001), (1000, 1000, 1288), (12500, 264, 520), (25000, 512, 512)])
def test_linear_where_a_workgroup_is_alone(m, k, n, dtype):
    """as many tiles as compute units, long reductions: four buffers, 64 x 64 and 128 x 128, each memory order, ragged ends"""
    check_linear(m, k, n, dtype, "gelu_tanh")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_linear_largest_tiles(dtype):
    """256 x 256 tiles in all three products, whole and cut by the ends, with and without splits"""
    check_linear(33000, 1032, 4104, dtype, "silu")
    check_linear(33001, 1031, 4103, dtype, "relu", bias=False)


def test_linear_largest_tiles_fp32():
    check_linear(16380, 2050, 1030, torch.float32, "silu")
    check_linear(16384, 2048, 1024, torch.float32, "gelu")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("m,k,n", [(971, 1, 3), (1, 700, 300), (5, 7, 900), (20000, 3, 2), (300, 2, 500), (17, 33, 20), (2, 64, 1000)])
def test_linear_gradients_of_few_values_are_rounded_once(m, k, n, act, dtype):
    """few values of dz, or few sums over it: nothing averages a rounding of dz out, so it stays in 32 bits.  Each gradient is
    then its own value rounded (half a step U at most) plus sums in fp32 and the activation's 2^-21 -- which cancellation among
    the terms magnifies, so they are taken relative to the sums of magnitudes"""
    from cinema_amd.models.mlp import linear_act
    x, w, b, _, dy = linear_data(m, k, n, dtype, seed=m + k + n, res=False)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(linear_act(*leaves, None, act), leaves, dy)
    z = x.double() @ w.double().t() + b.double()
    dz = dy.double() * slope64(z, act)
    e = dy.double().abs() * ((z.abs() + 4) ** 2 * 2.0 ** -21 + CURV * (k + 2) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t() + b.double().abs()))
    for g, v, err in ((got[0], dz @ w.double(), e @ w.double().abs()), (got[1], dz.t() @ x.double(), e.t() @ x.double().abs()), (got[2], dz.sum(0), e.sum(0))):
        sums = (max(m, n) + 2) * 2.0 ** -23 * (err / e.max().clamp_min(1e-30) * dz.abs().max())
        within(g, v, v.abs() * U[dtype] * 1.01 + 1.01 * (err + sums) + TINY[dtype], f"{m}x{k}x{n} {act}")
