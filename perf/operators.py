"""The operators of an MLP block's training step, and cases that time them: a linear layer with bias, activation and residual
in its epilogue, layer norm, both with their gradients, and the global gradient norm with clipping over many tensors.

`own` chooses what `run` computes with: elementary torch operations in 32 bits (False) or the package's kernels (True)."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
ACTIVATIONS = ("none", "relu", "gelu", "gelu_tanh", "silu")


def _linear(name, rows, inp, out, dtype, act, residual, train, bias=True):
    return {"name": name, "op": "linear", "rows": rows, "inp": inp, "out": out, "dtype": dtype, "act": act, "residual": residual,
            "bias": bias, "train": train}


def _norm(name, rows, width, dtype, train, weights="same"):
    return {"name": name, "op": "layer_norm", "rows": rows, "width": width, "dtype": dtype, "weights": weights, "train": train}


def _clip(name, sizes, dtype, max_norm, norm_type=2.0):
    return {"name": name, "op": "clip", "sizes": sizes, "dtype": dtype, "max_norm": max_norm, "norm_type": norm_type}


# parameter tensors of the decoder at hidden 512 with five hidden layers, three of them modulated by a 256-wide latent, then
# the latent table of 64 subjects and their rigid embeddings
DECODER = "9216,12,1536,512," + "262144,512,262144,1024," * 3 + "262144,512,262144,512,442368,384"


def listed():
    return [
        # the first layer of the latent regressor on the latents of 64 subjects: the smallest call, latency counts
        _linear("linear_regressor_fp32", 64, 256, 64, "fp32", "relu", False, False),
        # one sample through a wide layer, as a served model answers it: bound by reading the weights
        _linear("linear_one_row_bf16", 1, 1024, 4096, "bf16", "silu", False, False),
        # a residual block at the decoder's width on one training batch of coordinates, evaluated
        _linear("linear_block_bf16", 25000, 512, 512, "bf16", "gelu", True, False),
        # sizes that divide nothing (a latent with conditions appended, an odd hidden width)
        _linear("linear_odd_fp16", 8191, 257, 1283, "fp16", "silu", True, False),
        # the expanding product of a wide MLP over a dense evaluation's chunk of coordinates: the largest product
        _linear("linear_wide_bf16", 32768, 1024, 4096, "bf16", "gelu_tanh", False, False),
        # the same residual block in training: output, and every gradient
        _linear("linear_block_train_bf16", 25000, 512, 512, "bf16", "gelu", True, True),
        # training in exact 32-bit arithmetic with a latent plus one condition channel as input
        _linear("linear_train_fp32", 6400, 257, 512, "fp32", "silu", False, True),
        # normalising the latents of 64 subjects in training: the smallest call
        _norm("norm_latents_train_fp32", 64, 256, "fp32", True),
        # the residual stream at the decoder's width, evaluated
        _norm("norm_block_bf16", 25000, 512, "bf16", False),
        # a wide residual stream in training, 16-bit activations and 32-bit weights: the largest
        _norm("norm_wide_train_bf16", 16384, 4096, "bf16", True, "fp32"),
        # every gradient of the decoder's training step, above the bound
        _clip("clip_decoder_fp32", DECODER, "fp32", 0.25),
        # the gradients of a wide network in 16 bits, 60 ragged tensors
        _clip("clip_many_bf16", ",".join(["4194304,1048577,4096,1023"] * 15), "bf16", 1.0),
    ]


def _spread(rng, lo, hi):
    """A whole number, spread evenly over its logarithm; about half of them made odd."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n | 1 if rng.random() < 0.5 else n))


def draw(rng):
    op = rng.choice(["linear", "linear", "layer_norm", "clip"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "linear":
        train = rng.random() < 0.5
        rows, inp, out = _spread(rng, 1, 65536), _spread(rng, 1, 4096), _spread(rng, 1, 4096)
        # no more work than the largest listed product
        most = 32768 * 1024 * 4096 // ((3 if train else 1) * (8 if dtype == "fp32" else 1))
        rows = max(1, min(rows, most // (inp * out)))
        return _linear("", rows, inp, out, dtype, rng.choice(ACTIVATIONS), rng.random() < 0.5, train, rng.random() < 0.8) | {"name": "drawn"}
    if op == "layer_norm":
        width = _spread(rng, 4, 16384)   # below that dx is all cancellation
        rows = max(1, min(_spread(rng, 1, 65536), 16384 * 4096 * 2 // (BYTES[dtype] * width)))
        return _norm("drawn", rows, width, dtype, rng.random() < 0.6, rng.choice(["same", "fp32", "none"]))
    sizes = [_spread(rng, 1, 2000000) for _ in range(_spread(rng, 1, 60))]
    return _clip("drawn", ",".join(map(str, sizes)), dtype, rng.choice([0.1, 1.0, 1e6]), rng.choice([2.0, 2.0, 2.0, 1.0, math.inf]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 17)
    t = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=t):
        return (torch.randn(*shape, generator=g, device="cuda") * scale + mean).to(dtype)

    s = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inp"], case["out"]
        s["x"] = normal(m, k)                                       # what a layer norm hands on
        s["w"] = normal(n, k, scale=1.0 / math.sqrt(k))
        s["b"] = normal(n, scale=0.1) if case["bias"] else None
        s["r"] = normal(m, n) if case["residual"] else None
        if case["train"]:
            s["dy"] = normal(m, n, scale=0.01)
    elif case["op"] == "layer_norm":
        m, d = case["rows"], case["width"]
        s["x"] = normal(m, d, scale=1.5, mean=0.3)                  # a residual stream is off centre
        wt = torch.float32 if case["weights"] == "fp32" else t
        s["w"] = normal(d, scale=0.1, mean=1.0, dtype=wt) if case["weights"] != "none" else None
        s["b"] = normal(d, scale=0.1, dtype=wt) if case["weights"] != "none" else None
        if case["train"]:
            s["dy"] = normal(m, d, scale=0.01)
    else:
        s["params"] = [torch.empty(n, device="cuda", dtype=t) for n in map(int, case["sizes"].split(","))]
        for i, p in enumerate(s["params"]):
            p.grad = normal(p.numel(), scale=0.003 * (1 + i % 5))   # layers differ in the size of their gradients
    if case.get("train"):
        for k in ("x", "w", "b", "r"):
            if s.get(k) is not None:
                s[k].requires_grad_(True)
    return s


# ---- plain forms: `ft` is the type that everything is computed in ---------------------------------------------------------
def _act(z, act):
    """act(z) and its derivative."""
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        sg = torch.sigmoid(z)
        return z * sg, sg * (1 + z * (1 - sg))
    return z, None


def _plain_linear(s, ft):
    x, w = s["x"].detach().to(ft), s["w"].detach().to(ft)
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].detach().to(ft)
    y, slope = _act(z, s["case"]["act"])
    if s["r"] is not None:
        y = y + s["r"].detach().to(ft)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].to(ft)
    dz = dy if slope is None else dy * slope
    got = {"y": y, "dx": dz @ w, "dw": dz.t() @ x}
    if s["b"] is not None:
        got["db"] = dz.sum(0)
    if s["r"] is not None:
        got["dr"] = dy
    return got


def _plain_norm(s, ft, eps=1e-5):
    x = s["x"].detach().to(ft)
    c = x - x.mean(-1, keepdim=True)
    rs = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    h = c * rs
    y = h if s["w"] is None else h * s["w"].detach().to(ft) + s["b"].detach().to(ft)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].to(ft)
    gw = dy if s["w"] is None else dy * s["w"].detach().to(ft)
    got = {"y": y, "dx": rs * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))}
    if s["w"] is not None:
        got["dw"], got["db"] = (dy * h).sum(0), dy.sum(0)
    return got


def _norm_of(parts, p):
    """The p-norm of all parts' values, from each part's own."""
    if p == math.inf:
        return torch.stack([v.abs().max() for v in parts]).max()
    if p == 1.0:
        return torch.stack([v.abs().sum() for v in parts]).sum()
    return torch.sqrt(torch.stack([(v * v).sum() for v in parts]).sum())


def _plain_clip(s, ft):
    c = s["case"]
    parts = [p.grad.to(ft) for p in s["params"]]
    total = _norm_of(parts, c["norm_type"])
    scale = torch.clamp(c["max_norm"] / (total + 1e-6), max=1.0)
    return total, [v * scale for v in parts]


def _whole(tensors):
    """The tensors' values in one, so that 60 of them are one output."""
    return torch.cat([t.reshape(-1) for t in tensors])


def _rounded(got, s):
    """Each output in the type of what it belongs to, rounded once."""
    like = {"y": "x", "dx": "x", "dw": "w", "db": "b", "dr": "r"}
    return {k: v.to(s[like[k]].dtype) for k, v in got.items()}


def run(state):
    s, c = state, state["case"]
    if c["op"] == "clip":
        if own:
            from cinema_amd.optim import clip_grad_norm_
            total = clip_grad_norm_(s["params"], c["max_norm"], c["norm_type"])
        else:
            total, scaled = _plain_clip(s, torch.float32)
            [p.grad.copy_(v) for p, v in zip(s["params"], scaled)]
        grads = [p.grad for p in s["params"]]
        return {"norm": total, "grads": grads}
    if own:
        from cinema_amd.models.mlp import layer_norm, linear_act
        if not c["train"]:
            with torch.no_grad():
                return {"y": linear_act(s["x"], s["w"], s["b"], s["r"], c["act"]) if c["op"] == "linear" else layer_norm(s["x"], s["w"], s["b"])}
        y = linear_act(s["x"], s["w"], s["b"], s["r"], c["act"]) if c["op"] == "linear" else layer_norm(s["x"], s["w"], s["b"])
        names = [k for k in ("x", "w", "b", "r") if s.get(k) is not None]
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        return {"y": y.detach()} | {"d" + k: g for k, g in zip(names, grads)}
    with torch.no_grad():
        return _rounded(_plain_linear(s, torch.float32) if c["op"] == "linear" else _plain_norm(s, torch.float32), s)


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inp"], case["out"]
        values = m * k + n * k + m * n * (1 + case["residual"]) + n * case["bias"]
        if case["train"]:
            values += m * n + m * k + n * k + n * case["bias"]
        return {"bytes": b * values, "flops": 2 * m * n * k * (3 if case["train"] else 1)}
    if case["op"] == "layer_norm":
        m, d = case["rows"], case["width"]
        wb = {"same": b, "fp32": 4, "none": 0}[case["weights"]]
        return {"bytes": m * d * b * (4 if case["train"] else 2) + d * wb * (4 if case["train"] else 2), "flops": m * d * (20 if case["train"] else 8)}
    values = sum(map(int, case["sizes"].split(",")))
    return {"bytes": 2 * b * values, "flops": 3 * values}


# ---- the definitions in 64 bits, written apart from the plain forms --------------------------------------------------------
def _exact_act(z, act):
    """act by its definition; its derivative comes from differentiating this."""
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":
        return z / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z * 1.0


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        flat = _whole([p.grad for p in s["params"]]).double()
        p = case["norm_type"]
        total = flat.abs().max() if p == math.inf else flat.abs().pow(p).sum().pow(1 / p)
        flat = flat * min(1.0, case["max_norm"] / (float(total) + 1e-6))
        grads = list(torch.split(flat, [q.numel() for q in s["params"]]))
        return {"norm": total, "grads": grads}
    names = [k for k in ("x", "w", "b", "r") if s.get(k) is not None]
    d = {k: s[k].detach().double().requires_grad_(True) for k in names}
    with torch.enable_grad():
        if case["op"] == "linear":
            y = _exact_act(d["x"].matmul(d["w"].transpose(0, 1)) + d.get("b", 0.0), case["act"]) + d.get("r", 0.0)
        else:
            var, mu = torch.var_mean(d["x"], dim=-1, correction=0, keepdim=True)
            y = (d["x"] - mu) * torch.rsqrt(var + 1e-5) * d.get("w", 1.0) + d.get("b", 0.0)
        got = {"y": y.detach()}
        if case["train"]:
            got |= {"d" + k: v for k, v in zip(names, torch.autograd.grad(y, [d[k] for k in names], s["dy"].double()))}
    return got
