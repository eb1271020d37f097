"""torch.autograd.Functions that route the reference's module API into libcinema_hip.so."""
from __future__ import annotations

from typing import Optional

import ctypes as C

import torch

from . import _lib
from . import engine as E


class DecoderState:
    """Per-module mutable state shared between forward and backward."""

    def __init__(self, eng: E.SirenEngine):
        self.engine = eng
        self.k1 = E.TrilerpState()
        self.pack_sig = None
        self.keep_saved = True      # False for a forward under no_grad: the engine then keeps nothing for a backward


def _as_f32(t: torch.Tensor, device) -> torch.Tensor:
    return t.detach().to(device=device, dtype=torch.float32).contiguous()


def _maybe_pack(state: DecoderState, params):
    """Refresh the packed bf16/f32 weight copies.  Always: optimisers that write through raw pointers
    (HipAdamW) do not bump tensor version counters, and one pack launch costs ~25 us."""
    state.engine.pack()


class DecoderFunction(torch.autograd.Function):
    """INR_Decoder.forward of the reference (models/inr_decoder.py:24-36) as ONE autograd node:
    transform -> [idcs_df] gather -> trilinear interpolation -> Siren."""

    @staticmethod
    def forward(ctx, state: DecoderState, coords, latents, cond, tfs, idx, tf_per_sample: bool, *params):
        eng = state.engine
        dev = eng.device
        n = coords.shape[0]
        coords_c = _as_f32(coords, dev)
        lat_c = _as_f32(latents, dev)
        cond_c = _as_f32(cond, dev) if (cond is not None and cond.shape[-1] > 0) else None
        tfs_c = _as_f32(tfs, dev) if tfs is not None else None
        idx_c = idx.detach().to(device=dev, dtype=torch.int32).contiguous()
        eng.workspace(n)
        _maybe_pack(state, params)
        E.k1_forward(eng, state.k1, coords_c, idx_c, lat_c, cond_c, tfs_c, tf_per_sample, n)
        out = eng.forward(n, keep=state.keep_saved)[:n].clone()     # no_grad / inference: nothing is kept
        ctx.state, ctx.n, ctx.version = state, n, eng.version
        ctx.tf_per_sample = tf_per_sample
        ctx.lat_shape = tuple(lat_c.shape)
        ctx.cond_dims = 0 if cond_c is None else cond_c.shape[1]
        ctx.has_cond = cond is not None
        ctx.cond_shape = None if cond is None else tuple(cond.shape)
        ctx.save_for_backward(coords_c, idx_c, tfs_c if tfs_c is not None else coords_c.new_empty(0))
        ctx.has_tfs = tfs_c is not None
        return out

    @staticmethod
    def backward(ctx, gout):
        state, n = ctx.state, ctx.n
        eng = state.engine
        if eng.version != ctx.version:
            raise RuntimeError("cinema_amd: the saved activations of this forward were overwritten by a later forward of "
                               "the same module; call backward() before the next forward (or use a separate module copy)")
        coords_c, idx_c, tfs_c = ctx.saved_tensors
        tfs_c = tfs_c if ctx.has_tfs else None
        ws = eng.ws
        ws.ensure_backward()
        npad = E.round_up(n, E.ROW_ALIGN)
        ws.dout[:n].copy_(gout)
        if npad > n:
            ws.dout[n:npad].zero_()
        need = ctx.needs_input_grad
        want_w = any(need[7:])
        eng.backward(n, ws.dout, weight_grads=want_w)
        want_lat, want_cond, want_tf = need[2], ctx.has_cond and need[3], ctx.has_tfs and need[4]
        dlat, dtfs, dcond = E.k1_backward(eng, state.k1, coords_c, idx_c, ctx.lat_shape, ctx.cond_dims,
                                          tfs_c if want_tf else None, ctx.tf_per_sample, n,
                                          want_latents=want_lat, want_cond=want_cond)
        if ctx.has_cond and need[3] and dcond is None:   # zero-width condition tensor
            dcond = torch.zeros(ctx.cond_shape, device=eng.device)
        pgrads = [None] * (len(need) - 7)
        if want_w:
            g = eng.flat_grad.clone()
            for k, (key, off, shape) in enumerate(eng.layout):
                if need[7 + k]:
                    cnt = 1
                    for s in shape:
                        cnt *= s
                    pgrads[k] = g[off:off + cnt].view(shape)
        return (None, None, dlat, dcond, dtfs, None, None, *pgrads)


class SirenFunction(torch.autograd.Function):
    """Siren.forward of the reference (models/siren.py:59-61) on explicit (coords, latent) rows."""

    @staticmethod
    def forward(ctx, state: DecoderState, coords, latent, *params):
        eng = state.engine
        n = coords.shape[0]
        ws = eng.workspace(n)
        _maybe_pack(state, params)
        npad = E.round_up(n, E.ROW_ALIGN)
        ws.coords_t[:npad].zero_()
        ws.coords_t[:n].copy_(coords.detach())
        ws.lat[:npad].zero_()
        ws.lat[:n, :eng.desc.lat].copy_(latent.detach())
        out = eng.forward(n, keep=state.keep_saved)[:n].clone()
        ctx.state, ctx.n, ctx.version = state, n, eng.version
        return out

    @staticmethod
    def backward(ctx, gout):
        state, n = ctx.state, ctx.n
        eng = state.engine
        if eng.version != ctx.version:
            raise RuntimeError("cinema_amd: saved activations were overwritten by a later forward of the same Siren")
        ws = eng.ws
        ws.ensure_backward()
        npad = E.round_up(n, E.ROW_ALIGN)
        ws.dout[:n].copy_(gout)
        if npad > n:
            ws.dout[n:npad].zero_()
        need = ctx.needs_input_grad
        want_w = any(need[3:])
        eng.backward(n, ws.dout, weight_grads=want_w)
        dcoords = ws.dcoords[:n].clone() if need[1] else None
        dlat = ws.dlat[:n, :eng.desc.lat].clone() if need[2] else None
        pgrads = [None] * (len(need) - 3)
        if want_w:
            g = eng.flat_grad.clone()
            for k, (key, off, shape) in enumerate(eng.layout):
                if need[3 + k]:
                    cnt = 1
                    for s in shape:
                        cnt *= s
                    pgrads[k] = g[off:off + cnt].view(shape)
        return (None, dcoords, dlat, *pgrads)


class LossFunction(torch.autograd.Function):
    """Criterion's data terms (utils.py:84-95) with the gradient w.r.t. the network output
    produced in the same launch.  Returns (total_data, sr_mean, ce_mean); only `total_data`
    = sr_scale*sr_mean + seg_scale*ce_mean carries gradient."""

    @staticmethod
    def forward(ctx, output, target, sr_dims: int, loss_metric: str, class_w: Optional[torch.Tensor], sr_scale: float,
                seg_scale: float):
        n, od = output.shape
        dev = output.device
        out_c = output.detach().contiguous().float()
        tgt_c = target.detach().to(device=dev, dtype=torch.float32).contiguous()
        npad = E.round_up(n, E.ROW_ALIGN)
        dout = torch.empty(npad, od, device=dev, dtype=torch.float32)
        sums = torch.empty(4, device=dev, dtype=torch.float32)
        cw = None if class_w is None else class_w.detach().to(device=dev, dtype=torch.float32).contiguous()
        E.sample_loss(None, out_c, n, sr_dims, od - sr_dims, loss_metric, cw, sr_scale, seg_scale, dout, sums,
                      target=tgt_c)
        sr_mean = sums[0] / float(n * sr_dims)
        if seg_scale > 0:
            den = sums[2] if cw is not None else float(n)
            ce_mean = sums[1] / den
        else:
            ce_mean = torch.zeros((), device=dev)
        total = sr_scale * sr_mean + seg_scale * ce_mean
        ctx.save_for_backward(dout)
        ctx.n = n
        ctx.mark_non_differentiable(sr_mean, ce_mean)
        return total, sr_mean, ce_mean

    @staticmethod
    def backward(ctx, g_total, g_sr, g_ce):
        (dout,) = ctx.saved_tensors
        return dout[:ctx.n] * g_total, None, None, None, None, None, None


class SineLayerFunction(torch.autograd.Function):
    """SineLayer.forward of the reference (models/siren.py:26-36) as one C-ABI call each way
    (cinema_sine_layer_forward / _backward, include/cinema_hip.h).  latent / wl / bl are None for an unmodulated layer."""

    @staticmethod
    def forward(ctx, desc, x, latent, w, b, wl, bl):
        lib = _lib.load()
        n = x.shape[0]
        mod = desc.lat_feat > 0
        f32 = lambda t: None if t is None else t.detach().to(torch.float32).contiguous()
        x32, lat32, w32, b32, wl32, bl32 = f32(x), f32(latent) if mod else None, f32(w), f32(b), f32(wl) if mod else None, \
            f32(bl) if mod else None
        nbytes = lib.cinema_sine_layer_work_bytes(C.byref(desc), n)
        if nbytes < 0:
            _lib.check(-1, "cinema_sine_layer_work_bytes")
        work = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        out = torch.empty(n, desc.out_feat, dtype=torch.float32, device=x.device)
        stream = C.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)
        _lib.check(lib.cinema_sine_layer_forward(C.byref(desc), _lib.ptr(x32), _lib.ptr(lat32), _lib.ptr(w32), _lib.ptr(b32),
                                                 _lib.ptr(wl32), _lib.ptr(bl32), n, _lib.ptr(work), _lib.ptr(out), stream),
                   "cinema_sine_layer_forward")
        ctx.desc, ctx.n, ctx.work, ctx.w32, ctx.mod = desc, n, work, w32, mod
        return out

    @staticmethod
    def backward(ctx, gout):
        lib = _lib.load()
        d, n, dev = ctx.desc, ctx.n, gout.device
        z = lambda *shape: torch.empty(*shape, dtype=torch.float32, device=dev)
        dx, dw, db = z(n, d.in_feat), z(d.out_feat, d.in_feat), z(d.out_feat)
        dlat = z(n, d.lat_feat) if ctx.mod else None
        dwl = z(2 * d.out_feat, d.lat_feat) if ctx.mod else None
        dbl = z(2 * d.out_feat) if ctx.mod else None
        g32 = gout.detach().to(torch.float32).contiguous()
        stream = C.c_void_p(torch.cuda.current_stream(dev).cuda_stream)
        _lib.check(lib.cinema_sine_layer_backward(C.byref(d), _lib.ptr(ctx.w32), n, _lib.ptr(ctx.work), _lib.ptr(g32), _lib.ptr(dx),
                                                  _lib.ptr(dlat), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(dwl), _lib.ptr(dbl), stream),
                   "cinema_sine_layer_backward")
        return None, dx, dlat, dw, db, dwl, dbl


class ConvModFunction(torch.autograd.Function):
    """Modulator's Conv3d(C, C, k, padding='same') over the latent table (models/inr_decoder.py:109-123) through
    cinema_conv_mod_forward / _backward (include/cinema_hip.h)."""

    @staticmethod
    def forward(ctx, table, weight, bias, precision: int):
        lib = _lib.load()
        S, Cc, lx, ly, lz = table.shape
        k = weight.shape[2]
        f32 = lambda t: t.detach().to(torch.float32).contiguous()
        x, w, b = f32(table), f32(weight), f32(bias)
        nbytes = lib.cinema_conv_mod_work_bytes(S, Cc, lx, ly, lz, k, precision)
        if nbytes < 0:
            _lib.check(-1, "cinema_conv_mod_work_bytes")
        work = torch.empty(nbytes, dtype=torch.uint8, device=table.device)
        out = torch.empty_like(x)
        stream = C.c_void_p(torch.cuda.current_stream(table.device).cuda_stream)
        _lib.check(lib.cinema_conv_mod_forward(_lib.ptr(x), _lib.ptr(w), _lib.ptr(b), S, Cc, lx, ly, lz, k, precision, _lib.ptr(work),
                                               _lib.ptr(out), stream), "cinema_conv_mod_forward")
        ctx.save_for_backward(x, w)
        ctx.work, ctx.geom = work, (S, Cc, lx, ly, lz, k, precision)
        return out

    @staticmethod
    def backward(ctx, gout):
        lib = _lib.load()
        x, w = ctx.saved_tensors
        S, Cc, lx, ly, lz, k, precision = ctx.geom
        g = gout.detach().to(torch.float32).contiguous()
        din, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty(Cc, dtype=torch.float32, device=x.device)
        stream = C.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)
        _lib.check(lib.cinema_conv_mod_backward(_lib.ptr(x), _lib.ptr(w), _lib.ptr(g), S, Cc, lx, ly, lz, k, precision,
                                                _lib.ptr(ctx.work), _lib.ptr(din), _lib.ptr(dw), _lib.ptr(db), stream),
                   "cinema_conv_mod_backward")
        return din, dw, db, None


# ---- plain MLP operators (models/mlp.py) -----------------------------------------------------------------------------------
DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}


class _OnDevice:
    """Makes `device` current for a launch if it is not (a kernel goes to the device that is current at the call)."""

    def __init__(self, device):
        self.ctx = None if device.index == torch.cuda.current_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *a):
        if self.ctx is not None:
            self.ctx.__exit__(*a)


def _first_order_only(what: str):
    """A backward pass under create_graph=True: its results would silently carry no graph."""
    if torch.is_grad_enabled():
        raise RuntimeError(f"cinema_amd {what}: the gradients have no second derivative (create_graph=True)")


def _raw_stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _work(nbytes: int, device, what: str):
    if nbytes < 0:
        _lib.check(-1, what)
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _p(t):
    return None if t is None else t.data_ptr()


def _row_major(x2):
    """(x2 or its contiguous copy, row stride in elements) for the kernels: rows contiguous, any stride of at least a row."""
    m, k = x2.shape
    if (x2.stride(1) != 1 and k > 1) or (x2.stride(0) < k and m > 1):
        x2 = x2.contiguous()
    return x2, (x2.stride(0) if m > 1 else k)


def linear_act_forward(x2, w, bias, res2, act: int, keep: bool):
    """(y, z) of contiguous w and 2-d rows; z is None unless `keep` and there is an activation."""
    lib = _lib.load()
    (m, k), n, dev = x2.shape, w.shape[0], x2.device
    y = torch.empty((m, n), dtype=x2.dtype, device=dev)
    z = torch.empty((m, n), dtype=torch.float32 if x2.dtype == torch.float32 else torch.float16, device=dev) if keep and act else None
    if m == 0:
        return y, z
    x2, ldx = _row_major(x2)
    ldr = 0
    if res2 is not None:
        res2, ldr = _row_major(res2)
    dt = DTYPES[x2.dtype]
    with _OnDevice(dev):
        work = _work(lib.cinema_linear_work_bytes(m, k, n, dt, 0), dev, "cinema_linear_work_bytes")
        rc = lib.cinema_linear_forward(x2.data_ptr(), ldx, w.data_ptr(), _p(bias), int(bias is not None and bias.dtype == torch.float32),
                                       _p(res2), ldr, m, k, n, act, dt, _p(z), y.data_ptr(), _p(work), _raw_stream(dev))
    _lib.check(rc, "cinema_linear_forward")
    return y, z


class LinearActFunction(torch.autograd.Function):
    """y = act(x W^T + b) + r as one node (cinema_linear_forward / _backward).  Kept for the backward pass: x, W and, with an
    activation, the pre-activations (fp16 for 16-bit rows, fp32 for fp32)."""

    @staticmethod
    def forward(ctx, x2, w, bias, res2, act: int):
        need = ctx.needs_input_grad
        y, z = linear_act_forward(x2, w, bias, res2, act, need[0] or need[1] or need[2])
        ctx.save_for_backward(x2 if need[1] else None, w if need[0] else None, z)
        ctx.act, ctx.shape = act, (x2.shape[0], x2.shape[1], w.shape[0])
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    def backward(ctx, gout):
        _first_order_only("linear_act")
        need = ctx.needs_input_grad
        x2, w, z = ctx.saved_tensors
        m, k, n = ctx.shape
        dev = gout.device
        if not (need[0] or need[1] or need[2]):
            return None, None, None, gout, None
        new = torch.zeros if m == 0 else torch.empty
        dx = new((m, k), dtype=gout.dtype, device=dev) if need[0] else None
        dw = new((n, k), dtype=gout.dtype, device=dev) if need[1] else None
        db = new((n,), dtype=ctx.bias_dtype, device=dev) if need[2] else None
        if m:
            lib = _lib.load()
            g = gout.contiguous()
            ldx = k
            if x2 is not None:
                x2, ldx = _row_major(x2)
            dt = DTYPES[g.dtype]
            with _OnDevice(dev):
                work = _work(lib.cinema_linear_work_bytes(m, k, n, dt, 1), dev, "cinema_linear_work_bytes")
                rc = lib.cinema_linear_backward(g.data_ptr(), _p(z), _p(x2), ldx, _p(w), m, k, n, ctx.act, dt,
                                                int(ctx.bias_dtype == torch.float32), _p(dx), _p(dw), _p(db), _p(work), _raw_stream(dev))
            _lib.check(rc, "cinema_linear_backward")
        return dx, dw, db, gout if need[3] else None, None


def layer_norm_forward(x2, w, b, eps: float, keep: bool):
    """(y, mean, rstd) of 2-d rows; the statistics are None unless `keep`."""
    lib = _lib.load()
    (m, d), dev = x2.shape, x2.device
    y = torch.empty((m, d), dtype=x2.dtype, device=dev)
    mean, rstd = torch.empty((2, m), dtype=torch.float32, device=dev).unbind(0) if keep else (None, None)
    if m == 0:
        return y, mean, rstd
    x2, ldx = _row_major(x2)
    wt = w if w is not None else b
    with _OnDevice(dev):
        rc = lib.cinema_layer_norm_forward(x2.data_ptr(), ldx, _p(w), _p(b), int(wt is not None and wt.dtype == torch.float32), m, d, eps,
                                           DTYPES[x2.dtype], y.data_ptr(), _p(mean), _p(rstd), _raw_stream(dev))
    _lib.check(rc, "cinema_layer_norm_forward")
    return y, mean, rstd


class LayerNormFunction(torch.autograd.Function):
    """Layer norm over the last dimension as one node (cinema_layer_norm_forward / _backward).  Kept: x, w, the statistics."""

    @staticmethod
    def forward(ctx, x2, w, b, eps: float):
        y, mean, rstd = layer_norm_forward(x2, w, b, eps, True)
        ctx.save_for_backward(x2, w, mean, rstd)
        ctx.w_dtype = w.dtype if w is not None else (b.dtype if b is not None else x2.dtype)
        return y

    @staticmethod
    def backward(ctx, gout):
        _first_order_only("layer_norm")
        need = ctx.needs_input_grad
        x2, w, mean, rstd = ctx.saved_tensors
        (m, d), dev = x2.shape, gout.device
        new = torch.zeros if m == 0 else torch.empty
        dx = new((m, d), dtype=x2.dtype, device=dev) if need[0] else None
        dw = new((d,), dtype=ctx.w_dtype, device=dev) if need[1] else None
        db = new((d,), dtype=ctx.w_dtype, device=dev) if need[2] else None
        if m:
            lib = _lib.load()
            g = gout.contiguous()
            x2, ldx = _row_major(x2)
            dt = DTYPES[x2.dtype]
            with _OnDevice(dev):
                work = None
                if need[1] or need[2]:
                    work = _work(lib.cinema_layer_norm_work_bytes(m, d, dt), dev, "cinema_layer_norm_work_bytes")
                rc = lib.cinema_layer_norm_backward(g.data_ptr(), x2.data_ptr(), ldx, _p(w), int(ctx.w_dtype == torch.float32), mean.data_ptr(),
                                                    rstd.data_ptr(), m, d, dt, _p(dx), _p(dw), _p(db), _p(work), _raw_stream(dev))
            _lib.check(rc, "cinema_layer_norm_backward")
        return dx, dw, db, None
