"""RMSNorm: the root-mean-square norm with the residual's addition that stands before a layer or a feed-forward block, into 16 bits
(forward and gradients) or into 8-bit rows, on the HIP library. Every call enqueues on torch's current stream of the weight's
device; nothing synchronises."""
import ctypes

import torch
from torch import empty_like

from . import _lib as L
from .ffn import DTYPES, _current_device, _modes, _raw_stream, _tracing, eager_only, forward_ad, stream_here
from .q8 import ROW_DTYPES, Rows8

F32 = torch.float32
MOST_H = 16384


class RMSNorm:
    """y = v w / sqrt(mean(v^2) + eps) over the last dimension, v = x, or x + residual as the stream holds it: r = x + residual is
    summed in fp32 and rounded to residual's type, and the norm is of r.

    weight: [H] fp16, bf16 or fp32, contiguous on a device, H a multiple of 8 to 16,384; dtype: of y, fp16 or bf16 (default the
    weight's; fp32 weights need it). x and residual [..., H] of dtype or fp32 each, so that a MoELayer's fp32 output can go into a
    stream of 16 bits. forward(x) -> y; forward(x, residual) -> (y, r). Where autograd records, y and r carry the gradients of x,
    residual and weight (the rounding of r passes them as they are); the forward pass then keeps r (x without a residual), which must
    not be changed before the backward pass. Passes with gradients may be captured as GatedFFN's may. A row's squares are summed in
    fp32: one whose sum overflows (a norm past 1.8e19) has y 0."""

    def __init__(self, weight, eps=1e-6, dtype=None):
        self.weight, self.eps, self.dtype = weight, eps, dtype
        self._check()

    def _check(self):
        """The weight and options as they are now, and what follows from them."""
        w, eps, dtype = self.weight, self.eps, self.dtype
        if not torch.is_tensor(w) or w.dim() != 1 or w.dtype not in ROW_DTYPES or not w.is_cuda:
            raise ValueError("RMSNorm: weight must be an fp16, bf16 or fp32 device tensor [H]")
        if w.shape[0] <= 0 or w.shape[0] % 8 or w.shape[0] > MOST_H:
            raise ValueError(f"RMSNorm: H ({w.shape[0]}) must be a positive multiple of 8, at most {MOST_H}")
        if not w.is_contiguous() or w.data_ptr() % 16:
            raise ValueError("RMSNorm: weight must be contiguous and 16-byte aligned")
        out = w.dtype if dtype is None else dtype
        if out not in DTYPES or w.dtype not in (out, torch.float32):
            raise ValueError(f"RMSNorm: y must be fp16 or bf16 and the weight of that type or fp32, got {out} and {w.dtype}")
        # (what fp32 makes of it: the kernels get it so)
        if not 2.0 ** -149 <= eps <= torch.finfo(F32).max:
            raise ValueError(f"RMSNorm: eps must be positive and finite, got {eps}")
        self._out, self.hidden_size, self.device = out, w.shape[0], w.device
        self._checked = (w, eps, dtype, w.data_ptr(), w.dtype, w.shape[0])
        self._index, self._descs = w.device.index, {}

    def _current(self):
        """Checks again what was replaced since: an attribute, or what the weight tensor holds (Parameter.data)."""
        w, eps, dtype, at, wt, H = self._checked
        if not (w is self.weight and eps == self.eps and dtype is self.dtype and w.data_ptr() == at and w.dtype is wt and w.numel() == H and
                w.is_contiguous()):
            self._check()

    def __getstate__(self):
        """Without the calls' descriptors, which hold addresses: a copy has a weight of its own."""
        return {**self.__dict__, "_descs": {}, "_checked": (None,) * 6}

    def _desc(self, xt, rt):
        d = self._descs.get((xt, rt))
        if d is None:
            _, _, _, at, wt, H = self._checked
            d = self._descs[xt, rt] = ctypes.pointer(L.NormDesc(H, DTYPES[self._out], ROW_DTYPES[xt], ROW_DTYPES[rt], ROW_DTYPES[wt], self.eps, at))
        return d

    def _given(self, x, name):
        """x of [..., H], checked, contiguous and 16-byte aligned (a copy only where it is neither), and its address."""
        dt, H = x.dtype, self.hidden_size
        if (dt is not self._out and dt is not F32) or x.get_device() != self._index or not x.dim() or x.size(-1) != H:
            raise ValueError(f"RMSNorm: expected {name} {self._out} or fp32 [..., {H}] on {self.device}, got {dt} {tuple(x.shape)} on {x.device}")
        p = x.data_ptr()
        if p & 15 or not x.is_contiguous():
            x = x.clone(memory_format=torch.contiguous_format)
            p = x.data_ptr()
        return x, p

    # (a decode token's call is the host's time: 8.6 us, 3.9 of them the library's call and 2.3 the two results' allocations)
    def _run(self, x, residual, want_y, want_rows):
        """(y, rows, r), None what is not wanted. Behind _current()."""
        x, xp = self._given(x, "x")
        if _current_device() != self._index:    # (kernels go to the current device)
            with torch.cuda.device(self.device):
                return self._run(x, residual, want_y, want_rows)
        rt = xt = x.dtype
        rp = sp = yp = y = r = rows = to = None
        if residual is not None:
            residual, rp = self._given(residual, "residual")
            if residual.shape != x.shape:
                raise ValueError(f"RMSNorm: x {tuple(x.shape)} and residual {tuple(residual.shape)} must be of one shape")
            rt, r = residual.dtype, empty_like(residual)
            sp = r.data_ptr()
        if want_y:
            y = empty_like(x) if xt is self._out else empty_like(x, dtype=self._out)
            yp = y.data_ptr()
        T = x.numel() // self.hidden_size
        if want_rows:
            rows = Rows8._empty(T, self.hidden_size, self.device, self._out, x.shape)
            to = rows.struct
        if T:
            rc = L.lib().bmx_rms_norm(self._desc(xt, rt), xp, rp, T, sp, yp, to, _raw_stream(self._index))
            if rc:
                L.check(rc, "bmx_rms_norm")
        return y, rows, r

    def _enter(self, who, x, residual):
        """Checks that come before any work; whether autograd records."""
        self._current()
        if forward_ad._current_level >= 0 or _tracing() or _modes():
            eager_only(who, x, residual, self.weight)
        return ((x.requires_grad or self.weight.requires_grad or (residual is not None and residual.requires_grad)) and
                torch.is_grad_enabled())

    def forward(self, x, residual=None):
        if self._enter("RMSNorm", x, residual):
            got = _RMSNormFunction.apply(x, residual, self.weight, self)
            return got if residual is not None else got[0]
        y, _, r = self._run(x, residual, True, False)
        return y if residual is None else (y, r)

    __call__ = forward

    def rows8(self, x, residual=None):
        """The norm in 8 bits for ops.q8_linear and a GatedFFN of 8-bit weights: Rows8, or (Rows8, r) with a residual. The codes are
        of y before any rounding to 16 bits. No gradients."""
        self.refuse_grad(x, residual)
        _, rows, r = self._run(x, residual, False, True)
        return rows if residual is None else (rows, r)

    def both(self, x, residual=None):
        """y and its 8-bit rows in one pass: (y, Rows8), or (y, Rows8, r) with a residual. No gradients."""
        self.refuse_grad(x, residual)
        y, rows, r = self._run(x, residual, True, True)
        return (y, rows) if residual is None else (y, rows, r)

    def refuse_grad(self, x, residual):
        """What the forms without gradients refuse."""
        if self._enter("RMSNorm", x, residual):
            raise ValueError("RMSNorm: 8-bit rows have no gradients (torch.no_grad(), or forward)")


class _RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, norm):
        y, _, r = norm._run(x, residual, True, False)
        ctx.set_materialize_grads(False)
        v = x if r is None else r
        ctx.save_for_backward(weight, v)
        # (the descriptor holds the weight's address: asked for again below)
        ctx.desc, ctx.weight, ctx.device = norm._desc(x.dtype, v.dtype), weight, norm.device
        ctx.xt, ctx.vt, ctx.summed, ctx.shape = x.dtype, v.dtype, r is not None, v.shape
        return y, r

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dr):
        weight, v = ctx.saved_tensors
        d, dev, xt, rt, summed = ctx.desc, ctx.device, ctx.xt, ctx.vt, ctx.summed
        H = d.contents.H
        # (what hooks give back of the weight lies elsewhere; the weight itself does where its data was replaced)
        if weight.shape != (H,) or ROW_DTYPES.get(weight.dtype) != d.contents.weight_dtype or weight.device != dev or \
                (weight is ctx.weight and (weight.data_ptr() != d.contents.weight or not weight.is_contiguous())):
            raise RuntimeError("RMSNorm: the weight was replaced between the forward and the backward pass, or hooks gave its saved value back "
                               f"as {weight.dtype} {tuple(weight.shape)} on {weight.device}")
        if v.dtype is not rt or v.device != dev or v.shape != ctx.shape:
            raise RuntimeError(f"RMSNorm: hooks gave the saved rows back as {v.dtype} {tuple(v.shape)} on {v.device}")
        s = stream_here(dev)
        if s is None:                           # autograd's threads have a current device of their own
            with torch.cuda.device(dev):
                return _RMSNormFunction.backward(ctx, dy, dr)
        nx, nr, nw, _ = ctx.needs_input_grad
        if dy is None:                          # r alone was used (or neither)
            return dr.to(xt) if nx and dr is not None else None, dr if nr else None, torch.zeros_like(weight) if nw else None, None
        v, dy, weight = _dense(v), _dense(dy), _dense(weight)
        if weight.data_ptr() != d.contents.weight:
            c = d.contents
            d = L.NormDesc(c.H, c.dtype, c.x_dtype, c.residual_dtype, c.weight_dtype, c.eps, weight.data_ptr())
        if dr is not None:
            dr = _dense(dr)
        one = summed and rt is xt               # x's and residual's gradients are the same values
        dx = torch.empty_like(v, dtype=xt) if nx or (nr and one) else None
        dres = torch.empty_like(v) if nr and not one else None
        lib, T, dw, ws, need = L.lib(), v.numel() // H, None, None, 0
        if nw:
            dw = torch.empty_like(weight)
            need = lib.bmx_rms_norm_backward_workspace(d, T)
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
        ptr = lambda t: None if t is None else t.data_ptr()
        L.check(lib.bmx_rms_norm_backward(d, v.data_ptr(), summed, T, dy.data_ptr(), ptr(dr), ptr(dx), ptr(dres), ptr(dw), ptr(ws), need, s),
                "bmx_rms_norm_backward")
        return dx if nx else None, (dx if one else dres) if nr else None, dw, None


def _dense(t):
    """t contiguous and 16-byte aligned."""
    return t if t.is_contiguous() and not t.data_ptr() & 15 else t.clone(memory_format=torch.contiguous_format)
