"""GatedFFN: the gated feed-forward block y = act(x Wg^T, x Wu^T) Wd^T outside the routed experts (a model's leading dense
layers, a shared expert that the checkpoint keeps out of the trellis records), forward and backward, on the HIP library.

The reference runs these modules as exllamav3 MLPs beside its BlockSparseMLP hooks (engine/tiers.py:703-739 wraps the routed
experts only); here the block is a MoELayer's shared_ffn or a module of its own. Every call enqueues on torch's current
stream of the weights' device; nothing synchronises."""
import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib as L

DTYPES = {torch.float16: L.DT_FP16, torch.bfloat16: L.DT_BF16}


def rows_of(x, K, dtype, device, name):
    """x [..., K] as contiguous 16-byte aligned rows [T, K] (a copy only where x is neither)."""
    shape = x.shape
    if x.device != device or x.dtype != dtype or not shape or shape[-1] != K:
        raise ValueError(f"{name}: expected {dtype} [..., {K}] on {device}, got {x.dtype} {tuple(shape)} on {x.device}")
    if len(shape) != 2:
        x = x.reshape(-1, K)
    if not x.is_contiguous():
        x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


_raw_stream = torch._C._cuda_getCurrentRawStream
# (torch.cuda.current_device behind its check that CUDA runs, which it does where a device tensor is)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def stream_here(device):
    """The handle of the current stream of device if that is the current device, else None (the caller then enters it:
    kernels go to the current device). The handle is read without making a Stream object: that costs 2 us, as much as a
    decode call's other host work together."""
    index = device.index
    return _raw_stream(index) if _current_device() == index else None


# where a program is followed by its torch operations, one of these says so (asked before eager_only: 0.15 us of a call)
_tracing, _modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack


def eager_only(who, *tensors):
    """Refuses what follows a program by its torch operations: the kernels are called by address, so forward-mode
    derivatives would come out as none, and a traced program would hold the result's allocation and nothing that fills it.
    (torch.compile runs the calls between its graphs; other tracers have no addresses to give.)"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{who}: no forward-mode derivatives")
    if _tracing() or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise RuntimeError(f"{who}: cannot be traced")


class GatedFFN:
    """gate, up [I, H] and down [H, I]: contiguous fp16 or bf16 device tensors of one type (H, I multiples of 8), three Q4Matrix
    (gate and up of one group size), or three Q8Matrix (H, I multiples of 8; x and act(g, u) are quantized per token); with 4 or 8
    bits x may be fp16 or bf16, and there are no gradients. act: ACT_SILU, ACT_GELU (tanh), ACT_RELU2 or ACT_SILU_OAI; act_limit:
    the activation's clamp (0: none), both as MoELayer's.

    forward(x) -> y, x [..., H] of the weights' type (8-bit weights: or Rows8, as RMSNorm.rows8 gives them). Where autograd
    records (x or a weight requires grad), y carries the gradients of x and of the three weights; the forward pass then keeps
    x, g and u (fp32 [T, I]) and h (16 bits). Passes with gradients may be captured into a graph through torch.autograd.grad;
    with backward(), which accumulates into the leaves, only while no eager result of the same leaves is alive (torch's
    accumulation belongs to the stream that the leaf was first used on)."""

    def __init__(self, gate, up, down, act=L.ACT_SILU, act_limit=0.0):
        self.gate, self.up, self.down = gate, up, down
        self.act, self.act_limit = act, act_limit
        self._check()

    def _check(self):
        """The weights and options as they are now, and what follows from them."""
        gate, up, down = weights = self.gate, self.up, self.down
        quantized = not any(torch.is_tensor(w) for w in weights)
        bits = 16
        if quantized:
            from .q8 import Q8Matrix
            bits = 8 if isinstance(gate, Q8Matrix) else 4
            if any(isinstance(w, Q8Matrix) != (bits == 8) for w in weights):
                raise ValueError("GatedFFN: three tensors, three Q4Matrix or three Q8Matrix")
            I, H = gate.N, gate.K
            for name, q, shape in (("gate", gate, (I, H)), ("up", up, (I, H)), ("down", down, (H, I))):
                if (q.N, q.K) != shape or q.device != gate.device:
                    raise ValueError(f"GatedFFN: {name} must be {list(shape)} on {gate.device}, got {[q.N, q.K]} on {q.device}")
            if bits == 8 and (H % 8 or I % 8):
                raise ValueError(f"GatedFFN: H ({H}) and I ({I}) must be multiples of 8")
            if bits == 4 and gate.group != up.group:
                raise ValueError(f"GatedFFN: gate and up must have groups of one size, got {gate.group} and {up.group}")
        else:
            I, H = self._check_tensors(gate, up, down)
        if self.act not in (L.ACT_SILU, L.ACT_GELU, L.ACT_RELU2, L.ACT_SILU_OAI):
            raise ValueError(f"GatedFFN: unknown activation {self.act}")
        if not self.act_limit >= 0.0:
            raise ValueError(f"GatedFFN: act_limit must be 0 (off) or positive, got {self.act_limit}")
        self.act_limit = float(self.act_limit)
        self.quantized, self.bits = quantized, bits
        self.hidden_size, self.intermediate_size = H, I
        self.device = gate.device
        self.dtype = None if quantized else gate.dtype      # None: the input's
        self._checked = (*weights, self.act, self.act_limit)
        if not quantized:
            self._at = tuple(w.data_ptr() for w in weights), gate.shape, down.shape
        self._descs = {}

    def _current(self):
        """Checks again what was replaced since: an attribute, or (16 bits) what a weight tensor holds (Parameter.data). A call
        hands the kernels addresses, so one with unchecked sizes would read past them. (A weight on another device lies at another
        address.)"""
        g, u, d, act, limit = self._checked
        same = g is self.gate and u is self.up and d is self.down and act == self.act and limit == self.act_limit
        if same and not self.quantized:
            (at, gs, ds), dt = self._at, self.dtype
            same = ((g.data_ptr(), u.data_ptr(), d.data_ptr()) == at and g.shape == gs and u.shape == gs and d.shape == ds and
                    g.is_contiguous() and u.is_contiguous() and d.is_contiguous() and
                    g.dtype is dt and u.dtype is dt and d.dtype is dt)
        if not same:
            self._check()

    def __getstate__(self):
        """Without the calls' descriptors, which hold addresses: a copy has weights of its own."""
        return {**self.__dict__, "_descs": {}}

    @staticmethod
    def _check_tensors(gate, up, down):
        if not all(torch.is_tensor(w) for w in (gate, up, down)):
            raise ValueError("GatedFFN: three tensors, three Q4Matrix or three Q8Matrix")
        if gate.dim() != 2 or gate.dtype not in DTYPES:
            raise ValueError(f"GatedFFN: gate must be fp16 or bf16 [I, H], got {gate.dtype} {tuple(gate.shape)}")
        I, H = gate.shape
        for name, w, shape in (("gate", gate, (I, H)), ("up", up, (I, H)), ("down", down, (H, I))):
            if tuple(w.shape) != shape or w.dtype != gate.dtype or not w.is_cuda or w.device != gate.device:
                raise ValueError(f"GatedFFN: {name} must be {gate.dtype} {list(shape)} on {gate.device}, got {w.dtype} "
                                 f"{list(w.shape)} on {w.device}")
            if not w.is_contiguous() or w.data_ptr() % 16:
                raise ValueError(f"GatedFFN: {name} must be contiguous and 16-byte aligned")
        if H <= 0 or I <= 0 or H % 8 or I % 8:
            raise ValueError(f"GatedFFN: H ({H}) and I ({I}) must be positive multiples of 8")
        return I, H

    def _tensors(self):
        return () if self.quantized else (self.gate, self.up, self.down)

    def desc(self, dtype=None):
        """The call descriptor for an input of dtype (default: the weights')."""
        self._current()
        return self._desc(dtype)

    def _desc(self, dtype):
        """Of the weights as _current() has left them, kept for the next call."""
        d = self._descs.get(dtype)
        if d is None:
            if self.quantized:
                ref = lambda q: ctypes.pointer(q.struct)
                kind = L.Ffn8Desc if self.bits == 8 else L.Ffn4Desc
                d = kind(DTYPES[dtype], self.act, self.act_limit, 0, ref(self.gate), ref(self.up), ref(self.down))
            else:
                d = L.FfnDesc(self.hidden_size, self.intermediate_size, DTYPES[self.dtype], self.act, self.act_limit, 0, *self._at[0])
            self._descs[dtype] = d
        return d

    def _rows(self, x):
        if self.quantized and x.dtype not in DTYPES:
            raise ValueError(f"GatedFFN: x must be fp16 or bf16, got {x.dtype}")
        return rows_of(x, self.hidden_size, self.dtype or x.dtype, self.device, "GatedFFN: x")

    def _workspace(self, need):
        if need == 0:
            L.check(L.BMX_ERR_ARG, "GatedFFN")
        return torch.empty(need, dtype=torch.uint8, device=self.device)

    def forward(self, x):
        self._current()
        if self.bits == 8:
            return self._forward8(x)
        if forward_ad._current_level >= 0 or _tracing() or _modes():
            eager_only("GatedFFN", x, *self._tensors())
        if not self.quantized and torch.is_grad_enabled() and (x.requires_grad or self.gate.requires_grad or
                                                               self.up.requires_grad or self.down.requires_grad):
            return _GatedFFNFunction.apply(x, self.gate, self.up, self.down, self)
        if self.quantized and x.requires_grad and torch.is_grad_enabled():
            raise ValueError("GatedFFN: 4-bit weights have no gradients (detach x, or torch.no_grad())")
        return self._forward(x, None)

    __call__ = forward

    def _forward(self, x, keep):
        """y; keep: a list that receives x's rows and the saved g, u, h. Behind _current()."""
        r = self._rows(x)
        s = stream_here(self.device)
        if s is None:
            with torch.cuda.device(self.device):
                return self._forward(x, keep)
        T = r.shape[0]
        # of x's shape from the start: a view made in here could not be changed in place where autograd records
        y = torch.empty_like(r) if r is x else x.new_empty(x.shape)
        saved = None
        if keep is not None:
            g, u, h = (torch.empty((T, self.intermediate_size), dtype=dt, device=self.device)
                       for dt in (torch.float32, torch.float32, self.dtype))
            keep.extend((r, g, u, h))
            saved = L.FfnSaved(g.data_ptr(), u.data_ptr(), h.data_ptr())
        if T:
            d, lib = self._desc(r.dtype), L.lib()
            if self.quantized:
                ws = self._workspace(lib.bmx_ffn4_workspace(d, T))
                rc = lib.bmx_ffn4_forward(d, r.data_ptr(), T, y.data_ptr(), ws.data_ptr(), ws.numel(), s)
            else:
                ws = self._workspace(lib.bmx_ffn_workspace(d, T))
                rc = lib.bmx_ffn_forward(d, r.data_ptr(), T, y.data_ptr(), saved, ws.data_ptr(), ws.numel(), s)
            if rc:
                L.check(rc, "GatedFFN.forward")
        return y

    def _input8(self, x):
        """x's rows and Rows8 (one of them None), checked, with 8-bit weights."""
        if torch.is_tensor(x):
            if forward_ad._current_level >= 0 or _tracing() or _modes():
                eager_only("GatedFFN", x)
            if x.requires_grad and torch.is_grad_enabled():
                raise ValueError("GatedFFN: 8-bit weights have no gradients (detach x, or torch.no_grad())")
            return self._rows(x), None
        from .q8 import Rows8
        if not isinstance(x, Rows8) or x.K != self.hidden_size or x.device != self.device:
            raise ValueError(f"GatedFFN: x must be a tensor or Rows8 of {self.hidden_size} codes on {self.device}")
        if _tracing() or _modes():
            eager_only("GatedFFN")
        return None, x

    def _forward8(self, x):
        r, rows = self._input8(x)
        s = stream_here(self.device)
        if s is None:
            with torch.cuda.device(self.device):
                return self._forward8(x)
        y = torch.empty_like(r) if r is x else torch.empty(x.shape, dtype=x.dtype, device=self.device)
        T = rows.N if r is None else r.shape[0]
        if T:
            d, lib = self._desc(x.dtype), L.lib()
            ws = self._workspace(lib.bmx_ffn8_workspace(d, T))
            rc = lib.bmx_ffn8_forward(d, None if r is None else r.data_ptr(), None if rows is None else rows.struct, T, y.data_ptr(),
                                      ws.data_ptr(), ws.numel(), s)
            if rc:
                L.check(rc, "GatedFFN.forward")
        return y

    def check_added(self, x, out, gate_vec):
        """What add_to refuses of x, out, gate_vec (None: not there) and the weights, but for shapes and types."""
        self._current()
        given = (x, out, gate_vec, *self._tensors())
        if forward_ad._current_level >= 0 or _tracing() or _modes():
            eager_only("GatedFFN", *given)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in given):
            raise ValueError("GatedFFN: the added form has no gradients (torch.no_grad(), or out + forward(x))")

    def check_rows(self, rows, T):
        if self.bits != 8 or rows.N != T or rows.K != self.hidden_size or rows.device != self.device:
            raise ValueError(f"GatedFFN: rows must be {T} of {self.hidden_size} codes on {self.device}, for 8-bit weights")

    def add_to(self, out, x, gate_vec=None, rows=None):
        """out [T, H] (fp32, contiguous) += y, or sigmoid(x . gate_vec) * y with gate_vec [H] of x's type: the block as a
        layer's shared expert. y is not rounded to 16 bits. No gradients: refused where autograd records and x, gate_vec, out or a
        weight requires grad (torch.no_grad(), or forward()). rows: x's Rows8, with 8-bit weights, if they are there already
        (RMSNorm.both). Returns out."""
        self.check_added(x, out, gate_vec)
        r = self._rows(x)
        s = stream_here(self.device)
        if s is None:
            with torch.cuda.device(self.device):
                return self.add_to(out, x, gate_vec, rows)
        T = r.shape[0]
        if out.dtype != torch.float32 or out.device != self.device or not out.is_contiguous() or out.data_ptr() % 16 or \
                tuple(out.shape) != (T, self.hidden_size):
            raise ValueError(f"GatedFFN: out must be contiguous fp32 [{T}, {self.hidden_size}] on {self.device}")
        if gate_vec is not None and (gate_vec.dtype != r.dtype or gate_vec.device != self.device or
                                     gate_vec.numel() != self.hidden_size or not gate_vec.is_contiguous() or
                                     gate_vec.data_ptr() % 16):
            raise ValueError(f"GatedFFN: gate_vec must be a contiguous {r.dtype} tensor of {self.hidden_size} elements")
        if rows is not None:
            self.check_rows(rows, T)
        if T and self.bits == 8:
            d, lib = self._desc(r.dtype), L.lib()
            ws = self._workspace(lib.bmx_ffn8_workspace(d, T))
            L.check(lib.bmx_ffn8_add(d, r.data_ptr(), None if rows is None else rows.struct, T,
                                     gate_vec.data_ptr() if gate_vec is not None else None, out.data_ptr(), ws.data_ptr(), ws.numel(), s),
                    "GatedFFN.add_to")
        elif T:
            d, lib = self._desc(r.dtype), L.lib()
            ws = self._workspace(lib.bmx_ffn4_workspace(d, T) if self.quantized else lib.bmx_ffn_workspace(d, T))
            call = lib.bmx_ffn4_add if self.quantized else lib.bmx_ffn_add
            L.check(call(d, r.data_ptr(), T, gate_vec.data_ptr() if gate_vec is not None else None, out.data_ptr(),
                         ws.data_ptr(), ws.numel(), s), "GatedFFN.add_to")
        return out


class _GatedFFNFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, up, down, ffn):
        keep = []
        y = ffn._forward(x.detach(), keep)
        ctx.save_for_backward(gate, up, down, *keep)
        ctx.act, ctx.act_limit = ffn.act, ffn.act_limit
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        gate, up, down, x, g, u, h = ctx.saved_tensors
        I, H = gate.shape
        T, dev = x.shape[0], x.device
        if up.shape != gate.shape or down.shape != (H, I) or g.shape != (T, I) or x.shape[1] != H or \
                any(w.dtype != h.dtype or w.device != dev or not w.is_contiguous() for w in (gate, up, down)):
            raise RuntimeError("GatedFFN: a weight was replaced between the forward and the backward pass")
        s = stream_here(dev)
        if s is None:                           # autograd's threads have a current device of their own
            with torch.cuda.device(dev):
                return _GatedFFNFunction.backward(ctx, dy)
        r = rows_of(dy, H, gate.dtype, dev, "GatedFFN: the gradient of y")
        dx, dg, du, dd = [torch.empty_like(t) if n else None for t, n in zip((x, gate, up, down), ctx.needs_input_grad)]
        d, lib = L.FfnDesc(H, I, DTYPES[gate.dtype], ctx.act, ctx.act_limit, 0, gate.data_ptr(), up.data_ptr(),
                           down.data_ptr()), L.lib()
        ptr = lambda t: None if t is None else t.data_ptr()
        need = lib.bmx_ffn_backward_workspace(d, T)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        L.check(lib.bmx_ffn_backward(d, x.data_ptr(), T, L.FfnSaved(g.data_ptr(), u.data_ptr(), h.data_ptr()), r.data_ptr(),
                                     ptr(dx), ptr(dg), ptr(du), ptr(dd), ws.data_ptr(), need, s), "bmx_ffn_backward")
        return None if dx is None else dx.view(dy.shape), dg, du, dd, None
