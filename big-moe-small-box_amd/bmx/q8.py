"""Q8Matrix and Rows8: a linear's 8-bit weights with a scale per row, and tokens' rows in 8 bits with a scale each (bmx_q8 of
include/bmx.h), the two factors of the products in 8-bit integers."""
import torch

from . import _lib as L
from .ffn import DTYPES, eager_only, forward_ad, stream_here, _modes, _tracing

ROW_DTYPES = {**DTYPES, torch.float32: L.DT_FP32}
MOST_K = 131071


class _Codes8:
    """codes int8 in the kernels' order (bmx_q8) and scale fp32 [N], views of one allocation: what Q8Matrix and Rows8 have in
    common."""

    _fixed = ("N", "K", "device", "codes", "scale", "struct", "_held")

    def __setattr__(self, name, value):
        if name in self._fixed:
            raise AttributeError(f"{type(self).__name__}: {name} is read-only")
        super().__setattr__(name, value)

    def __reduce_ex__(self, protocol):
        raise TypeError(f"{type(self).__name__} cannot be pickled or copied (its struct holds device addresses)")

    def _make(self, N, K, device):
        """Codes and behind them scales of one allocation, not yet written."""
        n = (N + 15) // 16 * ((K + 63) // 64) * 1024
        held = torch.empty(n + 4 * N, dtype=torch.int8, device=device)
        p = held.data_ptr()
        d = self.__dict__
        d["N"], d["K"], d["device"], d["_held"], d["struct"] = N, K, device, held, L.Q8(N, K, p or None, p + n if p else None)

    @property
    def codes(self):
        return self._held[:self._held.numel() - 4 * self.N]

    @property
    def scale(self):
        return self._held[self._held.numel() - 4 * self.N:].view(torch.float32)

    def _given(self, codes, scale, rows):
        """A user's codes [N, K] and scales [N], copied into the kernels' order."""
        who = type(self).__name__
        if codes.dtype != torch.int8 or codes.dim() != 2 or not codes.is_cuda:
            raise ValueError(f"{who}: codes must be an int8 device tensor [{rows}, K], got {codes.dtype} {tuple(codes.shape)} on {codes.device}")
        N, K = codes.shape
        if (N <= 0 and rows == "N") or N > 1 << 24 or not 0 < K <= MOST_K:
            raise ValueError(f"{who}: {rows} ({N}) must be {'positive, ' if rows == 'N' else ''}at most 2^24, K ({K}) in [1, {MOST_K}]")
        if scale.dtype not in ROW_DTYPES or scale.numel() != N or scale.device != codes.device or scale.dim() not in (1, 2):
            raise ValueError(f"{who}: scale must be an fp32, fp16 or bf16 tensor of {N} values on {codes.device}, got {scale.dtype} "
                             f"{tuple(scale.shape)} on {scale.device}")
        self._make(N, K, codes.device)
        self.scale.copy_(scale.detach().reshape(-1))
        self._call("bmx_q8_pack", codes.detach().contiguous())

    def _call(self, name, *args):
        """A library call on this and args (tensors by address), on the current stream of its device; nothing for no rows."""
        if self.N:
            with torch.cuda.device(self.device):
                s = torch.cuda.current_stream().cuda_stream
                L.check(getattr(L.lib(), name)(self.struct, *(a.data_ptr() if torch.is_tensor(a) else a for a in args), s), name)

    def int8(self):
        """The codes, int8 [N, K]."""
        out = torch.empty((self.N, self.K), dtype=torch.int8, device=self.device)
        self._call("bmx_q8_unpack", out)
        return out

    def dequant(self, dtype=torch.float16):
        """The values [N, K] in fp16, bf16 or fp32, each rounded once."""
        if dtype not in ROW_DTYPES:
            raise ValueError(f"{type(self).__name__}.dequant: fp16, bf16 or fp32, got {dtype}")
        out = torch.empty((self.N, self.K), dtype=dtype, device=self.device)
        self._call("bmx_q8_dequant", ROW_DTYPES[dtype], out)
        return out


def _quantized(to, x, N, K):
    """to (a bare Q8Matrix or Rows8) of the contiguous rows x [N, K], on the current stream of x's device."""
    s = stream_here(x.device)
    if s is None:
        with torch.cuda.device(x.device):
            return _quantized(to, x, N, K)
    to._make(N, K, x.device)
    if N:
        rc = L.lib().bmx_q8_quantize(x.data_ptr(), ROW_DTYPES[x.dtype], to.struct, s)
        if rc:
            L.check(rc, "bmx_q8_quantize")
    return to


class Q8Matrix(_Codes8):
    """W[n, k] = scale[n] * code[n, k]. codes: int8 [N, K]; scale: fp32, fp16 or bf16 [N] (or [N, 1]); device tensors of one
    device, copied here (the given ones are not kept). K at most 131,071, N at most 2^20. Read-only: the kernels get the sizes and
    addresses that it was made with."""

    def __init__(self, codes, scale):
        if codes.dim() == 2 and codes.shape[0] > 1 << 20:
            raise ValueError(f"Q8Matrix: N ({codes.shape[0]}) must be at most 2^20")
        self._given(codes, scale, "N")

    @classmethod
    def quantize(cls, w):
        """The matrix of w (fp16, bf16 or fp32 [N, K]) with each row's largest magnitude at code 127. A row with an infinity or a NaN
        gets scale NaN."""
        if w.dim() != 2 or w.dtype not in ROW_DTYPES or not w.is_cuda or not w.numel() or w.shape[0] > 1 << 20 or w.shape[1] > MOST_K:
            raise ValueError(f"Q8Matrix.quantize: w must be an fp16, bf16 or fp32 device tensor [N, K], N to 2^20, K to {MOST_K}, got "
                             f"{w.dtype} {tuple(w.shape)} on {w.device}")
        w = w.detach().contiguous()
        return _quantized(cls.__new__(cls), w, *w.shape)


class Rows8(_Codes8):
    """Tokens [..., K] as value[t, k] = scale[t] * code[t, k]: what RMSNorm.rows8 and ops.quantize_rows give and the 8-bit products
    take in the place of x. codes: int8 [T, K]; scale: fp32, fp16 or bf16 [T] (or [T, 1]), copied here. dtype: fp16 or bf16, the
    type of the products' results; shape: of the tokens, [..., K] (default [T, K]). Read-only."""

    _fixed = _Codes8._fixed + ("dtype", "shape")

    def __init__(self, codes, scale, dtype=torch.float16, shape=None):
        if dtype not in DTYPES:
            raise ValueError(f"Rows8: dtype must be fp16 or bf16, got {dtype}")
        self._given(codes, scale, "T")
        shape = torch.Size((self.N, self.K) if shape is None else shape)
        if not shape or shape[-1] != self.K or shape.numel() != self.N * self.K:
            raise ValueError(f"Rows8: shape {tuple(shape)} is not that of {self.N} rows of {self.K}")
        self.__dict__.update(dtype=dtype, shape=shape)

    @classmethod
    def _empty(cls, T, K, device, dtype, shape):
        r = cls.__new__(cls)
        r._make(T, K, device)
        d = r.__dict__
        d["dtype"], d["shape"] = dtype, shape
        return r

    @classmethod
    def _of(cls, x):
        shape, K = x.shape, x.shape[-1]
        r = _quantized(cls.__new__(cls), x.reshape(-1, K).contiguous(), shape.numel() // K, K)
        r.__dict__.update(dtype=x.dtype, shape=shape)
        return r


def quantize_rows(x):
    """Rows8 of x [..., K] (fp16 or bf16): each token's largest magnitude at code 127. A token with an infinity or a NaN gets scale
    NaN, and all its products are NaN. No gradients."""
    if x.dtype not in DTYPES or not x.is_cuda or x.dim() < 1 or not 0 < x.shape[-1] <= MOST_K:
        raise ValueError(f"quantize_rows: x must be an fp16 or bf16 device tensor [..., K], K in [1, {MOST_K}], got {x.dtype} "
                         f"{tuple(x.shape)} on {x.device}")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError("quantize_rows: no gradients (detach x, or torch.no_grad())")
    if forward_ad._current_level >= 0 or _tracing() or _modes():
        eager_only("quantize_rows", x)
    return Rows8._of(x)
