"""Q4Matrix: a linear's 4-bit weights with group scales, in the kernels' order (bmx_q4 of include/bmx.h), for the matrices
that a checkpoint keeps neither in 16 bits nor as EXL3 trellis records."""
import torch

from . import _lib as L
from .ffn import DTYPES


class Q4Matrix:
    """W[n, k] = scale[n, k // group] * (code[n, k] - zero[n, k // group]).

    codes: uint8 [N, K / 2], the even column in a byte's low half; scale: fp16 or bf16 [N, K / group]; zero: uint8
    [N, K / group] or None (8 everywhere); group 32, 64 or 128, K a multiple of it. Contiguous device tensors of one device,
    copied into the kernels' order here (the given ones are not kept). Read-only: the kernels get the sizes and addresses that
    it was made with."""

    def __setattr__(self, name, value):
        if name in ("N", "K", "group", "device", "codes", "scale", "zero", "struct"):
            raise AttributeError(f"Q4Matrix: {name} is read-only")
        super().__setattr__(name, value)

    def __init__(self, codes, scale, zero=None, group=128):
        if group not in (32, 64, 128):
            raise ValueError(f"Q4Matrix: group must be 32, 64 or 128, got {group}")
        if codes.dtype != torch.uint8 or codes.dim() != 2 or not codes.is_cuda or not codes.is_contiguous():
            raise ValueError("Q4Matrix: codes must be a contiguous uint8 device tensor [N, K / 2]")
        N, K = codes.shape[0], 2 * codes.shape[1]
        if N <= 0 or K <= 0 or K % group or N > 1 << 20 or K > 1 << 20:
            raise ValueError(f"Q4Matrix: N ({N}) and K ({K}) must be positive, at most 2^20, K a multiple of the group ({group})")
        shape = (N, K // group)
        if scale.dtype not in DTYPES or tuple(scale.shape) != shape or scale.device != codes.device or not scale.is_contiguous():
            raise ValueError(f"Q4Matrix: scale must be a contiguous fp16 or bf16 tensor {list(shape)} on {codes.device}")
        if zero is not None and (zero.dtype != torch.uint8 or tuple(zero.shape) != shape or zero.device != codes.device or
                                 not zero.is_contiguous()):
            raise ValueError(f"Q4Matrix: zero must be a contiguous uint8 tensor {list(shape)} on {codes.device}")
        lib, device = L.lib(), codes.device
        n = lib.bmx_q4_group_count(N, K, group)
        own = dict(N=N, K=K, group=group, device=device,
                   codes=torch.empty(lib.bmx_q4_code_bytes(N, K), dtype=torch.uint8, device=device),
                   scale=torch.empty(n, dtype=scale.dtype, device=device),
                   zero=torch.empty(n, dtype=torch.uint8, device=device) if zero is not None else None)
        own["struct"] = L.Q4(N, K, group, DTYPES[scale.dtype], own["codes"].data_ptr(), own["scale"].data_ptr(),
                             own["zero"].data_ptr() if zero is not None else None)
        self.__dict__.update(own)
        with torch.cuda.device(self.device):
            s = torch.cuda.current_stream().cuda_stream
            L.check(lib.bmx_q4_pack(self.struct, codes.data_ptr(), scale.data_ptr(), zero.data_ptr() if zero is not None else None,
                                    s), "bmx_q4_pack")

    @classmethod
    def quantize(cls, w, group=128, symmetric=False):
        """The nearest 4-bit matrix of w (fp16 or bf16 [N, K]) with the scales and zero points that span each group's range
        (symmetric: zero point 8, the largest magnitude at code 0 or 15)."""
        if w.dim() != 2 or w.dtype not in DTYPES or not w.is_cuda or group not in (32, 64, 128) or w.shape[1] % group:
            raise ValueError("Q4Matrix.quantize: w must be an fp16 or bf16 device tensor [N, K], K a multiple of the group")
        if not w.numel():
            raise ValueError("Q4Matrix.quantize: w has no elements")
        w = w.detach().contiguous()
        v = w.float().view(w.shape[0], -1, group)
        if symmetric:
            scale, zero = v.abs().amax(2) / 7.5, None
        else:
            lo, hi = v.amin(2).clamp(max=0.0), v.amax(2).clamp(min=0.0)
            scale = (hi - lo) / 15.0
        # the stored scale decides the codes; one that is stored as 0 becomes 1 (every code the zero point)
        scale = scale.to(w.dtype)
        scale = torch.where(scale == 0, torch.ones_like(scale), scale)
        s = scale.float()
        if symmetric:
            z = torch.full_like(s, 8.0)
        else:
            z = (-lo / s).round().clamp(0, 15)
            zero = z.to(torch.uint8)
        c = (v / s[..., None] + z[..., None]).round().clamp(0, 15).to(torch.uint8).view(w.shape)
        return cls(c[:, 0::2] | (c[:, 1::2] << 4), scale, zero, group)

    def dequant(self, dtype=torch.float16):
        """W [N, K] in fp16 or bf16, each weight rounded once."""
        if dtype not in DTYPES:
            raise ValueError(f"Q4Matrix.dequant: fp16 or bf16, got {dtype}")
        out = torch.empty((self.N, self.K), dtype=dtype, device=self.device)
        with torch.cuda.device(self.device):
            s = torch.cuda.current_stream().cuda_stream
            L.check(L.lib().bmx_q4_dequant(self.struct, DTYPES[dtype], out.data_ptr(), s), "bmx_q4_dequant")
        return out
