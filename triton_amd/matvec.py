"""`matvec`: a few rows times a matrix of 4-bit weights with a scale, and possibly a zero point, per group along K.

`matmul` multiplies MXFP4 weights, whose scales are powers of two; the weights here are whole numbers with 16-bit scales per 32, 64
or 128 values, as weight-only quantisation of dense layers leaves them.  `pack_int4` lays them out once, when a model is loaded."""
import ctypes
from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib, _native

GROUP_SIZES = (32, 64, 128)
_TYPES = (torch.float32, torch.bfloat16, torch.float16)


@dataclass(frozen=True)
class Int4Weights:
    """4-bit weights [K, N] as the kernels read them (see `pack_int4`): blocks of 16 columns x 128 K of 1 KB each, the blocks of
    a strip of 16 columns one after the other; scales and zero points beside them in the same order.  K and N are padded."""
    data: torch.Tensor                 # uint8 [strips, blocks, 1024]
    scales: torch.Tensor               # bf16 / fp16 [strips, blocks, 16, 128 / group_size]
    zeros: Optional[torch.Tensor]      # uint8 like the scales, or None: 8 everywhere
    shape: tuple                       # (K, N)
    group_size: int

    def unpack(self):
        """(codes uint8 [K/2, N], scales [K/group_size, N], zeros or None): what `pack_int4` was given, with unit stride along N."""
        K, N = self.shape
        S, B = self.data.shape[:2]
        v = self.data.view(S, B, 4, 16, 4, 2, 2).permute(1, 4, 2, 6, 5, 0, 3)          # block, t, h, byte of the half, half, strip, column
        low, high = v[..., 0, :, :], v[..., 1, :, :]
        codes = torch.stack([(low & 15) | (high << 4), (low >> 4) | (high & 0xF0)], 4)  # block, t, h, byte of the half, byte of the pair, ...
        codes = codes.reshape(B * 64, S * 16)[:K // 2, :N].contiguous()
        groups = lambda t: t.permute(1, 3, 0, 2).reshape(-1, S * 16)[:K // self.group_size, :N].contiguous()  # noqa: E731
        return codes, groups(self.scales), None if self.zeros is None else groups(self.zeros)


def pack_int4(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, group_size: int = 128) -> Int4Weights:
    """
    Lays out weights w[k, n] = (q[k, n] - z[k // group_size, n]) * scales[k // group_size, n] for `matvec`.

    codes: uint8 [K/2, N], two values of 0..15 per byte along K (low nibble = even k); scales: bf16 / fp16 [K/group_size, N];
    zeros: uint8 [K/group_size, N] with values of 0..15, or None for 8 everywhere.  Any strides; K a multiple of group_size
    (32, 64 or 128).  The tensors are copied."""
    if codes.dtype != torch.uint8 or codes.ndim != 2:
        raise ValueError("codes must be uint8 [K/2, N]")
    if group_size not in GROUP_SIZES:
        raise NotImplementedError(f"groups of {group_size} are not built ({GROUP_SIZES} are)")
    if scales.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"scales of {scales.dtype} are not built (bfloat16 and float16 are)")
    K, N = 2 * codes.shape[0], codes.shape[1]
    if K == 0 or K % group_size:
        raise ValueError(f"K ({K}) must be a multiple of the group size ({group_size})")
    for t, name in ((scales, "scales"), (zeros, "zeros")):
        if t is not None and tuple(t.shape) != (K // group_size, N):
            raise ValueError(f"{name} shape {tuple(t.shape)} != {(K // group_size, N)}")
        if t is not None and t.device != codes.device:
            raise ValueError(f"{name} must live on the device of the codes")
    if zeros is not None and zeros.dtype != torch.uint8:
        raise ValueError("zeros must be uint8")
    S, B, per = -(-N // 16), -(-K // 128), 128 // group_size
    v = torch.nn.functional.pad(codes, (0, S * 16 - N, 0, B * 64 - K // 2)).view(B, 4, 4, 2, 2, S, 16)
    low, high = v[:, :, :, :, 0], v[:, :, :, :, 1]                                      # bytes 2 i and 2 i + 1 of a chunk of eight values
    data = torch.stack([(low & 15) | (high << 4), (low >> 4) | (high & 0xF0)], 3)       # block, t, h, half, byte of the half, strip, column
    data = data.permute(5, 0, 2, 6, 1, 3, 4).reshape(S, B, 1024).contiguous()

    def groups(t):
        t = torch.nn.functional.pad(t, (0, S * 16 - N, 0, B * per - t.shape[0]))
        return t.view(B, per, S, 16).permute(2, 0, 3, 1).contiguous()

    return Int4Weights(data, groups(scales), None if zeros is None else groups(zeros & 15), (K, N), group_size)


def matvec(x: torch.Tensor, w: Int4Weights, bias: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    y = x @ w + bias for a few rows x [M, K] (or one, [K]) of bf16 / fp16 and 4-bit weights of `pack_int4`.

    bias: [N] or None; out_dtype: float32, bfloat16 or float16 (default: x's type); out: where the result goes, which must not overlap
    an input.  Weights are not rounded, sums are float32, the result is rounded once; a row of x with a NaN or an infinity gives NaN,
    any finite one a finite result where float32 holds it (bf16: to a multiple of 2^-137).  The kernels are
    made for up to 64 rows.  Up to 16 read the weights once, and so do up to 64 where there are more than 32 columns per CU; with fewer columns 17 to
    64 rows are cut into parts of 16 to 48 that read them each, mostly from the caches.  More rows are cut alike, into parts of 64 at most."""
    if out is None:
        done = _native.matvec(x, w, bias, out_dtype)
        if done is not None:
            if type(done) is int:
                _lib.check(done, "matvec")
            return done
    _lib.require_gpu(x, "x")
    if x.ndim == 1:
        return matvec(x[None], w, bias, out_dtype, None if out is None else out[None])[0]
    assert x.ndim == 2, "x is [M, K] or [K]"
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"matvec is built for bfloat16 and float16 rows, not {x.dtype}")
    (K, N), M = w.shape, x.shape[0]
    assert x.shape[1] == K, f"inner dimensions differ: {x.shape[1]} vs {K}"
    for t, name in ((w.data, "the weights"), (w.scales, "the scales"), (w.zeros, "the zero points"), (bias, "bias")):
        assert t is None or t.device == x.device, f"{name} must live on the device of x"
    per = 128 // w.group_size
    S, B = -(-N // 16), -(-K // 128)
    for t, shape, dtypes in ((w.data, (S, B, 1024), (torch.uint8,)), (w.scales, (S, B, 16, per), (torch.bfloat16, torch.float16)), (w.zeros, (S, B, 16, per), (torch.uint8,))):
        assert t is None or (tuple(t.shape) == shape and t.dtype in dtypes and t.is_contiguous()), "weights as pack_int4 returns them"
    dtype = out_dtype or (out.dtype if out is not None else x.dtype)
    if dtype not in _TYPES:
        raise NotImplementedError(f"{dtype} outputs are not built")
    if bias is not None:
        assert tuple(bias.shape) == (N,), f"bias shape {tuple(bias.shape)} != {(N,)}"
        if bias.dtype not in _TYPES:
            raise NotImplementedError(f"a bias of {bias.dtype} is not built")
        bias = bias.contiguous()
    if out is None:
        out = torch.empty((M, N), dtype=dtype, device=x.device)
    else:
        assert out.dtype == dtype and out.device == x.device and tuple(out.shape) == (M, N) and (out.stride(1) == 1 or N <= 1) \
            and (M < 2 or out.stride(0) >= N), "out must be [M, N] of the output's type with unit stride along N"
    if M == 0 or N == 0:
        return out
    if x.stride(1) != 1 or (M > 1 and x.stride(0) % 8) or x.data_ptr() % 16 or (M > 1 and x.stride(0) >= 1 << 23):
        x = x.clone(memory_format=torch.contiguous_format)
    a = _lib.MatvecArgs(x=x.data_ptr(), x_stride_m=x.stride(0) if M > 1 else K, codes=w.data.data_ptr(), scales=w.scales.data_ptr(),
                        zeros=None if w.zeros is None else w.zeros.data_ptr(), bias=None if bias is None else bias.data_ptr(),
                        y=out.data_ptr(), y_stride_m=out.stride(0), x_dtype=_lib.dtype_code(x.dtype), scale_dtype=_lib.dtype_code(w.scales.dtype),
                        bias_dtype=_lib.F32 if bias is None else _lib.dtype_code(bias.dtype), y_dtype=_lib.dtype_code(dtype),
                        M=M, N=N, K=K, group=w.group_size)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().tamd_matvec(ctypes.byref(a), ctypes.sizeof(a), _lib.stream_ptr(x.device)), "matvec")
    return out
