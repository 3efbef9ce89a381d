"""Interleaved SwiGLU (swiglu.py of the reference): gate = even columns, linear =
odd columns, out = gate*sigmoid(alpha*gate) * (linear + 1) with clamping."""
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib, _native
from .numerics import InFlexData, OutFlexData


@dataclass(frozen=True)
class FlexCtx:
    out_data: OutFlexData = OutFlexData()
    inp_data: InFlexData = InFlexData()
    saturate_inf: bool = False


@dataclass(frozen=True)
class PrecisionConfig:
    limit: Optional[float]
    flex_ctx: FlexCtx = FlexCtx()


def swiglu_fn(*_args, **_kwargs):
    """Placeholder carried in FnSpecs("swiglu", swiglu_fn, ("alpha", "limit"), reduction_n=2);
    the fused epilogue is selected by the spec's name."""
    raise RuntimeError("swiglu_fn is a tag for the fused matmul epilogue, not a callable")


def swiglu(a: torch.Tensor, alpha: float, precision_config: PrecisionConfig, routing_data=None):
    _lib.require_gpu(a, "a")
    fc = precision_config.flex_ctx
    if fc.inp_data.scale is not None or fc.out_data.expected_scale is not None or fc.out_data.actual_scale is not None:
        raise NotImplementedError("flexpoint scaling in the standalone swiglu is not built")
    assert a.stride(-1) == 1
    assert a.shape[-1] % 2 == 0
    N = a.shape[-1]
    a2 = a.reshape(-1, N)
    M = a2.shape[0]
    out = torch.empty((M, N // 2), dtype=a.dtype, device=a.device)
    limit = precision_config.limit
    rc = _lib.lib().tamd_swiglu(_lib.ptr(a2), _lib.dtype_code(a.dtype), M, N // 2, a2.stride(0), _lib.ptr(out),
                                out.stride(0), float(alpha), float(limit if limit is not None else 0.0),
                                int(limit is not None), _lib.stream_ptr(a.device))
    _lib.check(rc, "swiglu")
    return out.view(*a.shape[:-1], N // 2)


_MX_GROUP = 32


def _limits(precision_config):
    """(limit, whether there is one) of a call without flexpoint scales."""
    fc = precision_config.flex_ctx
    out = fc.out_data
    if fc.inp_data.scale is not None or out.expected_scale is not None or out.actual_scale is not None or out.checksum_scale is not None:
        raise NotImplementedError("flexpoint scaling in the standalone swiglu is not built")
    limit = precision_config.limit
    if limit is not None and not limit >= 0:
        raise ValueError(f"limit of {limit}")
    return float(limit if limit is not None else 0.0), int(limit is not None)


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    """`t` as a matrix whose rows have unit stride."""
    assert t.ndim >= 1, f"{name} needs an axis of columns"
    rows = 1
    for n in t.shape[:-1]:
        rows *= n
    t = t.reshape(rows, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _check_type(t, name):
    _lib.require_gpu(t, name)
    if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise NotImplementedError(f"{name} of {t.dtype} is not built (float32, bfloat16 and float16 are)")


def swiglu_checkpoint(a: torch.Tensor, alpha: float, precision_config: PrecisionConfig) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """
    `swiglu(a, alpha, precision_config)` for training, which keeps a in 8 bits for `swiglu_backward`.

    a: [..., 2 N].  Returns (out [..., N] in a's type, values float8_e4m3fn [..., 2 N], scales uint8 [..., ceil(2 N / 32)]): values and
    scales are those of `downcast_to_mxfp(a, torch.float8_e4m3fn, -1)`, which `upcast_from_mxfp` reads, with a short last group
    where 32 does not divide 2 N (they may share one storage).  out is computed from a itself, in float32, and rounded once.  Unlike in `swiglu`, a NaN stays one beside a
    limit; the group of an infinity is NaN in what is kept."""
    done = _native.swiglu_checkpoint(a, alpha, precision_config)
    if done is not None:
        if type(done) is int:
            _lib.check(done, "swiglu_checkpoint")
        return done
    _check_type(a, "a")
    limit, has_limit = _limits(precision_config)
    assert a.shape[-1] % 2 == 0, "a has a gate and a linear column per value"
    L = a.shape[-1]
    a2 = _rows(a, "a")
    M, G = a2.shape[0], -(-L // _MX_GROUP)
    out = torch.empty((M, L // 2), dtype=a.dtype, device=a.device)
    values = torch.empty((M, L), dtype=torch.float8_e4m3fn, device=a.device)
    scales = torch.empty((M, G), dtype=torch.uint8, device=a.device)
    with torch.cuda.device(a.device):
        _lib.check(_lib.lib().tamd_swiglu_checkpoint(
            _lib.ptr(a2), _lib.dtype_code(a.dtype), M, L // 2, a2.stride(0), _lib.ptr(out), L // 2, _lib.ptr(values), L, _lib.ptr(scales), G, float(alpha),
            limit, has_limit, _lib.stream_ptr(a.device)), "swiglu_checkpoint")
    return out.view(*a.shape[:-1], L // 2), values.view(a.shape), scales.view(*a.shape[:-1], G)


def swiglu_backward(dout: torch.Tensor, values: torch.Tensor, scales: torch.Tensor, alpha: float, precision_config: PrecisionConfig,
                    return_out: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """
    The gradient of `swiglu` at what `swiglu_checkpoint` kept: (da [..., 2 N] in dout's type, out [..., N] or None).

    With a = values * 2^(scales - 127), g = min(a[2n], limit), l = clamp(a[2n+1], -limit, limit), s = sigmoid(alpha g):
      da[2n] = dout[n] * (l + 1) * s * (1 + alpha g (1 - s)),   da[2n+1] = dout[n] * g * s,   0 where the limit cut a off.
    return_out: also the activation at the kept values, for the gradient of the weights that it was multiplied with."""
    done = _native.swiglu_backward(dout, values, scales, alpha, precision_config, return_out)
    if done is not None:
        if type(done) is int:
            _lib.check(done, "swiglu_backward")
        return done
    _check_type(dout, "dout")
    limit, has_limit = _limits(precision_config)
    N = dout.shape[-1]
    L, G = 2 * N, -(-2 * N // _MX_GROUP)
    lead = tuple(dout.shape[:-1])
    assert values.dtype == torch.float8_e4m3fn and tuple(values.shape) == (*lead, L) and values.device == dout.device, \
        f"values are float8_e4m3fn {(*lead, L)} on the device of dout"
    assert scales.dtype == torch.uint8 and tuple(scales.shape) == (*lead, G) and scales.device == dout.device, \
        f"scales are uint8 {(*lead, G)} on the device of dout"
    d2, v2, s2 = _rows(dout, "dout"), _rows(values, "values"), _rows(scales, "scales")
    M = d2.shape[0]
    da = torch.empty((M, L), dtype=dout.dtype, device=dout.device)
    out = torch.empty((M, N), dtype=dout.dtype, device=dout.device) if return_out else None
    with torch.cuda.device(dout.device):
        _lib.check(_lib.lib().tamd_swiglu_backward(
            _lib.ptr(d2), _lib.dtype_code(dout.dtype), M, N, d2.stride(0), _lib.ptr(v2), v2.stride(0), _lib.ptr(s2), s2.stride(0), _lib.ptr(da), L, _lib.ptr(out), N,
            float(alpha), limit, has_limit, _lib.stream_ptr(dout.device)), "swiglu_backward")
    return da.view(*lead, L), None if out is None else out.view(*lead, N)
