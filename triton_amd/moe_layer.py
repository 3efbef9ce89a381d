"""`moe_layer`: a whole mixture-of-experts layer for a few tokens, in two or three launches.

The chain of `routing`, `matmul` (gathered rows, SwiGLU), `matmul` (gate weights, scatter) and `reduce` launches five or six
kernels and writes its rows to memory three times; with a handful of tokens that is most of a layer's time.  The kernels behind
this function pick the experts themselves, read every picked expert's weights once and add the experts' rows up where
they are made.  Arguments and options are those of `routing` and `matmul`."""
import ctypes
import math
from typing import Optional

import torch

from . import _lib, _native
from .matmul import FusedActivation, PrecisionConfig
from .tensor import FP4, Tensor
from .tensor_details.layout import CDNA4MXScaleLayout, CDNA4MXValueLayout

MAX_TOKENS, MAX_EXPERTS, MAX_PICKS, MAX_SLOTS = 64, 512, 16, 512
_BIAS_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _refuse_other_options(pc: PrecisionConfig, name: str):
    """Fields that would change the result and that the kernels do not take."""
    flex = pc.flex_ctx
    if (any(getattr(pc, f) is not None for f in ("a_mx_scale", "c_mx_scale", "a_mx_tensor_scale", "b_mx_tensor_scale", "out_dtype"))
            or pc.acc_scale != 1.0 or flex.lhs_data.scale is not None or flex.rhs_data.scale is not None or flex.acc_data.scale is not None
            or flex.lhs_data.dtype is not None or flex.rhs_data.dtype is not None
            or flex.out_data.expected_scale is not None or flex.out_data.actual_scale is not None):
        raise NotImplementedError(f"{name}: moe_layer takes b_mx_scale and b_microblock_size only")


def _weights(into, w, pc, bias, E, K, N, device, n):
    """Fills a `MoeWeights` from what `matmul` takes for MXFP4 weights [E, K, N]."""
    name = f"w{n}"
    if pc is None or pc.b_mx_scale is None:
        raise NotImplementedError(f"{name}: moe_layer is built for MXFP4 weights (precision_config{n}.b_mx_scale)")
    _refuse_other_options(pc, f"precision_config{n}")
    assert pc.b_microblock_size == 32, "Unsupported microscale block size"
    blocks = isinstance(w, Tensor) and isinstance(w.storage.layout, CDNA4MXValueLayout)
    data = w.storage.data if isinstance(w, Tensor) else w
    if (w.dtype != FP4) if isinstance(w, Tensor) else (w.dtype != torch.uint8):
        raise NotImplementedError(f"{name}: moe_layer is built for MXFP4 weights")
    if blocks:
        assert list(w.shape) == [E, K, N], f"{name} shape {list(w.shape)} != {[E, K, N]}"
        assert list(data.shape) == CDNA4MXValueLayout().storage_shape([E, K, N]) and data.is_contiguous(), \
            f"{name}: storage does not match the block layout"
        into.w_layout, into.w_stride_e, into.w_stride_n = _lib.W_CDNA4_BLOCKS, data.stride(0), 0
    else:
        assert data.ndim == 3 and list(data.shape) == [E, K // 2, N], f"{name}: storage {list(data.shape)} != {[E, K // 2, N]} (packed along K)"
        if data.stride(1) != 1:
            raise NotImplementedError(f"{name}: weights must be contiguous along K")
        into.w_layout, into.w_stride_e, into.w_stride_n = _lib.W_STRIDED, data.stride(0), data.stride(2)
    scale = pc.b_mx_scale
    shuffled = isinstance(scale, Tensor) and isinstance(scale.storage.layout, CDNA4MXScaleLayout)
    sd = scale.storage.data if isinstance(scale, Tensor) else scale
    assert sd.dtype == torch.uint8, f"Unsupported microscale dtype {sd.dtype}"
    want = [E, K // 32, N]
    assert math.prod(list(scale.shape)[:-2]) == E and list(scale.shape)[-2:] == want[1:], f"{name}: scale shape {list(scale.shape)} != {want}"
    if shuffled:
        assert list(sd.shape) == CDNA4MXScaleLayout().storage_shape(want) and (sd.stride(1) == 1 or sd.shape[1] == 1) \
            and (sd.stride(2) == sd.shape[1] or sd.shape[2] == 1), f"{name}: scale storage does not match the CDNA4 scale layout"
        into.scale_layout, into.scale_stride_e, into.scale_stride_n = _lib.SCALE_CDNA4, sd.stride(0), 0
    else:
        assert sd.ndim == 3
        if sd.stride(1) != 1 and sd.shape[1] != 1:
            raise NotImplementedError(f"{name}: scales must be contiguous along K")
        into.scale_layout, into.scale_stride_e, into.scale_stride_n = _lib.SCALE_STRIDED, sd.stride(0), sd.stride(2)
    assert data.device == device and sd.device == device, f"{name} and its scales must live on the device of x"
    into.w, into.scale = data.data_ptr(), sd.data_ptr()
    if bias is not None:
        assert bias.device == device and tuple(bias.shape) == (E, N) and (bias.stride(1) == 1 or N == 1), \
            f"bias{n}: a tensor of shape {(E, N)} with unit stride along its last axis, on the device of x"
        if bias.dtype not in _BIAS_TYPES:
            raise NotImplementedError(f"bias{n}: dtype {bias.dtype} is not built")
        if bias.data_ptr() % 4 or bias.stride(0) % 2:
            bias = bias.clone(memory_format=torch.contiguous_format)
        into.bias, into.bias_stride_e, into.bias_dtype = bias.data_ptr(), bias.stride(0), _lib.dtype_code(bias.dtype)
        return bias   # (alive until the launch)


def moe_layer(x: torch.Tensor, logits: torch.Tensor, n_expts_act: int, w1, bias1: Optional[torch.Tensor], w2,
              bias2: Optional[torch.Tensor], precision_config1: PrecisionConfig, precision_config2: PrecisionConfig,
              fused_activation: FusedActivation, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    y[t, :] = sum_j gate[t, j] * (swiglu(x[t, :] @ w1[e] + bias1[e]) @ w2[e] + bias2[e])   with e = pick j of token t

    x: [T, H] bf16 / fp16, T <= 64.  logits: [T, E] of the gate (float32 / bf16 / fp16), E <= 512; every token picks its
    n_expts_act <= 16 largest (ties: the lower expert; T * n_expts_act <= 512), gate is their softmax, in float32.  As in `routing`, a
    token whose logits are all -inf gets NaN gate weights.
    w1: [E, H, 2 I], w2: [E, I, H] MXFP4 weights as `matmul` takes them -- contiguous along K or in `CDNA4MXValueLayout` -- with
    precision_config{1,2}.b_mx_scale [E, K/32, N] (strided along K or in `CDNA4MXScaleLayout`) and b_microblock_size = 32.
    bias1: [E, 2 I], bias2: [E, H] or None.  fused_activation: "swiglu" with (alpha, limit), over the column pairs of w1.
    Returns [T, H] in x's type (`out`, if given, which must not overlap an input); sums are float32, the result is rounded once.
    More tokens: `routing`, `matmul`, `matmul`, `reduce`."""
    if out is None:
        done = _native.moe_layer(x, logits, n_expts_act, w1, bias1, w2, bias2, precision_config1, precision_config2, fused_activation)
        if done is not None:
            if type(done) is int:
                _lib.check(done, "moe_layer")
            return done
    _lib.require_gpu(x, "x")
    assert x.ndim == 2 and logits.ndim == 2 and logits.shape[0] == x.shape[0], "x is [tokens, hidden], logits [tokens, experts]"
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"moe_layer is built for bfloat16 and float16 activations, not {x.dtype}")
    T, H = x.shape
    E, k = logits.shape[1], int(n_expts_act)
    assert 1 <= k <= E, f"{k} picks of {E} experts"
    if T > MAX_TOKENS or E > MAX_EXPERTS or k > MAX_PICKS or T * k > MAX_SLOTS:
        raise NotImplementedError(f"moe_layer is built for up to {MAX_TOKENS} tokens, {MAX_EXPERTS} experts, {MAX_PICKS} picks and "
                                  f"{MAX_SLOTS} picks of all tokens: use routing, matmul and reduce")
    if fused_activation is None or fused_activation.specs.name != "swiglu":
        raise NotImplementedError("moe_layer is built for the swiglu activation")
    assert logits.device == x.device, "logits must live on the device of x"
    if logits.dtype not in _BIAS_TYPES:
        raise NotImplementedError(f"logits of {logits.dtype} are not built")
    two_inter = w1.shape[-1]
    assert len(w1.shape) == 3 and len(w2.shape) == 3, "w1 is [experts, hidden, 2 * inter], w2 [experts, inter, hidden]"
    assert two_inter % 2 == 0, "w1 has a gate and a linear column per value"
    inter = two_inter // 2
    if H % 32 or inter % 32 or not H or not inter:
        raise ValueError(f"hidden ({H}) and inter ({inter}) must be multiples of 32")
    a = _lib.MoeLayerArgs()
    held = [_weights(a.up, w1, precision_config1, bias1, E, H, two_inter, x.device, 1),
            _weights(a.down, w2, precision_config2, bias2, E, inter, H, x.device, 2)]  # noqa: F841
    if out is None:
        out = torch.empty((T, H), dtype=x.dtype, device=x.device)
    else:
        assert out.dtype == x.dtype and out.device == x.device and tuple(out.shape) == (T, H) and out.stride(1) == 1 and (T < 2 or out.stride(0) >= H)
    if T == 0:
        return out
    if x.stride(1) != 1 or x.stride(0) % 8 or x.data_ptr() % 16 or (T - 1) * x.stride(0) >= 1 << 23:
        x = x.clone(memory_format=torch.contiguous_format)
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    named = dict(zip(fused_activation.specs.fn_arg_names, fused_activation.fn_args))
    limit = named.get("limit")
    a.act_alpha, a.act_limit, a.act_has_limit = float(named["alpha"]), float(limit if limit is not None else 0.0), int(limit is not None)
    L = _lib.lib()
    with torch.cuda.device(x.device):
        workspace = torch.empty(L.tamd_moe_layer_workspace(T, k, inter), dtype=torch.uint8, device=x.device)
        a.x, a.x_stride_m, a.x_dtype = x.data_ptr(), x.stride(0) if T > 1 else H, _lib.dtype_code(x.dtype)
        a.logits, a.logits_stride, a.logits_dtype = logits.data_ptr(), logits.stride(0), _lib.dtype_code(logits.dtype)
        a.y, a.y_stride_m, a.workspace = out.data_ptr(), out.stride(0), workspace.data_ptr()
        a.n_tokens, a.n_experts, a.n_picks, a.hidden, a.inter = T, E, k, H, inter
        _lib.check(L.tamd_moe_layer(ctypes.byref(a), ctypes.sizeof(a), _lib.stream_ptr(x.device)), "moe_layer")
    return out
