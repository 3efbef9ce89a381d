"""`sample`: the token that follows, from a row of logits and a given uniform number.

Temperature, top-k, top-p and min-p in one call, beside `topk`, whose order (largest first, ties to the lower index) it shares."""
import ctypes
from typing import Union

import torch

from . import _lib, _native

MAX_VOCABULARY = MAX_ROWS = 1 << 20


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0, top_k: Union[int, torch.Tensor] = 0,
           top_p: Union[float, torch.Tensor] = 1.0, min_p: Union[float, torch.Tensor] = 0.0) -> torch.Tensor:
    """
    Token indices int32 [R] for logits [R, V] (float32 / bf16 / fp16, V <= 2^20) and uniform numbers u [R] (float32, of [0, 1)).

    In a row's order -- the largest logit first, equal ones by index -- with w = exp((x - max) / temperature), kept are
      the first top_k (0 or less: all),
      of these the shortest prefix that holds top_p of their mass (1 or more: all of them),
      of these what has w >= min_p, that is at least min_p times the largest probability,
    and always the first.  The token is the first kept one whose running sum of w exceeds u times the sum of all kept, so the same
    u gives the same token however large the batch.  w is held to the nearest multiple of 2^-44 of the largest for V up to 2^18 - 1, of 2^-41 for
    2^20, which leaves sums of V logits within V / 2 of these (and 2^-38 of themselves); the settings are taken as float32.

    temperature, top_k, top_p, min_p: a number for all rows, or a tensor [R] (float32; top_k int32).  temperature 0 takes the
    first of the order.  NaN logits count as -inf; a row with nothing but -inf gives -1; +inf logits share the mass alike.
    In tensors, which are not looked at on the host, a temperature below 0 or NaN counts as 0, a NaN top_p as 1, min_p is
    clamped to [0, 1], u to [0, 1)."""
    done = _native.sample(logits, u, temperature, top_k, top_p, min_p)
    if done is not None:
        if type(done) is int:
            _lib.check(done, "sample")
        return done
    _lib.require_gpu(logits, "logits")
    assert logits.ndim == 2, "logits are [rows, vocabulary]"
    R, V = logits.shape
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise NotImplementedError(f"logits of {logits.dtype} are not built")
    assert 1 <= V, "an empty vocabulary"
    if V > MAX_VOCABULARY or R > MAX_ROWS:
        raise NotImplementedError(f"sample is built for vocabularies of up to {MAX_VOCABULARY} and as many rows")
    assert tuple(u.shape) == (R,) and u.dtype == torch.float32 and u.device == logits.device, "u is float32 [rows] on the device of the logits"
    u = u.contiguous()
    a = _lib.SampleArgs(logits_dtype=_lib.dtype_code(logits.dtype), R=R, V=V)
    held = []
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32), ("top_p", top_p, torch.float32),
                               ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            assert tuple(value.shape) == (R,) and value.dtype == dtype and value.device == logits.device, \
                f"{name} is a number or {dtype} [rows] on the device of the logits"
            held.append(value.contiguous())
            setattr(a, name, held[-1].data_ptr())
        elif name == "top_k":
            a.top_k_value = max(0, min(int(value), MAX_VOCABULARY))
        else:
            if not value >= 0 or (name == "min_p" and value > 1):
                raise ValueError(f"{name} of {value}")
            setattr(a, name + "_value", float(value))
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    tokens = torch.empty(R, dtype=torch.int32, device=logits.device)
    if R == 0:
        return tokens
    L = _lib.lib()
    with torch.cuda.device(logits.device):
        workspace = torch.empty(L.tamd_sample_workspace_exact(R, V), dtype=torch.uint8, device=logits.device)
        a.logits, a.logits_stride, a.u = logits.data_ptr(), logits.stride(0), u.data_ptr()
        a.tokens, a.workspace = tokens.data_ptr(), workspace.data_ptr()
        _lib.check(L.tamd_sample(ctypes.byref(a), ctypes.sizeof(a), _lib.stream_ptr(logits.device)), "sample")
    return tokens
