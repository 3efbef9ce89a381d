"""Rows of tokens to the rows of their experts and back, with gate weights, and the gradients of both.

`matmul` gathers and scatters rows by itself in the forward pass, and `reduce` adds them up; a training step needs the sorted rows as
a tensor of their own (the weights' gradient is a product over an expert's rows) and everything in the other direction.  All four
functions take `row_indx` [T, k], the expert row of every pick of every token, which is `routing(...).row_sorted_indx.view(T, k)`:

  dispatch            rows[row_indx[t, j]] = gates[t, j] * x[t]
  combine             y[t] = sum_j gates[t, j] * rows[row_indx[t, j]]
  dispatch_backward   gradients of x and gates from that of the rows
  combine_backward    gradients of the rows and gates from that of y

A pick whose index is outside [0, number of rows) -- routing leaves -1 where there is none -- takes no part: it adds nothing, and its
gate weight's gradient is 0.  In `dispatch` and `combine_backward` every row is named by at most one pick; rows that none
names are not written.  Types: float32, bfloat16 or float16 rows; gate weights of any of the three; sums are float32."""
import ctypes
from typing import Optional, Tuple

import torch

from . import _lib, _native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _by_row(t: torch.Tensor, name: str) -> torch.Tensor:
    """[n, H] with unit stride along H."""
    _lib.require_gpu(t, name)
    assert t.ndim == 2, f"{name} is a matrix of rows"
    if t.dtype not in _TYPES:
        raise NotImplementedError(f"{name} of {t.dtype} is not built (float32, bfloat16 and float16 are)")
    if t.shape[1] >= 1 << 31:
        raise NotImplementedError(f"{name}: rows of 2^31 elements and more are not built")
    return t if t.stride(1) == 1 or t.shape[1] <= 1 else t.contiguous()


def _pitch(t):
    return t.stride(0) if t.shape[0] > 1 else 0


def _run(spread, src, dst, row_indx, gates, other, n_rows, what):
    """One call of the library: `src` to `dst`, and with `other` the products [T, k] that are the gradient of the gates."""
    dev = src.device
    assert row_indx.ndim == 2 and row_indx.dtype == torch.int32 and row_indx.device == dev, "row_indx is int32 [tokens, picks] on the device of the rows"
    T, k = row_indx.shape
    assert (src if spread else dst).shape[0] == T, f"{(src if spread else dst).shape[0]} tokens, but row_indx has {T}"
    if n_rows >= 1 << 31 or T >= 1 << 31:
        raise NotImplementedError(f"{what}: 2^31 rows and more are not built")
    if gates is not None:
        assert tuple(gates.shape) == (T, k) and gates.device == dev, f"gates are [{T}, {k}] on the device of the rows"
        if gates.dtype not in _TYPES:
            raise NotImplementedError(f"gates of {gates.dtype} are not built (float32, bfloat16 and float16 are)")
        gates = gates if k <= 1 or gates.stride(1) == 1 else gates.contiguous()
    row_indx = row_indx if k <= 1 or row_indx.stride(1) == 1 else row_indx.contiguous()
    dots = None if other is None else torch.empty((T, k), dtype=gates.dtype, device=dev)
    a = _lib.TokenRowsArgs(src=src.data_ptr(), src_stride=_pitch(src), dst=dst.data_ptr(), dst_stride=_pitch(dst),
                           row_indx=row_indx.data_ptr(), row_indx_stride=_pitch(row_indx), dtype=_lib.dtype_code(src.dtype), T=T, k=k, H=src.shape[1],
                           n_rows=n_rows)
    if gates is not None:
        a.gates, a.gates_stride, a.gates_dtype = gates.data_ptr(), _pitch(gates), _lib.dtype_code(gates.dtype)
    if dots is not None:
        a.other, a.other_stride, a.dots, a.dots_stride = other.data_ptr(), _pitch(other), dots.data_ptr(), k
    L = _lib.lib()
    with torch.cuda.device(dev):
        _lib.check((L.tamd_dispatch if spread else L.tamd_combine)(ctypes.byref(a), ctypes.sizeof(a), _lib.stream_ptr(dev)), what)
    return dots


def _rows_out(like: torch.Tensor, row_indx: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
    H = like.shape[1]
    if out is None:
        return torch.empty((row_indx.numel(), H), dtype=like.dtype, device=like.device)
    assert out.ndim == 2 and out.shape[1] == H and out.dtype == like.dtype and out.device == like.device, f"out holds rows of {H} {like.dtype} on the same device"
    assert (out.stride(1) == 1 or H <= 1) and (out.shape[0] < 2 or out.stride(0) >= H), "out must have unit stride along its rows, which do not overlap"
    return out


def _kept(t, rows, H, like, name):
    t = _by_row(t, name)
    assert tuple(t.shape) == (rows, H) and t.dtype == like.dtype and t.device == like.device, f"{name} must be {like.dtype} [{rows}, {H}] on the same device"
    return t


def dispatch(x: torch.Tensor, row_indx: torch.Tensor, gates: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    rows[row_indx[t, j]] = gates[t, j] * x[t]: the tokens' rows [T, H] sorted by expert.

    Returns [T * k, H] in x's type, or writes to `out` (any number of rows; it must not overlap an input).  Rows that no pick
    names are left as they are -- in a new tensor: undefined.  Without gates rows are copied bit for bit."""
    done = _native.dispatch(x, row_indx, gates, out)
    if done is not None:
        if type(done) is int:
            _lib.check(done, "dispatch")
        return done
    x = _by_row(x, "x")
    out = _rows_out(x, row_indx, out)
    _run(True, x, out, row_indx, gates, None, out.shape[0], "dispatch")
    return out


def combine(rows: torch.Tensor, row_indx: torch.Tensor, gates: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """
    y[t] = sum_j gates[t, j] * rows[row_indx[t, j]]: the experts' rows [n, H] added up per token.

    Returns [T, H] in the rows' type (`out`, if given, which must not overlap an input); the sum is float32, in the order of j,
    and rounded once.  A token none of whose picks has a row gets zeros."""
    done = _native.combine(rows, row_indx, gates, out)
    if done is not None:
        if type(done) is int:
            _lib.check(done, "combine")
        return done
    rows = _by_row(rows, "rows")
    T, H = row_indx.shape[0], rows.shape[1]
    if out is None:
        out = torch.empty((T, H), dtype=rows.dtype, device=rows.device)
    else:
        assert tuple(out.shape) == (T, H) and out.dtype == rows.dtype and out.device == rows.device, f"out must be {rows.dtype} [{T}, {H}] on the same device"
        assert (out.stride(1) == 1 or H <= 1) and (T < 2 or out.stride(0) >= H), "out must have unit stride along its rows, which do not overlap"
    _run(False, rows, out, row_indx, gates, None, rows.shape[0], "combine")
    return out


def dispatch_backward(drows: torch.Tensor, row_indx: torch.Tensor, x: Optional[torch.Tensor] = None,
                      gates: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """
    The gradients of `dispatch(x, row_indx, gates)` from drows [n, H], that of its rows:

      dx[t] = sum_j gates[t, j] * drows[row_indx[t, j]]        dgates[t, j] = <x[t], drows[row_indx[t, j]]>

    Returns (dx [T, H] in drows' type, dgates [T, k] in the gates' type).  dgates is None without gates, and without x, which
    nothing else needs."""
    done = _native.dispatch_backward(drows, row_indx, x, gates, None)
    if done is not None:
        if type(done) is int:
            _lib.check(done, "dispatch_backward")
        return done
    drows = _by_row(drows, "drows")
    T, H = row_indx.shape[0], drows.shape[1]
    x = None if x is None or gates is None else _kept(x, T, H, drows, "x")
    dx = torch.empty((T, H), dtype=drows.dtype, device=drows.device)
    return dx, _run(False, drows, dx, row_indx, gates, x, drows.shape[0], "dispatch_backward")


def combine_backward(dy: torch.Tensor, row_indx: torch.Tensor, rows: Optional[torch.Tensor] = None, gates: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """
    The gradients of `combine(rows, row_indx, gates)` from dy [T, H]:

      drows[row_indx[t, j]] = gates[t, j] * dy[t]        dgates[t, j] = <dy[t], rows[row_indx[t, j]]>

    Returns (drows, dgates [T, k] in the gates' type).  drows is [T * k, H] in dy's type, or `out`, as in `dispatch`: rows that no pick names
    are left as they are.  out may be `rows` itself, which the gradient then takes the place of.  dgates is None without gates, and without rows, which nothing else needs and which are as many as drows."""
    done = _native.combine_backward(dy, row_indx, rows, gates, out)
    if done is not None:
        if type(done) is int:
            _lib.check(done, "combine_backward")
        return done
    dy = _by_row(dy, "dy")
    drows = _rows_out(dy, row_indx, out)
    rows = None if rows is None or gates is None else _kept(rows, drows.shape[0], dy.shape[1], dy, "rows")
    return drows, _run(True, dy, drows, row_indx, gates, rows, drows.shape[0], "combine_backward")
