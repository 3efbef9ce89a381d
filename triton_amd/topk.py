"""Top-k over experts with optional softmax over the picked k (topk.py of the reference)."""
from typing import Optional, Union

import torch

from . import _lib, _native
from .tensor import BIT, SparseMatrix, Tensor, wrap_torch_tensor


def topk_forward(x, k, apply_softmax=True, dim=1, y_indx=None, n_rows=None):
    """Returns (vals [T,k], indx [T,k] int16, bit matrix Tensor).  The bit matrix
    storage is uint32 [ceil(E/32), pad32(T)] viewed transposed, as in topk.py:52-57."""
    if isinstance(x, Tensor):
        n_rows = x.shape[0] if n_rows is None else n_rows
        x = x.storage.data
    assert x.ndim == 2
    assert dim == 1
    assert x.shape[-1] < 32768
    _lib.require_gpu(x, "x")
    if x.stride(1) != 1:
        x = x.contiguous()
    n_rows_max, n_cols = x.shape
    n_rows = n_rows_max if n_rows is None else int(n_rows)
    dev = x.device
    y_vals = torch.empty((n_rows_max, k), dtype=x.dtype, device=dev)
    provided = y_indx is not None
    if provided:
        assert y_indx.dtype == torch.int16 and y_indx.is_contiguous() and tuple(y_indx.shape) == (n_rows_max, k)
    else:
        y_indx = torch.empty((n_rows_max, k), dtype=torch.int16, device=dev)
    n_words = -(-n_cols // 32)
    bits_store = torch.empty((n_words, -(-n_rows_max // 32) * 32), dtype=torch.int32, device=dev)
    bits = bits_store.transpose(0, 1)[:n_rows_max]
    rc = _lib.lib().tamd_topk_forward(_lib.ptr(x), _lib.dtype_code(x.dtype), x.stride(0), n_rows, n_cols, k,
                                      int(apply_softmax), int(provided), _lib.ptr(y_vals), _lib.ptr(y_indx), k,
                                      _lib.ptr(bits_store), bits.stride(0), bits.stride(1), _lib.stream_ptr(dev))
    _lib.check(rc, "topk")
    bitmatrix = wrap_torch_tensor(bits.view(torch.uint32), dtype=BIT, shape=[n_rows, n_cols],
                                  shape_max=[n_rows_max, n_cols])
    return y_vals, y_indx, bitmatrix


def topk(x: Union[Tensor, torch.Tensor], k: int, apply_softmax: bool = True, dim: int = 1,
         y_indx: Optional[torch.Tensor] = None, n_rows: Optional[int] = None, all_gather: bool = False,
         symm_mem_pool=None) -> SparseMatrix:
    """Sparse matrix equal to `x` with all but the k largest entries of every row
    dropped (values optionally replaced by their softmax).  Ties go to the lower
    column; entries are ordered by value, largest first."""
    if all_gather or symm_mem_pool is not None:
        raise NotImplementedError("all_gather needs more than one GPU")
    vals, indx, mask = topk_forward(x, k, apply_softmax, dim, y_indx, n_rows)
    return SparseMatrix(indx=indx, vals=vals, mask=mask)


def topk_backward(x: Union[Tensor, torch.Tensor], indx: torch.Tensor, dvals: torch.Tensor, apply_softmax: bool = True,
                  n_rows: Optional[int] = None) -> torch.Tensor:
    """
    The gradient of `topk(x, k, apply_softmax)` (topk_details/_topk_backward.py:5-51 of the reference) from dvals [T, k], that of its values:

      dx[t, indx[t, j]] = p_j * (dvals[t, j] - sum_m p_m * dvals[t, m]),  p = softmax(x[t, indx[t]]);   without the softmax: dvals[t, j]

    and 0 elsewhere and in rows from n_rows on, which were not routed.  x: the logits [T, E] (float32 / bf16 / fp16, E < 32768), of which the
    picked ones are read; indx: int16 [T, k] as `topk` and `routing` return it, k <= 64 (an index outside [0, E) is no pick); dvals
    may be of another floating type than x.  Returns [T, E] in x's type; arithmetic is float32, rounded once."""
    if n_rows is None and type(x) is torch.Tensor:
        done = _native.topk_backward(x, indx, dvals, apply_softmax)
        if done is not None:
            if type(done) is int:
                _lib.check(done, "topk_backward")
            return done
    if isinstance(x, Tensor):
        n_rows = x.shape[0] if n_rows is None else n_rows
        x = x.storage.data
    _lib.require_gpu(x, "x")
    assert x.ndim == 2 and x.shape[1] < 32768, "x is [rows, columns], with fewer than 32768 columns"
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16) or dvals.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise NotImplementedError(f"logits of {x.dtype} with gradients of {dvals.dtype} are not built (float32, bfloat16 and float16 are)")
    T, E = x.shape
    assert indx.ndim == 2 and indx.dtype == torch.int16 and indx.shape[0] == T and indx.device == x.device, "indx is int16 [rows, k] on the device of x"
    k = indx.shape[1]
    if k > 64:
        raise NotImplementedError("topk_backward is built for up to 64 picks")
    assert tuple(dvals.shape) == (T, k) and dvals.device == x.device, f"dvals are [{T}, {k}] on the device of x"
    live = T if n_rows is None else int(n_rows)
    assert 0 <= live <= T, f"{live} of {T} rows"
    x, d, i = (t if t.shape[1] <= 1 or t.stride(1) == 1 else t.contiguous() for t in (x, dvals, indx))
    dx = torch.empty((T, E), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().tamd_topk_backward(
            _lib.ptr(x), _lib.dtype_code(x.dtype), x.stride(0), T, live, E, k, int(apply_softmax), _lib.ptr(i), i.stride(0), _lib.ptr(d),
            _lib.dtype_code(d.dtype), d.stride(0), _lib.ptr(dx), E, _lib.stream_ptr(x.device)), "topk_backward")
    return dx
