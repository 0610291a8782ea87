"""Products with one matrix for each group of rows, and their gradients (``csrc/cuda/grouped.cu``).

The rows of ``X [T, K]`` are sorted by the group that they belong to (segment, cluster, expert): group ``e`` has the rows
``offsets[e] <= t < offsets[e + 1]``, any number of them, and the matrix ``W[e]`` of ``W [E, N, K]``.

* ``grouped_nt(X, W, offsets)``   ``Y[t] = W[e] x[t]``, the values of a layer whose weights depend on the row's group;
* ``grouped_nn(dY, W, offsets)``  ``dX[t] = W[e]^T dy[t]``, its gradient with respect to the rows;
* ``grouped_tn(dY, X, offsets)``  ``dW[e] = sum over the group's rows of dy[t] x[t]^T``, and to the matrices.

Rows and matrices are bfloat16 or float16, both the same; sums are held in float32, and rounded once into ``out_dtype``
(the inputs' type, or ``torch.float32``).  The tensor cores cut what they add to their fp32 sums off rather than round it, so the
relative error of an fp32 result grows with the length of the sum: 5e-7 at 512 terms, 2e-6 at 2048, 9e-6 at 8192 (3.5e-5 where all terms have one sign).  There it
stays: longer sums are made of parts of 8192 terms that are added up rounded.
Like the other products of this package these know nothing of torch's autograd: call the gradients.

``offsets`` (``E + 1`` int32 or int64 numbers on the device) is read by the kernels only, so that a batch can be cut up
without the host.  They stay inside the tensors whatever it holds: a bound below the one before it, or outside of ``0 .. T``,
is moved to the nearest that is allowed, and ``check_status`` raises for it.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._calls import calls

TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_GROUPS = 1024
MAX_ROWS = (1 << 31) - 512


def check_status(device=None) -> None:
    """Raise if a grouped product on ``device`` met bounds that it had to move, or gave up on a wait (synchronises the
    current stream).

    The device keeps one report for all streams and threads, the first since it was last asked: it is raised once, to whoever asks first.  What runs on
    other streams counts once it has run, and what a graph's replay reports as well."""
    read_status("pcl_grouped_status", device, "grouped product")


def read_status(entry: str, device, what: str) -> None:
    index = None if device is None else torch.device(device).index
    index = torch.cuda.current_device() if index is None else index
    status = torch.empty(4, dtype=torch.int64, device=f"cuda:{index}")
    _lib.call_on(index, entry, status.data_ptr())
    _lib.raise_status(status.cpu(), what)


def check_operand(t: torch.Tensor, name: str, dims: int, dtype=None) -> None:
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got {t.dim()}")
    if dtype is None:
        if t.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"{name} must be bfloat16 or float16, got {t.dtype}")
    elif t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def check_offsets(offsets: torch.Tensor) -> int:
    """Number of groups."""
    if offsets.dim() != 1 or offsets.dtype not in (torch.int32, torch.int64) or not offsets.is_contiguous():
        raise ValueError("offsets must be a contiguous one-dimensional tensor of int32 or int64")
    groups = offsets.numel() - 1
    if not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"offsets must have 2 to {MAX_GROUPS + 1} numbers, got {offsets.numel()}")
    return groups


def check_devices(**tensors) -> torch.device:
    """The one CUDA device that all of them are on (None: not given)."""
    device = None
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device.type != "cuda":
            raise ValueError(f"{name} must be a CUDA tensor")
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}")
    return device


def result_type(out: Optional[torch.Tensor], out_dtype: Optional[torch.dtype], default: torch.dtype, allowed) -> torch.dtype:
    dtype = out_dtype if out_dtype is not None else default if out is None else out.dtype
    if dtype not in allowed:
        raise ValueError(f"out_dtype must be one of {', '.join(map(str, allowed))}, got {dtype}")
    return dtype


def check_out(out: Optional[torch.Tensor], shape, dtype) -> None:
    """``out`` may be strided, but its rows are contiguous and apart."""
    if out is None:
        return
    check_operand(out, "out", len(shape), dtype)
    if tuple(out.shape) != tuple(shape):
        raise ValueError(f"out must be {tuple(shape)}, got {tuple(out.shape)}")
    if len(shape) == 3:
        if not out.is_contiguous():
            raise ValueError("out must be contiguous")
    elif (shape[1] > 1 and out.stride(1) != 1) or (shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError("out must have contiguous rows that do not overlap")


def aligned(x: torch.Tensor) -> torch.Tensor:
    """The 16-bit matrix or matrices ``x`` if the last dimension is contiguous and every row starts at a multiple of 16 bytes, as
    the tensor copies need it, else a copy that does."""
    if x.shape[-1] > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    if x.data_ptr() % 16 == 0 and all(s % 8 == 0 and s > 0 for s, n in zip(x.stride()[:-1], x.shape[:-1]) if n > 1):
        return x
    *mats, rows, cols = x.shape
    pitch = (cols + 7) // 8 * 8
    buf = torch.empty(*mats, rows, pitch, dtype=x.dtype, device=x.device)
    if not x.is_cuda:
        buf[..., :cols] = x
        return buf[..., :cols]
    step = stride_of(x, -2, pitch)
    step_e = stride_of(x, 0, rows * step) if mats else rows * step
    _lib.call_on(x.get_device(), "pcl_grouped_pad", x.data_ptr(), step_e, step, mats[0] if mats else 1, rows, cols, buf.data_ptr(),
                 0, 0, 0, 0, 0, 0, 0, 0, 0)
    return buf[..., :cols]


def stride_of(x: torch.Tensor, dim: int, size: int) -> int:
    """Elements from one index of ``dim`` to the next; a dimension of one index may report any stride."""
    return x.stride(dim) if x.shape[dim] > 1 else size


def _check_sizes(rows: int, **sizes) -> None:
    for name, v in sizes.items():
        if not 1 <= v < 1 << 30:
            raise ValueError(f"{name} must be 1 to 2^30 - 1, got {v}")
    if rows >= MAX_ROWS:
        raise ValueError(f"at most 2^31 - 513 rows, got {rows}")


def _check_rows(mode: int, X, W, offsets, out, dtype) -> None:
    """Raise for what is wrong with the operands of ``_rows``."""
    name = "X" if mode == 0 else "dY"
    check_operand(X, name, 2)
    check_operand(W, "W", 3, X.dtype)
    groups = check_offsets(offsets)
    E, N, K = W.shape
    if E != groups:
        raise ValueError(f"W has {E} matrices, offsets {groups} groups")
    given, cols = (K, N) if mode == 0 else (N, K)
    if X.shape[1] != given:
        raise ValueError(f"{name} must have {given} columns, got {X.shape[1]}")
    _check_sizes(X.shape[0], N=N, K=K)
    dtype = result_type(out, dtype, X.dtype, (X.dtype, torch.float32))
    check_out(out, (X.shape[0], cols), dtype)
    check_devices(**{name: X, "W": W, "offsets": offsets, "out": out})


def _rows(mode: int, X, W, offsets, out, out_dtype):
    # A call is a few microseconds on the device, and the long way costs the host about 11 (the plain one 6).
    if out is None and X.is_cuda:
        out = calls().grouped_rows(mode, X, W, offsets, out_dtype)
        if out is not None:
            _lib.count_launch()
            return out
    xs, ws, dtype, device = X.shape, W.shape, X.dtype, X.get_device()
    if not (len(xs) == 2 and len(ws) == 3 and (dtype == torch.bfloat16 or dtype == torch.float16) and W.dtype == dtype
            and xs[1] == ws[2 - mode] and 0 < ws[1] < 1 << 30 and 0 < ws[2] < 1 << 30 and xs[0] < MAX_ROWS
            and offsets.dim() == 1 and offsets.shape[0] == ws[0] + 1 and 0 < ws[0] <= MAX_GROUPS
            and (offsets.dtype == torch.int32 or offsets.dtype == torch.int64) and offsets.is_contiguous()
            and device >= 0 and W.get_device() == device and offsets.get_device() == device
            and out is None and (out_dtype is None or out_dtype == dtype or out_dtype == torch.float32)):
        _check_rows(mode, X, W, offsets, out, out_dtype)
    T, (E, N, K) = xs[0], ws
    cols = ws[1 + mode]
    fill = out is None
    if fill:
        out = torch.empty(T, cols, dtype=dtype if out_dtype is None else out_dtype, device=X.device)
    if T == 0:
        return out
    x, w = X.data_ptr(), W.data_ptr()
    ldx, unit = X.stride()
    ws_e, ws_n, w_unit = W.stride()
    if x & 15 or w & 15 or unit != 1 or w_unit != 1 or ldx & 7 or ws_n & 7 or ws_e & 7 or not (ldx and ws_n and ws_e):
        X, W = aligned(X), aligned(W)
        x, w = X.data_ptr(), W.data_ptr()
        ldx = stride_of(X, 0, (xs[1] + 7) // 8 * 8)
        ws_n = stride_of(W, 1, (K + 7) // 8 * 8)
        ws_e = stride_of(W, 0, ws_n * N)
    _lib.call_on(device, "pcl_grouped_rows", mode, TYPES[dtype], TYPES[out.dtype], x, ldx, w, ws_e, ws_n, offsets.data_ptr(),
                 offsets.dtype == torch.int64, out.data_ptr(), out.stride(0), T, E, N, K, fill)
    return out


def _check_tn(dY, X, offsets, out, dtype) -> None:
    """Raise for what is wrong with the operands of ``grouped_tn``."""
    check_operand(X, "X", 2)
    check_operand(dY, "dY", 2, X.dtype)
    E = check_offsets(offsets)
    if dY.shape[0] != X.shape[0]:
        raise ValueError(f"dY has {dY.shape[0]} rows, X {X.shape[0]}")
    _check_sizes(X.shape[0], N=dY.shape[1], K=X.shape[1])
    dtype = result_type(out, dtype, X.dtype, (X.dtype, torch.float32))
    check_out(out, (E, dY.shape[1], X.shape[1]), dtype)
    check_devices(dY=dY, X=X, offsets=offsets, out=out)


def grouped_nt(X: torch.Tensor, W: torch.Tensor, offsets: torch.Tensor, out: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``Y [T, N]`` with ``Y[t] = W[e] x[t]`` for the rows of every group ``e``.

    ``X [T, K]`` and ``W [E, N, K]`` may be strided; where rows do not start at multiples of 16 bytes (an odd K) they are copied
    first.  Rows that no group has, before ``offsets[0]`` or from ``offsets[E]`` on, are zero in a new result, and are
    left as they were in ``out``, which must not overlap an operand."""
    return _rows(0, X, W, offsets, out, out_dtype)


def grouped_nn(dY: torch.Tensor, W: torch.Tensor, offsets: torch.Tensor, out: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``dX [T, K]`` with ``dX[t] = W[e]^T dy[t]``: the gradient of ``grouped_nt`` with respect to ``X``, or the product with
    the matrices as they lie.  ``dY [T, N]``; otherwise as ``grouped_nt``."""
    return _rows(1, dY, W, offsets, out, out_dtype)


def grouped_tn(dY: torch.Tensor, X: torch.Tensor, offsets: torch.Tensor, out: Optional[torch.Tensor] = None,
               out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``dW [E, N, K]``, ``dW[e]`` the sum of ``dy[t] x[t]^T`` over the rows of group ``e`` (zero where it has none): the
    gradient of ``grouped_nt`` with respect to ``W``.  ``dY [T, N]``, ``X [T, K]``; ``out`` must be contiguous."""
    if out is None and X.is_cuda:
        out = calls().grouped_tn(dY, X, offsets, out_dtype)
        if out is not None:
            _lib.count_launch()
            return out
    xs, ys, dtype, device = X.shape, dY.shape, X.dtype, X.get_device()
    if not (len(xs) == 2 and len(ys) == 2 and (dtype == torch.bfloat16 or dtype == torch.float16) and dY.dtype == dtype
            and xs[0] == ys[0] and xs[0] < MAX_ROWS and 0 < xs[1] < 1 << 30 and 0 < ys[1] < 1 << 30
            and offsets.dim() == 1 and 1 < offsets.shape[0] <= MAX_GROUPS + 1
            and (offsets.dtype == torch.int32 or offsets.dtype == torch.int64) and offsets.is_contiguous()
            and device >= 0 and dY.get_device() == device and offsets.get_device() == device
            and out is None and (out_dtype is None or out_dtype == dtype or out_dtype == torch.float32)):
        _check_tn(dY, X, offsets, out, out_dtype)
    T, K, N, E = xs[0], xs[1], ys[1], offsets.shape[0] - 1
    if out is None:
        out = torch.empty(E, N, K, dtype=dtype if out_dtype is None else out_dtype, device=X.device)
    if T == 0:
        return out.zero_()
    x, y = X.data_ptr(), dY.data_ptr()
    ldx, unit = X.stride()
    ldy, y_unit = dY.stride()
    if x & 15 or y & 15 or unit != 1 or y_unit != 1 or ldx & 7 or ldy & 7 or not (ldx and ldy):
        X, dY = aligned(X), aligned(dY)
        x, y = X.data_ptr(), dY.data_ptr()
        ldx, ldy = stride_of(X, 0, (K + 7) // 8 * 8), stride_of(dY, 0, (N + 7) // 8 * 8)
    _lib.call_on(device, "pcl_grouped_tn", TYPES[dtype], TYPES[out.dtype], y, ldy, x, ldx, offsets.data_ptr(),
                 offsets.dtype == torch.int64, out.data_ptr(), T, E, N, K)
    return out
