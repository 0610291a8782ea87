"""Matrices in four bits with a shared scale for every 32 values of a row, and their products (``csrc/cuda/mx4.cu``).

The format is OCP's MXFP4: elements E2M1 (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign), scales E8M0 (code c stands for 2^(c - 127), 255 for
NaN).  A table of factors, or the matrices of trained experts, take 17/32 of a byte a value: an eighth of fp32's.

* ``mx4_quantize(X)``                    ``Mx4Matrix`` of a float32, bfloat16 or float16 matrix;
* ``mx4_dequantize(Q)``                  its values;
* ``mx4_gemm_nt(A, B)``                  ``A @ B.T``, as ``gemm_nt``, on the tensor cores' four-bit instructions;
* ``mx4_grouped_nt(A, B, offsets)``      the same with one matrix for each group of rows, as ``grouped_nt``.

A block's scale is 2^(floor(log2 m) - 2) for its largest magnitude m (at least 2^-127), its values are divided by it and rounded to the
nearest element, ties to the even code, what is beyond 6 to 6.  A block that holds an infinity or a NaN is NaN as a whole.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib
from ._calls import calls
from .grouped import MAX_GROUPS, MAX_ROWS, TYPES, check_devices, check_offsets, check_out, read_status, result_type

BLOCK = 32


class Mx4Matrix:
    """``rows x cols`` values in four bits.

    ``data [rows, 16 ceil(cols / 32)]`` (uint8): value ``2 j`` of a row in the low half of its byte ``j``, value ``2 j + 1`` in the
    high half, zeros behind the last.  ``scales [ceil(cols / 128), rows, 4]`` (uint8): ``scales[b, r, i]`` is the code of block
    ``4 b + i`` of row ``r`` (255, which stands for NaN, only where the row has such a block)."""

    # _data and _scales are None where both lie in _buf, until they are asked for
    __slots__ = ("_data", "_scales", "_buf", "_device", "rows", "cols", "_data_ptr", "_scales_ptr")

    def __init__(self, data: torch.Tensor, scales: torch.Tensor, cols: int):
        ds, ss = data.shape, scales.shape
        data_ptr, scales_ptr, device = data.data_ptr(), scales.data_ptr(), data.get_device()
        if not (0 < cols < 1 << 30 and data.dtype == torch.uint8 and scales.dtype == torch.uint8 and len(ds) == 2 and len(ss) == 3
                and ds[1] == (cols + 31) // 32 * 16 and ss[0] == (cols + 127) // 128 and ss[1] == ds[0] and ss[2] == 4
                and ds[0] < MAX_ROWS and data.is_contiguous() and scales.is_contiguous()
                and not (data_ptr | scales_ptr) & 15 and scales.get_device() == device):
            self._refuse(data, scales, cols)
        self._data, self._scales, self._buf, self._device = data, scales, None, device
        self.rows, self.cols, self._data_ptr, self._scales_ptr = ds[0], cols, data_ptr, scales_ptr

    @classmethod
    def _of(cls, buf: torch.Tensor, device: int, rows: int, cols: int, data_ptr: int, scales_ptr: int) -> "Mx4Matrix":
        """One whose parts lie in ``buf``, the scales behind the data, and are looked at as tensors only when asked for."""
        q = cls.__new__(cls)
        q._data, q._scales, q._buf, q._device, q.rows, q.cols = None, None, buf, device, rows, cols
        q._data_ptr, q._scales_ptr = data_ptr, scales_ptr
        return q

    @property
    def data(self) -> torch.Tensor:
        if self._data is None:
            width = (self.cols + 31) // 32 * 16
            self._data = self._buf[:self.rows * width].view(self.rows, width)
        return self._data

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._buf[self.rows * ((self.cols + 31) // 32 * 16):].view((self.cols + 127) // 128, self.rows, 4)
        return self._scales

    @staticmethod
    def _refuse(data, scales, cols):
        if not 1 <= cols < 1 << 30:
            raise ValueError(f"cols must be 1 to 2^30 - 1, got {cols}")
        for t, name in ((data, "data"), (scales, "scales")):
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be contiguous uint8 that starts at a multiple of 16 bytes")
        if data.dim() != 2 or data.shape[1] != (cols + 31) // 32 * 16:
            raise ValueError(f"data must be [rows, {(cols + 31) // 32 * 16}] for {cols} columns, got {tuple(data.shape)}")
        if tuple(scales.shape) != ((cols + 127) // 128, data.shape[0], 4):
            raise ValueError(f"scales must be {((cols + 127) // 128, data.shape[0], 4)}, got {tuple(scales.shape)}")
        if scales.device != data.device:
            raise ValueError(f"scales must be on {data.device}, got {scales.device}")
        raise ValueError(f"at most 2^31 - 513 rows, got {data.shape[0]}")

    @property
    def device(self) -> torch.device:
        return (self._data if self._buf is None else self._buf).device

    def __reduce__(self):
        # copies and pickles are made of the two tensors: addresses are not theirs
        return Mx4Matrix, (self.data, self.scales, self.cols)

    def nbytes(self) -> int:
        return self.rows * ((self.cols + 31) // 32 * 16 + (self.cols + 127) // 128 * 4)

    def __repr__(self):
        return f"Mx4Matrix({self.rows} x {self.cols}, {self.device})"


def check_status(device=None) -> None:
    """Raise if a grouped four-bit product on ``device`` met bounds that it had to move, or one of these products gave up on
    a wait (synchronises the current stream; one report for all streams and threads, as ``ops.grouped.check_status`` says)."""
    read_status("pcl_mx4_status", device, "four-bit product")


def mx4_quantize(X: torch.Tensor) -> Mx4Matrix:
    """``X [rows, K]`` (float32, bfloat16, float16) in four bits; ``X [E, N, K]``, the matrices of E groups, becomes one
    of ``E N`` rows."""
    if X.is_cuda:
        parts = calls().quantize(X)
        if parts is not None:
            _lib.count_launch()
            return Mx4Matrix._of(*parts)
    shape, kind, device = X.shape, TYPES.get(X.dtype), X.get_device()
    if kind is None:
        raise ValueError(f"X must be float32, bfloat16 or float16, got {X.dtype}")
    if len(shape) != 2 and len(shape) != 3:
        raise ValueError(f"X must have 2 or 3 dimensions, got {len(shape)}")
    K = shape[-1]
    if not 1 <= K < 1 << 30:
        raise ValueError(f"X must have 1 to 2^30 - 1 columns, got {K}")
    if device < 0:
        check_devices(X=X)
    if len(shape) == 3:
        X = X.reshape(-1, K)
    X, ldx = _row_stride(X)
    rows = X.shape[0]
    if rows >= MAX_ROWS:
        raise ValueError(f"at most 2^31 - 513 rows, got {rows}")
    size = rows * ((K + 31) // 32 * 16)                  # a multiple of 16
    buf = torch.empty(size + (K + 127) // 128 * rows * 4, dtype=torch.uint8, device=X.device)
    q = Mx4Matrix._of(buf, device, rows, K, buf.data_ptr(), buf.data_ptr() + size)
    if rows:
        _lib.call_on(device, "pcl_mx4_quantize", X.data_ptr(), ldx, kind, q._data_ptr, q._scales_ptr, rows, K)
    return q


def _row_stride(X: torch.Tensor):
    """(``X``, or a copy of it, with contiguous rows; values from one row to the next)"""
    ldx, unit = X.stride()
    if unit != 1 and X.shape[1] > 1:
        X = X.contiguous()
        ldx = X.shape[1]
    return X, ldx


def mx4_dequantize(q: Mx4Matrix, dtype: torch.dtype = torch.float32, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values of ``q`` as ``[rows, cols]``.  float32 and bfloat16 hold every value exactly (but for those of 2^128 and more, infinite in
    either); float16 rounds."""
    if dtype not in TYPES:
        raise ValueError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    if out is None and q._device >= 0:
        out = calls().dequantize(q._data if q._buf is None else q._buf, q._data_ptr, q._scales_ptr, q.rows, q.cols, dtype)
        if out is not None:
            _lib.count_launch()
            return out
    if out is not None or q._device < 0:
        check_out(out, (q.rows, q.cols), dtype)
        check_devices(q=q, out=out)
    if out is None:
        out = torch.empty(q.rows, q.cols, dtype=dtype, device=q.device)
    if q.rows:
        _lib.call_on(q._device, "pcl_mx4_dequantize", q._data_ptr, q._scales_ptr, out.data_ptr(), out.stride(0), TYPES[dtype], q.rows,
                     q.cols)
    return out


def _check_product(A, B, offsets, out, dtype) -> None:
    """Raise for what is wrong with the operands of ``_product``."""
    if not isinstance(B, Mx4Matrix):
        raise ValueError("B must be an Mx4Matrix: quantise it once with mx4_quantize")
    packed = isinstance(A, Mx4Matrix)
    if not packed and (A.dim() != 2 or A.dtype not in TYPES):
        raise ValueError(f"A must be an Mx4Matrix or a matrix of float32, bfloat16 or float16, got {A.dtype} {tuple(A.shape)}")
    T, cols = (A.rows, A.cols) if packed else A.shape
    if cols != B.cols:
        raise ValueError(f"A has {cols} columns, B {B.cols}")
    groups = 1 if offsets is None else check_offsets(offsets)
    if B.rows == 0 or B.rows % groups:
        raise ValueError(f"B must have the same number of rows for each of the {groups} groups, at least one, got {B.rows}")
    if T >= MAX_ROWS:
        raise ValueError(f"at most 2^31 - 513 rows, got {T}")
    dtype = result_type(out, dtype, torch.float32 if packed else A.dtype, tuple(TYPES))
    check_out(out, (T, B.rows // groups), dtype)
    check_devices(A=A, B=B, offsets=offsets, out=out)


def _product(A, B: Mx4Matrix, offsets, out, out_dtype):
    packed = isinstance(A, Mx4Matrix)
    if not isinstance(B, Mx4Matrix):
        _check_product(A, B, offsets, out, out_dtype)
    K, rows, device = B.cols, B.rows, B._device
    if out is None and not packed and A.is_cuda:
        out = calls().mx4_rows(A, B._data_ptr, B._scales_ptr, rows, K, device, offsets, out_dtype)
        if out is not None:
            _lib.count_launch()
            return out
    if packed:
        T, cols, kind, place, own = A.rows, A.cols, -1, A._device, torch.float32
    else:
        T, cols = A.shape if A.dim() == 2 else (0, 0)
        own = A.dtype
        kind, place = TYPES.get(own), A.get_device()
    dtype = out_dtype if out_dtype is not None else out.dtype if out is not None else own
    groups = 1 if offsets is None else offsets.numel() - 1
    if not (cols == K and kind is not None and dtype in TYPES and out is None and T < MAX_ROWS
            and 0 < groups <= rows and rows % groups == 0 and device >= 0 and place == device
            and (offsets is None or offsets.dim() == 1 and groups <= MAX_GROUPS and offsets.get_device() == device
                 and (offsets.dtype == torch.int32 or offsets.dtype == torch.int64) and offsets.is_contiguous())):
        _check_product(A, B, offsets, out, out_dtype)
    N = rows // groups
    fill = out is None
    if fill:
        out = torch.empty(T, N, dtype=dtype, device=B.device)
    if T == 0:
        return out
    if packed:
        x, ldx, a, sa = 0, 0, A._data_ptr, A._scales_ptr
    else:
        # A in four bits, for the length of the call
        A, ldx = _row_stride(A)
        size = T * ((K + 31) // 32 * 16)
        work = torch.empty(_lib.load().pcl_mx4_room(kind, T, groups, N, K), dtype=torch.uint8, device=out.device)
        x, a = A.data_ptr(), work.data_ptr()
        sa = a + size
    _lib.call_on(device, "pcl_mx4_rows", x, ldx, kind, a, sa, B._data_ptr, B._scales_ptr, None if offsets is None else offsets.data_ptr(),
                 offsets is not None and offsets.dtype == torch.int64, out.data_ptr(), out.stride(0), TYPES[dtype], T, groups, N, K, fill)
    return out


def mx4_gemm_nt(A: Union[torch.Tensor, Mx4Matrix], B: Mx4Matrix, out: Optional[torch.Tensor] = None,
                out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``A @ B.T`` for ``A [M, K]`` and ``B [N, K]`` in four bits; an ``A`` in float32, bfloat16 or float16 is quantised here.
    Products are exact, and sums are held in float32: sums of blocks with scales that lie close together are exact as well, others off by 3e-7 at 32768 terms and
    9e-6 at 131072 (3e-5 of one sign).  ``out`` must not overlap an operand.  The result has ``out``'s type, ``out_dtype``, ``A``'s own, or float32 if A is in four bits."""
    return _product(A, B, None, out, out_dtype)


def mx4_grouped_nt(A: Union[torch.Tensor, Mx4Matrix], B: Mx4Matrix, offsets: torch.Tensor, out: Optional[torch.Tensor] = None,
                   out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``Y[t] = B[e] a[t]`` for the rows ``offsets[e] <= t < offsets[e + 1]`` of ``A [T, K]``; ``B`` holds the N rows of every
    group one after the other (``mx4_quantize`` of an ``[E, N, K]`` tensor).  Offsets and rows that no group has are
    treated as in ``grouped_nt``."""
    if offsets is None:
        raise ValueError("offsets must be a CUDA tensor; a product without groups is mx4_gemm_nt")
    return _product(A, B, offsets, out, out_dtype)
