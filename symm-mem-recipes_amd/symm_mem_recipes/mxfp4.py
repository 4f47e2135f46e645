"""4-bit microscaled operands (OCP MXFP4: e2m1 elements, one power-of-two scale per 32 of
them along the contracted axis): quantisation, the values back, and the product of two
operands.  The next narrower type after the e4m3fn switch of the all-gather matmul
(symm_mem_recipes/triton_all_gather_matmul.py:115,123,188); that product takes no 4-bit operands, this one multiplies
what one GPU holds.

For training, the two products of a linear layer's backward pass contract over the layer's
outputs and over the tokens; ``mxfp4_quantize(..., transpose=True)`` gives their operands::

    y  = mxfp4_matmul(x, mxfp4_quantize(w))                       # x [T, K], w [N, K]
    dx = mxfp4_matmul(dy, mxfp4_quantize(w, transpose=True))      # contracts over N
    dw = mxfp4_matmul(mxfp4_quantize(dy, transpose=True),         # contracts over T
                      mxfp4_quantize(x, transpose=True))

Nothing here is recorded by autograd.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib

#: elements that share a scale; rows and contracted extent of a storage unit
BLOCK, UNIT_ROWS, SLAB = 32, 16, 256
#: rows of ``b`` that the product of a few bf16 or fp32 rows takes in one launch
_ROWS_MAX_N = 2 ** 28 - 64

_DTYPE_CODE = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_FP32}
#: the current stream's handle without building a torch.cuda.Stream object around it
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _call(index: int, what: str, fn, *args) -> None:
    """``fn(*args, stream)`` on the current stream of GPU ``index``, with that GPU current."""
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        _lib.check(rc, what)


def _span(t: torch.Tensor):
    """First and last byte + 1 that a tensor's elements lie in."""
    first = t.data_ptr()
    return first, first + (1 + sum((n - 1) * step for n, step in zip(t.shape, t.stride()))) * t.element_size()


def _check_apart(out: torch.Tensor, *inputs: torch.Tensor) -> None:
    """``out`` shares no memory with ``inputs``: workgroups write while others still read."""
    if out.numel() == 0:
        return
    first, end = _span(out)
    for t in inputs:
        if t.numel() != 0:
            t_first, t_end = _span(t)
            assert end <= t_first or t_end <= first, "out must not overlap an input"


def _units(rows: int, cols: int) -> int:
    return -(-rows // UNIT_ROWS) * -(-cols // SLAB)


def _check_extents(rows: int, cols: int) -> None:
    assert 0 <= rows < 2 ** 31 and 0 <= cols < 2 ** 31, "rows and cols must be in 0..2^31-1"
    assert rows or cols, "rows and cols must not both be 0"


class MxFp4Tensor:
    """A matrix ``[rows, cols]`` in 4-bit microscaled floats, ``cols`` the axis that a product
    contracts, kept in the order the matrix cores take it (``smr.h``: ``smr_mxfp4_code_bytes``).
    Made by :func:`mxfp4_quantize` or :meth:`from_blocks`; ``storage`` (uint8) holds its codes and,
    behind them, its scales."""

    __slots__ = ("storage", "rows", "cols")

    def __init__(self, storage: torch.Tensor, rows: int, cols: int):
        """``storage`` as smr.h lays it out, 16-byte aligned."""
        _check_extents(rows, cols)
        assert storage.dtype == torch.uint8 and storage.is_contiguous(), "storage must be contiguous uint8"
        assert storage.shape == (_units(rows, cols) * 2176,), "storage must be [units * 2176]"
        assert storage.data_ptr() % 16 == 0, "storage must be aligned to 16 bytes"
        self.storage, self.rows, self.cols = storage, rows, cols

    @property
    def shape(self) -> torch.Size:
        return torch.Size((self.rows, self.cols))

    @property
    def device(self) -> torch.device:
        return self.storage.device

    @property
    def codes(self) -> torch.Tensor:
        return self.storage[:_units(self.rows, self.cols) * 2048]

    @property
    def scales(self) -> torch.Tensor:
        return self.storage[_units(self.rows, self.cols) * 2048:]

    def _ptrs(self):
        codes = self.storage.data_ptr()
        return codes, codes + _units(self.rows, self.cols) * 2048

    def __repr__(self) -> str:
        return f"MxFp4Tensor(rows={self.rows}, cols={self.cols}, device={self.device})"

    @staticmethod
    def empty(rows: int, cols: int, device) -> "MxFp4Tensor":
        """Storage for a matrix, its values undefined."""
        _check_extents(rows, cols)
        q = MxFp4Tensor.__new__(MxFp4Tensor)
        q.storage = torch.empty(_units(rows, cols) * 2176, dtype=torch.uint8, device=device)
        q.rows, q.cols = rows, cols
        return q

    @staticmethod
    def from_blocks(codes: torch.Tensor, scales: torch.Tensor, cols: Optional[int] = None) -> "MxFp4Tensor":
        """From the layout checkpoints use: ``codes`` uint8 [rows, blocks * 16], two elements a
        byte, the first in the low half, and ``scales`` uint8 [rows, blocks] biased exponents,
        a block being 32 columns.  ``cols`` (default: blocks * 32) says how many columns are
        real; what the last block holds past them is taken as zero."""
        assert codes.dtype == torch.uint8 and scales.dtype == torch.uint8, "codes and scales must be uint8"
        assert codes.dim() == 2 and scales.dim() == 2 and codes.shape[0] == scales.shape[0]
        assert codes.device == scales.device, "codes and scales must be on one device"
        rows, blocks = scales.shape
        assert codes.shape[1] == blocks * (BLOCK // 2), "codes must have 16 bytes per block"
        cols = blocks * BLOCK if cols is None else int(cols)
        assert blocks == -(-cols // BLOCK), "cols must end in the last block"
        _check_extents(rows, cols)
        row_units, slabs = -(-rows // UNIT_ROWS), -(-cols // SLAB)
        padded = torch.zeros(row_units * UNIT_ROWS, slabs * SLAB // 2, dtype=torch.uint8, device=codes.device)
        used = -(-cols // 2)
        padded[:rows, :used] = codes[:, :used]
        if cols % 2:
            padded[:rows, used - 1] &= 15
        padded = padded.view(row_units, UNIT_ROWS, slabs, 2, 4, 16)          # unit row, row, slab, step, block, byte
        exponents = torch.zeros(row_units * UNIT_ROWS, slabs * 8, dtype=torch.uint8, device=codes.device)
        exponents[:rows, :blocks] = scales
        exponents = exponents.view(row_units, UNIT_ROWS, slabs, 2, 4)
        return MxFp4Tensor(torch.cat((padded.permute(2, 0, 3, 4, 1, 5).reshape(-1),
                                      exponents.permute(2, 0, 4, 1, 3).reshape(-1))), rows, cols)

    def to_blocks(self):
        """``(codes, scales)`` in the layout :meth:`from_blocks` takes."""
        row_units, slabs = -(-self.rows // UNIT_ROWS), -(-self.cols // SLAB)
        blocks = -(-self.cols // BLOCK)
        codes = self.codes.view(slabs, row_units, 2, 4, UNIT_ROWS, 16).permute(1, 4, 0, 2, 3, 5)
        scales = self.scales.view(slabs, row_units, 4, UNIT_ROWS, 2).permute(1, 3, 0, 4, 2)
        return (codes.reshape(row_units * UNIT_ROWS, slabs * SLAB // 2)[:self.rows, :blocks * 16].contiguous(),
                scales.reshape(row_units * UNIT_ROWS, slabs * 8)[:self.rows, :blocks].contiguous())

    def dequantize(self, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The values, ``[rows, cols]`` bf16 or fp32: exact in both, but for those of a checkpoint's scale codes 253 and
        254 that are past both types and become infinite."""
        storage = self.storage
        if out is None:
            assert dtype in _DTYPE_CODE, "Only bfloat16 and float32 are supported for now."
            out = torch.empty((self.rows, self.cols), dtype=dtype, device=storage.device)
        else:
            assert out.dtype in _DTYPE_CODE, "Only bfloat16 and float32 are supported for now."
            assert tuple(out.shape) == (self.rows, self.cols) and out.is_contiguous(), "out must be contiguous [rows, cols]"
            assert out.device == storage.device, "out must be on the operand's device"
            _check_apart(out, storage)
        assert storage.is_cuda, "the operand must be on a GPU"
        codes, scales = self._ptrs()
        _call(storage.get_device(), "mxfp4_dequantize", _lib.load().smr_mxfp4_dequantize, codes, scales, out.data_ptr(),
              self.rows, self.cols, _DTYPE_CODE[out.dtype])
        return out


def _check_rows(x: torch.Tensor) -> int:
    """Validates a matrix whose rows are to be quantised; elements from row to row."""
    assert x.dtype in _DTYPE_CODE, "Only bfloat16 and float32 are supported for now."
    assert x.dim() == 2, "x must be a matrix"
    rows, cols = x.shape
    assert cols <= 1 or x.stride(1) == 1, "the elements of a row must be adjacent"
    if rows <= 1:
        return cols
    row_stride = x.stride(0)
    assert row_stride >= cols, "the rows of x must not overlap"
    return row_stride


def mxfp4_quantize(x: torch.Tensor, *, transpose: bool = False, out: Optional[MxFp4Tensor] = None) -> MxFp4Tensor:
    """``x`` [rows, cols] bf16 or fp32, elements of a row adjacent (rows may be apart), in 4-bit
    microscaled floats with blocks of 32 along its rows.

    ``transpose`` blocks along the columns: the operand of ``x.T``, for products that contract
                  over ``x``'s rows.
    ``out``       an operand of the result's shape to write into, apart from ``x``.

    A block's scale is ``2 ** (floor(log2(max |block|)) - 2)``, at least 2^-127; its elements round
    to nearest even and saturate at 6 scales.  A block with an infinity or a NaN becomes NaN."""
    row_stride = _check_rows(x)
    rows, cols = x.shape
    assert x.is_cuda, "x must be on a GPU"
    if out is None:
        out = MxFp4Tensor.empty(cols, rows, x.device) if transpose else MxFp4Tensor.empty(rows, cols, x.device)
    else:
        assert (out.rows, out.cols) == ((cols, rows) if transpose else (rows, cols)), "out has another shape"
        assert out.device == x.device, "out must be on x's device"
        _check_apart(out.storage, x)
    codes, scales = out._ptrs()
    _call(x.get_device(), "mxfp4_quantize", _lib.load().smr_mxfp4_quantize, x.data_ptr(), row_stride, codes, scales, rows,
          cols, _DTYPE_CODE[x.dtype], 1 if transpose else 0)
    return out


def mxfp4_matmul(a: Union[MxFp4Tensor, torch.Tensor], b: MxFp4Tensor, *, out_dtype: torch.dtype = torch.bfloat16,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a @ b.T`` for ``a`` [M, K] and ``b`` [N, K], accumulated in fp32 - in an order that depends
    on the sizes only - and rounded once to ``out_dtype`` (bf16 or fp32).  A bf16 or fp32 ``a`` is
    quantised on the way, as by :func:`mxfp4_quantize`; for up to 16 rows the order of the sum may
    then be another.  ``out`` may not overlap an operand.  K = 0 (a weight's gradient over no tokens)
    gives zeros."""
    assert isinstance(b, MxFp4Tensor), "b must be an MxFp4Tensor"
    quantised = isinstance(a, MxFp4Tensor)
    shape = a.shape
    assert len(shape) == 2 and shape[1] == b.cols, "a and b must be matrices with one contracted extent"
    device = b.device
    assert a.device == device, "a and b must be on one device"
    assert device.type == "cuda", "the operands must be on a GPU"
    M, N = shape[0], b.rows
    if out is None:
        assert out_dtype in _DTYPE_CODE, "Only bfloat16 and float32 are supported for now."
        out = torch.empty(M, N, dtype=out_dtype, device=device)
    else:
        assert out.dtype in _DTYPE_CODE, "Only bfloat16 and float32 are supported for now."
        assert tuple(out.shape) == (M, N) and out.is_contiguous(), "out must be contiguous [M, N]"
        assert out.device == device, "out must be on the operands' device"
        _check_apart(out, a.storage if quantised else a, b.storage)
        out_dtype = out.dtype
    if b.cols == 0:
        if not quantised:
            _check_rows(a)
        return out.zero_()
    lib = _lib.load()
    if not quantised:
        if M <= UNIT_ROWS and N <= _ROWS_MAX_N and M <= lib.smr_mxfp4_matmul_rows_limit(b.cols):
            row_stride = _check_rows(a)
            _call(a.get_device(), "mxfp4_matmul", lib.smr_mxfp4_matmul_rows, a.data_ptr(), row_stride, _DTYPE_CODE[a.dtype],
                  *b._ptrs(), out.data_ptr(), M, N, b.cols, _DTYPE_CODE[out_dtype])
            return out
        a = mxfp4_quantize(a)
    _call(device.index, "mxfp4_matmul", lib.smr_mxfp4_matmul, *a._ptrs(), *b._ptrs(), out.data_ptr(), M, N, b.cols,
          _DTYPE_CODE[out_dtype])
    return out
