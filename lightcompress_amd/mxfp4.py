"""Microscaled 4-bit numbers (MXFP4, OCP microscaling formats): quantization, and products on the matrix pipe that takes them as they are.

Blocks of 32 values along the last dimension share a power of two.  Next to ``FloatQuantizer('e2m1', ...)`` (quant.py:962-1080), whose
scales are floating-point numbers per group or channel and which leaves running the result to others, this is the form that MI355X
multiplies natively: four bits a value and a byte per block, for weights and activations alike.
All of this is forward only: nothing here records a gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .w8a8 import MOST_COLS, _at, _code, _cols, _here, _rows, _whole, _with, _workspace

BLOCK = 32
MOST_DISTANCE = 1 << 22


class Mxfp4(NamedTuple):
    """codes uint8 [..., 16 B]: two e2m1 codes a byte, the lower half first, B = ceil(cols / 32) blocks of 16 bytes, zeros behind the
    last column; scales uint8 [..., B]: byte s stands for 2^(s - 127), 255 for NaN.  cols None: 32 B.  (Tensors of torch's own
    float4_e2m1fn_x2 and float8_e8m0fnu are taken too.)"""
    codes: torch.Tensor
    scales: torch.Tensor
    cols: Optional[int] = None


_U8 = torch.uint8
_BYTES = (getattr(torch, 'float4_e2m1fn_x2', None), getattr(torch, 'float8_e8m0fnu', None))


def _plain(t, name):
    """t as bytes."""
    if t.dtype is _U8:
        return t
    if t.dtype not in _BYTES:
        raise L.LcqError(f'{name} are bytes (torch.uint8), got {t.dtype}')
    return t.view(_U8)


def _parts(q, name):
    """-> codes and scales as bytes, the number of columns."""
    codes, scales, cols = q.codes, q.scales, q.cols
    if codes.dtype is not _U8 or scales.dtype is not _U8:
        codes, scales = _plain(codes, f'{name} codes'), _plain(scales, f'{name} scales')
    shape, rows = scales.shape, codes.shape
    dims = len(shape)
    B = shape[-1] if dims else 0
    # (slices of a torch.Size cost half a microsecond each)
    if not B or len(rows) != dims or rows[-1] != 16 * B or (rows[0] != shape[0] if dims == 2 else rows[:-1] != shape[:-1]):
        raise ValueError(f'{name}: codes {tuple(rows)} and scales {tuple(shape)} are not blocks of 16 bytes and one')
    if cols is None:
        cols = BLOCK * B
    elif not BLOCK * (B - 1) < cols <= BLOCK * B:
        raise ValueError(f'{name}: {cols} columns in {B} blocks of {BLOCK}')
    return codes, scales, cols


def _byte_rows(t, width, step=1):
    """-> (t or a contiguous copy that starts on a multiple of `step` bytes, rows of `width`, distance between rows, such a multiple)."""
    if t.is_contiguous():
        return t if t.data_ptr() % step == 0 else t.clone(), t.numel() // width, width
    t, rows, ld = _rows(t, width)
    if rows == 1:
        ld = width
    if not width <= ld <= MOST_DISTANCE or ld % step:          # (rows on top of each other, far apart or off alignment)
        t, ld = t.contiguous(), width
    if t.data_ptr() % step:
        t, ld = t.clone(memory_format=torch.contiguous_format), width
    return t, rows, ld


def quantize_mxfp4(x):
    """The codes of x [..., K] (fp32, bf16, fp16): Mxfp4.  With m the largest magnitude of a block of 32 the scale is 2^(floor(log2 m) - 2)
    (at least 2^-127); codes are the nearest, a tie goes to the even one, what lies beyond 6 is 6.  A block with an
    infinity or a NaN is NaN throughout."""
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f'a last dimension of at least one column is needed, got shape {tuple(shape)}')
    K = shape[-1]
    code = _code(x.dtype)
    if not _here(x):
        with torch.cuda.device(x.device):
            return quantize_mxfp4(x)
    rows, T, ld = _rows(x, K)
    B = (K + BLOCK - 1) // BLOCK
    codes, scales = x.new_empty(_with(shape, 16 * B), dtype=torch.uint8), x.new_empty(_with(shape, B), dtype=torch.uint8)
    if T:
        L.check(L.lib().lcq_mxfp4_quant(rows.data_ptr(), code, T, K, ld, codes.data_ptr(), scales.data_ptr(), B, L.stream()), 'lcq_mxfp4_quant')
    return Mxfp4(codes, scales, K)


def dequantize_mxfp4(q, dtype=torch.bfloat16):
    """What q stands for, [..., cols] of `dtype` (fp32 and bf16 hold every value below 2^128, which quantize_mxfp4 does not pass; larger ones - 4 and
    6 with scale byte 253, 2 to 6 with 254 - are infinite.  fp16 rounds or overflows)."""
    codes, scales, K = _parts(q, 'q')
    code = _code(dtype)
    if not _here(codes, scales):
        with torch.cuda.device(codes.device):
            return dequantize_mxfp4(q, dtype)
    B = scales.shape[-1]
    codes, T, ldc = _byte_rows(codes, 16 * B, 4)
    scales, _, lds = _byte_rows(scales, B)
    y = codes.new_empty(_with(q.scales.shape, K), dtype=dtype)
    if T:
        L.check(L.lib().lcq_mxfp4_dequant(codes.data_ptr(), ldc, scales.data_ptr(), lds, T, K, y.data_ptr(), code, L.stream()), 'lcq_mxfp4_dequant')
    return y


def _check_weight(weight, bias, K):
    codes, scales, cols = _parts(weight, 'weight')
    if codes.dim() != 2 or cols != K:
        raise ValueError(f'a weight of {tuple(codes.shape[:-1])} rows and {cols} columns does not take tokens of {K} columns')
    N = codes.shape[0]
    if bias is not None and bias.shape != (N,):
        raise ValueError(f'the bias of {N} channels has shape {tuple(bias.shape)}')
    return codes, scales, N


def mxfp4_matmul(tokens, weight, bias=None, out_dtype=torch.bfloat16):
    """Tokens (Mxfp4, [..., K]) times a weight (Mxfp4, [N, K]), plus a bias [N] (fp32, bf16, fp16): [..., N] of `out_dtype`.  Products of codes and scales
    are exact, the sums are fp32, the result is rounded once.  Rows may lie apart; operands off 16 bytes are copied."""
    a, sa, K = _parts(tokens, 'tokens')
    if K > MOST_COLS:
        raise ValueError(f'at most {MOST_COLS} columns, got {K}')
    w, sw, N = _check_weight(weight, bias, K)
    code = _code(out_dtype)
    if not _here(a, sa, w, sw, bias):
        with torch.cuda.device(a.device):
            return mxfp4_matmul(tokens, weight, bias, out_dtype)
    shape, B = sa.shape, sa.shape[-1]
    a, M, lda = _byte_rows(a, 16 * B, 16)
    sa, _, ldsa = _byte_rows(sa, B)
    y = a.new_empty(_with(shape, N), dtype=out_dtype)
    if M and N:
        w, _, ldw = _byte_rows(w, 16 * B, 16)
        sw, _, ldsw = _byte_rows(sw, B)
        bias = _whole(bias)
        aligned = not (sa.data_ptr() | ldsa | sw.data_ptr() | ldsw) % 16
        ws = _workspace(a, 'lcq_mxfp4_matmul_workspace_bytes', M, N, K, aligned)
        L.check(L.lib().lcq_mxfp4_matmul(a.data_ptr(), lda, sa.data_ptr(), ldsa, w.data_ptr(), ldw, sw.data_ptr(), ldsw, _at(bias),
                                         0 if bias is None else _code(bias.dtype), M, N, K, y.data_ptr(), code, _at(ws), L.stream()),
                'lcq_mxfp4_matmul')
    return y


def mxfp4_linear(x, weight, bias=None, out_dtype=None):
    """A Linear with an MXFP4 weight [N, K] on x [..., K]: quantize_mxfp4(x), then mxfp4_matmul to x's type (or `out_dtype`)."""
    shape = x.shape
    K = _cols(shape)
    x_code = _code(x.dtype)
    if out_dtype is None:
        out_dtype = x.dtype
    code = _code(out_dtype)
    w, sw, N = _check_weight(weight, bias, K)
    if not _here(x, w, sw, bias):
        with torch.cuda.device(x.device):
            return mxfp4_linear(x, weight, bias, out_dtype)
    rows, M, ld = _rows(x, K)
    y = x.new_empty(_with(shape, N), dtype=out_dtype)
    if M and N:
        B = sw.shape[-1]
        w, _, ldw = _byte_rows(w, 16 * B, 16)
        sw, _, ldsw = _byte_rows(sw, B)
        bias = _whole(bias)
        ws = _workspace(x, 'lcq_mxfp4_linear_workspace_bytes', M, N, K)
        L.check(L.lib().lcq_mxfp4_linear(rows.data_ptr(), x_code, ld, w.data_ptr(), ldw, sw.data_ptr(), ldsw, _at(bias),
                                         0 if bias is None else _code(bias.dtype), M, N, K, y.data_ptr(), code, _at(ws), L.stream()),
                'lcq_mxfp4_linear')
    return y
