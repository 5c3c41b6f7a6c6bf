"""Running a w8a8 model: int8 codes of tokens, the int8 product with a scale for each token and channel, and the norm
between two blocks that can hand its result on as codes.

``VllmRealQuantLinear`` (module_utils.py:855-955) holds such a Linear's int8 weight and its scale per channel; the
reference leaves running it to the serving engine, here its ``forward`` is ``int8_linear``.  The codes of activations
are those of ``IntegerQuantizer`` with granularity per_token (quant.py:544-558, 698-716) on fp32 rows.
All of this is forward only: nothing here records a gradient.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional

import torch

from . import _lib as L

NORM_LAYER, NORM_POST_WEIGHT_F32, NORM_POST_BIAS_F32, NORM_WEIGHT_F32, NORM_BIAS_F32, NORM_RESIDUAL_F32 = 1, 2, 4, 8, 16, 32
NORM_OUT_F32, NORM_ASYM = 64, 128
MOST_COLS = 65536


class QuantizedTokens(NamedTuple):
    """(codes - zeros) * scales stands for the tokens; zero points are within -128 .. 127."""
    codes: torch.Tensor                       # int8 [..., K]
    scales: torch.Tensor                      # fp32 [..., 1], or one for all tokens
    zeros: Optional[torch.Tensor] = None      # int32 [..., 1]; None: 0


class ResidualNorm(NamedTuple):
    out: object                               # a tensor, or QuantizedTokens
    residual: torch.Tensor


_CODES = {torch.float32: L.F32, torch.bfloat16: L.BF16, torch.float16: L.F16}
_current = torch._C._cuda_getDevice


def _code(dtype):
    code = _CODES.get(dtype)
    return L.dtype_code(dtype) if code is None else code


def _here(x, *others):
    """Checks that all tensors are on x's GPU.  -> is that the current one?  (If not, the caller runs again with it made current:
    kernels go to the current device's current stream.)"""
    index = x.get_device()
    if index < 0:
        raise L.LcqError('liblcq operates on GPU tensors only (no CPU fallback)')
    for t in others:
        if t is not None and t.get_device() != index:
            raise L.LcqError(f'a tensor of the call is on {t.device}, the tokens are on {x.device}')
    return index == _current()


@lru_cache(maxsize=1024)
def _bytes(entry, *sizes):
    """What a workspace entry of the library answers for these sizes (its answer depends on nothing else)."""
    return getattr(L.lib(), entry)(*sizes)


def _workspace(x, entry, *sizes):
    size = _bytes(entry, *sizes)
    return x.new_empty(size, dtype=torch.uint8) if size else None


def _like(x, dtype):
    """A new contiguous tensor of x's shape.  (empty_like keeps strides, so only where they are those; it costs a third less.)"""
    if x.is_contiguous():
        return torch.empty_like(x) if dtype is x.dtype else torch.empty_like(x, dtype=dtype)
    return torch.empty(x.shape, dtype=dtype, device=x.device)


def _rows(t, K):
    """-> (t or a contiguous copy, number of rows of K elements, distance between rows)."""
    if t.is_contiguous():
        return t, t.numel() // K, K
    if t.dim() == 2 and t.stride(1) == 1:
        return t, t.shape[0], t.stride(0)
    t = t.contiguous()
    return t, t.numel() // K, K


def _with(shape, n):
    """`shape` with n columns.  (Slicing a torch.Size costs half a microsecond.)"""
    return (shape[0], n) if len(shape) == 2 else (*shape[:-1], n)


def _cols(shape):
    """-> the last of a shape's sizes, the columns of the tokens."""
    if not shape or shape[-1] == 0:
        raise ValueError(f'tokens need a last dimension of at least one column, got shape {tuple(shape)}')
    K = shape[-1]
    if K > MOST_COLS:
        raise ValueError(f'at most {MOST_COLS} columns, got {K}')
    return K


def _given(scale, symmetric):
    if not symmetric:
        raise ValueError('a given scale is a symmetric one')
    if scale.numel() != 1:
        raise ValueError(f'one scale for all tokens, got {tuple(scale.shape)}')
    return scale.reshape(1).float()


def quantize_tokens(x, symmetric=True, scale=None):
    """Int8 codes of the tokens x [..., K] (fp32, bf16, fp16), one fp32 scale per token (and, not symmetric, one zero
    point): QuantizedTokens.  `scale`: one given fp32 scale for all tokens (static activations, symmetric)."""
    shape = x.shape
    K = _cols(shape)
    code = _code(x.dtype)
    given = None if scale is None else _given(scale, symmetric)
    if not _here(x, given):
        with torch.cuda.device(x.device):
            return quantize_tokens(x, symmetric, scale)
    rows, T, ld = _rows(x, K)
    one = _with(shape, 1)
    codes = _like(x, torch.int8)
    scales = x.new_empty(one, dtype=torch.float32) if given is None else given
    zeros = None if symmetric else x.new_empty(one, dtype=torch.int32)
    if T:
        L.check(L.lib().lcq_quant_tokens(rows.data_ptr(), code, T, K, ld, not symmetric, None if given is None else given.data_ptr(),
                                         codes.data_ptr(), scales.data_ptr(), None if symmetric else zeros.data_ptr(), L.stream()),
                'lcq_quant_tokens')
    return QuantizedTokens(codes, scales, zeros)


def _at(t):
    return None if t is None else t.data_ptr()


def _whole(t):
    """t (or None), or a contiguous copy."""
    return t if t is None or t.is_contiguous() else t.contiguous()


def _on16(t):
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _check_weight(weight, weight_scales, bias, K):
    if weight.dtype != torch.int8:
        raise L.LcqError(f'an int8 weight is needed, got {weight.dtype}')
    shape = weight.shape
    if len(shape) != 2 or shape[1] != K:
        raise ValueError(f'weight {tuple(shape)} does not take tokens of {K} columns')
    N = shape[0]
    if weight_scales.numel() not in (1, N):
        raise ValueError(f'{N} weight scales (or one) are needed, got {tuple(weight_scales.shape)}')
    if bias is not None and bias.shape != (N,):
        raise ValueError(f'the bias of {N} channels has shape {tuple(bias.shape)}')
    return N


def int8_matmul(tokens, weight, weight_scales, bias=None, out_dtype=torch.bfloat16):
    """Tokens as codes (QuantizedTokens, codes [..., K]) times an int8 weight [N, K] with a scale per channel ([N], [N, 1], or
    one for all; fp32, bf16, fp16), plus a bias [N]: [..., N] of `out_dtype`.  The sums are exact integers, scales and bias
    are applied in fp32, the result is rounded once.  Operands with strides (the last token's codes of each sequence) are copied, a
    weight too, and in every call."""
    codes, scales, zeros = tokens
    shape = codes.shape
    K = _cols(shape)
    if codes.dtype != torch.int8 or scales.dtype != torch.float32 or (zeros is not None and zeros.dtype != torch.int32):
        raise L.LcqError('tokens are int8 codes with fp32 scales and int32 zero points')
    N = _check_weight(weight, weight_scales, bias, K)
    M = codes.numel() // K
    if scales.numel() not in (1, M) or (zeros is not None and zeros.numel() != M):
        raise ValueError(f'{M} token scales and zero points are needed, got {tuple(scales.shape)}'
                         + ('' if zeros is None else f' and {tuple(zeros.shape)}'))
    code = _code(out_dtype)
    if not _here(codes, scales, zeros, weight, weight_scales, bias):
        with torch.cuda.device(codes.device):
            return int8_matmul(tokens, weight, weight_scales, bias, out_dtype)
    codes, scales, zeros = _whole(codes), _whole(scales), _whole(zeros)
    weight, weight_scales, bias = _whole(weight), _whole(weight_scales), _whole(bias)
    if K % 16 == 0:                           # (rows of other widths may start anywhere)
        codes, weight = _on16(codes), _on16(weight)
    y = codes.new_empty(_with(shape, N), dtype=out_dtype)
    if M and N:
        ws = _workspace(codes, 'lcq_int8_matmul_workspace_bytes', M, N, K)
        L.check(L.lib().lcq_int8_matmul(codes.data_ptr(), scales.data_ptr(), scales.numel() == 1, _at(zeros), weight.data_ptr(),
                                        weight_scales.data_ptr(), _code(weight_scales.dtype), weight_scales.numel() == 1, _at(bias),
                                        0 if bias is None else _code(bias.dtype), M, N, K, y.data_ptr(), code, _at(ws),
                                        L.stream()), 'lcq_int8_matmul')
    return y


def int8_linear(x, weight, weight_scales, bias=None, symmetric=True, scale=None, out_dtype=None):
    """A w8a8 Linear on x [..., K]: quantize_tokens(x, symmetric, scale), then int8_matmul to x's type (or `out_dtype`)."""
    shape = x.shape
    K = _cols(shape)
    x_code = code = _code(x.dtype)
    if out_dtype is None:
        out_dtype = x.dtype
    else:
        code = _code(out_dtype)
    given = None if scale is None else _given(scale, symmetric)
    N = _check_weight(weight, weight_scales, bias, K)
    if not _here(x, given, weight, weight_scales, bias):
        with torch.cuda.device(x.device):
            return int8_linear(x, weight, weight_scales, bias, symmetric, scale, out_dtype)
    rows, M, ld = _rows(x, K)
    weight, weight_scales, bias = _whole(weight), _whole(weight_scales), _whole(bias)
    if K % 16 == 0:                           # (rows of other widths may start anywhere)
        weight = _on16(weight)
    y = x.new_empty(_with(shape, N), dtype=out_dtype)
    if M and N:
        ws = _workspace(x, 'lcq_int8_linear_workspace_bytes', M, N, K)
        L.check(L.lib().lcq_int8_linear(rows.data_ptr(), x_code, ld, not symmetric, _at(given), weight.data_ptr(),
                                        weight_scales.data_ptr(), _code(weight_scales.dtype), weight_scales.numel() == 1, _at(bias),
                                        0 if bias is None else _code(bias.dtype), M, N, K, y.data_ptr(), code, _at(ws),
                                        L.stream()), 'lcq_int8_linear')
    return y


def _affine(name, t, K, dtype, flag):
    """The flag of a [K] parameter of a norm: of the tokens' type, or fp32."""
    if t.shape != (K,):
        raise ValueError(f'{name} of {K} columns has shape {tuple(t.shape)}')
    if t.dtype is dtype:
        return 0
    if t.dtype != torch.float32:
        raise L.LcqError(f'{name} is {t.dtype}: the tokens\' {dtype} or float32 is needed')
    return flag


def _meets(t, out, read_before):
    """Does t lie where the contiguous `out` is written?  What is read before that (read_before) may lie there element on element."""
    if not t.numel() or (read_before and t.data_ptr() == out.data_ptr() and t.dtype == out.dtype and t.shape == out.shape and t.is_contiguous()):
        return False
    span = (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    return t.data_ptr() < out.data_ptr() + out.numel() * out.element_size() and out.data_ptr() < t.data_ptr() + span


def residual_norm(x, residual=None, weight=None, bias=None, *, gate=None, post_weight=None, post_bias=None, scale=1.0,
                  eps=1e-6, kind='rms', weight_offset=0.0, quantize=None, out_dtype=None, inplace=False):
    """The end of one block and the start of the next, for the block's output x [..., K], in one pass:

        b = x, or norm(x) with post_weight / post_bias where post_weight is given
        h = residual + scale * (gate * b)                       the residual stream
        out = norm(h) with weight / bias                        the next block's input

    kind 'rms': norm(v) = v / sqrt(mean v^2 + eps) * (w + weight_offset) + b;  'layer': the same of v - mean v.
    residual: like x, in x's type or fp32 (the stream keeps it); None: 0.  gate: like x, or [K]; None: 1.  A missing
    weight is 1 without an offset.  quantize 'symmetric' / 'asymmetric': out is quantize_tokens of the unrounded norm.
    out_dtype: x's type (default) or fp32.  inplace: h is written over residual, which may be x itself.  -> ResidualNorm(out, residual = h)"""
    shape, dtype = x.shape, x.dtype
    K = _cols(shape)
    code = _code(dtype)
    if kind not in ('rms', 'layer') or quantize not in (None, 'symmetric', 'asymmetric'):
        raise ValueError(f'kind {kind!r}, quantize {quantize!r}')
    if post_bias is not None and post_weight is None:
        raise ValueError('post_bias goes with post_weight')
    flags = NORM_LAYER if kind == 'layer' else 0
    if weight is not None:
        flags |= _affine('weight', weight, K, dtype, NORM_WEIGHT_F32)
        weight = _whole(weight)
    if bias is not None:
        flags |= _affine('bias', bias, K, dtype, NORM_BIAS_F32)
        bias = _whole(bias)
    if post_weight is not None:
        flags |= _affine('post_weight', post_weight, K, dtype, NORM_POST_WEIGHT_F32)
        post_weight = _whole(post_weight)
    if post_bias is not None:
        flags |= _affine('post_bias', post_bias, K, dtype, NORM_POST_BIAS_F32)
        post_bias = _whole(post_bias)
    stream_dtype = dtype
    if residual is not None:
        if residual.shape != shape:
            raise ValueError(f'residual {tuple(residual.shape)} next to x {tuple(shape)}')
        if residual.dtype is not dtype:
            if residual.dtype != torch.float32:
                raise L.LcqError(f'residual is {residual.dtype}: x\'s {dtype} or float32 is needed')
            stream_dtype = torch.float32
            flags |= NORM_RESIDUAL_F32
    if inplace:
        if residual is None or not residual.is_contiguous():
            raise ValueError('inplace needs a contiguous residual')
        if residual.requires_grad and torch.is_grad_enabled():
            raise ValueError('inplace would change a residual that autograd keeps')
        for t in (x, gate, post_weight, post_bias, weight, bias):
            if t is not None and _meets(t, residual, t is not weight and t is not bias):      # (the last norm reads its own behind h)
                raise ValueError('inplace would write over a part of another operand that is still read')
    if gate is not None:
        if gate.dtype is not dtype:
            raise L.LcqError(f'gate is {gate.dtype}, x is {dtype}')
        if gate.shape != shape and gate.shape != (K,):
            raise ValueError(f'gate {tuple(gate.shape)} next to x {tuple(shape)}')
    if out_dtype is None or out_dtype == dtype:
        out_dtype = dtype
    elif out_dtype == torch.float32:
        flags |= NORM_OUT_F32
    else:
        raise L.LcqError(f'out_dtype {out_dtype}: x\'s {dtype} or float32 is needed')
    if not _here(x, residual, weight, bias, gate, post_weight, post_bias):
        with torch.cuda.device(x.device):
            return residual_norm(x, residual, weight, bias, gate=gate, post_weight=post_weight, post_bias=post_bias, scale=scale,
                                 eps=eps, kind=kind, weight_offset=weight_offset, quantize=quantize, out_dtype=out_dtype, inplace=inplace)
    rows, T, ldx = _rows(x, K)
    res, ldr, g, ldg = residual, 0, gate, 0
    if residual is not None:
        res, _, ldr = _rows(residual, K)
    if gate is not None:
        g, _, ldg = (_whole(gate), 1, 0) if gate.dim() == 1 else _rows(gate, K)
    h = residual if inplace else _like(x, stream_dtype)
    out = codes = scales = zeros = None
    if quantize is None:
        out = _like(x, out_dtype)
    else:
        codes = _like(x, torch.int8)
        scales = x.new_empty(_with(shape, 1), dtype=torch.float32)
        if quantize == 'asymmetric':
            flags |= NORM_ASYM
            zeros = x.new_empty(_with(shape, 1), dtype=torch.int32)
    if T:
        L.check(L.lib().lcq_residual_norm(
            rows.data_ptr(), code, T, K, ldx, _at(res), ldr, _at(g), ldg, _at(post_weight), _at(post_bias), _at(weight), _at(bias),
            scale, eps, weight_offset, flags, h.data_ptr(), _at(out), _at(codes), _at(scales), _at(zeros), L.stream()), 'lcq_residual_norm')
        if inplace:                           # (so that a backward pass which kept the old values says so)
            torch.autograd.graph.increment_version(residual)
    return ResidualNorm(out if quantize is None else QuantizedTokens(codes, scales, zeros), h)
