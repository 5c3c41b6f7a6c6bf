"""A mixture-of-experts layer on MXFP4 experts, for the few tokens of a decoding step, and the router in front of it.

The quantizers take the experts of a layer several at a time (``quant.experts_as_rows``); what ``quantize_mxfp4`` makes of their stacked
weights runs here: tokens that chose the same expert share one pass over its bytes, activations keep their precision.
All of this is forward only: nothing here records a gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib as L
from .mxfp4 import BLOCK, MOST_DISTANCE, Mxfp4, _parts
from .w8a8 import _at, _code, _cols, _here, _rows, _whole, _with, _workspace

MOST_EXPERTS, MOST_TOP = 1024, 32
_SCORING = {'softmax': 0, 'sigmoid': 1}
_RENORMALIZE = 2
_ACTIVATIONS = {'silu': 0, 'gelu': 1}


class Router(NamedTuple):
    """How tokens choose: by their `top` largest of logits [..., E] (fp32, bf16, fp16), equal ones by the lowest index, a NaN first, -inf last.

    Scores are softmax(logits) or sigmoid(logits).  With a correction [E] (fp32) the choice is by score + correction, and the weights are
    the scores alone.  renormalize: the chosen scores over their sum (0 where that is 0); all weights times scale."""
    logits: torch.Tensor
    top: int
    scoring: str = 'softmax'
    renormalize: bool = True
    correction: Optional[torch.Tensor] = None
    scale: float = 1.0


class Routing(NamedTuple):
    experts: torch.Tensor                     # int32 [..., top], best first
    weights: torch.Tensor                     # fp32 [..., top]


def _check_router(r):
    shape = r.logits.shape
    if not shape or not 0 < shape[-1] <= MOST_EXPERTS:
        raise ValueError(f'logits of 1 to {MOST_EXPERTS} experts are needed, got shape {tuple(shape)}')
    if not 0 < r.top <= min(MOST_TOP, shape[-1]):
        raise ValueError(f'top {r.top}: between 1 and {min(MOST_TOP, shape[-1])}')
    if r.scoring not in _SCORING:
        raise ValueError(f'scoring {r.scoring!r}: one of {sorted(_SCORING)}')
    if r.correction is not None:
        if r.correction.shape != (shape[-1],):
            raise ValueError(f'the correction of {shape[-1]} experts has shape {tuple(r.correction.shape)}')
        if r.correction.dtype != torch.float32:
            raise L.LcqError(f'the correction is fp32, got {r.correction.dtype}')
    return shape[-1], _code(r.logits.dtype), _SCORING[r.scoring] | (_RENORMALIZE if r.renormalize else 0)


def route_tokens(router):
    """-> Routing of a Router: the experts of each token and their weights."""
    r = router
    E, code, flags = _check_router(r)
    if not _here(r.logits, r.correction):
        with torch.cuda.device(r.logits.device):
            return route_tokens(router)
    rows, T, ld = _rows(r.logits, E)
    shape = _with(r.logits.shape, r.top)
    experts, weights = rows.new_empty(shape, dtype=torch.int32), rows.new_empty(shape, dtype=torch.float32)
    if T:
        correction = _whole(r.correction)
        L.check(L.lib().lcq_route(rows.data_ptr(), code, T, E, ld, r.top, flags, _at(correction), r.scale, experts.data_ptr(), weights.data_ptr(),
                                  L.stream()), 'lcq_route')
    return Routing(experts, weights)


def _experts(t, step, most=MOST_DISTANCE):
    """Bytes [E, rows, width] -> (t or a contiguous copy, distance between experts, between rows), on multiples of `step` bytes (as widths are)."""
    E, rows, width = t.shape
    lde, ld = rows * width, width
    if not t.is_contiguous():
        e, r, w = t.stride()
        if rows == 1:
            r = width
        if E == 1:
            e = rows * r
        if w != 1 or not width <= r <= most or r % step or e % step:
            t = t.contiguous()
        else:
            lde, ld = e, r
    if t.data_ptr() % step:
        t = t.clone(memory_format=torch.contiguous_format)
        lde, ld = rows * width, width
    return t, lde, ld


def mxfp4_moe(x, router, gate_up, down, *, gate_up_bias=None, down_bias=None, activation='silu', out_dtype=None):
    """A mixture-of-experts layer on x [..., K] (bf16, fp16, fp32):

        y = sum over the chosen experts e of weight * (down_e (act(gate_e x + b) * (up_e x + b)) + b)

    router: a Router over logits [..., E] of the same tokens, or a Routing (an index outside 0 .. E - 1 is no expert; the same expert several
    times counts once, with the sum of the weights).  gate_up: Mxfp4 of [E, 2 I, K], the gates' rows and then the ups';  down: Mxfp4 of [E, N, I].
    gate_up_bias [E, 2 I], down_bias [E, N]: of one type.  activation 'silu' or 'gelu' (by erf).  -> [..., N] of x's type or `out_dtype`.

    Activations are not quantized, sums and act(...) * (...) are fp32.  An expert whose weight is 0 is not asked; a token without experts gives 0.
    Weights of 2^128 and more (4 and 6 with scale byte 253, 2 to 6 with 254) count as infinite.  This is for few tokens: up to 128 at a time share a
    pass over the experts' bytes.  Operands with strides are copied (experts and their rows may lie apart)."""
    shape = x.shape
    K = _cols(shape)
    code = _code(x.dtype)
    if out_dtype is None:
        out_dtype = x.dtype
    out_code = _code(out_dtype)
    if activation not in _ACTIVATIONS:
        raise ValueError(f'activation {activation!r}: one of {sorted(_ACTIVATIONS)}')
    gw, gs, cols = _parts(gate_up, 'gate_up')
    dw, ds, I = _parts(down, 'down')
    if gw.dim() != 3 or dw.dim() != 3 or gw.shape[0] != dw.shape[0]:
        raise ValueError(f'gate_up {tuple(gw.shape)} and down {tuple(dw.shape)} are not experts one behind the other')
    E, N = dw.shape[0], dw.shape[1]
    if cols != K or gw.shape[1] != 2 * I:
        raise ValueError(f'gate_up of {gw.shape[1]} rows and {cols} columns between tokens of {K} columns and down of {I}')
    if max(I, N) > 65536:
        raise ValueError(f'at most 65536 channels, got {I} and {N}')
    for name, bias, n in (('gate_up_bias', gate_up_bias, 2 * I), ('down_bias', down_bias, N)):
        if bias is not None and bias.shape != (E, n):
            raise ValueError(f'{name} is [{E}, {n}], got {tuple(bias.shape)}')
    if gate_up_bias is not None and down_bias is not None and gate_up_bias.dtype != down_bias.dtype:
        raise L.LcqError(f'biases of one type are needed, got {gate_up_bias.dtype} and {down_bias.dtype}')
    bias = gate_up_bias if gate_up_bias is not None else down_bias
    bias_code = 0 if bias is None else _code(bias.dtype)
    routed = isinstance(router, Routing)
    if routed:
        experts, weights = router
        top, flags, scale, logits_code = experts.shape[-1] if experts.dim() else 0, 0, 1.0, 0
        if experts.dtype != torch.int32 or weights.dtype != torch.float32:
            raise L.LcqError(f'experts are int32 and weights fp32, got {experts.dtype} and {weights.dtype}')
        if experts.shape != weights.shape or experts.shape[:-1] != shape[:-1] or not 0 < top <= MOST_TOP:
            raise ValueError(f'experts {tuple(experts.shape)} and weights {tuple(weights.shape)} of tokens {tuple(shape)}: 1 to {MOST_TOP} for each')
        if not 0 < E <= MOST_EXPERTS or top > E:
            raise ValueError(f'{top} of {E} experts')
        on = (experts, weights)
    else:
        chosen_of, logits_code, flags = _check_router(router)
        if chosen_of != E or router.logits.shape[:-1] != shape[:-1]:
            raise ValueError(f'logits {tuple(router.logits.shape)} of {E} experts and tokens {tuple(shape)}')
        top, scale = router.top, router.scale
        on = (router.logits, router.correction)
    if not _here(x, gw, gs, dw, ds, gate_up_bias, down_bias, *on):
        with torch.cuda.device(x.device):
            return mxfp4_moe(x, router, gate_up, down, gate_up_bias=gate_up_bias, down_bias=down_bias, activation=activation, out_dtype=out_dtype)
    rows, T, ld = _rows(x, K)
    y = rows.new_empty(_with(shape, N), dtype=out_dtype)
    if T and N:
        logits = correction = experts = weights = None
        ldl = 0
        if routed:
            experts, weights = _whole(on[0]), _whole(on[1])
        else:
            logits, _, ldl = _rows(on[0], E)
            correction = _whole(on[1])
        gw, g_lde, g_ld = _experts(gw, 16)
        gs, g_ldse, g_lds = _experts(gs, 1, (1 << 30) // (I + 64))
        dw, d_lde, d_ld = _experts(dw, 16)
        ds, d_ldse, d_lds = _experts(ds, 1)
        gate_up_bias, down_bias = _whole(gate_up_bias), _whole(down_bias)
        ws = _workspace(rows, 'lcq_mxfp4_moe_workspace_bytes', T, top, E, K, I, N, code)
        L.check(L.lib().lcq_mxfp4_moe(rows.data_ptr(), code, T, K, ld, _at(logits), logits_code, ldl, flags, _at(correction), scale, _at(experts),
                                      _at(weights), E, top, gw.data_ptr(), g_lde, g_ld, gs.data_ptr(), g_ldse, g_lds, _at(gate_up_bias),
                                      dw.data_ptr(), d_lde, d_ld, ds.data_ptr(), d_ldse, d_lds, _at(down_bias), bias_code, I, N,
                                      _ACTIVATIONS[activation], y.data_ptr(), out_code, _at(ws), L.stream()), 'lcq_mxfp4_moe')
    return y
