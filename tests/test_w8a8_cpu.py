"""What the operators of a running w8a8 model refuse, before any launch (CPU: nothing reaches a GPU)."""
import ctypes

import pytest
import torch

from lightcompress_amd import _lib as L
from lightcompress_amd.logprobs import token_logprobs
from lightcompress_amd.module_utils import AutoawqRealQuantLinear, VllmRealQuantLinear, _act_form
from lightcompress_amd.w8a8 import QuantizedTokens, int8_linear, int8_matmul, quantize_tokens, residual_norm

BUF = ctypes.create_string_buffer(256)
P = ctypes.addressof(BUF) & ~15                  # stands for a device pointer: every call below returns before it is used


ROWS = torch.zeros(3, 64)


def tokens(M=2, K=64):
    return QuantizedTokens(torch.zeros(M, K, dtype=torch.int8), torch.ones(M, 1))


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 64), torch.zeros(8, 64, dtype=torch.int8)
    for call in (lambda: quantize_tokens(x), lambda: int8_matmul(tokens(), w, torch.ones(8)), lambda: int8_linear(x, w, torch.ones(8)),
                 lambda: residual_norm(x, x), lambda: token_logprobs(x)):
        with pytest.raises(L.LcqError, match='GPU tensors only'):
            call()


@pytest.mark.parametrize('call, error', [
    (lambda: quantize_tokens(torch.zeros(2, 0)), ValueError),
    (lambda: quantize_tokens(torch.zeros(())), ValueError),
    (lambda: quantize_tokens(torch.zeros(1, 65537)), ValueError),
    (lambda: quantize_tokens(torch.zeros(2, 64, dtype=torch.float64)), L.LcqError),
    (lambda: quantize_tokens(torch.zeros(2, 64), scale=torch.ones(2)), ValueError),
    (lambda: quantize_tokens(torch.zeros(2, 64), symmetric=False, scale=torch.ones(1)), ValueError),
    (lambda: int8_matmul(tokens(), torch.zeros(8, 64), torch.ones(8)), L.LcqError),
    (lambda: int8_matmul(tokens(), torch.zeros(8, 64, dtype=torch.uint8), torch.ones(8)), L.LcqError),
    (lambda: int8_matmul(tokens(), torch.zeros(8, 63, dtype=torch.int8), torch.ones(8)), ValueError),
    (lambda: int8_matmul(tokens(), torch.zeros(8, 64, dtype=torch.int8), torch.ones(7)), ValueError),
    (lambda: int8_matmul(tokens(), torch.zeros(8, 64, dtype=torch.int8), torch.ones(8), torch.zeros(1)), ValueError),
    (lambda: int8_matmul(QuantizedTokens(torch.zeros(3, 64, dtype=torch.int8), torch.ones(2, 1)), torch.zeros(8, 64, dtype=torch.int8),
                         torch.ones(8)), ValueError),
    (lambda: int8_matmul(QuantizedTokens(torch.zeros(3, 64, dtype=torch.uint8), torch.ones(3, 1)), torch.zeros(8, 64, dtype=torch.int8),
                         torch.ones(8)), L.LcqError),
    (lambda: int8_matmul(QuantizedTokens(torch.zeros(3, 64, dtype=torch.int8), torch.ones(3, 1), torch.zeros(3, 1)),
                         torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)), L.LcqError),
    (lambda: residual_norm(torch.zeros(2, 64), torch.zeros(2, 63)), ValueError),
    (lambda: residual_norm(torch.zeros(2, 64), torch.zeros(2, 64, dtype=torch.bfloat16)), L.LcqError),
    (lambda: residual_norm(torch.zeros(2, 64), weight=torch.zeros(63)), ValueError),
    (lambda: residual_norm(torch.zeros(2, 64), weight=torch.zeros(64, dtype=torch.bfloat16)), L.LcqError),
    (lambda: residual_norm(torch.zeros(2, 64), post_bias=torch.zeros(64)), ValueError),
    (lambda: residual_norm(torch.zeros(2, 64), gate=torch.zeros(2, 1)), ValueError),
    (lambda: residual_norm(torch.zeros(2, 64), kind='batch'), ValueError),
    (lambda: residual_norm(torch.zeros(2, 64), quantize='int4'), ValueError),
    (lambda: residual_norm(torch.zeros(2, 64), out_dtype=torch.bfloat16), L.LcqError),
    (lambda: residual_norm(torch.zeros(2, 64), inplace=True), ValueError),
    (lambda: residual_norm(ROWS[1:], ROWS[:2], inplace=True), ValueError),
    (lambda: residual_norm(ROWS[:2].clone(), ROWS[:2], ROWS[1], inplace=True), ValueError),
    (lambda: residual_norm(ROWS.view(torch.bfloat16)[:1, :64], ROWS[:1], inplace=True), ValueError),
    (lambda: residual_norm(ROWS[:2].clone(), ROWS[:2], gate=ROWS[1:], inplace=True), ValueError),
    (lambda: residual_norm(torch.zeros(2, 64), torch.zeros(64, 2).t(), inplace=True), ValueError),
    (lambda: residual_norm(torch.zeros(2, 64), torch.zeros(2, 64, requires_grad=True), inplace=True), ValueError),
    (lambda: token_logprobs(torch.zeros(2, 0)), ValueError),
    (lambda: token_logprobs(torch.zeros(2, 8), top=9), ValueError),
    (lambda: token_logprobs(torch.zeros(2, 80), top=65), ValueError),
    (lambda: token_logprobs(torch.zeros(2, 8), top=-1), ValueError),
    (lambda: token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.int32)), L.LcqError),
    (lambda: token_logprobs(torch.zeros(2, 8), torch.zeros(3, dtype=torch.int64)), ValueError),
    (lambda: token_logprobs(torch.zeros(2, 8, dtype=torch.int64)), L.LcqError),
])
def test_calls_that_are_refused(call, error):
    with pytest.raises(error):
        call()


def test_the_c_entries_refuse_before_a_launch():
    lib = L.lib()
    quant = lambda x=P, d=0, T=2, K=64, ld=64, asym=0, sc=None, c=P, s=P, z=None: lib.lcq_quant_tokens(x, d, T, K, ld, asym, sc, c, s, z, None)  # noqa: E731
    assert quant(x=None) == quant(T=0) == quant(K=0) == quant(c=None) == quant(s=None) == quant(asym=1) == quant(ld=-1) == -1
    assert quant(asym=1, sc=P, z=P) == -1 and quant(d=3) == -3 and quant(K=65537) == -6
    mm = lambda a=P, s=P, w=P, ws=P, wd=0, b=None, bd=0, M=2, N=8, K=64, y=P, d=0: lib.lcq_int8_matmul(  # noqa: E731
        a, s, 0, None, w, ws, wd, 0, b, bd, M, N, K, y, d, None, None)
    assert mm(a=None) == mm(s=None) == mm(w=None) == mm(ws=None) == mm(y=None) == mm(M=0) == mm(N=0) == mm(K=0) == mm(M=-1) == -1
    assert mm(wd=5) == mm(d=-1) == mm(b=P, bd=9) == -3 and mm(K=65537) == -6
    assert lib.lcq_int8_matmul_workspace_bytes(0, 8, 64) == lib.lcq_int8_matmul_workspace_bytes(2, 8, 65537) == 0
    lin = lambda x=P, xd=0, asym=0, sc=None, w=P, ld=64, M=9, K=64, ws=None: lib.lcq_int8_linear(  # noqa: E731
        x, xd, ld, asym, sc, w, P, 0, 0, None, 0, M, 8, K, P, 0, ws, None)
    assert lin(x=None) == lin(w=None) == lin(ld=-1) == lin(asym=1, sc=P) == lin(M=0) == -1 and lin(xd=5) == -3 and lin(K=65537) == -6
    assert lin(w=P + 8) == -2 and lin() == -5 and lin(ws=P + 8) == -2 and mm(w=P + 1) == mm(a=P + 4) == -2 and mm(M=65, K=63) == mm(K=15) == -5
    assert lib.lcq_int8_linear_workspace_bytes(1, 8, 64) == lib.lcq_int8_linear_workspace_bytes(8, 8, 64) == 0 < lib.lcq_int8_linear_workspace_bytes(9, 8, 64)
    norm = lambda x=P, d=0, T=2, K=64, pw=None, pb=None, f=0, h=P, o=P, c=None, s=None, z=None: lib.lcq_residual_norm(  # noqa: E731
        x, d, T, K, 64, None, 0, None, 0, pw, pb, None, None, 1.0, 1e-6, 0.0, f, h, o, c, s, z, None)
    assert norm(x=None) == norm(h=None) == norm(o=None) == norm(c=P) == norm(T=0) == norm(pb=P) == norm(f=256) == -1
    assert norm(f=128, c=P, s=P) == -1 and norm(d=7) == -3 and norm(K=65537) == -6
    lp = lambda x=P, d=0, T=2, V=100, ld=100, t=None, m=0, o=None, k=0, tv=None, ti=None: lib.lcq_token_logprobs(  # noqa: E731
        x, d, T, V, ld, t, m, -100, o, None, k, tv, ti, None)
    assert lp(x=None) == lp(T=0) == lp(V=0) == lp(m=1) == lp(k=1) == lp(k=65, tv=P, ti=P) == lp(V=3, k=4, tv=P, ti=P) == lp(m=-1) == -1
    assert lp(d=4) == -3 and lp(V=1 << 31) == -6


def test_which_containers_run():
    w8 = dict(bit=8, symmetric=True, granularity='per_channel')
    a8 = dict(bit=8, symmetric=True, granularity='per_token')
    assert _act_form({'weight': w8, 'act': a8}) == 'symmetric'
    assert _act_form({'weight': w8, 'act': dict(a8, symmetric=False)}) == 'asymmetric'
    assert _act_form({'weight': w8, 'act': dict(a8, granularity='per_tensor', static=True)}) == 'static'
    for weight, act in ((w8, None), (dict(w8, symmetric=False), a8), (dict(w8, bit=4), a8), (dict(w8, granularity='per_group'), a8),
                        (dict(w8, need_pack=True), a8), (dict(w8, bit='e4m3', quant_type='float-quant'), a8), (w8, dict(a8, bit=4)),
                        (w8, dict(a8, granularity='per_tensor')), (w8, dict(a8, granularity='per_tensor', static=True, symmetric=False)),
                        (w8, dict(a8, calib_algo='mse')), (w8, dict(a8, int_range=[-8, 7])), (w8, dict(a8, round_zp=False))):
        assert _act_form({'weight': weight, 'act': act} if act else {'weight': weight}) is None
    with pytest.raises(NotImplementedError):
        VllmRealQuantLinear(torch.zeros(2, 8), None, torch.ones(2, 1), None, False, 'weight_scale')(torch.zeros(1, 8))
    with pytest.raises(NotImplementedError):
        AutoawqRealQuantLinear(torch.zeros(8, 1), None, torch.ones(1, 8), torch.zeros(1, 1))(torch.zeros(1, 8))
