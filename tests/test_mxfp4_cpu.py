"""What the operators on 4-bit numbers refuse, before any launch (CPU: nothing reaches a GPU)."""
import ctypes

import pytest
import torch

from lightcompress_amd import _lib as L
from lightcompress_amd.moe import Router, Routing, mxfp4_moe, route_tokens
from lightcompress_amd.mxfp4 import Mxfp4, dequantize_mxfp4, mxfp4_linear, mxfp4_matmul, quantize_mxfp4

BUF = ctypes.create_string_buffer(256)
P = ctypes.addressof(BUF) & ~15                  # stands for a device pointer: every call below returns before it is used
EINVAL, EALIGN, EDTYPE, EWORKSPACE, ESIZE = -1, -2, -3, -5, -6


def mx(*shape):
    """[..., K] of zeros"""
    B = -(-shape[-1] // 32)
    return Mxfp4(torch.zeros(*shape[:-1], 16 * B, dtype=torch.uint8), torch.zeros(*shape[:-1], B, dtype=torch.uint8), shape[-1])


def moe(x=None, router=None, gate_up=None, down=None, **other):
    x = torch.zeros(2, 64) if x is None else x
    return mxfp4_moe(x, router or Router(torch.zeros(2, 4), 2), gate_up or mx(4, 80, 64), down or mx(4, 48, 40), **other)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64)
    for call in (lambda: quantize_mxfp4(x), lambda: dequantize_mxfp4(mx(2, 64)), lambda: mxfp4_matmul(mx(2, 64), mx(8, 64)), lambda: mxfp4_linear(x, mx(8, 64)),
                 lambda: route_tokens(Router(x, 2)), moe, lambda: moe(router=Routing(torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2)))):
        with pytest.raises(L.LcqError, match='GPU tensors only'):
            call()


@pytest.mark.parametrize('call, error', [
    (lambda: quantize_mxfp4(torch.zeros(2, 0)), ValueError),
    (lambda: quantize_mxfp4(torch.zeros(())), ValueError),
    (lambda: quantize_mxfp4(torch.zeros(2, 64, dtype=torch.float64)), L.LcqError),
    (lambda: dequantize_mxfp4(mx(2, 64), torch.float64), L.LcqError),
    (lambda: dequantize_mxfp4(Mxfp4(torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2, 2, dtype=torch.uint8))), L.LcqError),
    (lambda: dequantize_mxfp4(Mxfp4(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 3, dtype=torch.uint8))), ValueError),
    (lambda: dequantize_mxfp4(Mxfp4(torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(3, 2, dtype=torch.uint8))), ValueError),
    (lambda: dequantize_mxfp4(Mxfp4(torch.zeros(2, 0, dtype=torch.uint8), torch.zeros(2, 0, dtype=torch.uint8))), ValueError),
    (lambda: dequantize_mxfp4(mx(2, 64)._replace(cols=32)), ValueError),
    (lambda: dequantize_mxfp4(mx(2, 64)._replace(cols=65)), ValueError),
    (lambda: mxfp4_matmul(mx(2, 64), mx(8, 96)), ValueError),
    (lambda: mxfp4_matmul(mx(2, 64), mx(8, 63)), ValueError),
    (lambda: mxfp4_matmul(mx(2, 64), mx(2, 8, 64)), ValueError),
    (lambda: mxfp4_matmul(mx(2, 64), mx(8, 64), torch.zeros(7)), ValueError),
    (lambda: mxfp4_matmul(mx(1, 65537), mx(1, 65537)), ValueError),
    (lambda: mxfp4_matmul(mx(2, 64), mx(8, 64), out_dtype=torch.float64), L.LcqError),
    (lambda: mxfp4_linear(torch.zeros(2, 64, dtype=torch.int8), mx(8, 64)), L.LcqError),
    (lambda: mxfp4_linear(torch.zeros(2, 63), mx(8, 64)), ValueError),
    (lambda: mxfp4_linear(torch.zeros(()), mx(8, 64)), ValueError),
    (lambda: route_tokens(Router(torch.zeros(2, 1025), 2)), ValueError),
    (lambda: route_tokens(Router(torch.zeros(2, 0), 1)), ValueError),
    (lambda: route_tokens(Router(torch.zeros(2, 8), 0)), ValueError),
    (lambda: route_tokens(Router(torch.zeros(2, 8), 9)), ValueError),
    (lambda: route_tokens(Router(torch.zeros(2, 64), 33)), ValueError),
    (lambda: route_tokens(Router(torch.zeros(2, 8), 2, 'tanh')), ValueError),
    (lambda: route_tokens(Router(torch.zeros(2, 8), 2, correction=torch.zeros(7))), ValueError),
    (lambda: route_tokens(Router(torch.zeros(2, 8), 2, correction=torch.zeros(8, dtype=torch.bfloat16))), L.LcqError),
    (lambda: moe(x=torch.zeros(2, 32)), ValueError),
    (lambda: moe(x=torch.zeros(3, 64)), ValueError),
    (lambda: moe(x=torch.zeros(2, 64, dtype=torch.float64)), L.LcqError),
    (lambda: moe(gate_up=mx(4, 79, 64)), ValueError),
    (lambda: moe(gate_up=mx(3, 80, 64)), ValueError),
    (lambda: moe(gate_up=mx(80, 64)), ValueError),
    (lambda: moe(down=mx(4, 1, 65537), gate_up=mx(4, 2 * 65537, 64)), ValueError),
    (lambda: moe(router=Router(torch.zeros(2, 5), 2)), ValueError),
    (lambda: moe(activation='relu'), ValueError),
    (lambda: moe(gate_up_bias=torch.zeros(4, 40)), ValueError),
    (lambda: moe(down_bias=torch.zeros(48)), ValueError),
    (lambda: moe(gate_up_bias=torch.zeros(4, 80), down_bias=torch.zeros(4, 48, dtype=torch.bfloat16)), L.LcqError),
    (lambda: moe(router=Routing(torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 2))), L.LcqError),
    (lambda: moe(router=Routing(torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 1))), ValueError),
    (lambda: moe(router=Routing(torch.zeros(2, 5, dtype=torch.int32), torch.zeros(2, 5))), ValueError),
    (lambda: moe(out_dtype=torch.float64), L.LcqError),
])
def test_python_refusals(call, error):
    with pytest.raises(error):
        call()


def test_the_entries_of_quantization_refuse_before_a_launch():
    quant = lambda x=P, d=0, rows=2, K=64, ld=64, c=P, s=P, lds=2: L.lib().lcq_mxfp4_quant(x, d, rows, K, ld, c, s, lds, None)  # noqa: E731
    assert quant(x=None) == quant(c=None) == quant(s=None) == quant(rows=0) == quant(K=0) == quant(ld=-1) == quant(lds=1) == EINVAL
    assert quant(d=3) == EDTYPE and quant(c=P + 2) == EALIGN and quant(rows=1 << 36) == ESIZE
    back = lambda c=P, ldc=32, s=P, lds=2, rows=2, K=64, y=P, d=0: L.lib().lcq_mxfp4_dequant(c, ldc, s, lds, rows, K, y, d, None)  # noqa: E731
    assert back(c=None) == back(s=None) == back(y=None) == back(rows=0) == back(K=0) == back(ldc=-4) == back(lds=-1) == EINVAL
    assert back(d=-1) == EDTYPE and back(c=P + 2) == back(ldc=33) == EALIGN and back(rows=1 << 37) == ESIZE


def test_the_entries_of_products_refuse_before_a_launch():
    def product(a=P, lda=32, sa=P, ldsa=2, w=P, ldw=32, sw=P, ldsw=2, b=None, bd=0, M=2, N=8, K=64, y=P, d=0, ws=None):
        return L.lib().lcq_mxfp4_matmul(a, lda, sa, ldsa, w, ldw, sw, ldsw, b, bd, M, N, K, y, d, ws, None)
    assert product(a=None) == product(sa=None) == product(w=None) == product(sw=None) == product(y=None) == product(M=0) == product(N=0) == product(K=0) == EINVAL
    assert product(lda=16) == product(ldsa=1) == product(ldw=16) == product(ldsw=1) == EINVAL
    assert product(a=P + 8) == product(w=P + 8) == product(lda=40) == product(ldw=40) == EALIGN
    assert product(d=3) == product(b=P, bd=3) == EDTYPE
    assert product(K=65537, lda=1 << 20, ldw=1 << 20, ldsa=1 << 20, ldsw=1 << 20) == product(M=(1 << 28) + 1) == product(N=1 << 28) == ESIZE
    assert product(lda=(1 << 22) + 16) == product(ldw=(1 << 22) + 16) == product(ldsa=(1 << 22) + 1) == product(ldsw=(1 << 22) + 1) == ESIZE
    assert product(M=5000, N=5000) == EWORKSPACE and product(M=5000, N=5000, ws=P + 8) == EALIGN

    def linear(x=P, xd=1, ld=64, w=P, ldw=32, sw=P, ldsw=2, b=None, bd=0, M=400, N=8, K=64, y=P, d=0, ws=None):
        return L.lib().lcq_mxfp4_linear(x, xd, ld, w, ldw, sw, ldsw, b, bd, M, N, K, y, d, ws, None)
    assert linear(x=None) == linear(ld=-1) == linear(w=None) == linear(M=0) == EINVAL
    assert linear(xd=3) == linear(d=-1) == EDTYPE and linear() == EWORKSPACE and linear(ws=P + 4) == EALIGN and linear(w=P + 4) == EALIGN


def test_the_entries_of_experts_refuse_before_a_launch():
    route = lambda x=P, d=0, T=2, E=8, ld=8, top=2, f=0, c=None, e=P, w=P: L.lib().lcq_route(x, d, T, E, ld, top, f, c, 1.0, e, w, None)  # noqa: E731
    assert route(x=None) == route(e=None) == route(w=None) == route(T=0) == route(E=0) == route(top=0) == route(top=9) == route(ld=-1) == EINVAL
    assert route(d=3) == EDTYPE and route(E=1025) == route(E=64, top=33) == route(T=1 << 26) == ESIZE

    def layer(x=P, d=1, T=2, K=64, ldx=64, lg=P, lgd=0, ldl=4, f=0, c=None, e=None, w=None, E=4, top=2, g=P, gle=2560, gld=32, gs=P, gse=160, gsd=2, gb=None,
              dn=P, dle=1536, dld=32, ds=P, dse=96, dsd=2, db=None, bd=0, I=40, N=48, act=0, y=P, od=1, ws=P):
        return L.lib().lcq_mxfp4_moe(x, d, T, K, ldx, lg, lgd, ldl, f, c, 1.0, e, w, E, top, g, gle, gld, gs, gse, gsd, gb, dn, dle, dld, ds, dse, dsd, db, bd, I, N,
                                     act, y, od, ws, None)
    assert layer(x=None) == layer(g=None) == layer(gs=None) == layer(dn=None) == layer(ds=None) == layer(y=None) == layer(lg=None) == layer(e=P, w=P) == EINVAL
    assert layer(lg=None, e=P) == layer(T=0) == layer(K=0) == layer(I=0) == layer(N=0) == layer(act=2) == layer(top=5) == layer(ldx=-1) == EINVAL
    assert layer(gld=16) == layer(gsd=1) == layer(dld=16) == layer(dsd=1) == EINVAL
    assert layer(d=3) == layer(od=3) == layer(lgd=3) == layer(db=P, bd=3) == EDTYPE
    assert layer(K=65537) == layer(I=65537) == layer(N=65537) == layer(gld=(1 << 22) + 16) == layer(dsd=(1 << 22) + 1) == layer(gsd=1 << 24) == ESIZE
    assert layer(g=P + 8) == layer(gld=40) == layer(gle=2568) == layer(dn=P + 8) == layer(dld=40) == layer(dle=1544) == layer(ws=P + 8) == EALIGN
    assert layer(ws=None) == EWORKSPACE
    need = L.lib().lcq_mxfp4_moe_workspace_bytes
    assert need(0, 2, 4, 64, 40, 48, 1) == need(2, 33, 64, 64, 40, 48, 1) == need(2, 2, 4, 65537, 40, 48, 1) == need(2, 2, 4, 64, 40, 48, 3) == 0
    assert need(2, 2, 4, 64, 40, 48, 1) > 0 and need(128, 32, 32, 32, 65536, 4, 0) < 2 ** 31 + 2 ** 28 and need(1 << 25, 2, 4, 64, 40, 48, 1) == need(128, 2, 4, 64, 40, 48, 1)


def test_sizes_whose_products_pass_64_bits_are_refused():
    """Distances that a multiplication would wrap, and the rows that a quantization takes at most."""
    layer = lambda gsd: L.lib().lcq_mxfp4_moe(P, 1, 2, 64, 64, P, 0, 4, 0, None, 1.0, None, None, 4, 2, P, 2560, 32, P, 160, gsd, None, P, 1536, 32, P, 96, 2, None, 0,  # noqa: E731
                                              40, 48, 0, P, 1, P, None)
    assert {layer(gsd) for gsd in ((1 << 30) // 104 + 1, 1 << 60, 1 << 61, 1 << 62, (1 << 63) - 1)} == {ESIZE}
    for rows, K in ((1 << 30, 1), (1 << 30, 33), (1 << 32, 32), ((1 << 36) // 64 + 1, 64)):
        assert L.lib().lcq_mxfp4_quant(P, 0, rows, K, K, P, P, -(-K // 32) + 1, None) == ESIZE
        assert L.lib().lcq_mxfp4_dequant(P, 1 << 20, P, 1 << 20, rows, K, P, 0, None) == ESIZE
