"""Calls of the operators of a running w8a8 model that are refused before any launch: operands that meet, forms that are unknown."""
import ctypes

import pytest
import torch

from lightcompress_amd import _lib as L
from lightcompress_amd.logprobs import _sequences
from lightcompress_amd.module_utils import VllmRealQuantLinear
from lightcompress_amd.w8a8 import residual_norm

BUF = ctypes.create_string_buffer(256)
P = ctypes.addressof(BUF) & ~15                  # stands for a device pointer: every call below returns before it is used


@pytest.mark.parametrize('name', ['weight', 'bias'])
def test_in_place_over_what_the_last_norm_reads(name):
    """One token as a vector: its weight or bias is read behind h, so it may not lie on the residual, not even element on element."""
    v, base = torch.zeros(64), torch.zeros(80)
    for residual, other in ((v, v), (v, v.view(8, 8).view(64)), (base[:64], base[16:])):
        with pytest.raises(ValueError, match='write over'):
            residual_norm(torch.zeros(64), residual, inplace=True, **{name: other})
    with pytest.raises(ValueError, match='write over'):                      # (one tensor in both roles: the later reading counts)
        residual_norm(torch.zeros(64), v, inplace=True, post_weight=v, **{name: v})


def test_in_place_over_what_is_read_before():
    """x, gate and the norm in front read their elements before h takes their place: such calls get as far as a GPU."""
    v = torch.zeros(64)
    for call in (lambda: residual_norm(v, v, inplace=True), lambda: residual_norm(torch.zeros(64), v, gate=v, inplace=True),
                 lambda: residual_norm(torch.zeros(64), v, post_weight=v, post_bias=v, inplace=True)):
        with pytest.raises(L.LcqError, match='GPU tensors only'):
            call()


def test_strided_logits_are_one_call():
    """Views of logits as sequences of rows, without a copy wherever two strides say where the rows are."""
    x = torch.arange(4 * 6 * 5 * 7.0).view(4, 6, 5, 7)
    flat = x.view(24, 5, 7)

    def form(v, copied=False):
        t, B, S, lds, ldx = _sequences(v)
        assert B * S * v.shape[-1] == v.numel() and (t is v) != copied
        at = torch.arange(B)[:, None, None] * lds + torch.arange(S)[:, None] * ldx + torch.arange(v.shape[-1])
        got = torch.as_strided(t, (t.untyped_storage().size() // 4,), (1,), 0)[at + t.storage_offset()]
        assert torch.equal(got.reshape(v.shape), v)
        return B, S

    assert form(x) == (1, 120) and form(flat[0, 2]) == (1, 1) and form(flat[:, 1]) == (1, 24) and form(flat[:, -1:]) == (1, 24)
    assert form(flat[:, :-1]) == (24, 4) and form(flat[:1, :-1]) == (1, 4) and form(flat[3:, 1:3, 2:]) == (21, 2)
    assert form(x[:, :, :-1]) == (24, 4) and form(x[:, :-1]) == (4, 25) and form(x[:, 2]) == (4, 5) and form(x[..., 3:]) == (1, 120)
    assert form(flat.transpose(0, 1)) == (5, 24) and form(flat[:1].expand(3, 5, 7)) == (3, 5) and form(flat[0, :1].expand(9, 7)) == (1, 9)
    assert form(x[..., :1]) == (1, 120) and form(x[:, :-1, :-1], copied=True) == (1, 80) and form(x.transpose(2, 3), copied=True) == (1, 168)
    assert form(x[0, 0].t(), copied=True) == (1, 7)


def test_the_entry_of_sequences_refuses_before_a_launch():
    call = lambda x=P, d=0, B=2, S=3, V=100, lds=300, ld=100, t=None, m=0, o=None, k=0: L.lib().lcq_token_logprobs_of(  # noqa: E731
        x, d, B, S, V, lds, ld, t, m, -100, o, None, k, None, None, None)
    assert call(x=None) == call(B=0) == call(S=0) == call(V=0) == call(lds=-1) == call(ld=-1) == call(m=1) == call(k=1) == call(k=65) == -1
    assert call(d=4) == -3 and call(B=1 << 16, S=1 << 15) == call(B=1 << 31, S=1) == call(S=1 << 31) == call(V=1 << 29) == -6
    assert call(x=P + 1) == -2


def test_products_of_more_lanes_than_a_launch_has_are_refused():
    """2^24 workgroups of 256 lanes are 2^32: one block of channels, or one tile, too many."""
    linear = lambda M, N, K: L.lib().lcq_int8_linear(P, 0, K, 0, None, P, P, 0, 0, None, 0, M, N, K, P, 0, P, None)  # noqa: E731
    product = lambda M, N, K: L.lib().lcq_int8_matmul(P, P, 0, None, P, P, 0, 0, None, 0, M, N, K, P, 0, P, None)  # noqa: E731
    assert linear(1, (1 << 28) - 15, 64) == linear(1, 1 << 28, 64) == linear(1, (1 << 27) - 15, 8208) == linear(1, 1 << 29, 64) == -6
    assert product(4095 * 128, 4097 * 128, 64) == product(1, 1 << 28, 64) == product(1 << 29, 1, 64) == -6


def test_containers_that_are_told_their_form():
    """Made by the constructor around saved buffers: with a form they get as far as a GPU, one that is unknown or lacks its scale is refused."""
    def made(form, scale=None):
        c = VllmRealQuantLinear(torch.zeros(8, 64, dtype=torch.int8), None, torch.ones(8, 1), scale, False, 'weight_scale')
        c.act_form = form
        return c

    for form, scale in (('symmetric', None), ('asymmetric', None), ('static', torch.ones(1))):
        with pytest.raises(L.LcqError, match='GPU tensors only'):
            made(form, scale)(torch.zeros(2, 64))
    for form, scale in (('per_token', None), ('asym', None), ('static', None)):
        with pytest.raises(ValueError, match='act_form'):
            made(form, scale)(torch.zeros(2, 64))
    with pytest.raises(NotImplementedError):
        made(None)(torch.zeros(2, 64))
