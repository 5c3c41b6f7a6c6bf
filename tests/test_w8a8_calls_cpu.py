"""Calls of the operators of a running w8a8 model that are refused before any launch: operands that meet, forms that are unknown."""
import pytest
import torch

from lightcompress_amd import _lib as L
from lightcompress_amd.w8a8 import residual_norm


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
