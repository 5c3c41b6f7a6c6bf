"""Calls of the operators of a running w8a8 model as a program makes them: beside autograd, on views, captured, of many shapes."""
import pytest
import torch

from lightcompress_amd.w8a8 import residual_norm
from tests.helpers import gen

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize('mode', ['no_grad', 'grad'])
@pytest.mark.parametrize('cut', [False, True])
def test_in_place_is_seen_by_a_backward_pass_that_kept_the_residual(dev, mode, cut):
    """As torch's own in-place operations: the backward pass raises instead of using the new values, also where a view was written."""
    x, whole = torch.randn(4, 64, generator=gen(1)).to(dev), torch.randn(8, 64, generator=gen(2)).to(dev)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = (whole * w).sum()                            # keeps `whole`, which has no gradient of its own
    residual = whole[:4] if cut else whole
    before = whole._version
    with torch.set_grad_enabled(mode == 'grad'):
        got = residual_norm(x if cut else torch.cat([x, x]), residual, inplace=True)
    assert got.residual is residual and whole._version > before
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


def test_in_place_leaves_versions_alone_that_it_does_not_write(dev):
    x, r = torch.randn(4, 64, generator=gen(3)).to(dev), torch.randn(4, 64, generator=gen(4)).to(dev)
    residual_norm(x, r)
    residual_norm(x[:0], r[:0], inplace=True)
    assert x._version == r._version == 0
    with torch.inference_mode():                     # (tensors made here have no version)
        t = torch.randn(4, 64, device=dev)
        want = t + x
        assert torch.equal(residual_norm(x, t, inplace=True).residual, want)
