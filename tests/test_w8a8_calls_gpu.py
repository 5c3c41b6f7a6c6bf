"""Calls of the operators of a running w8a8 model as a program makes them: beside autograd, on views, captured, of many shapes."""
import pytest
import torch

from lightcompress_amd.w8a8 import QuantizedTokens, int8_linear, int8_matmul, quantize_tokens, residual_norm
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


# -- strides ----------------------------------------------------------------------------------------------------------------
def same(got, want):
    return all((a is None and b is None) or (torch.equal(a, b) and a.shape == b.shape) for a, b in zip(got, want))


@pytest.mark.parametrize('symmetric', [True, False])
@pytest.mark.parametrize('K', [64, 63])
@pytest.mark.parametrize('B', [1, 3, 70])
def test_codes_of_the_last_tokens(dev, B, K, symmetric):
    """Codes, scales and zero points of [B, S, K] cut to one token of each sequence, as in front of a head; operands with strides."""
    x = (torch.randn(B, 5, K, generator=gen(B + K)) + 0.5).to(BF).to(dev)
    w = torch.randint(-127, 128, (40, K), generator=gen(7), dtype=torch.int8).to(dev)
    ws, bias = torch.rand(40, generator=gen(8)).to(dev), torch.randn(40, generator=gen(9)).to(dev)
    spread = lambda t: torch.stack([t, t], -1).flatten(-2)[..., ::2]  # noqa: E731  (t in twice the room)
    q = quantize_tokens(x, symmetric)
    for cut in ((slice(None), -1), (slice(None), slice(1, 3)), (slice(None, None, 2),)):
        part = QuantizedTokens(*(None if t is None else t[cut] for t in q))
        whole = QuantizedTokens(*(None if t is None else t[cut].contiguous() for t in q))
        want = int8_matmul(whole, w, ws, bias)
        assert torch.equal(int8_matmul(part, w, ws, bias), want)
        assert torch.equal(int8_matmul(part, spread(w), spread(ws), spread(bias)), want)
        assert torch.equal(int8_matmul(part, w.t().contiguous().t(), spread(ws)[:, None], spread(bias)), want)
    want = int8_linear(x, w, ws, bias, symmetric)
    assert torch.equal(int8_linear(x, spread(w), spread(ws), spread(bias), symmetric), want)
    one = ws[:1]
    assert torch.equal(int8_linear(x, w, one.expand(40), bias, symmetric), int8_linear(x, w, one, bias, symmetric))


def test_norm_parameters_with_strides(dev):
    x, r = torch.randn(3, 96, generator=gen(5)).to(dev), torch.randn(3, 96, generator=gen(6)).to(dev)
    p = torch.randn(96, 5, generator=gen(7)).to(dev)
    names = ('weight', 'bias', 'post_weight', 'post_bias', 'gate')
    kw = {n: p[:, i] for i, n in enumerate(names)}
    assert same(residual_norm(x, r, **kw), residual_norm(x, r, **{n: t.contiguous() for n, t in kw.items()}))
