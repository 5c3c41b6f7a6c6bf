"""Int8 codes of tokens, the int8 product, the norm between blocks and their run together, against 64-bit arithmetic."""
import pytest
import torch

from lightcompress_amd import IntegerQuantizer
from lightcompress_amd.logprobs import token_logprobs
from lightcompress_amd.module_utils import VllmRealQuantLinear
from lightcompress_amd.rtn import RTN
from lightcompress_amd.w8a8 import QuantizedTokens, int8_linear, int8_matmul, quantize_tokens, residual_norm
from tests.helpers import assert_bit_equal, gen

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24                                     # half a step of fp32, relative
TINY = {BF: 2.0 ** -134, HF: 2.0 ** -25, F32: 2.0 ** -150}   # half the distance of subnormals


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def acts(T, K, dtype, seed=0, shift=0.0):
    g = gen(seed)
    return ((torch.randn(T, K, generator=g) * torch.exp(0.7 * torch.randn(K, generator=g))) + shift).to(dtype)


# -- codes of tokens ------------------------------------------------------------------------------------------------
def codes_of(x, symmetric):
    """The formulas in fp32 on the CPU, every operation rounded as IEEE 754 says (tensor divisors: no reciprocals)."""
    x = x.float()
    if symmetric:
        s = x.abs().amax(1, keepdim=True).clamp_min(1e-5) / torch.tensor([127.0])
        return torch.round(x / s).clamp(-128, 127).to(torch.int8), s, None
    lo, hi = x.amin(1, keepdim=True), x.amax(1, keepdim=True)
    s = (hi - lo).clamp_min(1e-5) / torch.tensor([255.0])
    z = (-128 - torch.round(lo / s)).clamp(-128, 127)
    return (torch.round(x / s) + z).clamp(-128, 127).to(torch.int8), s, z.to(torch.int32)


@pytest.mark.parametrize('symmetric', [True, False])
@pytest.mark.parametrize('dtype', [BF, HF, F32])
@pytest.mark.parametrize('T,K', [(1, 1), (1, 4096), (5, 63), (3, 64), (7, 1000), (4, 1025), (2, 2048), (3, 5121), (2, 14336), (2, 16386),
                                 (1, 65536), (1, 65535), (130, 520)])
def test_codes_equal_the_formula(dev, T, K, dtype, symmetric):
    x = acts(T, K, dtype, seed=T + K, shift=0.3)
    got = quantize_tokens(x.to(dev), symmetric)
    codes, s, z = codes_of(x, symmetric)
    assert torch.equal(got.codes.cpu(), codes)
    assert_bit_equal(got.scales, s, 'scales')
    assert (got.zeros is None) == symmetric and (symmetric or torch.equal(got.zeros.cpu(), z))


@pytest.mark.parametrize('symmetric', [True, False])
def test_codes_equal_the_class_quantizer_on_fp32_rows(dev, symmetric):
    x = acts(33, 1024, F32, seed=5).to(dev)
    got = quantize_tokens(x, symmetric)
    codes, s, z = IntegerQuantizer(8, symmetric, 'per_channel').real_quant_weight_dynamic(x)
    assert torch.equal(got.codes.int(), codes.int() - (0 if symmetric else 128))
    assert_bit_equal(got.scales, s, 'scales')
    assert symmetric or torch.equal(got.zeros, z.int() - 128)


@pytest.mark.parametrize('rows', [
    torch.zeros(1, 40), torch.full((1, 40), 1e-9), torch.full((1, 40), 5.0), torch.full((1, 40), -5.0), torch.full((1, 40), 3e38),
    torch.linspace(4, 5, 40)[None], torch.cat([torch.zeros(1, 39), torch.full((1, 1), -1.0)], 1), torch.linspace(-3e38, 3e38, 40)[None] / 4,
    torch.linspace(-3, 3, 40)[None] * 2.5e37])
@pytest.mark.parametrize('symmetric', [True, False])
def test_rows_at_the_edges(dev, rows, symmetric):
    got = quantize_tokens(rows.to(dev), symmetric)
    if not bool(torch.isfinite(rows).all()):       # (linspace of a range that overflows is not finite: only that is promised)
        assert not bool(torch.isfinite(got.scales).any())
        return
    codes, s, z = codes_of(rows, symmetric)
    assert torch.equal(got.codes.cpu(), codes) and torch.equal(got.scales.cpu(), s) and (symmetric or torch.equal(got.zeros.cpu(), z))


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
@pytest.mark.parametrize('symmetric', [True, False])
def test_a_token_that_is_not_finite_gives_a_row_that_is_not(dev, bad, symmetric):
    x = acts(3, 200, BF, seed=2)
    x[1, 77] = bad
    w = torch.randint(1, 127, (9, 200), generator=gen(3), dtype=torch.int8)
    y = int8_linear(x.to(dev), w.to(dev), torch.ones(9, device=dev), symmetric=symmetric)
    assert not bool(torch.isfinite(y[1]).any()) and bool(torch.isfinite(y[[0, 2]]).all())


def test_given_scale(dev):
    x = acts(6, 264, BF, seed=8)
    x[0, 0], x[0, 1], x[0, 2] = float('inf'), -float('inf'), 3e38
    s = torch.tensor(0.05, device=dev, dtype=BF)
    got = quantize_tokens(x.to(dev), scale=s)
    assert torch.equal(got.codes.cpu(), torch.round(x.float() / s.float().cpu()).clamp(-128, 127).to(torch.int8))
    assert got.scales.numel() == 1 and got.zeros is None and float(got.scales) == float(s)


def test_rows_apart_and_off_alignment(dev):
    wide = acts(9, 700, BF, seed=4).to(dev)
    for view in (wide[:, :512], wide[:, 1:514], wide[::2, 8:520], wide[:, 3:67], wide.t()[:64].t(), wide.view(3, 3, 700)[:, 1:, :256], wide[:1].expand(5, 700)):
        a, b = quantize_tokens(view), quantize_tokens(view.clone(memory_format=torch.contiguous_format))
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and a.codes.shape == view.shape


# -- the product ----------------------------------------------------------------------------------------------------
def check_product(got, q, s, z, w, ws, bias, dtype):
    """y against 64 bits.  fp32 steps of the kernel: the sum to fp32, the product of the scales, their product, the bias: each off
    by at most U relative to its own result; then half a step of the output type."""
    assert got.dtype == dtype
    f = torch.float64
    q = q.to(f).reshape(-1, q.shape[-1])
    if z is not None:
        q = q - z.to(f).reshape(-1, 1)
    prod = (q @ w.to(f).t()) * s.to(f).reshape(-1, 1) * ws.to(f).reshape(1, -1)
    want = prod if bias is None else prod + bias.to(f)
    err32 = 3.01 * U * prod.abs() + 1.01 * U * want.abs()
    tol = err32 + half_step(dtype) * (want.abs() + err32) + TINY[dtype]
    err = (got.to(f).reshape(want.shape) - want).abs()
    assert bool((err <= tol).all()), f'{float((err / tol).max())} of the tolerance'


def product_inputs(M, N, K, asym, bias, ws_dtype=F32, seed=0, dev=None):
    g = torch.Generator(device=dev)
    g.manual_seed(seed + M + 7 * N + 13 * K)
    q = torch.randint(-128, 128, (M, K), generator=g, dtype=torch.int8, device=dev)
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device=dev)
    s = 0.001 + 0.01 * torch.rand(M, 1, generator=g, device=dev)
    ws = (0.001 + 0.01 * torch.rand(N, 1, generator=g, device=dev)).to(ws_dtype)
    z = torch.randint(-128, 128, (M, 1), generator=g, dtype=torch.int32, device=dev) if asym else None
    b = torch.randn(N, generator=g, device=dev) if bias else None
    return q, s, z, w, ws, b


SIZES = [(1, 1, 1), (1, 64, 64), (1, 1000, 4096), (2, 17, 63), (3, 4096, 128), (7, 100, 2050), (8, 256, 1024), (15, 33, 80), (16, 4096, 4096),
         (17, 130, 272), (31, 64, 4112), (32, 512, 512), (33, 257, 1040), (48, 1024, 2048), (64, 64, 64), (65, 1001, 2047), (100, 300, 4096),
         (127, 129, 144), (128, 128, 16), (129, 2048, 512), (200, 96, 14336), (255, 511, 1008), (256, 256, 4096), (257, 4096, 1024),
         (300, 5000, 48), (513, 513, 513), (1000, 777, 2064), (2048, 1024, 4096), (4097, 300, 256), (20, 24, 65536), (300, 264, 65536),
         (17, 4112, 528), (32, 5001, 272), (25, 9000, 4112), (5, 9001, 2064)]


@pytest.mark.parametrize('asym,bias,dtype', [(False, False, BF), (True, True, F32), (True, False, HF), (False, True, F32)])
@pytest.mark.parametrize('M,N,K', SIZES)
def test_product(dev, M, N, K, asym, bias, dtype):
    q, s, z, w, ws, b = product_inputs(M, N, K, asym, bias, dev=dev)
    if dtype == HF:
        ws = ws / K                                # (sums of K products of 128 by 128 stay within fp16)
    check_product(int8_matmul(QuantizedTokens(q, s, z), w, ws, b, out_dtype=dtype), q, s, z, w, ws, b, dtype)


# sizes of each tile (test_int8_cut_cpu.py holds the rule to them): 256 x 256, 256 x 192, 128 x 128 in parts of K
TILED = [(1000, 14300, 1040), (4090, 4090, 528), (1500, 6100, 640), (2048, 6144, 4096), (700, 14300, 1040), (70, 4100, 4112), (300, 1000, 14336)]


@pytest.mark.parametrize('asym,dtype', [(False, BF), (True, F32), (True, HF)])
@pytest.mark.parametrize('M,N,K', TILED)
def test_product_in_every_tile(dev, M, N, K, asym, dtype):
    q, s, z, w, ws, b = product_inputs(M, N, K, asym, True, dev=dev)
    if dtype == HF:
        ws = ws / K
    check_product(int8_matmul(QuantizedTokens(q, s, z), w, ws, b, out_dtype=dtype), q, s, z, w, ws, b, dtype)


# few tokens: one to four blocks of 16 of them by one or two of 16 channels, rows that start on 16 bytes and such that do not
FEW = [(16, 4096, 1040), (2, 4100, 528), (16, 8192, 4112), (7, 8200, 272), (1, 14339, 528), (17, 4096, 528), (24, 4097, 1040), (32, 8192, 4112),
       (31, 8200, 272), (32, 14339, 16), (9, 14336, 1040), (3, 28673, 48),
       (16, 4096, 1041), (1, 300, 17), (5, 4100, 4111), (2, 70, 15), (9, 14339, 300), (32, 300, 31), (20, 4096, 1023), (31, 8193, 2047), (25, 6200, 513),
       (33, 1000, 1024), (48, 4096, 2064), (64, 600, 512), (50, 2048, 2048), (40, 300, 1041), (64, 1001, 2047), (64, 100, 15), (49, 4095, 300)]


@pytest.mark.parametrize('asym,dtype', [(False, BF), (True, F32), (True, HF)])
@pytest.mark.parametrize('M,N,K', FEW)
def test_product_of_few_tokens(dev, M, N, K, asym, dtype):
    q, s, z, w, ws, b = product_inputs(M, N, K, asym, True, dev=dev)
    if dtype == HF:
        ws = ws / K
    check_product(int8_matmul(QuantizedTokens(q, s, z), w, ws, b, out_dtype=dtype), q, s, z, w, ws, b, dtype)


@pytest.mark.parametrize('M', [1, 16, 40, 300])
def test_product_at_the_ends_of_the_range(dev, M):
    """All codes -128 at K = 65536, zero points 127: the largest sums there are."""
    K, N = 65536, 40
    q = torch.full((M, K), -128, dtype=torch.int8, device=dev)
    w = torch.full((N, K), -128, dtype=torch.int8, device=dev)
    s, ws, z = torch.ones(M, 1, device=dev), torch.ones(N, device=dev), torch.full((M, 1), 127, dtype=torch.int32, device=dev)
    assert bool((int8_matmul(QuantizedTokens(q, s), w, ws, out_dtype=F32) == 16384.0 * K).all())
    assert bool((int8_matmul(QuantizedTokens(q, s, z), w, ws, out_dtype=F32) == 255.0 * 128 * K).all())


@pytest.mark.parametrize('M,N,K', [(1, 200, 256), (40, 200, 300), (300, 520, 512)])
@pytest.mark.parametrize('ws_dtype', [BF, HF, F32])
def test_product_scale_and_bias_types(dev, M, N, K, ws_dtype):
    q, s, _, w, ws, b = product_inputs(M, N, K, False, True, ws_dtype, dev=dev)
    check_product(int8_matmul(QuantizedTokens(q, s), w, ws, b.to(ws_dtype), out_dtype=F32), q, s, None, w, ws, b.to(ws_dtype), F32)
    one, wone = s[:1], ws[:1]
    check_product(int8_matmul(QuantizedTokens(q, one), w, wone), q, one.expand(M, 1), None, w, wone.expand(N, 1), None, BF)


@pytest.mark.parametrize('M,N,K', [(5, 80, 512), (70, 300, 1024), (300, 300, 2048)])
def test_product_off_alignment(dev, M, N, K):
    """Operands that start on any byte."""
    q, s, z, w, ws, b = product_inputs(M, N, K, True, False, dev=dev)
    for off in (1, 4, 8):
        qb, wb = torch.empty(M * K + off, dtype=torch.int8, device=dev), torch.empty(N * K + off, dtype=torch.int8, device=dev)
        qb[off:], wb[off:] = q.view(-1), w.view(-1)
        got = int8_matmul(QuantizedTokens(qb[off:].view(M, K), s, z), wb[off:].view(N, K), ws, out_dtype=F32)
        check_product(got, q, s, z, w, ws, None, F32)


@pytest.mark.parametrize('M,N,K', [(1, 80, 513), (5, 4100, 17), (20, 300, 1023), (40, 70, 258), (60, 33, 1041), (90, 300, 515), (3, 5, 9)])
def test_product_of_odd_rows_off_alignment(dev, M, N, K):
    """Rows of odd widths in operands that start on any byte, next to other bytes on both sides."""
    q, s, z, w, ws, b = product_inputs(M, N, K, True, False, dev=dev)
    for off in (0, 1, 2, 3):
        qb = torch.full((M * K + 32,), 77, dtype=torch.int8, device=dev)
        wb = torch.full((N * K + 32,), -99, dtype=torch.int8, device=dev)
        qb[16 + off:16 + off + M * K], wb[19 - off:19 - off + N * K] = q.view(-1), w.view(-1)
        got = int8_matmul(QuantizedTokens(qb[16 + off:16 + off + M * K].view(M, K), s, z), wb[19 - off:19 - off + N * K].view(N, K), ws, out_dtype=F32)
        check_product(got, q, s, z, w, ws, None, F32)


@pytest.mark.parametrize('dtype', [BF, HF, F32])
@pytest.mark.parametrize('M,K', [(1, 1), (1, 16), (1, 4096), (1, 16400), (1, 40960), (1, 40976), (1, 65536), (2, 1040), (3, 4096), (4, 10240), (4, 10256), (4, 1000),
                                 (5, 512), (16, 4096), (33, 1024), (300, 528), (2, 16), (8, 1024), (6, 1008), (4, 4112)])
def test_linear_is_codes_and_product(dev, M, K, dtype):
    """However few the tokens, however they lie: the same bits as by the codes."""
    g = gen(M + K)
    w = torch.randint(-128, 128, (72, K), generator=g, dtype=torch.int8).to(dev)
    ws, b = (0.01 * torch.rand(72, 1, generator=g)).to(dev), torch.randn(72, generator=g).to(dev)
    wide = acts(M, K + 24, dtype, seed=K, shift=0.2).to(dev)
    for x in (wide[:, :K], wide[:, 3:K + 3], wide[:, :K].contiguous()):
        for kw in (dict(symmetric=True), dict(symmetric=False), dict(scale=torch.tensor([0.03], device=dev))):
            want = int8_matmul(quantize_tokens(x, **kw), w, ws, b, out_dtype=F32)
            assert_bit_equal(int8_linear(x, w, ws, b, out_dtype=F32, **kw), want, f'{kw}')
        assert int8_linear(x, w, ws).dtype == dtype


@pytest.mark.parametrize('N,K', [(8200, 512), (8193, 4096), (9000, 16400), (4096, 8208), (1, 8192), (17, 16), (9000, 8192), (300, 32768)])
@pytest.mark.parametrize('symmetric', [True, False])
def test_one_token(dev, N, K, symmetric):
    g = torch.Generator(device=dev)
    g.manual_seed(N)
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8, device=dev)
    ws = 0.01 * torch.rand(N, 1, generator=g, device=dev)
    x = acts(1, K, BF, seed=N, shift=0.2).to(dev)
    q = quantize_tokens(x, symmetric)
    check_product(int8_linear(x, w, ws, symmetric=symmetric, out_dtype=F32), q.codes, q.scales, q.zeros, w, ws, None, F32)


def test_product_shapes_and_nothing(dev):
    q, s, _, w, ws, _ = product_inputs(6, 40, 128, False, False, dev=dev)
    flat = int8_matmul(QuantizedTokens(q, s), w, ws)
    assert torch.equal(int8_matmul(QuantizedTokens(q.view(2, 3, 128), s.view(2, 3, 1)), w, ws), flat.view(2, 3, 40))
    assert torch.equal(int8_matmul(QuantizedTokens(q[0], s[0]), w, ws), flat[0])
    assert int8_matmul(QuantizedTokens(q[:0], s[:0]), w, ws).shape == (0, 40)
    assert int8_matmul(QuantizedTokens(q, s), w[:0], ws[:0]).shape == (6, 0)
    assert quantize_tokens(torch.zeros(0, 64, device=dev)).codes.shape == (0, 64)


def test_product_behind_two_to_the_31(dev):
    """Codes and outputs of more than 2^31 elements: the last rows and columns."""
    M, K, N = 600_000, 4096, 8
    q = torch.zeros(M, K, dtype=torch.int8, device=dev)
    q[-300:] = torch.randint(-128, 128, (300, K), device=dev, dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), device=dev, dtype=torch.int8)
    s, ws = torch.rand(M, 1, device=dev), torch.rand(N, 1, device=dev)
    y = int8_matmul(QuantizedTokens(q, s), w, ws, out_dtype=F32)
    check_product(y[-300:], q[-300:], s[-300:], None, w, ws, None, F32)
    del q, y
    q, w = torch.randint(-128, 128, (17000, 64), device=dev, dtype=torch.int8), torch.randint(-128, 128, (140_000, 64), device=dev, dtype=torch.int8)
    s, ws = torch.rand(17000, 1, device=dev), torch.rand(140_000, 1, device=dev)
    y = int8_matmul(QuantizedTokens(q, s), w, ws)
    check_product(y[-200:, -500:].contiguous(), q[-200:], s[-200:], None, w[-500:], ws[-500:], None, BF)


# -- the norm between two blocks --------------------------------------------------------------------------------------
def norm64(v, dv, kind, w, b, offset, eps):
    """-> norm of v in 64 bits, and how far the kernel's may be from it where its v is within dv of this one.  A sum over a row in
    fp32: at most 64 terms in a lane, then 6 + 4 levels, so within 80 U of the sum of the terms' magnitudes."""
    if kind == 'layer':
        dv = dv + 80 * U * v.abs().mean(1, keepdim=True) + U * (v - v.mean(1, keepdim=True)).abs() + dv.mean(1, keepdim=True)
        v = v - v.mean(1, keepdim=True)
    ms = v.square().mean(1, keepdim=True)
    inv = 1 / torch.sqrt(ms + eps)
    dms = 2 * (v.abs() * dv).mean(1, keepdim=True) + dv.square().mean(1, keepdim=True) + 84 * U * ms
    rel = 0.5 * dms / (ms + eps) + 4 * U
    f = torch.ones_like(v[:1]) if w is None else w.double()[None] + offset
    y = v * inv * f
    dy = dv * inv * f.abs() + y.abs() * (rel + 4 * U)
    if w is not None and offset:
        dy = dy + (v * inv).abs() * U * f.abs()
    if b is not None:
        y = y + b.double()[None]
        dy = dy + U * (y.abs() + dy)
    return y, 1.02 * dy


def norm_inputs(T, K, dtype, dev, *, residual='same', gate=None, post=True, layer=False, affine32=False, seed=0):
    x = acts(T, K, dtype, seed + 1).to(dev)
    a = lambda i, mean: (mean + 0.3 * torch.randn(K, generator=gen(seed + i))).to(F32 if affine32 else dtype).to(dev)  # noqa: E731
    r = None if residual is None else acts(T, K, F32 if residual == 'f32' else dtype, seed + 2).to(dev)
    g = None if gate is None else torch.randn(*((T, K) if gate == 'rows' else (K,)), generator=gen(seed + 3)).to(dtype).to(dev)
    return x, dict(residual=r, weight=a(4, 1.0), bias=a(5, 0.0) if layer else None, gate=g, post_weight=a(6, 1.0) if post else None,
                   post_bias=a(7, 0.0) if layer and post else None, kind='layer' if layer else 'rms')


def check_norm(got, x, kw, scale=1.0, eps=1e-6, offset=0.0):
    f = torch.float64
    K = x.shape[-1]
    b = x.reshape(-1, K).to(f)
    db = torch.zeros_like(b)
    if kw['post_weight'] is not None:
        b, db = norm64(b, db, kw['kind'], kw['post_weight'], kw['post_bias'], offset, eps)
    if kw['gate'] is not None:
        g = kw['gate'].to(f).reshape(-1, K)
        b = b * g
        db = db * g.abs() + U * b.abs()
    h, dh = b * scale, db * abs(scale)
    if kw['residual'] is not None:
        h = h + kw['residual'].reshape(-1, K).to(f)
    dh = dh + U * (h.abs() + dh)
    y, dy = norm64(h, dh, kw['kind'], kw['weight'], kw['bias'], offset, eps)
    for name, t, want, tol in (('residual', got.residual, h, dh), ('out', got.out, y, dy)):
        tol = tol + half_step(t.dtype) * (want.abs() + tol) + TINY[t.dtype]
        err = (t.to(f).reshape(want.shape) - want).abs()
        assert bool((err <= tol).all()), f'{name}: {float((err / tol).max())} of the tolerance'


@pytest.mark.parametrize('dtype', [BF, HF, F32])
@pytest.mark.parametrize('layer', [False, True])
@pytest.mark.parametrize('T,K', [(1, 1), (3, 2), (2, 63), (5, 64), (9, 512), (4, 520), (3, 1000), (6, 1023), (2, 2048), (1, 4096), (3, 4095), (2, 7168),
                                 (2, 14336), (1, 20000), (1, 32769), (1, 65536)])
def test_norm(dev, T, K, dtype, layer):
    x, kw = norm_inputs(T, K, dtype, dev, layer=layer, seed=K)
    if layer and K == 1:
        kw['post_weight'] = kw['post_bias'] = None       # (of a norm of one column nothing is left but its bias)
    check_norm(residual_norm(x, scale=0.5, **kw), x, kw, scale=0.5)


@pytest.mark.parametrize('residual', [None, 'same', 'f32'])
@pytest.mark.parametrize('gate', [None, 'rows', 'row'])
@pytest.mark.parametrize('post', [True, False])
def test_norm_forms(dev, residual, gate, post):
    for dtype, K, affine32 in ((BF, 768, False), (HF, 771, True), (F32, 4100, False), (BF, 4096, True)):
        x, kw = norm_inputs(5, K, dtype, dev, residual=residual, gate=gate, post=post, affine32=affine32)
        got = residual_norm(x, scale=-0.75, eps=1e-3, weight_offset=1.0, **kw)
        assert got.out.dtype == dtype and got.residual.dtype == (F32 if residual == 'f32' else dtype)
        check_norm(got, x, kw, scale=-0.75, eps=1e-3, offset=1.0)
        check_norm(residual_norm(x, out_dtype=F32, **kw), x, kw)


def test_norm_without_weights_in_place_and_in_shapes(dev):
    x, kw = norm_inputs(6, 256, BF, dev, post=False)
    kw['weight'] = None
    got = residual_norm(x, **kw)
    check_norm(got, x, kw)
    stream = kw['residual'].clone()
    again = residual_norm(x, stream, inplace=True)
    assert again.residual is stream and torch.equal(stream, got.residual) and torch.equal(again.out, got.out)
    cube = residual_norm(x.view(2, 3, 256), kw['residual'].view(2, 3, 256))
    assert torch.equal(cube.out, got.out.view(2, 3, 256))
    assert residual_norm(x[:0], kw['residual'][:0]).out.shape == (0, 256)
    assert torch.equal(residual_norm(x[0], kw['residual'][0]).out, got.out[0])


def test_norm_rows_apart_and_off_alignment(dev):
    wide, other, gates = (acts(8, 900, BF, seed=i).to(dev) for i in range(3))
    for cut in (slice(0, 512), slice(1, 513), slice(8, 808), slice(5, 6)):
        views = [t[::2, cut] for t in (wide, other, gates)]
        plain = [t.contiguous() for t in views]
        a, b = residual_norm(views[0], views[1], gate=views[2]), residual_norm(plain[0], plain[1], gate=plain[2])
        assert torch.equal(a.out, b.out) and torch.equal(a.residual, b.residual)


@pytest.mark.parametrize('dtype', [BF, HF, F32])
@pytest.mark.parametrize('quantize', ['symmetric', 'asymmetric'])
@pytest.mark.parametrize('K', [40, 1023, 4096, 9000])
def test_norm_to_codes(dev, dtype, quantize, K):
    """The codes are those of the norm before it is rounded."""
    x, kw = norm_inputs(7, K, dtype, dev, gate='rows')
    plain = residual_norm(x, out_dtype=F32, **kw)
    fused = residual_norm(x, quantize=quantize, **kw)
    want = quantize_tokens(plain.out, quantize == 'symmetric')
    assert torch.equal(fused.out.codes, want.codes) and torch.equal(fused.out.scales, want.scales) and torch.equal(fused.residual, plain.residual)
    assert quantize == 'symmetric' or torch.equal(fused.out.zeros, want.zeros)


def test_norm_rows_that_are_not_finite_stay_by_themselves(dev):
    x, kw = norm_inputs(4, 256, BF, dev, post=False)
    x[1, 3], x[2, 9] = float('nan'), float('inf')
    got = residual_norm(x, **kw)
    assert bool(torch.isnan(got.out[1]).all()) and bool(torch.isnan(got.out[2, 9])) and bool(torch.isfinite(got.out[[0, 3]]).all())
    zero = residual_norm(torch.zeros(2, 256, device=dev), weight=torch.ones(256, device=dev))
    assert bool((zero.out == 0).all())


def test_norm_behind_two_to_the_31(dev):
    T, K = 530_000, 4096
    x = torch.zeros(T, K, dtype=BF, device=dev)
    x[-9:] = acts(9, K, BF, seed=1).to(dev)
    kw = dict(residual=None, weight=None, bias=None, gate=None, post_weight=None, post_bias=None, kind='rms')
    got = residual_norm(x)
    check_norm(type(got)(got.out[-9:], got.residual[-9:]), x[-9:], kw)


# -- the container, and all of it together ------------------------------------------------------------------------------
def test_more_rows_than_a_launch(dev):
    """2^21 rows and more: those around the seam and the last ones."""
    T, K = 2 ** 22 + 70, 16
    x, r = torch.randn(T, K, device=dev), torch.randn(T, K, device=dev)
    rows = torch.cat([torch.arange(300), 2 ** 21 + torch.arange(-200, 200), T - 1 - torch.arange(200)]).to(dev)
    got, want = quantize_tokens(x, False), quantize_tokens(x[rows], False)
    assert torch.equal(got.codes[rows], want.codes) and torch.equal(got.scales[rows], want.scales) and torch.equal(got.zeros[rows], want.zeros)
    codes, s, z = codes_of(x[rows].cpu(), False)
    assert torch.equal(want.codes.cpu(), codes)
    got = residual_norm(x, r)
    part = residual_norm(x[rows], r[rows])
    assert_bit_equal(got.out[rows], part.out, 'out')
    assert_bit_equal(got.residual[rows], part.residual, 'residual')
    q, s, z, w, ws, b = product_inputs(2 ** 21 + 300, 3, 17, True, True, dev=dev)
    check_product(int8_matmul(QuantizedTokens(q, s, z), w, ws, b, out_dtype=F32), q, s, z, w, ws, b, F32)


def linear(N, K, dtype, seed, bias=True):
    m = torch.nn.Linear(K, N, bias=bias, dtype=dtype)
    m.weight.data = (torch.randn(N, K, generator=gen(seed)) * 0.02).to(dtype)
    if bias:
        m.bias.data = torch.randn(N, generator=gen(seed + 1)).to(dtype)
    return m.cuda()


@pytest.mark.parametrize('dtype', [BF, HF, F32])
@pytest.mark.parametrize('act', [dict(symmetric=True, granularity='per_token'), dict(symmetric=False, granularity='per_token'),
                                 dict(symmetric=True, granularity='per_tensor', static=True)])
@pytest.mark.parametrize('granularity', ['per_channel', 'per_tensor'])
def test_the_container_runs(dev, dtype, act, granularity):
    rtn = RTN({'weight': dict(bit=8, symmetric=True, granularity=granularity), 'act': dict(bit=8, **act)})
    fc = linear(96, 160, dtype, 3)
    x = acts(10, 160, dtype, 4).to(dev).view(2, 5, 160)
    if rtn.act_static:
        rtn.register_act_qparams({'fc': fc}, [x])
    real = VllmRealQuantLinear.new(fc, **rtn.get_replacement_params('vllm_quant'))
    y = real(x)
    q = quantize_tokens(x.view(10, 160), act['symmetric'], real.input_scale if rtn.act_static else None)
    ws = real.weight_scale.reshape(-1, 1).expand(96, 1)
    check_product(y.view(10, 96), q.codes, q.scales.reshape(-1, 1).expand(10, 1), q.zeros, real.weight, ws, fc.bias.data, dtype)
    fake = rtn.a_qdq(x, fc, rtn.aquantizer) @ rtn.w_qdq(fc, rtn.wquantizer).t() + fc.bias.data
    assert float((y - fake).float().norm() / fake.float().norm()) < 0.02      # (the fake-quantized stand-in, itself in the row type)


def test_a_w8a8_block_and_its_answer(dev):
    """norm -> codes -> Linear -> norm with its gate -> Linear -> logits -> log probabilities, each step against 64 bits from the
    tensors that the step before it gave; eager, on a side stream and captured, which all give the same bits."""
    T, D, H, V = 37, 512, 1024, 1003
    cfg = {'weight': dict(bit=8, symmetric=True, granularity='per_channel'), 'act': dict(bit=8, symmetric=True, granularity='per_token')}
    rtn = RTN(cfg)
    up, down, head = (VllmRealQuantLinear.new(linear(n, k, BF, s, bias=False), **rtn.get_replacement_params('vllm_quant'))
                      for n, k, s in ((H, D, 1), (D, H, 2), (V, D, 3)))
    x, kw = norm_inputs(T, D, BF, dev, post=False)
    gate = torch.rand(D, generator=gen(9)).to(BF).to(dev)
    tokens = torch.randint(0, V, (T,), generator=gen(10)).to(dev)

    def run():
        a = residual_norm(x, kw['residual'], kw['weight'], quantize='symmetric')
        u = up(a.out)
        d = down(torch.relu(u))
        b = residual_norm(d, a.residual, kw['weight'], gate=gate, post_weight=kw['weight'], scale=0.5)
        logits = head(b.out)
        return [a.out.codes, a.out.scales, a.residual, u, d, b.out, b.residual, logits, *token_logprobs(logits, tokens, top=4)]

    codes, scales, h, u, d, out, h2, logits, logp, entropy, top_logp, top = first = run()
    check_product(u, codes, scales, None, up.weight, up.weight_scale, None, BF)
    q = quantize_tokens(torch.relu(u))
    check_product(d, q.codes, q.scales, None, down.weight, down.weight_scale, None, BF)
    check_norm(residual_norm(d, h, kw['weight'], gate=gate, post_weight=kw['weight'], scale=0.5), d,
               dict(residual=h, weight=kw['weight'], bias=None, gate=gate, post_weight=kw['weight'], post_bias=None, kind='rms'), scale=0.5)
    want = torch.log_softmax(logits.double(), 1)
    assert float((logp - want.gather(1, tokens[:, None])[:, 0]).abs().max()) < 1e-5
    assert torch.equal(top[:, 0], logits.float().argmax(1)) and float((top_logp - want.gather(1, top)).abs().max()) < 1e-5

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = run()
    for rep in range(3):
        x.mul_(1.0 + rep)                          # eager work between the replays
        fresh = run()
        torch.cuda.synchronize()
        for t in third:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(fresh, third)), rep


def test_two_graphs_side_by_side(dev):
    """Calls that take a workspace, captured in two graphs and replayed in turn on two streams."""
    inputs = [product_inputs(M, 200, 4096, True, False, seed=M, dev=dev) for M in (3, 40)]
    call = lambda q, s, z, w, ws, b: int8_matmul(QuantizedTokens(q, s, z), w, ws, out_dtype=F32)  # noqa: E731
    want = [call(*i) for i in inputs]
    graphs, outs = [], []
    for i in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(*i))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))
