"""Microscaled 4-bit codes, their products and their refusals, against the definitions in 64 bits."""
import pytest
import torch

from lightcompress_amd._lib import LcqError
from lightcompress_amd.mxfp4 import Mxfp4, dequantize_mxfp4, mxfp4_linear, mxfp4_matmul, quantize_mxfp4
from tests.helpers import gen

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
f64 = torch.float64
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=f64)
TINY = {BF: 2.0 ** -134, HF: 2.0 ** -25, F32: 2.0 ** -150}   # half the distance of subnormals


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def acts(T, K, dtype, seed=0):
    g = gen(seed)
    return (torch.randn(T, K, generator=g) * torch.exp(0.7 * torch.randn(K, generator=g))).to(dtype)


def quantized(x):
    """codes [T, B, 32] and scale bytes [T, B] of x [T, K] by the definition: the nearest of the grid, a tie the even code."""
    T, K = x.shape
    B = (K + 31) // 32
    v = torch.zeros(T, 32 * B, dtype=f64)
    v[:, :K] = x.to(f64)
    v = v.view(T, B, 32)
    most = v.abs().amax(2)
    bad = ~torch.isfinite(most)
    e = torch.where((most > 0) & ~bad, torch.frexp(torch.where(bad, 1.0, most))[1] - 1, -200)
    scale = (e - 2 + 127).clamp_min(0)
    r = v.abs().nan_to_num(0, 0, 0) / torch.exp2(scale.to(f64) - 127)[..., None]
    mid = (GRID[1:] + GRID[:-1]) / 2
    up = torch.tensor([i % 2 == 0 for i in range(1, 8)])
    code = ((r[..., None] > mid) | ((r[..., None] == mid) & up)).sum(-1) + 8 * torch.signbit(v)
    code[bad] = 0
    return code.to(torch.uint8), torch.where(bad, 255, scale).to(torch.uint8)


def packed(code):
    c = code.flatten(-2)
    return c[..., 0::2] | c[..., 1::2] << 4


def values(q, cols=None):
    """What an Mxfp4 stands for, in 64 bits on its device."""
    codes, scales = q.codes.view(torch.uint8), q.scales.view(torch.uint8)
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    table = torch.cat([GRID, -GRID]).to(codes.device)
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.to(f64) - 127))
    return (table[both] * s.repeat_interleave(32, -1))[..., :q.cols if cols is None else cols]


def random_mx(rows, K, g, dev, low=118, high=130):
    """Random codes (zeros behind K) and scales."""
    B = (K + 31) // 32
    codes = torch.randint(0, 256, (rows, 16 * B), generator=g, dtype=torch.uint8, device=dev)
    if K % 32:
        codes[:, (K + 1) // 2:] = 0
        if K % 2:
            codes[:, K // 2] &= 15
    return Mxfp4(codes, torch.randint(low, high, (rows, B), generator=g, dtype=torch.uint8, device=dev), K)


def gpu_gen(seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return g


# -- codes ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', [BF, HF, F32])
@pytest.mark.parametrize('T,K', [(1, 1), (1, 7), (1, 32), (2, 33), (5, 63), (3, 64), (7, 1000), (4, 1025), (2, 2048), (3, 5121), (2, 14336), (1, 65536),
                                 (130, 520), (1000, 31), (33, 4096), (1, 70001)])
def test_codes_equal_the_definition(dev, T, K, dtype):
    x = acts(T, K, dtype, seed=T + K)
    got = quantize_mxfp4(x.to(dev))
    code, scale = quantized(x)
    assert got.cols == K and torch.equal(got.scales.cpu(), scale) and torch.equal(got.codes.cpu(), packed(code))
    for out in (F32, BF, HF):
        y = dequantize_mxfp4(got, out)
        assert y.dtype == out and torch.equal(y.cpu(), values(Mxfp4(packed(code), scale, K)).float().to(out))


def test_rows_at_the_edges(dev):
    """Ties of every pair of codes, both signs; zeros; subnormals; the largest numbers; each in a block of its own."""
    mid = ((GRID[1:] + GRID[:-1]) / 2).float()
    rows = []
    for e in (0, -20, 100, -126, -127, 121):
        v = torch.cat([mid, -mid, GRID.float(), -GRID.float(), mid[:2]]) * torch.tensor(2.0, dtype=f64).pow(e).float()
        rows.append(v)
        rows.append(torch.nextafter(v, torch.full((32,), torch.inf)))
        rows.append(torch.nextafter(v, torch.full((32,), -torch.inf)))
    for top in (1.0, 1.9999999, 2.0, 1.7e38, 1.2e-38, 1e-40, 1.5e-45, 5e-39):
        v = torch.linspace(-top, top, 32)
        v[5] = top
        rows.append(v)
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), torch.finfo(F32).max)]
    x = torch.stack(rows)
    assert bool(torch.isfinite(x).all())
    code, scale = quantized(x)
    got = quantize_mxfp4(x.to(dev))
    assert torch.equal(got.scales.cpu(), scale)
    assert torch.equal(got.codes.cpu(), packed(code))
    assert torch.equal(dequantize_mxfp4(got, F32).cpu(), values(Mxfp4(packed(code), scale, 32)).float())
    y = quantize_mxfp4(x.to(BF).to(dev))           # (the largest rounds to infinity)
    code, scale = quantized(x.to(BF).float())
    assert torch.equal(y.scales.cpu(), scale) and torch.equal(y.codes.cpu(), packed(code))


@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_a_block_that_is_not_finite_is_nan(dev, bad):
    for dtype in (BF, HF, F32):
        x = acts(3, 100, dtype, seed=2)
        x[1, 40] = bad
        got = quantize_mxfp4(x.to(dev))
        code, scale = quantized(x)
        assert int(scale[1, 1]) == 255 and torch.equal(got.scales.cpu(), scale) and torch.equal(got.codes.cpu(), packed(code))
        y = dequantize_mxfp4(got, dtype)
        assert bool(torch.isnan(y[1, 32:64]).all()) and int(torch.isnan(y).sum()) == 32
        w = quantize_mxfp4(acts(70, 100, dtype, seed=3).to(dev))
        for tokens in (x, x[1:2], x.repeat(40, 1)):
            p = mxfp4_linear(tokens.to(dev), w)
            spoilt = torch.isnan(tokens.float()).any(1) | torch.isinf(tokens.float()).any(1)
            assert torch.equal(torch.isnan(p).all(1).cpu(), spoilt) and torch.equal(torch.isnan(p).any(1).cpu(), spoilt)


@pytest.mark.parametrize('dtype', [BF, F32])
def test_rows_apart_and_off_alignment(dev, dtype):
    big = acts(9, 700, dtype, seed=4).to(dev)
    for view in (big[:, :512], big[:, 1:514], big[::2, 8:520], big[:, 3:67], big.t()[:64].t(), big.view(3, 3, 700)[:, 1:, :256], big[:1].expand(5, 700),
                 big[:, ::2]):
        a, b = quantize_mxfp4(view), quantize_mxfp4(view.clone(memory_format=torch.contiguous_format))
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and a.codes.shape[:-1] == view.shape[:-1]
    q = quantize_mxfp4(big)
    part = Mxfp4(q.codes[:, 32:160], q.scales[:, 2:10])            # columns 64 .. 319
    assert torch.equal(dequantize_mxfp4(part, dtype), dequantize_mxfp4(q, dtype)[:, 64:320])
    part = Mxfp4(q.codes[::3, 32:160], q.scales[::3, 2:10], 250)
    assert torch.equal(dequantize_mxfp4(part, dtype), dequantize_mxfp4(q, dtype)[::3, 64:314])


def test_more_values_than_31_bits(dev):
    x = torch.zeros(9, 1 << 28, dtype=BF, device=dev)
    x[8, -40:] = torch.arange(40, device=dev)
    q = quantize_mxfp4(x)
    y = dequantize_mxfp4(q)
    assert torch.equal(y[8, -64:], dequantize_mxfp4(quantize_mxfp4(x[8, -64:]))) and int(torch.count_nonzero(y)) == int(torch.count_nonzero(y[8, -64:]))


def test_scales_at_both_ends(dev):
    """Every code with the least and the largest scales.  Above the largest fp32 number: 4 and 6 with byte 253, 2 to 6 with 254; those are infinite."""
    low = torch.arange(16, dtype=torch.uint8, device=dev)
    codes = (low | low.flip(0) << 4).expand(12, 16).contiguous()
    scales = torch.tensor([0, 1, 2, 3, 7, 127, 250, 251, 252, 253, 254, 255], dtype=torch.uint8, device=dev)[:, None]
    q = Mxfp4(codes, scales)
    want = values(q)
    for out in (F32, BF, HF):
        y = dequantize_mxfp4(q, out)
        torch.testing.assert_close(y, want.float().to(out), rtol=0, atol=0, equal_nan=True)
    y = dequantize_mxfp4(q, F32)
    assert [int(torch.isinf(r).sum()) for r in y] == [0] * 9 + [8, 16, 0] and bool(torch.isnan(y[11]).all())
    assert torch.equal(y[:9].to(f64), want[:9])


@pytest.mark.parametrize('M', [1, 20, 100, 300])
def test_products_of_the_largest_scales(dev, M):
    """The product takes all scales as they are: sums of tokens of 2^-110 or so with weights that fp32 does not hold are ordinary numbers."""
    g = gpu_gen(M)
    N, K = 130, 544
    a, w = random_mx(M, K, g, dev, 15, 18), random_mx(N, K, g, dev, 252, 255)
    va, vw = values(a), values(w)
    assert bool((vw.abs() > torch.finfo(F32).max).any())
    size = va.abs() @ vw.abs().t()
    assert bool(((mxfp4_matmul(a, w, out_dtype=F32).to(f64) - va @ vw.t()).abs() <= (K / 64 + 16) * 2.0 ** -23 * size).all())


# -- the product ----------------------------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 64, 64), (1, 1000, 4096), (2, 17, 63), (3, 4096, 128), (7, 100, 2050), (8, 256, 1024), (15, 33, 80), (16, 4096, 4096),
         (17, 130, 272), (31, 64, 4112), (32, 512, 512), (33, 257, 1040), (48, 1024, 2048), (64, 64, 64), (65, 1001, 2047), (100, 300, 4096),
         (127, 129, 144), (128, 128, 32), (129, 2048, 512), (200, 96, 14336), (255, 511, 1008), (256, 256, 4096), (257, 4096, 1024),
         (300, 5000, 48), (513, 513, 513), (1000, 777, 2064), (2048, 1024, 4096), (4097, 300, 256), (300, 264, 65536), (20, 24, 65536),
         (4000, 4000, 1030), (4096, 4096, 512), (3900, 4001, 64), (5000, 3333, 1536), (70, 4100, 4112), (300, 1000, 14336)]


@pytest.mark.parametrize('bias,dtype', [(False, F32), (True, F32), (True, BF), (False, HF)])
@pytest.mark.parametrize('M,N,K', SIZES)
def test_product(dev, M, N, K, bias, dtype):
    """Steps of the pipe's sums: one per 64 codes at least, each off by at most 2^-23 of the magnitudes that went into them; then the
    waves' or parts' sums and the bias, and half a step of the output type."""
    g = gpu_gen(M + 7 * N + 13 * K)
    a, w = random_mx(M, K, g, dev), random_mx(N, K, g, dev, 110, 122)
    b = torch.randn(N, generator=g, device=dev) if bias else None
    got = mxfp4_matmul(a, w, b, out_dtype=dtype)
    assert got.dtype == dtype and got.shape == (M, N)
    va, vw = values(a), values(w)
    want, size = va @ vw.t(), va.abs() @ vw.abs().t()
    if bias:
        want, size = want + b.to(f64), size + b.to(f64).abs()
    err32 = (K / 64 + 16) * 2.0 ** -23 * size
    tol = err32 + half_step(dtype) * (want.abs() + err32) + TINY[dtype]
    err = (got.to(f64) - want).abs()
    if dtype == HF:
        over = want.abs() + err32 >= 65504
        err = err.masked_fill(over, 0)
    assert bool((err <= tol).all()), f'{float((err / tol).max())} of the tolerance'


CUTS = [(5, 14336, 520), (9, 6145, 4100), (13, 300017, 96), (20, 14300, 1100), (25, 7170, 2050), (45, 14335, 300), (90, 2500, 16000), (61, 40001, 200),
        (211, 4000, 14300), (300, 3000, 10000), (1000, 14300, 4100),
        (4900, 66, 14470), (66, 12450, 11050), (2790, 66, 21800), (6730, 17, 6420), (2070, 16, 3811), (33, 17, 487), (67, 10694, 140), (7000, 14501, 1100)]          # (the last one's outputs go past the caches)


@pytest.mark.parametrize('dtype', [F32, BF])
@pytest.mark.parametrize('M,N,K', CUTS)
def test_product_of_every_cut(dev, M, N, K, dtype):
    test_product(dev, M, N, K, True, dtype)


@pytest.mark.parametrize('M,N,K', [(1, 300, 2048), (2, 77, 1000), (5, 100, 1999), (16, 515, 2048), (30, 64, 1056), (64, 200, 2048), (65, 130, 2000),
                                   (200, 600, 1537), (3000, 4100, 1030), (257, 255, 1024), (4097, 4097, 544)])
def test_sums_that_fit_are_exact(dev, M, N, K):
    """Scales within a factor of two: all sums are multiples of 2^-4 below 2^19, which 24 bits hold, so any order gives them exactly."""
    g = gpu_gen(K)
    a, w = random_mx(M, K, g, dev, 126, 129), random_mx(N, K, g, dev, 126, 129)
    assert float((values(a).abs() @ values(w).abs().t()).max()) < 2 ** 19
    assert torch.equal(mxfp4_matmul(a, w, out_dtype=F32).to(f64), values(a) @ values(w).t())


@pytest.mark.parametrize('dtype', [BF, HF, F32])
@pytest.mark.parametrize('M,N,K', [(1, 300, 2048), (2, 4096, 4096), (2, 70, 999), (3, 130, 4000), (8, 500, 1024), (16, 64, 14336), (40, 300, 70), (100, 257, 2080),
                                   (1, 40, 32768), (1, 40, 65536), (513, 700, 1111), (4096, 4096, 520)])
def test_linear_is_codes_and_product(dev, M, N, K, dtype):
    """The codes of a Linear are those of quantize_mxfp4.  Sums may be cut differently: up to their steps."""
    g = gpu_gen(N)
    x = acts(M, K, dtype, seed=K).to(dev)
    w = random_mx(N, K, g, dev, 110, 122)
    b = torch.randn(N, generator=g, device=dev).to(dtype)
    got = mxfp4_linear(x, w, b, out_dtype=F32)
    va, vw = values(quantize_mxfp4(x)), values(w)
    size = va.abs() @ vw.abs().t() + b.to(f64).abs()
    err = (got.to(f64) - (va @ vw.t() + b.to(f64))).abs()
    assert bool((err <= ((K / 64 + 16) * 2.0 ** -23 + 2.0 ** -24) * size).all())
    y = mxfp4_linear(x, w, b)
    assert y.dtype == dtype and torch.equal(y, got.to(dtype))
    assert torch.equal(mxfp4_linear(x.view(1, M, K), w, b), y.view(1, M, N))


@pytest.mark.parametrize('M,K', [(1, 1024), (5, 1000), (100, 1024), (300, 1056)])
def test_operands_apart_and_off_alignment(dev, M, K):
    g = gpu_gen(M)
    big, bw = random_mx(M + 3, 2 * K, g, dev), random_mx(203, 2 * K, g, dev, 110, 122)
    B = K // 32
    cut = lambda q, r, at: Mxfp4(q.codes[r:, 16 * at:16 * (at + B)], q.scales[r:, at:at + B])  # noqa: E731
    whole = lambda q: Mxfp4(q.codes.contiguous(), q.scales.contiguous())                       # noqa: E731
    for a, w in ((cut(big, 3, 1), cut(bw, 3, 2)), (whole(cut(big, 2, 0)), cut(bw, 0, 3)), (cut(big, 1, 5), whole(cut(bw, 1, 0)))):
        assert torch.equal(mxfp4_matmul(a, w), mxfp4_matmul(whole(a), whole(w)))
    flat = torch.zeros(203 * 16 * B + 5, dtype=torch.uint8, device=dev)
    off = flat[5:].view(203, 16 * B)
    off.copy_(cut(bw, 0, 0).codes)
    a = whole(cut(big, 0, 0))
    sc = cut(bw, 0, 0).scales
    flat = torch.zeros(sc.numel() + 3, dtype=torch.uint8, device=dev)
    sc_off = flat[3:].view(sc.shape)
    sc_off.copy_(sc)
    assert torch.equal(mxfp4_matmul(a, Mxfp4(off, sc_off)), mxfp4_matmul(a, whole(cut(bw, 0, 0))))


@pytest.mark.parametrize('M', [1, 3, 20, 100])
def test_a_nan_scale_spoils_its_row_alone(dev, M):
    """Also where the blocks behind a row's last would be."""
    g = gpu_gen(M)
    for K in (32, 100, 544, 1024, 2080):
        a, w = random_mx(M, K, g, dev), random_mx(150, K, g, dev)
        w.scales[7, -1] = 255
        w.scales[149, 0] = 255
        a.scales[M - 1, 0] = 255
        y = torch.isnan(mxfp4_matmul(a, w, out_dtype=F32))
        want = torch.zeros(M, 150, dtype=torch.bool, device=dev)
        want[:, [7, 149]] = True
        want[M - 1] = True
        assert torch.equal(y, want)


def test_types_of_torch_and_empty_calls(dev):
    g = gpu_gen(1)
    a, w = random_mx(5, 256, g, dev), random_mx(9, 256, g, dev)
    typed = Mxfp4(w.codes.view(torch.float4_e2m1fn_x2), w.scales.view(torch.float8_e8m0fnu))
    assert torch.equal(mxfp4_matmul(a, typed), mxfp4_matmul(a, w)) and torch.equal(dequantize_mxfp4(typed), dequantize_mxfp4(w))
    assert quantize_mxfp4(torch.zeros(0, 64, device=dev)).codes.shape == (0, 32)
    assert mxfp4_linear(torch.zeros(0, 256, device=dev), w).shape == (0, 9)
    assert mxfp4_matmul(a, Mxfp4(w.codes[:0], w.scales[:0])).shape == (5, 0)
    assert dequantize_mxfp4(Mxfp4(w.codes[:0], w.scales[:0])).shape == (0, 256)


def test_another_stream_and_a_graph(dev):
    """Two products whose workspaces a graph keeps, and quantization, replayed between eager calls of the same sizes."""
    g = gpu_gen(2)
    w, w2 = random_mx(1000, 2000, g, dev, 110, 122), random_mx(600, 1000, g, dev, 110, 122)
    x = acts(100, 2000, BF, seed=1).to(dev)
    run = lambda x: mxfp4_linear(mxfp4_linear(x, w), w2)  # noqa: E731
    want = run(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x)
    for i in range(4):
        x.copy_(acts(100, 2000, BF, seed=10 + i).to(dev))
        want = run(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_every_kind_of_cut_in_two_graphs(dev):
    """Streamed, tiles of each size, parts and their join: two graphs replayed in turn, with eager calls of the same operands between."""
    g = gpu_gen(4)
    sizes = [(9, 300, 1000), (40, 520, 2048), (70, 3000, 2000), (300, 264, 9190), (211, 14336, 1056), (1000, 14300, 600)]
    operands = [(random_mx(M, K, g, dev, 110, 122), random_mx(N, K, g, dev, 110, 122), torch.randn(N, generator=g, device=dev)) for M, N, K in sizes]
    run = lambda: [mxfp4_matmul(a, w, b) for a, w, b in operands]  # noqa: E731
    run()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(run())
    for i in range(3):
        for a, _, _ in operands:
            a.codes.copy_(a.codes.roll(1, 0))
        want = run()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.parametrize('M', [1, 40, 100, 300])
def test_weights_behind_2_gigabytes(dev, M):
    g = gpu_gen(5)
    N, K = 66000, 65536
    a, w = random_mx(M, K, g, dev), random_mx(N, K, g, dev, 110, 122)
    assert w.codes.numel() > 2 ** 31
    got = mxfp4_matmul(a, w, out_dtype=F32)
    for at in (slice(0, 70), slice(N - 70, N)):
        va, vw = values(a), values(Mxfp4(w.codes[at], w.scales[at], K))
        err = (got[:, at].to(f64) - va @ vw.t()).abs()
        assert bool((err <= (K / 64 + 16) * 2.0 ** -23 * (va.abs() @ vw.abs().t()) + TINY[F32]).all())


def test_outputs_behind_2_31(dev):
    g = gpu_gen(6)
    M, N, K = 300, 8000000, 32
    a, w = random_mx(M, K, g, dev), random_mx(N, K, g, dev, 110, 122)
    got = mxfp4_matmul(a, w)
    assert got.numel() > 2 ** 31
    for at in (slice(0, 999), slice(N - 999, N)):
        assert torch.equal(got[:, at], mxfp4_matmul(a, Mxfp4(w.codes[at].contiguous(), w.scales[at].contiguous(), K)))


@pytest.mark.parametrize('M,N,dtype', [(64, 150000000, BF), (130, 143165600, HF), (64, 155000000, F32)])
def test_rows_of_a_store_behind_2_32_bytes(dev, M, N, dtype):
    """64 x 64 tiles whose stores reach over 15 rows of two bytes, or 7 of four: 2^32 bytes and more."""
    g = gpu_gen(8)
    K = 32
    a, w = random_mx(M, K, g, dev), random_mx(N, K, g, dev, 110, 122)
    got = mxfp4_matmul(a, w, out_dtype=dtype)
    for at in (0, 1 << 20, N // 2 // 64 * 64, N - 64 - 1000):
        rows = slice(at, at + 1000)
        assert torch.equal(got[:, rows], mxfp4_matmul(a, Mxfp4(w.codes[rows].contiguous(), w.scales[rows].contiguous(), K), out_dtype=dtype))


@pytest.mark.parametrize('dtype', [BF, HF, F32])
def test_one_row_for_all(dev, dtype):
    """Expanded operands: rows that lie on top of each other."""
    g = gpu_gen(7)
    w = random_mx(50, 160, g, dev, 110, 122)
    for T in (3, 40, 200):
        x = torch.randn(1, 160, generator=g, device=dev).to(dtype).expand(T, 160)
        q = quantize_mxfp4(x)
        assert torch.equal(q.codes, quantize_mxfp4(x[:1]).codes.expand(T, -1)) and torch.equal(mxfp4_linear(x, w), mxfp4_linear(x.contiguous(), w))
        one = quantize_mxfp4(x[:1])
        wide = Mxfp4(one.codes.expand(T, -1), one.scales.expand(T, -1), 160)
        assert torch.equal(mxfp4_matmul(wide, w), mxfp4_matmul(q, w)) and torch.equal(dequantize_mxfp4(wide), dequantize_mxfp4(q))
        rows = Mxfp4(w.codes[:1].expand(50, -1), w.scales[:1].expand(50, -1), 160)
        assert torch.equal(mxfp4_matmul(q, rows), mxfp4_matmul(q, Mxfp4(rows.codes.contiguous(), rows.scales.contiguous(), 160)))


# -- refusals -------------------------------------------------------------------------------------------------------
def test_refusals(dev):
    g = gpu_gen(3)
    a, w = random_mx(5, 256, g, dev), random_mx(9, 256, g, dev)
    for bad in (lambda: mxfp4_matmul(a, random_mx(9, 250, g, dev)), lambda: mxfp4_matmul(a, w, torch.zeros(8, device=dev)),
                lambda: mxfp4_matmul(Mxfp4(a.codes[:, :-16], a.scales), w), lambda: mxfp4_matmul(Mxfp4(a.codes, a.scales, 224), w),
                lambda: mxfp4_matmul(a, Mxfp4(w.codes[None], w.scales[None])), lambda: mxfp4_linear(torch.zeros(3, 250, device=dev), w),
                lambda: quantize_mxfp4(torch.zeros(3, 0, device=dev)), lambda: mxfp4_linear(torch.zeros(3, 70000, device=dev), w)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: quantize_mxfp4(torch.zeros(3, 32, dtype=torch.int32, device=dev)), lambda: dequantize_mxfp4(a, torch.float64),
                lambda: mxfp4_matmul(Mxfp4(a.codes.to(torch.int8), a.scales), w), lambda: mxfp4_matmul(a, Mxfp4(w.codes.cpu(), w.scales.cpu())),
                lambda: mxfp4_matmul(a, w, torch.zeros(9, dtype=torch.int32, device=dev))):
        with pytest.raises(LcqError):
            bad()
