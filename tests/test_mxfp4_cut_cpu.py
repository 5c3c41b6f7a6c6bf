"""The rules by which products of 4-bit numbers are cut (csrc/launch_rules.h), over sizes: compiled with the host compiler, no GPU needed."""
import ctypes
import itertools
import shutil
import subprocess

import pytest

from lightcompress_amd import _lib as L
from lightcompress_amd.build import CSRC

WRAPPERS = '''
#include "launch_rules.h"
extern "C" int cut(long long M, long long N, long long B) { const lcq::Mxfp4Cut c = lcq::mxfp4_cut(M, N, B); return c.stream * 1024 + c.tile * 256 + c.parts; }
extern "C" int waves(long long M, long long N, long long B) { return lcq::mxfp4_waves(M, N, B); }
template <int FN, int E> long long lost(long long N) {         // of the largest offset of a store, in the type that the kernel has for it
  typedef lcq::Mxfp4Store<FN, E> S;
  const long long of = ((S::TOKENS - 1) * N + 64 * FN - 16 / E) * E;
  return of - (long long)(typename S::Offset)of;
}
extern "C" long long lost_of(long long FN, long long E, long long N) {
  return FN == 4 ? (E == 2 ? lost<4, 2>(N) : lost<4, 4>(N)) : FN == 2 ? (E == 2 ? lost<2, 2>(N) : lost<2, 4>(N)) : E == 2 ? lost<1, 2>(N) : lost<1, 4>(N);
}
extern "C" long long units(long long M, long long N, long long KS) { return lcq::mxfp4_units(M, N, (int)KS); }
'''
WIDTHS = (1, 15, 16, 100, 200, 300, 1000, 4096, 6144, 14336, 140000, 1 << 24)
DEPTHS = (1, 32, 33, 255, 256, 257, 2047, 4096, 14336, 65536)


def blocks(K):
    return -(-K // 32)


@pytest.fixture(scope='module')
def rules(tmp_path_factory):
    if not shutil.which('g++'):
        pytest.skip('no host compiler')
    d = tmp_path_factory.mktemp('cut')
    (d / 'w.cpp').write_text(WRAPPERS)
    subprocess.run(['g++', '-std=c++17', '-shared', '-fPIC', f'-I{CSRC}', str(d / 'w.cpp'), '-o', str(d / 'w.so')], check=True)
    so = ctypes.CDLL(str(d / 'w.so'))
    for f in (so.cut, so.waves, so.units, so.lost_of):
        f.argtypes = [ctypes.c_longlong] * 3
    so.units.restype = so.lost_of.restype = ctypes.c_longlong
    return so


@pytest.fixture(scope='module')
def cut(rules):
    """-> (streamed, tile, parts)"""
    def of(M, N, K):
        v = rules.cut(M, N, blocks(K))
        return v // 1024, v // 256 % 4, v % 256
    return of


def test_cuts_are_whole(rules, cut):
    for M, N, K in itertools.product((1, 16, 17, 32, 33, 64, 65, 129, 300, 1000, 5000, 100000, 1 << 28), WIDTHS, DEPTHS):
        streamed, tile, parts = cut(M, N, K)
        assert streamed or M > 32
        if streamed:
            KS = rules.waves(M, N, blocks(K))
            assert KS in (1, 2, 4) and M <= 2048
            group = 16 if M <= 16 else 32
            assert rules.units(M, N, KS) == -(-(-(-N // 16)) // (4 // KS)) * -(-M // group) < 2 ** 31
        if not streamed and -(-M // 128) * -(-N // 128) <= (1 << 24) - 8:    # (what the product takes) fewer than 2^32 lanes
            side = (256, 128, 64)[tile]
            assert -(-M // side) * -(-N // side) * parts <= (1 << 24) - 8, (M, N, K)
        if not streamed and parts > 1:             # parts of 128 x 128 and 64 x 64 tiles only, at least two periods of 16 blocks each
            assert tile in (1, 2) and parts <= 8 and -(-blocks(K) // 16) >= 2 * parts


def test_the_workspace_follows_the_rules(cut):
    need, linear = L.lib().lcq_mxfp4_matmul_workspace_bytes, L.lib().lcq_mxfp4_linear_workspace_bytes
    for M, N, K in itertools.product((1, 16, 17, 33, 64, 65, 300, 5000), WIDTHS[:-1], DEPTHS):
        streamed, tile, parts = cut(M, N, K)
        scales = -(-blocks(K) // 16) * 16 * (M + N)
        sums = -(-4 * M * N * parts // 256) * 256 if parts > 1 else 0
        assert need(M, N, K, 0) == (0 if streamed else sums + scales)
        assert need(M, N, K, 1) == (0 if streamed else sums + (scales if tile == 0 or blocks(K) % 16 else 0))
        codes = M <= 16 and M * K <= (8192 if K % 8 else 16384)
        assert linear(M, N, K) == 0 if codes else linear(M, N, K) >= need(M, N, K, 0) + 16 * M * blocks(K) + M * blocks(K)
    assert need(0, 1, 1, 0) == need(1, 0, 1, 0) == need(1, 1, 0, 0) == need(1, 1, 65537, 0) == linear(1, 1, 65537) == 0


def test_measured_choices(rules, cut):
    """The sizes at which the cuts were timed against each other: the fastest, or one within a few percent of it."""
    for (M, N, K), want in {(64, 4096, 4096): (1,), (128, 4096, 4096): (0, 2, 1), (211, 4096, 4096): (0, 2, 1), (2048, 4096, 4096): (0, 1, 1),
                            (128, 1001, 2047): (1,), (1333, 1001, 2047): (0, 2, 1), (64, 14336, 4096): (0, 2, 1), (211, 14336, 4096): (0, 1, 1),
                            (1024, 14336, 4096): (0, 0, 1), (1024, 4096, 14336): (0, 1, 1), (64, 4096, 14336): (0, 2, 4), (128, 4096, 14336): (0, 2, 2),
                            (211, 2048, 7168): (0, 2, 1), (8192, 14336, 4096): (0, 0, 1)}.items():
        assert cut(M, N, K)[:len(want)] == want, (M, N, K)
    for (N, K), KS in {(1024, 1024): 4, (4096, 4096): 4, (7168, 2048): 2, (6144, 4096): 2, (14336, 4096): 1, (2048, 7168): 4, (4096, 14336): 4}.items():
        assert rules.waves(16, N, blocks(K)) == rules.waves(32, N, blocks(K)) == KS, (N, K)


def test_sizes_of_the_gpu_tests_reach_every_cut(rules, cut):
    from tests.test_mxfp4_gpu import CUTS, SIZES
    got = [(s, cut(*s)) for s in SIZES + CUTS]
    tiles = [(c[1], c[2]) for _, c in got if not c[0]]
    assert set(tiles) == {(0, 1)} | {(t, p) for t in (1, 2) for p in (1, 2, 4, 8)}
    streams = {(1 if M <= 16 else 2 if M <= 32 else 3, rules.waves(M, N, blocks(K))) for (M, N, K), c in got if c[0]}
    assert streams == {(t, KS) for t in (1, 2, 3) for KS in (1, 2, 4)}
    ragged = [(M, N, K) for (M, N, K), c in got if c[0] and M > 32 and M % 32 and N % 16 and K % 256]
    many = [(M, N, K) for (M, N, K), c in got if c[0] and rules.units(M, N, rules.waves(M, N, blocks(K))) > 256]
    assert len(ragged) >= 3 and {M > 32 for M, _, _ in many} == {True, False}


def test_offsets_of_stores_keep_their_bits(rules, cut):
    """Tiles of 64 x 64 are what more channels than 32 bits have bytes for get: 15 rows of two bytes or 7 of four to a store, 2^32 bytes from 143 165 577 channels on."""
    most = (1 << 28) - 16
    for N in (143165577, 150000000, 153391690, 160000000, 200000000, most):
        for E, FN in itertools.product((2, 4), (1, 2, 4)):
            assert rules.lost_of(FN, E, N) == 0, (N, E, FN)
    assert {cut(64, N, K)[:2] for N in (150000000, 155000000, most) for K in (32, 512)} == {(0, 2)}
    assert 15 * 2 * 150000000 > 1 << 32 and 7 * 4 * 155000000 > 1 << 32
