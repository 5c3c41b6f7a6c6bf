"""The rule by which the int8 product is cut (csrc/launch_rules.h), over sizes: compiled with the host compiler, no GPU needed."""
import ctypes
import itertools
import shutil
import subprocess

import pytest

from lightcompress_amd import _lib as L
from lightcompress_amd.build import CSRC

WRAPPERS = '''
#include "launch_rules.h"
extern "C" int cut(long long M, long long N, long long K) { const lcq::Int8Cut c = lcq::int8_cut(M, N, K); return c.tile * 256 + c.parts; }
extern "C" int streams(long long M, long long N, long long K) { return lcq::int8_streams(M, N, K); }
'''


@pytest.fixture(scope='module')
def rules(tmp_path_factory):
    if not shutil.which('g++'):
        pytest.skip('no host compiler')
    d = tmp_path_factory.mktemp('cut')
    (d / 'w.cpp').write_text(WRAPPERS)
    subprocess.run(['g++', '-std=c++17', '-shared', '-fPIC', f'-I{CSRC}', str(d / 'w.cpp'), '-o', str(d / 'w.so')], check=True)
    so = ctypes.CDLL(str(d / 'w.so'))
    for f in (so.cut, so.streams):
        f.argtypes = [ctypes.c_longlong] * 3
    return so


@pytest.fixture(scope='module')
def cut(rules):
    return lambda *s: divmod(rules.cut(*s), 256)


def test_parts_are_whole_fit_the_chip_and_the_workspace(cut):
    for M, N, K in itertools.product((33, 64, 129, 300, 1000, 5000, 100000), (1, 16, 100, 4096, 6144, 14336, 140000), (16, 128, 2048, 4096, 14336, 65536)):
        tile, parts = cut(M, N, K)
        tiles = -(-M // 128) * -(-N // 128)
        assert tile in (0, 1, 2) and 1 <= parts <= 16
        if parts > 1:                              # parts of 128 x 128 tiles only, at least two stages each, one per CU, sums in the workspace
            assert tile == 2 and parts * tiles <= 256 and -(-K // 128) // parts >= 2


def test_the_workspace_follows_the_rules(cut, rules):
    need = L.lib().lcq_int8_matmul_workspace_bytes
    for M, N, K in itertools.product((1, 16, 17, 33, 64, 65, 300, 5000), (1, 100, 4096, 14336), (1, 15, 16, 17, 1024, 4097, 14336, 65536)):
        streams = rules.streams(M, N, K)
        parts = 1 if streams else cut(M, N, -(-K // 16) * 16)[1]
        padded = K % 16 and (not streams or K < 16)
        assert streams == 1 if M <= 16 else True
        assert not streams or M <= 64
        assert (need(M, N, K) == 0) == (parts == 1 and not padded)
        assert need(M, N, K) >= (4 * M * N * parts if parts > 1 else 0) + ((M + N) * -(-K // 16) * 16 if padded else 0)


def test_measured_streams(rules):
    """The sizes at which streams and tiles were timed against each other."""
    for (M, N, K), streams in {(64, 512, 512): 1, (33, 2048, 2048): 1, (64, 2048, 2048): 1, (33, 4096, 4096): 1, (64, 4096, 4096): 0,
                               (32, 14336, 4096): 0, (32, 4096, 14336): 0, (16, 14336, 4096): 1, (65, 512, 512): 0}.items():
        assert rules.streams(M, N, K) == streams, (M, N, K)


def test_measured_choices(cut):
    """The sizes at which the tiles were timed against each other: the fastest, or one within a few percent of it."""
    for (M, N), tile in {(1024, 4096): 2, (2048, 4096): 2, (1024, 6144): 2, (2048, 6144): 1, (512, 14336): 2, (1024, 14336): 0,
                         (2048, 14336): 0, (8192, 14336): 0}.items():
        assert cut(M, N, 4096)[0] == tile, (M, N)
    assert cut(64, 4096, 4096)[1] > 1 and cut(2048, 4096, 4096)[1] == 1


def test_sizes_of_the_gpu_tests_reach_every_tile(cut):
    from tests.test_w8a8_gpu import SIZES, TILED
    assert {cut(*s)[0] for s in TILED} == {0, 1, 2} and {cut(M, N, -(-K // 16) * 16)[0] for M, N, K in SIZES if M > 32} >= {2}
    assert sum(cut(*s)[1] > 1 for s in TILED) >= 2 and [cut(*s)[0] for s in TILED[:5]] == [0, 0, 1, 1, 1]
