"""Byte offsets of the matrix operators' operand layouts at the sizes where 32 bits end.  The kernels take them from one header that
needs no GPU compiler: it is compiled here for the host."""
import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'objectdetection_amd', 'csrc')
LARGEST = 2 ** 31 - 2 ** 16                     # values of a row, at most


@pytest.fixture(scope='module')
def offsets(tmp_path_factory):
    at = tmp_path_factory.mktemp('offsets')
    source = at / 'offsets.cpp'
    source.write_text('#include "offsets.h"\n'
                      'extern "C" long long pair_offset(int k) { return split_at(k); }\n'
                      'extern "C" long long column_offset(int col, int cols) { return column_at(col, cols); }\n')
    subprocess.run(['g++', '-std=c++17', '-O2', '-fPIC', '-shared', '-Wall', '-Werror', '-I', CSRC, str(source), '-o', str(at / 'offsets.so')],
                   check=True)
    lib = C.CDLL(str(at / 'offsets.so'))
    for f in (lib.pair_offset, lib.column_offset):
        f.restype = C.c_longlong
    return lib


@pytest.mark.parametrize('k', [0, 31, 32, 2 ** 29 - 32, 2 ** 29, 2 ** 30 + 40, LARGEST - 8])
def test_pairs_of_a_long_row(offsets, k):
    assert offsets.pair_offset(k) == k // 32 * 128 + k % 32 * 2


@pytest.mark.parametrize('cols', [8, 1000, 2 ** 30, 2 ** 30 + 4096, LARGEST])
def test_columns_of_a_long_row(offsets, cols):
    last = (cols - 1) // 8 * 8
    for col in (0, cols // 16 * 8, last, last + 8, last + 248):
        assert offsets.column_offset(col, cols) == 2 * min(col, last)
