"""The "around" form of the accumulating min (dgs_spmm_csr_acc_min_around_f32) on rows that hold their local result alone: a NaN that ends
the local chain leaves its arg, and the virtual entry that stands for it must not lose it.  (Rows with halo entries are redone by
dgs_spmm_min_merge_f32 when the data holds a NaN; a row without any is not.)  Over the emulation, like tests/test_emu_cpu.py."""
import os
import sys

import numpy as np
import pytest

import oracle
from util import around_matrix, assert_bitexact

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), 'emu'))
import emu_lib as E  # noqa: E402

pytestmark = pytest.mark.skipif(not os.path.exists('/opt/rocm/lib/llvm/bin/clang++'), reason='the emulation builds with ROCm\'s clang')


@pytest.mark.parametrize('N', [4, 5])
def test_a_nan_in_the_local_result_keeps_its_arg(N):
    M, K, a, b = 6, 8, 2, 6
    rp = np.array([0, 2, 4, 5, 5, 7, 8], np.int32)
    #               [fine, NaN] [NaN, fine] [NaN] [] [fine, inf] [inf]: all local columns
    col = np.array([2, 3, 3, 4, 3, 4, 5, 5], np.int32)
    X = np.full((K, N), 0.5, np.float32)
    X[3], X[5] = np.nan, np.inf
    val, deg, nl = np.ones(col.size, np.float32), np.diff(rp), b - a
    Xe = np.ascontiguousarray(np.concatenate([X[a:b], X[:a], X[b:]]))
    lcol = (col - a).astype(np.int32)
    Co, Eo = oracle.spmm('min', rp, lcol, val, Xe)
    C, Ei = E.spmm(E.MIN, rp, lcol, val, np.ascontiguousarray(Xe[:nl]))
    assert_bitexact(Ei, Eo, 'local arg ids')
    arp, acol, aval, arows = around_matrix(rp, col, val, deg, a, b, M, compact=False)
    E.spmm_acc_min_around(arp, acol, aval, np.ascontiguousarray(Xe[nl:]), C, Ei, arows, nl, a, M)
    assert_bitexact(C, Co, 'values')
    assert_bitexact(Ei, Eo, 'arg ids')
