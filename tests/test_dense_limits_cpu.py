"""The dense operators' entries at the ends of their ranges, and the layers' host logic, without a GPU."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_workspace_of_sizes_that_the_entry_refuses():
    """A child with a time limit: the answer is a number, whatever the sizes."""
    code = ("import ctypes\n"
            f"L = ctypes.CDLL({os.path.join(ROOT, 'dgsparse-lib_amd', 'dgsparse', 'libdgsparse_hip.so')!r})\n"
            "f = L.dgs_embedding_bwd_workspace_bytes\n"
            "f.argtypes, f.restype = [ctypes.c_int64] * 3, ctypes.c_size_t\n"
            "big = [2 ** 31 - 1, 2 ** 31, 2 ** 62, 2 ** 63 - 1]\n"
            "assert all(f(*s) == 0 for v in big for s in ((1, v, 8), (v, 1, 8), (1, 1, v), (v, v, v)))\n"
            "assert f(2 ** 31 - 2, 2 ** 31 - 2, 1) > 4 * 4 * (2 ** 31 - 2) and f(1, 1, 1) > 0 and f(0, 5, 8) > 0\n")
    subprocess.run([sys.executable, '-c', code], check=True, timeout=60)
