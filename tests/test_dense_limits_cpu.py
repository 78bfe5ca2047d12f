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


@pytest.fixture
def quantize_here(monkeypatch):
    """quantize_fp8 on the CPU, one scale for each 128 x 128."""
    from dgsparse.nn import dense as layers

    def quantize(x, rows=1):
        scale = torch.stack([torch.stack([t.abs().max() / 448 for t in r.split(128, 1)]) for r in x.detach().split(rows, 0)])
        wide = scale.repeat_interleave(rows, 0)[:x.shape[0]].repeat_interleave(128, 1)[:, :x.shape[1]]
        return (x.detach() / wide).to(torch.float8_e4m3fn), scale
    monkeypatch.setattr(layers.dense, 'quantize_fp8', quantize)
    return quantize


@pytest.mark.parametrize('change', [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: m.type(torch.float16),
                                    lambda m: torch.nn.Sequential(m).to('cpu', torch.float16)[0]])
def test_a_change_of_type_leaves_an_8_bit_weight_alone(quantize_here, change):
    import dgsparse.nn as nn
    lin = nn.LinearFP8(torch.randn(200, 150))
    weight, scale = lin.weight.clone(), lin.weight_scale.clone()
    assert change(lin) is lin
    assert lin.weight.dtype == torch.float8_e4m3fn and torch.equal(lin.weight.view(torch.uint8), weight.view(torch.uint8))
    assert lin.weight_scale.dtype == torch.float32 and torch.equal(lin.weight_scale, scale)
    assert list(lin.state_dict()) == ['weight', 'weight_scale']
    assert lin.to('meta').weight.is_meta and lin.weight.dtype == torch.float8_e4m3fn  # another device is one
