"""The dense products against 64 bits in every tile shape that a size can select, split over K and not, and over walks along K that are long enough
for every buffer to come round again.  Each case says which tiles it is there for, and asks the library whether it takes them."""
import ctypes
import os

import pytest
import torch

from test_gpu_dense import TYPES, check_ffn, check_mm8, ids_of, rand

pytestmark = pytest.mark.gpu
DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def tiles(entry, *sizes):
    lib = ctypes.CDLL(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'dgsparse-lib_amd', 'dgsparse', 'libdgsparse_hip.so'))
    f = getattr(lib, entry)
    f.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.POINTER(ctypes.c_int32)]
    out = (ctypes.c_int32 * 6)(*[-1] * 6)
    assert f(*sizes, out) == 0
    return [(out[i], out[i + 1]) for i in range(0, 6, 2) if out[i] >= 0]


# sizes -> (edge, splits of K) of the forward product, dx, dW: 16 bits, and 32 bits.  (Widths and rows that end inside a tile, a hidden size whose
# rows of dg and du are padded.)
FFN = [((4100, 2992, 2100), [(256, 1), (256, 1), (256, 1)], [(128, 1), (128, 1), (128, 1)]),
       ((3080, 1544, 2056), [(256, 1), (256, 4), (256, 3)], [(128, 1), (128, 1), (128, 1)]),
       ((2100, 1000, 2052), [(128, 1), (128, 4), (128, 1)], [(128, 1), (128, 4), (128, 1)]),
       ((700, 520, 1030), [(64, 1), (64, 6), (64, 1)], [(64, 1), (64, 6), (64, 1)])]


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('sizes,half,full', FFN, ids=lambda v: 'x'.join(map(str, v)) if isinstance(v, tuple) else '')
def test_gated_ffn_in_every_tile(sizes, half, full, t):
    T, D, F = sizes
    assert tiles('dgs_gated_ffn_tiles', DTYPE[t], T, D, F) == (full if t == torch.float32 else half)
    check_ffn(rand(T, D, t=t, seed=1), rand(F, D, t=t, seed=2, scale=D ** -0.5), rand(F, D, t=t, seed=3, scale=D ** -0.5), 'gelu' if T == 3080 else 'silu')


# sizes -> tiles of a result in 16 bits and in 32, and the blocks of 128 that a workgroup walks (the scales come in windows of 8): more than two
# windows, one and a bit, several; whole operands and ones that are copied (K no multiple of 16)
MM8 = [((3000, 4100, 2192), (256, 1), (128, 1)), ((2049, 6001, 1300), (256, 1), (128, 1)), ((2050, 2050, 9000), (256, 4), (128, 1)),
       ((1030, 1030, 8208), (128, 4), (128, 4)), ((1500, 1000, 3000), (64, 1), (64, 1)), ((300, 1000, 11008), (64, 7), (64, 7))]


@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('sizes,half,full', MM8, ids=lambda v: 'x'.join(map(str, v)))
def test_matmul_fp8_through_many_windows_of_scales(sizes, half, full, t):
    import dgsparse
    M, N, K = sizes
    want = full if t == torch.float32 else half
    assert tiles('dgs_matmul_fp8_tiles', DTYPE[t], M, N, K) == [want] and -(-K // 128) / want[1] > 8
    # a scale of its own for every row and block, none like its neighbours': one that is taken from another step shows
    g = torch.Generator(device='cuda').manual_seed(K)
    a, sa = dgsparse.quantize_fp8(rand(M, K, t=torch.float32, seed=1))
    b, sb = dgsparse.quantize_fp8(rand(N, K, t=torch.float32, seed=2), 128)
    sa = sa * torch.exp2(torch.randint(-3, 4, sa.shape, generator=g, device='cuda'))
    sb = sb * torch.exp2(torch.randint(-3, 4, sb.shape, generator=g, device='cuda'))
    check_mm8(a, sa, b, sb, t)


def test_every_tile_is_covered():
    seen = {(which, e, s > 1) for sizes, half, full in FFN for plan in (half, full) for which, (e, s) in zip(('forward', 'dx', 'dw'), plan)}
    assert seen >= {('forward', e, False) for e in (64, 128, 256)} | {('dx', e, True) for e in (64, 128, 256)} | {('dx', 128, False), ('dx', 256, False), ('dw', 256, True)} \
        | {('dw', e, False) for e in (64, 128, 256)}
    seen = {(e, s > 1) for _, half, full in MM8 for e, s in (half, full)}
    assert seen >= {(256, False), (256, True), (128, False), (128, True), (64, False), (64, True)}
