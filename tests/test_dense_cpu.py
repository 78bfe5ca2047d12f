"""The dense operators without a GPU: what they refuse, through the Python functions, the operator registry and the C entries (which look at
their arguments before anything is launched), and the layers' host logic."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, EINVAL, EWORKSPACE, ERANGE = 0, -1, -2, -4
F32, F16, BF16 = 0, 1, 2
P = 1 << 20  # a pointer that is 16-byte aligned and never followed


@pytest.fixture(scope='module')
def lib():
    L = ctypes.CDLL(os.path.join(ROOT, 'dgsparse-lib_amd', 'dgsparse', 'libdgsparse_hip.so'))
    vp, i64, i32, f, sz = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
    L.dgs_embedding.argtypes = [i32, i32, i64, i64, i64, vp, vp, i64, f, vp, vp]
    L.dgs_embedding_bwd.argtypes = [i32, i32, i64, i64, i64, vp, i64, vp, i64, f, vp, vp, sz, vp]
    L.dgs_rms_norm.argtypes = [i32, i64, i64, vp, i64, vp, i64, vp, f, vp, vp, vp, vp, vp]
    L.dgs_rms_norm_bwd.argtypes = [i32, i64, i64, vp, vp, f, vp, vp, vp, vp, vp, sz, vp]
    L.dgs_gated_ffn.argtypes = [i32, i32, i64, i64, i64, vp, i64, vp, vp, i64, vp, vp, vp, sz, vp]
    L.dgs_gated_ffn_bwd.argtypes = [i32, i32, i64, i64, i64, vp, i64, vp, vp, i64, vp, vp, vp, vp, vp, vp, sz, vp]
    L.dgs_quantize_fp8.argtypes = [i32, i64, i64, vp, i64, i32, vp, vp, vp]
    L.dgs_matmul_fp8.argtypes = [i32, i64, i64, i64, vp, i64, vp, vp, i64, vp, vp, vp, sz, vp]
    for name, args in (('dgs_embedding_bwd_workspace_bytes', [i64] * 3), ('dgs_rms_norm_bwd_workspace_bytes', [i32, i64, i64]),
                       ('dgs_gated_ffn_workspace_bytes', [i32, i64, i64, i64, i32]), ('dgs_matmul_fp8_workspace_bytes', [i64] * 3)):
        getattr(L, name).argtypes, getattr(L, name).restype = args, sz
    return L


def test_embedding_entries_refuse(lib):
    good = dict(dtype=F32, idb=8, n=4, V=10, D=8, ids=P, table=P, ld=8, scale=1.0, out=P, stream=None)
    call = lambda **k: lib.dgs_embedding(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=3), dict(dtype=-1), dict(idb=2), dict(n=-1), dict(V=-1), dict(D=0), dict(ids=None), dict(table=None), dict(out=None)):
        assert call(**bad) == EINVAL, bad
    for bad in (dict(n=2 ** 31), dict(V=2 ** 31), dict(D=2 ** 26)):
        assert call(**bad) == ERANGE, bad
    assert call(n=0, ids=None, out=None) == OK
    good = dict(dtype=BF16, idb=4, n=4, V=10, D=8, ids=P, pad=-1, dout=P, ld=8, scale=1.0, dtable=P, ws=P, wsb=1 << 30, stream=None)
    call = lambda **k: lib.dgs_embedding_bwd(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=7), dict(idb=3), dict(D=-3), dict(ids=None), dict(dout=None), dict(dtable=None)):
        assert call(**bad) == EINVAL, bad
    need = lib.dgs_embedding_bwd_workspace_bytes(4, 10, 8)
    assert call(wsb=need - 1) == EWORKSPACE and call(ws=None) == EWORKSPACE and call(n=2 ** 31) == ERANGE
    assert call(V=0, dtable=None) == OK
    # the workspace goes by the positions, not by the table
    assert lib.dgs_embedding_bwd_workspace_bytes(100000, 10, 64) < 100000 * 64 + (1 << 22)
    assert need <= lib.dgs_embedding_bwd_workspace_bytes(9000, 10, 8)


def test_norm_entries_refuse(lib):
    good = dict(dtype=F16, rows=4, D=8, x=P, ldx=8, res=P, ldr=8, w=P, eps=1e-6, y=P, s=P, q=None, sc=None, stream=None)
    call = lambda **k: lib.dgs_rms_norm(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=5), dict(rows=-1), dict(D=0), dict(eps=-1.0), dict(eps=float('nan')), dict(x=None), dict(w=None), dict(s=None), dict(res=None), dict(y=None),
                dict(q=P), dict(y=None, q=P), dict(sc=P)):
        assert call(**bad) == EINVAL, bad
    assert call(rows=2 ** 32) == ERANGE and call(rows=0) == OK
    good = dict(dtype=F32, rows=4, D=8, s=P, w=P, eps=1e-6, dy=P, ds=None, dx=P, dw=P, ws=P, wsb=1 << 30, stream=None)
    call = lambda **k: lib.dgs_rms_norm_bwd(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=5), dict(rows=0), dict(D=0), dict(s=None), dict(w=None), dict(dy=None), dict(dx=None)):
        assert call(**bad) == EINVAL, bad
    assert call(wsb=lib.dgs_rms_norm_bwd_workspace_bytes(F32, 4, 8) - 1) == EWORKSPACE and call(ws=None) == EWORKSPACE


def test_ffn_entries_refuse(lib):
    good = dict(dtype=BF16, act=0, rows=4, D=8, F=16, x=P, ldx=8, wg=P, wu=P, ldw=8, h=P, pre=None, ws=P, wsb=1 << 30, stream=None)
    call = lambda **k: lib.dgs_gated_ffn(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=4), dict(act=3), dict(act=-1), dict(rows=-1), dict(D=0), dict(F=0), dict(ldx=-8), dict(x=None), dict(wg=None), dict(wu=None), dict(h=None),
                dict(h=P + 8), dict(pre=P + 4), dict(x=P + 2), dict(ldx=12), dict(ldw=9), dict(ldx=0)):
        assert call(**bad) == EINVAL, bad
    assert call(D=2 ** 23, ldx=2 ** 23, ldw=2 ** 23) == ERANGE and call(F=2 ** 23) == ERANGE and call(rows=2 ** 31) == ERANGE
    assert call(rows=0, x=None) == OK
    assert call(D=7, ldx=7, ldw=7, wsb=lib.dgs_gated_ffn_workspace_bytes(BF16, 4, 7, 16, 0) - 1) == EWORKSPACE
    good = dict(dtype=F32, act=1, rows=4, D=8, F=16, x=P, ldx=8, wg=P, wu=P, ldw=8, pre=None, dh=P, dx=P, dwg=P, dwu=P, ws=P, wsb=1 << 30, stream=None)
    call = lambda **k: lib.dgs_gated_ffn_bwd(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=4), dict(act=9), dict(rows=0), dict(dh=None), dict(dh=P + 4), dict(dx=P + 4), dict(dwg=None), dict(dwu=None), dict(dwu=P + 8), dict(ldx=6)):
        assert call(**bad) == EINVAL, bad
    assert call(wsb=lib.dgs_gated_ffn_workspace_bytes(F32, 4, 8, 16, 1) - 1) == EWORKSPACE and call(ws=None) == EWORKSPACE


def test_fp8_entries_refuse(lib):
    good = dict(dtype=F16, rows=4, cols=8, x=P, ld=8, block=1, q=P, sc=P, stream=None)
    call = lambda **k: lib.dgs_quantize_fp8(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=4), dict(rows=-1), dict(cols=0), dict(block=2), dict(block=0), dict(x=None), dict(q=None), dict(sc=None), dict(q=P + 1), dict(ld=-1)):
        assert call(**bad) == EINVAL, bad
    assert call(rows=0) == OK
    good = dict(dtype=BF16, M=4, N=8, K=32, a=P, lda=32, sa=P, b=P, ldb=32, sb=P, out=P, ws=P, wsb=1 << 30, stream=None)
    call = lambda **k: lib.dgs_matmul_fp8(*{**good, **k}.values())  # noqa: E731
    for bad in (dict(dtype=4), dict(M=-1), dict(N=-1), dict(K=0), dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(out=None), dict(out=P + 4), dict(a=P + 8), dict(lda=33),
                dict(ldb=40), dict(lda=-1)):
        assert call(**bad) == EINVAL, bad
    assert call(M=0) == OK and call(N=0) == OK and call(K=2 ** 24) == ERANGE and call(M=2 ** 31) == ERANGE
    assert call(K=33, wsb=lib.dgs_matmul_fp8_workspace_bytes(4, 8, 33) - 1) == EWORKSPACE


def test_rows_that_overlap_or_run_backwards_and_grids_beyond_32_bits_are_refused(lib):
    # (an 8-bit operand that is read in place: a row distance below the row's length would end the last row early)
    good = dict(dtype=BF16, M=4, N=8, K=32, a=P, lda=32, sa=P, b=P, ldb=32, sb=P, out=P, ws=P, wsb=1 << 30, stream=None)
    for bad in (dict(lda=16), dict(ldb=16), dict(lda=0), dict(ldb=0)):
        assert lib.dgs_matmul_fp8(*{**good, **bad}.values()) == EINVAL, bad
    assert lib.dgs_matmul_fp8(*{**good, **dict(N=2 ** 27 + 64, wsb=1 << 62)}.values()) == ERANGE
    good = dict(dtype=F16, rows=4, D=8, x=P, ldx=8, res=P, ldr=8, w=P, eps=1e-6, y=P, s=P, q=None, sc=None, stream=None)
    for bad in (dict(ldx=-8), dict(ldr=-8)):
        assert lib.dgs_rms_norm(*{**good, **bad}.values()) == EINVAL, bad
    assert lib.dgs_rms_norm(*{**good, **dict(rows=2 ** 25, D=4096, ldx=4096, ldr=4096)}.values()) == ERANGE
    good = dict(dtype=F32, idb=8, n=4, V=10, D=8, ids=P, table=P, ld=-8, scale=1.0, out=P, stream=None)
    assert lib.dgs_embedding(*good.values()) == EINVAL
    assert lib.dgs_embedding(*{**good, **dict(ld=4096, D=4096, n=2 ** 25)}.values()) == ERANGE
    good = dict(dtype=BF16, idb=4, n=4, V=10, D=8, ids=P, pad=-1, dout=P, ld=-8, scale=1.0, dtable=P, ws=P, wsb=1 << 30, stream=None)
    assert lib.dgs_embedding_bwd(*good.values()) == EINVAL
    assert lib.dgs_quantize_fp8(F16, 2 ** 30, 128, P, 128, 1, P, P, None) == ERANGE
    good = dict(dtype=BF16, act=0, rows=4, D=8, F=2 ** 23 - 2 ** 10, x=P, ldx=8, wg=P, wu=P, ldw=8, h=P, pre=None, ws=P, wsb=1 << 30, stream=None)
    assert lib.dgs_gated_ffn(*{**good, **dict(F=2 ** 23)}.values()) == ERANGE


def test_an_8_bit_projection_ends_with_the_weight_it_was_made_of(monkeypatch):
    """Training drops it: the layer would go on with the projection of the old weight after the next eval()."""
    import dgsparse.nn as nn
    from dgsparse.nn import dense as layers
    monkeypatch.setattr(layers.dense, 'quantize_fp8', lambda x, rows=1: (x.clone(), torch.ones(1, 1)))
    layer = nn.ResidualGCN(8, 16).quantize()
    assert layer.conv8 is not None and not layer.training
    layer.eval()
    assert layer.conv8 is not None
    layer.train()
    assert layer.conv8 is None
    assert layer.eval().conv8 is None


def test_python_functions_refuse():
    import dgsparse
    x, w, ids = torch.rand(4, 8), torch.rand(8), torch.zeros(3, dtype=torch.long)
    f8 = x.to(torch.float8_e4m3fn)
    for call in (lambda: dgsparse.embedding(ids, x), lambda: dgsparse.rms_norm(x, w), lambda: dgsparse.add_rms_norm(x, x, w), lambda: dgsparse.add_rms_norm_fp8(x, x, w),
                 lambda: dgsparse.gated_ffn(x, x, x), lambda: dgsparse.quantize_fp8(x), lambda: dgsparse.matmul_fp8(f8, w[:1].expand(4, 1), f8, w[:1].view(1, 1))):
        with pytest.raises(RuntimeError, match='no CPU fallback'):
            call()
    with pytest.raises(ValueError, match='padding_idx'):
        dgsparse.embedding(ids, x, padding_idx=-1)
    with pytest.raises(ValueError, match='activation'):
        dgsparse.gated_ffn(x, x, x, activation='tanh')
    with pytest.raises(ValueError, match='block_rows'):
        dgsparse.quantize_fp8(x, 64)
    with pytest.raises(RuntimeError, match='not a row of the table'):
        dgsparse.embedding(ids, x, padding_idx=4)


def test_layers_are_built_without_a_gpu():
    from dgsparse import nn as dnn
    e = dnn.Embedding(10, 4, padding_idx=3)
    assert e.weight[3].eq(0).all() and e.weight.requires_grad
    block = dnn.ResidualGCN(16, 40)
    assert sorted(n for n, _ in block.named_parameters()) == ['conv.W.weight', 'ffn.down.weight', 'ffn.w_gate', 'ffn.w_up', 'norm1.weight', 'norm2.weight']
    assert block.ffn.down.weight.shape == (16, 40) and dnn.GatedFFN(8, 24, 5).down.weight.shape == (5, 24)
    assert isinstance(dnn.GINConv(apply_func=dnn.GatedFFN(8, 24)).apply_func, dnn.GatedFFN)
