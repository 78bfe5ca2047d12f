"""The dense operators where values and calls are out of the ordinary."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwad

from test_gpu_dense import E32, TYPES, U, check_mm8, ids_of, norm_want, rand, tiny, within

pytestmark = pytest.mark.gpu


# ---- what an infinity or a NaN reaches ----------------------------------------------------------------------------------------
@pytest.mark.parametrize('t', TYPES, ids=ids_of)
@pytest.mark.parametrize('T,D,F', [(80, 40, 50), (300, 264, 136), (10, 24, 70)])
def test_gated_ffn_a_bad_gradient_stays_in_its_row(T, D, F, t):
    """dh[r, f] enters row r of dx and row f of the weights' gradients, and nothing else: every other row keeps its bits."""
    import dgsparse
    leaves = [a.requires_grad_() for a in (rand(T, D, t=t, seed=1), rand(F, D, t=t, seed=2, scale=D ** -0.5), rand(F, D, t=t, seed=3, scale=D ** -0.5))]
    dh = rand(T, F, t=t, seed=4)
    places = [(0, 0, math.inf), (T - 1, F - 1, -math.inf), (3, 7, math.nan), (5, 12, math.inf), (T // 2, 33, math.nan)]
    bad = dh.clone()
    for r, f, v in places:
        bad[r, f] = v
    rows, cols = torch.ones(T, dtype=torch.bool, device='cuda'), torch.ones(F, dtype=torch.bool, device='cuda')
    rows[[p[0] for p in places]] = False
    cols[[p[1] for p in places]] = False
    for again in (False, True):
        h = dgsparse.gated_ffn(*leaves, activation='silu', recompute=again)
        want = torch.autograd.grad(h, leaves, dh, retain_graph=True)
        got = torch.autograd.grad(h, leaves, bad)
        for a, b, keep, what in zip(got, want, (rows, cols, cols), ('dx', 'dw_gate', 'dw_up')):
            assert torch.equal(a[keep], b[keep]), (what, again, 'a row that the value does not enter')
            assert not a[~keep].isfinite().any(), (what, again, 'a row that it enters')


def test_gated_ffn_a_closed_unit_stays_in_its_column():
    """A weight of -inf under relu closes a hidden unit for rows with a positive feature: g = -inf, h = dg = du = 0.  Of dx it enters column d
    alone (0 x inf there)."""
    import dgsparse
    T, D, F = 10, 24, 40
    x = rand(T, D, t=torch.float32, seed=1).abs() + 0.1
    wg, wu, dh = rand(F, D, t=torch.float32, seed=2), rand(F, D, t=torch.float32, seed=3), rand(T, F, t=torch.float32, seed=4)
    for f, d in ((3, 6), (8, 11), (39, 23)):
        wg[f, d] = -math.inf
    leaves = [a.requires_grad_() for a in (x, wg, wu)]
    h = dgsparse.gated_ffn(*leaves, activation='relu', recompute=False)
    assert h.isfinite().all() and h[:, [3, 8, 39]].eq(0).all()
    dx, = torch.autograd.grad(h, leaves[:1], dh)
    open_ = torch.ones(D, dtype=torch.bool, device='cuda')
    open_[[6, 11, 23]] = False
    assert dx[:, ~open_].isnan().all() and dx[:, open_].isfinite().all()


# ---- magnitudes ---------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('t', [torch.float32, torch.bfloat16], ids=ids_of)
@pytest.mark.parametrize('scale,eps', [(1e13, 1e-6), (1e15, 1e-6), (1e16, 1e-6), (1e-12, 0.0), (1e-14, 0.0), (1e-16, 0.0), (1e-14, 1e-30)])
@pytest.mark.parametrize('rows,D', [(5, 64), (9, 1000), (3, 4096), (2, 16390)])
def test_rms_norm_gradient_at_any_magnitude(rows, D, scale, eps, t):
    """s, its squares' sum and the gradient are all within the type's range (s^2 sums to at most 2e4 * 1e32, at least 64 * 1e-32)."""
    import dgsparse
    x = rand(rows, D, t=t, seed=1, scale=scale).requires_grad_()
    w = (1 + rand(D, t=torch.float32, seed=3, scale=0.1)).to(t).requires_grad_()
    dy, ds = rand(rows, D, t=t, seed=4), rand(rows, D, t=t, seed=5, scale=1 / scale)
    y, s = dgsparse.add_rms_norm(x, torch.zeros_like(x), w, eps)
    assert torch.equal(s, x)
    dx, dw = torch.autograd.grad((y, s), (x, w), (dy, ds))
    eps = torch.tensor(eps, dtype=torch.float32).double().item()  # (the entry takes a float)
    wy, wdx, mag, wdw, wmag = norm_want(s.detach(), w.detach(), eps, dy, ds)
    n = D + 16  # as at ordinary magnitudes: a mean over D, its root, some products
    within(y, wy, wy.abs() * (U(t) + n * E32) + tiny(t), 'y')
    within(dx, wdx, wdx.abs() * U(t) + 2 * n * E32 * mag + tiny(t), 'dx')
    within(dw, wdw, wdw.abs() * U(t) + (n + rows) * E32 * wmag + tiny(t), 'dw')


# ---- forward-mode derivatives ---------------------------------------------------------------------------------------------------
def test_forward_mode_derivatives_are_refused():
    """They have none: a tangent that came back empty would stand for 0."""
    import dgsparse
    x, w, m = rand(6, 16, t=torch.float32, seed=1), rand(16, t=torch.float32, seed=2), rand(8, 16, t=torch.float32, seed=3)
    ids = torch.arange(4, device='cuda')
    calls = [(x, lambda a: dgsparse.embedding(ids, a)), (x, lambda a: dgsparse.rms_norm(a, w)), (w, lambda a: dgsparse.rms_norm(x, a)),
             (x, lambda a: dgsparse.add_rms_norm(a, x, w)), (x, lambda a: dgsparse.add_rms_norm(x, a, w)), (w, lambda a: dgsparse.add_rms_norm(x, x, a)),
             (x, lambda a: dgsparse.gated_ffn(a, m, m)), (m, lambda a: dgsparse.gated_ffn(x, a, m)), (m, lambda a: dgsparse.gated_ffn(x, m, a))]
    for i, (primal, f) in enumerate(calls):
        for needs_grad in (False, True):
            with fwad.dual_level():
                dual = fwad.make_dual(primal.clone().requires_grad_(needs_grad), torch.ones_like(primal))
                with pytest.raises(RuntimeError, match='forward-mode'):
                    f(dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match='forward-mode'):
                    f(dual)
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (primal,), (torch.ones_like(primal),))
        with fwad.dual_level():  # a dual level alone is no reason
            f(primal)


# ---- rows far apart -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('t,L,D', [(torch.bfloat16, 2049, 2048), (torch.float32, 2049, 1024), (torch.float32, 2100, 1001)], ids=str)
def test_gated_ffn_of_every_sequence_s_last_token(t, L, D):
    """[batch, length, features][:, -1]: rows further apart than a tile's 32-bit offsets reach."""
    import dgsparse
    x = rand(3, L, D, t=t, seed=1)[:, -1]
    assert x.stride(0) * 256 * t.itemsize > 2 ** 31
    leaves = [a.requires_grad_() for a in (rand(40, D, t=t, seed=2, scale=D ** -0.5), rand(40, D, t=t, seed=3, scale=D ** -0.5))]
    dh = rand(3, 40, t=t, seed=4)
    outs = []
    for v in (x, x.contiguous()):
        v = v.detach().requires_grad_()
        h = dgsparse.gated_ffn(v, *leaves)
        outs.append((h,) + torch.autograd.grad(h, [v] + leaves, dh))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


@pytest.mark.parametrize('L,K', [(4097, 2048), (4400, 2000), (4300, 2001)])
def test_matmul_fp8_of_every_sequence_s_last_token(L, K):
    import dgsparse
    a, sa = dgsparse.quantize_fp8(rand(3, L, K, t=torch.bfloat16, seed=1))
    b, sb = dgsparse.quantize_fp8(rand(130, K, t=torch.float32, seed=2), 128)
    a, sa = a[:, -1], sa[:, -1]
    assert a.stride(0) * 256 > 2 ** 31
    out = check_mm8(a, sa, b, sb, torch.bfloat16)
    assert torch.equal(out, dgsparse.matmul_fp8(a.view(torch.uint8).contiguous().view(a.dtype), sa.contiguous(), b, sb, torch.bfloat16))


# ---- long lists -----------------------------------------------------------------------------------------------------------------
def test_embedding_gradient_of_more_than_2_30_positions():
    """A frequent token's partial sums are joined at the borders of chunks of 64: behind position 2^30 they are more than a launch has workgroups.
    Token 999's places, sorted, run from 2^30 - 5 to the list's end.  Whole numbers: every sum is exact."""
    import dgsparse
    n, V = 2 ** 30 + 100, 1000
    ids = torch.arange(n, dtype=torch.int32, device='cuda').remainder_(999)
    ids[torch.arange(105, device='cuda') * 10000019] = 999
    dout = torch.arange(n, dtype=torch.int32, device='cuda').remainder_(3).to(torch.float32).view(n, 1)
    table = torch.zeros(V, 1, device='cuda', requires_grad=True)
    grad, = torch.autograd.grad(dgsparse.embedding(ids, table, scale=0.5), table, dout)
    want = torch.zeros(V, dtype=torch.float64, device='cuda')
    for at in range(0, n, 1 << 27):
        want += torch.bincount(ids[at:at + (1 << 27)], weights=dout[at:at + (1 << 27), 0].double(), minlength=V)
    assert want.max() < 2 ** 24 and int((ids == 999).sum()) == 105
    assert torch.equal(grad[:, 0].double(), 0.5 * want)
