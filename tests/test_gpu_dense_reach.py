"""The dense operators where values and calls are out of the ordinary."""
import math

import pytest
import torch

from test_gpu_dense import TYPES, ids_of, rand

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
