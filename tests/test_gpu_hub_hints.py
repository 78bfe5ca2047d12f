"""What Storage tells the launches about its longest row and column, with a threshold that the library takes (DGS_HUB_CHAIN is clamped to 1024 and
above): hints while no row is a hub row, none for the rows once one is, the same bits either way."""
import numpy as np
import pytest
import torch

from util import assert_close

pytestmark = pytest.mark.gpu


def test_storage_drops_the_row_hint_when_a_row_becomes_a_hub_row(monkeypatch):
    import dgsparse
    import oracle
    from dgsparse import _capi
    monkeypatch.delenv('DGS_HUB_CHAIN', raising=False)
    rng = np.random.default_rng(9)
    M = K = 6000
    deg = rng.integers(0, 10, M)
    deg[17], deg[4000] = 1300, 78
    rp = np.zeros(M + 1, np.int32)
    rp[1:] = np.cumsum(deg)
    col = np.concatenate([np.sort(rng.choice(K, d, replace=False)) for d in deg]).astype(np.int32)
    col[-1] = K - 1
    val = rng.random(col.size, dtype=np.float32)
    drp, dcol, dval = (torch.from_numpy(a).cuda() for a in (rp, col, val))
    A = dgsparse.SparseTensor(rowptr=drp, col=dcol, values=dval, has_value=True)
    st = A.storage
    assert st._max_row_len == 1300
    torch.cuda.synchronize()
    both = _capi.ALG_NO_HUB_ROWS | _capi.ALG_NO_HUB_COLS
    assert st.hub_hints() == both and st._hints == (16384, both)
    assert st._max_col_len == int(np.bincount(col, minlength=K).max()) < 1024
    X = torch.rand((K, 64), device='cuda', requires_grad=True)
    out = dgsparse.spmm_sum(A, X, 0)
    plain, _ = _capi.spmm(_capi.SUM, drp, dcol, dval, X.detach())
    assert torch.equal(out.detach(), plain)
    G = torch.rand_like(out)
    out.backward(G)
    colptr, row, tval, _ = oracle.csr2csc(rp, col, val, K)
    gX, _ = oracle.spmm('sum', colptr, row, tval, G.cpu().numpy(), fma=True)
    assert_close(X.grad.cpu().numpy(), gX, 1e-5, 2e-6, 'dX with the column hint')
    monkeypatch.setenv('DGS_HUB_CHAIN', '1024')  # row 17 is a hub row now; no column is one
    bits = st.hub_hints()
    assert not bits & _capi.ALG_NO_HUB_ROWS and bits & _capi.ALG_NO_HUB_COLS
    out2 = dgsparse.spmm_sum(A, X.detach(), 0)
    ref, _ = oracle.spmm('sum', rp, col, val, X.detach().cpu().numpy(), fma=True)
    assert np.array_equal(out2.cpu().numpy()[17].view(np.int32), ref[17].view(np.int32)), 'the hub row is chained'
    assert_close(out2.cpu().numpy(), ref, 1e-5, 2e-6, 'the other rows')
