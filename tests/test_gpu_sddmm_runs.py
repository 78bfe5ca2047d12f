"""SDDMM over the plan (csrc/sddmm_fused.h) where the runs of short rows between long ones hold fewer entries than a wave has groups, or end in the
middle of a batch: a group without an entry of its own makes the wave's batches all the same and stores nothing."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('F', [32, 36, 64, 128, 256])
@pytest.mark.parametrize('mean', [False, True])
def test_sddmm_over_the_plan_on_runs_of_every_length(F, mean, monkeypatch):
    from dgsparse import _capi as capi
    monkeypatch.setenv('DGS_SDDMM_FUSED', '1')
    rng = np.random.default_rng(F)
    # runs of 0 .. 70 entries (rows of 0 .. 3), each ended by a row that the units take
    deg = []
    for total in list(range(71)) * 140:
        while total > 0:
            deg.append(min(total, int(rng.integers(0, 4))))
            total -= deg[-1]
        deg.append(int(rng.integers(65, 90)))
    deg = np.array(deg)
    M, K = deg.size, 1000
    rp = np.concatenate([[0], np.cumsum(deg)]).astype(np.int32)
    col = rng.integers(0, K, rp[-1]).astype(np.int32)
    D1, D2 = rng.random((M, F), dtype=np.float32), rng.random((K, F), dtype=np.float32)
    rpt, colt, d1, d2 = (torch.from_numpy(a).cuda() for a in (rp, col, D1, D2))
    plan = capi.spmm_plan(rpt, colt, K, F, force=True)
    assert plan is not None
    got = capi.sddmm(rpt, colt, d1, d2, reduce_op=capi.MEAN if mean else capi.SUM, plan=plan)
    row = torch.repeat_interleave(torch.arange(M, device='cuda'), torch.from_numpy(deg).cuda())
    want = torch.empty(rp[-1], dtype=torch.float64, device='cuda')
    for at in range(0, rp[-1], 1 << 18):
        want[at:at + (1 << 18)] = (d1[row[at:at + (1 << 18)]].double() * d2[colt[at:at + (1 << 18)].long()].double()).sum(1)
    if mean:
        want /= torch.from_numpy(deg).cuda()[row]
    # F products and additions of positive terms (and a division) in 32 bits
    assert ((got.double() - want).abs() <= (F + 2) * 2.0 ** -24 * want).all()
