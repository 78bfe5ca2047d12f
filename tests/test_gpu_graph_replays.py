"""Captured products replayed again and again with new inputs, the program's own eager calls and synchronizations in between: every replay clears what it
counts with (unit and long-row counters, barrier counters, the scattered gradients) as the first one did."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def captured(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


def replay_and_compare(step, inputs, exact):
    graph, out = captured(step)
    for k in range(5):
        for x in inputs:
            x.copy_(torch.randint(-8, 9, x.shape, device='cuda') / 8)
        if k % 2:
            torch.cuda.synchronize()
        eager = [v.clone() for v in step()]
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(out, eager)):
            if exact[i]:
                assert torch.equal(a, b), (k, i)
            else:  # fp32 atomics: sums of multiples of 2^-9, exact in whatever order below 2^15
                assert torch.equal(a, b) or (a - b).abs().max() <= 1e-5 * b.abs().max(), (k, i)


@pytest.fixture
def matrix():
    from bench import graphgen
    rp, col, st = graphgen.powerlaw_csr(40000, 700000, alpha=1.9, dmax=9000, seed=3)
    rp, col = torch.from_numpy(rp).cuda(), torch.from_numpy(col).cuda()
    val = (torch.randint(1, 9, (st['nnz'] if 'nnz' in st else col.numel(),), device='cuda') / 8)
    return rp, col, val, rp.numel() - 1, int(st['K'])


def test_products_of_every_kind(matrix):
    from dgsparse import _capi as c
    rp, col, val, M, K = matrix
    X = torch.empty(K, 64, device='cuda')
    plan = c.spmm_plan(rp, col, K, 64, force=True)

    def step():
        out = []
        for op in (c.SUM, c.MEAN, c.MAX, c.MIN):
            for p in (None, plan):
                C, E = c.spmm(op, rp, col, val, X, plan=p)
                out += [C] + ([E] if op in (c.MAX, c.MIN) else [])
        out.append(c.spmm(c.SUM, rp, col, val, X, algorithm=c.ALG_STRICT_SUM)[0])
        return out

    X.normal_()
    n = len(step())
    replay_and_compare(step, [X], [True] * n)


def test_backward_products(matrix):
    from dgsparse import _capi as c
    rp, col, val, M, K = matrix
    X, G = torch.randn(K, 32, device='cuda'), torch.randn(M, 32, device='cuda')
    colptr, row, tval, _ = c.csr2csc(rp, col, val, K)

    def step():
        _, E = c.spmm(c.MAX, rp, col, val, X)
        gX, gW = c.spmm_arg_backward(rp, col, val, E, G, X)
        return [c.spmm_mask(colptr, row, tval, G, E), c.sddmm(rp, col, G, X), c.sddmm(rp, col, G, X, E=E), gX, gW]

    replay_and_compare(step, [X, G], [True, True, True, False, False])


def test_panel_schedules(monkeypatch):
    from bench import graphgen
    from dgsparse import _capi as c
    monkeypatch.setenv('DGS_PANEL', '1')
    monkeypatch.setenv('DGS_PANEL_KB', '64')
    monkeypatch.setenv('DGS_PANEL_TLONG', '512')
    rp, col, st = graphgen.dataset_shaped('arxiv', seed=1, device='cuda', as_torch=True)
    assert c.spmm_schedule(c.SUM, st['M'], st['K'], 64, st['nnz']) == 'panel'
    val = torch.randint(1, 9, (st['nnz'],), device='cuda') / 8
    X, D1 = torch.randn(st['K'], 64, device='cuda'), torch.randn(st['M'], 64, device='cuda')

    def step():
        C, E = c.spmm(c.MAX, rp, col, val, X)
        return [C, E, c.spmm(c.SUM, rp, col, val, X)[0], c.sddmm(rp, col, D1, X)]

    replay_and_compare(step, [X, D1], [True] * 4)


def test_autograd_of_the_public_product(matrix):
    import dgsparse
    rp, col, val, M, K = matrix
    A = dgsparse.SparseTensor(rowptr=rp, col=col, values=val.clone().requires_grad_(), has_value=True)
    X, G = torch.randn(K, 48, device='cuda', requires_grad=True), torch.randn(M, 48, device='cuda')
    leaf = A.storage._values if hasattr(A.storage, '_values') else None
    src = X.detach()

    def step():
        out = dgsparse.spmm_sum(A, X, 0)
        return [out.detach()] + list(torch.autograd.grad(out, [X] + ([leaf] if leaf is not None and leaf.requires_grad else []), G))

    n = len(step())
    replay_and_compare(step, [src, G], [True] * n)
