"""The layers on the dense operators against the functions they are made of (bit for bit: each function has its own test against 64 bits), and
what the operators refuse when they are given GPU tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def graph(n=300, e=2500, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.unique(torch.randint(0, n, (2, e), generator=g), dim=1).cuda(), n


def leaves(*shapes, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return [torch.randn(*s, generator=g, device='cuda').requires_grad_() for s in shapes]


def test_residual_gcn_is_its_parts_forward_and_backward():
    import dgsparse
    from dgsparse import nn as dnn
    ei, n = graph()
    torch.manual_seed(1)
    block = dnn.ResidualGCN(32, 72, activation='gelu').cuda()
    dcsr = dnn.get_gcn_dcsr_from_edge_index(ei, n)
    x, r = leaves((n, 32), (n, 32), seed=2)
    do, dr = (v.detach() for v in leaves((n, 32), (n, 32), seed=3))
    out, s2 = block(dcsr, x, r)
    params = list(block.parameters())
    got = torch.autograd.grad((out, s2), [x, r] + params, (do, dr))
    # the same by hand, its backward pass too
    y1, s1 = dgsparse.add_rms_norm(x, r, block.norm1.weight, 1e-6)
    m = dnn.spmm_sum_fused(dcsr, block.conv.W(y1), relu=True)
    y2, s = dgsparse.add_rms_norm(m, s1, block.norm2.weight, 1e-6)
    want_out = torch.nn.functional.linear(dgsparse.gated_ffn(y2, block.ffn.w_gate, block.ffn.w_up, 'gelu'), block.ffn.down.weight)
    want = torch.autograd.grad((want_out, s), [x, r] + params, (do, dr))
    assert torch.equal(s2, s) and torch.equal(out, want_out)
    for a, b, name in zip(got, want, ['x', 'residual'] + [n for n, _ in block.named_parameters()]):
        assert torch.equal(a, b) and torch.isfinite(a).all(), name


def test_residual_gcn_in_8_bits():
    import dgsparse
    from dgsparse import nn as dnn
    ei, n = graph(seed=4)
    torch.manual_seed(2)
    block = dnn.ResidualGCN(160, 200).cuda()
    dcsr = dnn.get_gcn_dcsr_from_edge_index(ei, n)
    x, r = (v.detach() for v in leaves((n, 160), (n, 160), seed=5))
    full, s_full = block.eval()(dcsr, x, r)
    out, s2 = block.quantize()(dcsr, x, r)
    q, scale, s1 = dgsparse.add_rms_norm_fp8(x, r, block.norm1.weight)
    w8, ws = dgsparse.quantize_fp8(block.conv.W.weight, 128)
    m = dnn.spmm_sum_fused(dcsr, dgsparse.matmul_fp8(q, scale, w8, ws, torch.float32), relu=True)
    y, s = dgsparse.add_rms_norm(m, s1, block.norm2.weight)
    assert torch.equal(s2, s) and torch.equal(out, block.ffn(y)) and not out.requires_grad
    # both factors off by at most 2^-4 of themselves: the sum of the residual differs by less than that of its parts
    assert (s2 - s_full).norm() <= 2.0 ** -3 * (s_full - (x + r)).norm()
    assert block.train()(dcsr, x, r)[0].requires_grad  # training goes on in full precision


def test_gin_update_and_embedding_layers():
    import dgsparse
    from dgsparse import nn as dnn
    ei, n = graph(seed=6)
    torch.manual_seed(3)
    emb = dnn.Embedding(50, 24, padding_idx=7, scale=2.0).cuda()
    conv = dnn.GINConv(apply_func=dnn.GatedFFN(24, 40, 10, activation='silu'), aggregator_type='sum').cuda()
    ids = torch.randint(-1, 50, (n,), device='cuda')
    ids[0] = 7
    h = emb(ids)
    assert torch.equal(h, dgsparse.embedding(ids, emb.weight, 2.0, 7)) and h[0].eq(0).all()
    out = conv(ei, h, n)
    assert out.shape == (n, 10)
    out.square().sum().backward()
    assert emb.weight.grad[7].eq(0).all() and emb.weight.grad.isfinite().all() and emb.weight.grad.ne(0).any()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in conv.parameters() if p.requires_grad)
    lin = dnn.LinearFP8(torch.randn(30, 24, device='cuda'), torch.float16)
    a = torch.randn(5, 24, device='cuda')
    assert torch.equal(lin(a), lin(dgsparse.quantize_fp8(a))) and lin(a).dtype == torch.float16


def test_what_the_operators_refuse_on_the_gpu():
    import dgsparse
    x, w, ids = torch.rand(4, 8, device='cuda'), torch.rand(8, device='cuda'), torch.zeros(3, dtype=torch.long, device='cuda')
    f8, s = dgsparse.quantize_fp8(x)
    b8, bs = dgsparse.quantize_fp8(x, 128)
    cases = {
        'int32 or int64': lambda: dgsparse.embedding(ids.float(), x),
        'table must be': lambda: dgsparse.embedding(ids, w),
        'float32, float16 or bfloat16': lambda: dgsparse.embedding(ids, x.double()),
        'no CPU fallback': lambda: dgsparse.embedding(ids.cpu(), x),
        'residual must have the shape': lambda: dgsparse.add_rms_norm(x, x[:1], w),
        'weight must be \\[8\\]': lambda: dgsparse.rms_norm(x, w[:7]),
        'weight must have the type': lambda: dgsparse.rms_norm(x, w.half()),
        'residual must have the type': lambda: dgsparse.add_rms_norm(x, x.half(), w),
        'eps must not be negative': lambda: dgsparse.rms_norm(x, w, -1e-3),
        'at least one feature': lambda: dgsparse.rms_norm(x[:, :0], w[:0]),
        'w_gate must be': lambda: dgsparse.gated_ffn(x, x[:, :4], x[:, :4]),
        'w_up must have the shape': lambda: dgsparse.gated_ffn(x, x, x[:2]),
        'w_up must have the type': lambda: dgsparse.gated_ffn(x, x, x.bfloat16()),
        'block_rows is 1, or 128': lambda: dgsparse.quantize_fp8(x[None], 128),
        'must be float8_e4m3fn': lambda: dgsparse.matmul_fp8(x, s, b8, bs),
        'scales must be float32': lambda: dgsparse.matmul_fp8(f8, s.half(), b8, bs),
        'a must be': lambda: dgsparse.matmul_fp8(f8[:, :4], s, b8, bs),
        'a_scale must be': lambda: dgsparse.matmul_fp8(f8, s[:3], b8, bs),
        'b_scale must be': lambda: dgsparse.matmul_fp8(f8, s, b8, bs.expand(2, 1)),
        'the result must be': lambda: dgsparse.matmul_fp8(f8, s, b8, bs, torch.float64),
    }
    for match, call in cases.items():
        with pytest.raises(RuntimeError, match=match):
            call()
    # a saved operand that is overwritten before the backward pass is noticed
    a, g = torch.rand(70, 8, device='cuda', requires_grad=True), torch.rand(8, 8, device='cuda')
    h = dgsparse.gated_ffn(a, g, g)
    g.add_(1)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        h.sum().backward()
