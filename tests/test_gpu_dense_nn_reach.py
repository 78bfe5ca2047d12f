"""The layers on the dense operators between calls: weights that are loaded, types that are changed."""
import pytest
import torch

from test_gpu_dense_nn import graph, leaves

pytestmark = pytest.mark.gpu


def test_residual_gcn_in_8_bits_takes_a_loaded_weight_in_place():
    """Behind load_state_dict the layer answers with the new weight, called and in a graph that was captured before."""
    from dgsparse import nn as dnn
    ei, n = graph(seed=4)
    torch.manual_seed(2)
    block, other = dnn.ResidualGCN(160, 200).cuda().quantize(), dnn.ResidualGCN(160, 200).cuda().quantize()
    dcsr = dnn.get_gcn_dcsr_from_edge_index(ei, n)
    x, r = (v.detach() for v in leaves((n, 160), (n, 160), seed=5))
    want, first = other(dcsr, x, r)[0], block(dcsr, x, r)[0]
    assert not torch.equal(want, first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(dcsr, x, r)
    torch.cuda.current_stream().wait_stream(side)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        out = block(dcsr, x, r)[0]
    captured.replay()
    assert torch.equal(out, first)
    held = block.conv8.weight
    block.load_state_dict(other.state_dict())
    assert block.conv8.weight is held
    for _ in range(3):
        assert torch.equal(block(dcsr, x, r)[0], want)
        captured.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_linear_fp8_in_a_module_of_another_type():
    from dgsparse import nn as dnn
    a = torch.randn(5, 200, device='cuda')
    lin = dnn.LinearFP8(torch.randn(30, 200, device='cuda'), torch.float16)
    want = lin(a)
    for change in (lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.cpu().cuda()):
        assert torch.equal(change(lin)(a), want)
    assert lin(a.half()).dtype == torch.float16
