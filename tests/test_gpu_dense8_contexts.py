"""weights_laid_out on the device: calls on another stream and captured calls use weights of their own."""
import pytest
import torch

from test_gpu_dense8_paths import batch_of, pair

pytestmark = pytest.mark.gpu


@torch.no_grad()
def test_other_streams_and_graphs():
    _, m = pair(dense_inference="int8")
    batch = batch_of(400)
    want = m(batch)
    side = torch.cuda.Stream()
    graph, inside = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with m.weights_laid_out():
        assert m._weights8 is not None and torch.equal(m(batch), want)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert m._weights8 is None
            other = m(batch)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, want)
        with torch.cuda.graph(graph):
            assert m._weights8 is None
            out = m(batch)
    with torch.cuda.graph(inside):
        with m.weights_laid_out():
            assert m._weights8 is not None
            outs = [m(batch), m(batch)]
    assert m._weights8 is None
    for i in range(3):
        torch.full((1 << 22,), 7, dtype=torch.int8, device="cuda")  # over what the context held
        for p in m.parameters():
            p.mul_(1.0 - 0.01 * i)
        want = m(batch)
        for g in (graph, inside):
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(v, want) for v in (out, *outs))
