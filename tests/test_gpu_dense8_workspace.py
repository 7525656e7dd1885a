"""What a linear8 call takes of the device's memory: its result, and a workspace only where its kernel has one."""
import pytest
import torch

from test_gpu_dense8 import dense, make, weight8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,k,act,out,workspace", [
    (256, 256, "relu", torch.bfloat16, False), (100, 64, None, torch.float32, False), (64, 256, "relu", torch.int8, False),
    (256, 700, "relu", torch.float32, False), (256, 256, "sigmoid", torch.float32, True), (3, 256, None, torch.float32, True)])
def test_peak(n, k, act, out, workspace, dtype):
    d = dense()
    rows = 20000
    x = make(rows, k, dtype)
    q, s = weight8(n, k, 1)
    w, b = d.pack_weight8(q.cuda(), s.cuda()), torch.zeros(n, device="cuda")
    d.linear8([x], [w], [b], act, out=out)
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_stats()["requested_bytes.all.current"]
    y = d.linear8([x], [w], [b], act, out=out)
    peak = torch.cuda.memory_stats()["requested_bytes.all.peak"] - base
    ld = (n + 15) // 16 * 16
    result = rows * ld + 128 + rows * 4 if out == torch.int8 else rows * n * out.itemsize
    q8 = -(-(rows * ((k + 15) // 16 * 16) + 128) // 256) * 256 + -(-rows * 4 // 256) * 256
    assert y.shape == (rows, n) and peak == result + (q8 if workspace else 0)
