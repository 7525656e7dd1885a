"""bf16 results are the fp32 results rounded, and scales are the largest value by the fp32 number next to 1 / 127."""
import numpy as np
import pytest
import torch

from test_gpu_dense8 import dense, make, weight8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k", [(3, 5), (200, 300), (4, 5000)])
def test_rows8(rows, k):
    d = dense()
    x = make(rows, k, torch.float32, k)
    r = d.quantize_rows(x)
    assert torch.equal(r.scale.cpu(), x.abs().amax(1).cpu() * torch.tensor(np.float32(1) / np.float32(127)))
    v = r.q.float() * r.scale[:, None]
    assert torch.equal(r.restore(), v) and torch.equal(r.restore(torch.bfloat16), v.bfloat16())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("rows,n,k", [(7, 40, 300), (300, 90, 100), (300, 100, 500), (16400, 130, 200), (9000, 1000, 100)])
def test_linear8(rows, n, k, dtype):
    d = dense()
    x = make(rows, k, torch.float32 if dtype == torch.int8 else dtype, n)
    x = d.quantize_rows(x) if dtype == torch.int8 else x
    q, s = weight8(n, k, 2)
    w, b = d.pack_weight8(q.cuda(), s.cuda()), torch.randn(n, generator=torch.Generator().manual_seed(1)).cuda()
    for act in (None, "relu", "sigmoid"):
        want = d.linear8([x], [w], [b], act).bfloat16()
        assert torch.equal(d.linear8([x], [w], [b], act, out=torch.bfloat16), want)
