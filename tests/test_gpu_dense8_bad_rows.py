"""Rows with an infinity or a NaN: NaN in all of that row's results, and in no other row's."""
import pytest
import torch

from test_gpu_dense8 import dense, leaves

pytestmark = pytest.mark.gpu

BAD = (float("inf"), -float("inf"), float("nan"))


@pytest.mark.parametrize("act", [None, "relu", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(40, 3, 30), (200, 40, 33), (16500, 200, 70), (65300, 130, 33)])
def test_checkpointed_layer(rows, n, k, dtype, act):
    d = dense()
    xs, ws, bs, dy = leaves(rows, n, (k,), dtype, n)
    x = xs[0].detach().clone()
    fine = d.linear([(x, 0, 0)], ws, bs, act, checkpoint="int8").detach()
    at = torch.tensor([0, 9, 11, 17, 18, rows - 1])
    for i, m in enumerate(at):
        x[m, (7 * i) % k] = BAD[i % 3]
    with torch.no_grad():
        ws[0][: n // 3 + 1].abs_()  # (weights of one sign, and of both)
        want = d.linear([(xs[0], 0, 0)], ws, bs, act, checkpoint="int8")
    y = d.linear([(x, 0, 0)], ws, bs, act, checkpoint="int8")
    others = torch.ones(rows, dtype=torch.bool)
    others[at] = False
    assert torch.isnan(y[at.cuda()]).all() and torch.equal(y[others.cuda()], want[others.cuda()])
    assert fine.isfinite().all()
    # what those rows give the weight's gradient is NaN as well; a gradient next to them is its own
    g = torch.autograd.grad(y, ws[0], dy)[0]
    assert torch.isnan(g).all()
    # the same rows made before, of another call
    y2 = d.linear([(x, 0, 0)], ws, bs, act, checkpoint=[d.quantize_rows(x)])
    assert torch.equal(torch.isnan(y2), torch.isnan(y)) and torch.equal(y2[others.cuda()], y[others.cuda()])
