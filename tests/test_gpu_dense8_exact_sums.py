"""The checkpointed layer's sums over many rows, by equality: a lost, doubled or misplaced part of the rows shows.

x holds whole multiples of 1/128 below one, 127/128 in each row's first column, so that its 8 bits are exact; dy whole
numbers up to 2.  A sum over 33,001 rows is a multiple of 1/128 below 33,001 * 2 * 127 / 128, 2^23 steps: exact in fp32 in
any order.  Weights are multiples of 2^-5 up to 1, so that outputs (up to 300 products, multiples of 2^-12) and dx
are exact too, and each ReLU's border is known.  A sigmoid of zero weights and biases is 1/2, its slope 1/4."""
import pytest
import torch

from test_gpu_dense8 import dense

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [None, "relu", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,widths", [(33000, 130, (1,)), (32769, 256, (256,)), (33001, 66, (300,)), (4099, 3, (64,)),
                                           (33000, 3, (256,)), (16385, 200, (40, 257)), (70, 40, (30,)), (31, 5, (7,))])
def test_sums_are_exact(rows, n, widths, dtype, act):
    d = dense()
    g = torch.Generator().manual_seed(rows + n)
    xs, ws, bs = [], [], []
    for k in widths:
        x = torch.randint(-127, 128, (rows, k), generator=g).float() / 128
        x[:, 0] = torch.where(x[:, 0] < 0, -127 / 128, 127 / 128)
        xs.append(x.to(dtype).cuda().requires_grad_())
        w, b = torch.randint(-32, 33, (n, k), generator=g) / 32.0, torch.randint(-32, 33, (n,), generator=g) / 32.0
        ws.append((w * (act != "sigmoid")).cuda().requires_grad_())
        bs.append((b * (act != "sigmoid")).cuda().requires_grad_())
    dy = torch.randint(-2, 3, (rows, n), generator=g).float().cuda()
    y = d.linear([(x, i, 0) for i, x in enumerate(xs)], ws, bs, act, checkpoint="int8")
    grads = [t.cpu().double() for t in torch.autograd.grad(y, [*xs, *ws, *bs], dy)]
    x64, w64 = [[t.detach().cpu().double() for t in ts] for ts in (xs, ws)]
    z = sum(x @ w.t() for x, w in zip(x64, w64)) + sum(b.detach().cpu().double() for b in bs)
    dz = dy.cpu().double()
    if act == "relu":
        assert torch.equal(y.detach().cpu().double(), z.clamp_min(0))
        dz = dz * (z > 0)
    elif act == "sigmoid":
        assert (y == 0.5).all()
        dz = dz / 4
    else:
        assert torch.equal(y.detach().cpu().double(), z)
    m = len(widths)
    for x, w, dx, dw, db in zip(x64, w64, grads[:m], grads[m:2 * m], grads[2 * m:]):
        assert torch.equal(dx, (dz @ w).to(dtype).double())
        assert torch.equal(dw, dz.t() @ x) and torch.equal(db, dz.sum(0))


@pytest.mark.parametrize("rows", [1, 33000])
def test_bias_gradient_alone(rows):
    """Frozen weights: db by a kernel of its own."""
    d = dense()
    g = torch.Generator().manual_seed(rows)
    x, w = torch.randint(-127, 128, (rows, 20), generator=g) / 128.0, torch.randint(-32, 33, (70, 20), generator=g) / 32.0
    b = torch.zeros(70, device="cuda", requires_grad=True)
    dy = torch.randint(-2, 3, (rows, 70), generator=g).float()
    y = d.linear([(x.cuda(), 0, 0)], [w.cuda()], [b], "relu", checkpoint="int8")
    dz = dy * (x.double() @ w.double().t() > 0)
    assert torch.equal(torch.autograd.grad(y, b, dy.cuda())[0].cpu().double(), dz.double().sum(0))
