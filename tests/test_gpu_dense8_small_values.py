"""The checkpointed layer where values come near the end of fp32's range.

dW: dz s is rounded once (2^-24 of it, 2^-150 where it is subnormal) and cut into three bf16 pieces, whose subnormals
end at 2^-133: a term is off by less than (2^-133 + 2^-150) |q|, below 2^-126 and a millionth, beside the bound of
test_gpu_dense8.  The result is rounded to at most 2^-150.  y and dx: rows are scaled by powers of two, so
that their own size costs nothing but the result's rounding, 2^-150 a part; a row of x of scale 0 is a row of zeros."""
import pytest
import torch

from test_gpu_dense8 import U32, dense, far_below, rows64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("exponent", [-90, -105, -110, -115, -120, -126, -132, -140, -148])
def test_small_gradients(exponent):
    d = dense()
    rows, n, k = 256, 64, 70
    g = torch.Generator().manual_seed(exponent)
    x, w = torch.randn((rows, k), generator=g).cuda().requires_grad_(), torch.randn((n, k), generator=g).cuda().requires_grad_()
    dy = (torch.randn((rows, n), generator=g).double() * 2.0 ** exponent).float().cuda()
    y = d.linear([(x, 0, 0)], [w], [], None, checkpoint="int8")
    dx, dw = (t.cpu().double() for t in torch.autograd.grad(y, [x, w], dy))
    q, s = rows64(x.detach())
    dz, v = dy.cpu().double(), q * s[:, None]
    lim = (3 * rows + 8) * U32 * (dz.abs().t() @ v.abs()) + 2.0 ** -133 * (1 + 1e-4) * q.abs().sum(0)[None] + 2.0 ** -149
    assert ((dw - dz.t() @ v).abs() <= lim).all()
    w64 = w.detach().cpu().double()
    lim = (3 * n + 8) * U32 * (dz.abs() @ w64.abs()) + far_below(dz, w64) + 2.0 ** -149
    assert ((dx - dz @ w64).abs() <= lim).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("exponent", [-100, -120, -126, -132, -136, -143, -148])
def test_small_inputs(exponent, dtype):
    d = dense()
    rows, n, k = 200, 40, 30
    g = torch.Generator().manual_seed(exponent)
    x = (torch.randn((rows, k), generator=g).double() * 2.0 ** exponent).to(dtype).cuda()
    w = (torch.randn((n, k), generator=g) * 2.0 ** 10).cuda()
    y = d.linear([(x, 0, 0)], [w], [], None, checkpoint="int8").cpu().double()
    r = d.quantize_rows(x)
    top = x.abs().amax(1).cpu().double()
    gone = top < 2.0 ** -143
    assert torch.equal(r.scale.cpu() == 0, gone)
    x64, w64 = x.cpu().double() * ~gone[:, None], w.cpu().double()
    lim = (3 * k + 8) * U32 * (x64.abs() @ w64.abs().t()) + far_below(x64, w64.t()) + 2.0 ** -149
    assert ((y - x64 @ w64.t()).abs() <= lim).all()
