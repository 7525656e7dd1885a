"""The checkpointed layer on inputs and gradients of unusual layout, against the same values laid out plainly."""
import pytest
import torch

from test_gpu_dense8 import dense, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [0, 1, 2])
@pytest.mark.parametrize("act", [None, "relu", "sigmoid"])
def test_rows_far_apart(rows, act):
    """Rows 2^21 values apart and more, one or none of them as well, of x and of the gradient."""
    d = dense()
    far = (1 << 21) + 9
    near_x, near_dy = make(rows, 50, torch.float32, 1), make(rows, 20, torch.float32, 3)
    w = torch.randn((20, 50), generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    x = torch.zeros(2 * far, device="cuda").as_strided((rows, 50), (far, 1), 7).copy_(near_x).requires_grad_()
    dy = torch.zeros(2 * far, device="cuda").as_strided((rows, 20), (far, 1), 3).copy_(near_dy)
    near_x.requires_grad_()
    got = d.linear([(x, 0, 0)], [w], [], act, checkpoint="int8")
    want = d.linear([(near_x, 0, 0)], [w], [], act, checkpoint="int8")
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, [x, w], dy), torch.autograd.grad(want, [near_x, w], near_dy)):
        assert torch.equal(a, b)
