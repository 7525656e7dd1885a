"""How the 8-bit dense layers take their inputs' layouts, without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("rows", [0, 1, 2])
def test_rows_far_apart_are_copied_whatever_their_number(rows):
    import dense
    far = (1 << 21) + 8
    base = torch.arange(float(far + 8))
    x = base.as_strided((rows, 8), (far, 1))
    near = dense._near(x)
    assert near.shape == x.shape and near.stride() == (8, 1) and torch.equal(near, x)
    kept = base.as_strided((rows, 8), ((1 << 21) - 1, 1))
    assert dense._near(kept) is kept
    x.requires_grad_()
    near = dense._near(x)
    assert torch.equal(torch.autograd.grad(near, x, torch.ones_like(near))[0], torch.ones(rows, 8))


def test_dual_tensors_are_told_apart():
    import dense
    from torch.autograd import forward_ad
    x = torch.ones(2, 3)
    assert not dense._has_tangent(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert not dense._has_tangent(x) and dense._has_tangent(dual)
        with torch.no_grad():
            assert dense._has_tangent(dual) and dense._has_tangent(dual[:, 1:].t())
        assert not dense._has_tangent(forward_ad.unpack_dual(dual).primal)
