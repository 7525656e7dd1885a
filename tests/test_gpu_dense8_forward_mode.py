"""Forward-mode differentiation through the 8-bit dense layers is refused, not silently without its tangent."""
import pytest
import torch
from torch.autograd import forward_ad

from test_gpu_dense8 import dense, make
from test_gpu_dense8_paths import batch_of, pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("recorded", [True, False])
def test_dual_tensors_are_refused(recorded):
    d = dense()
    x, w, b = make(8, 16, torch.float32), make(4, 16, torch.float32, 1), torch.zeros(4).cuda()
    w8 = d.quantize_weight(w)
    want = d.linear8([x], [w8], [b])
    with torch.set_grad_enabled(recorded), forward_ad.dual_level():
        dx, dw, db = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w, b))
        for call in (lambda: d.linear8([dx], [w8], [b]), lambda: d.linear8([x], [w8], [db]),
                     lambda: d.linear8([d.quantize_rows(x), dx], [w8, w8], [b], out=torch.int8),
                     lambda: d.quantize_rows(dx), lambda: d.quantize_weight(dw),
                     lambda: d.linear([(dx, 0, 0)], [w], [b], None, checkpoint="int8"),
                     lambda: d.linear([(x, 0, 0)], [dw], [b], None, checkpoint="int8")):
            with pytest.raises(RuntimeError):  # (NotImplementedError of a Function without one is one too)
                call()
        # tensors without a tangent are taken, in a dual level as well
        assert torch.equal(d.linear8([x], [w8], [b]), want)
        assert torch.equal(d.linear8([forward_ad.unpack_dual(dx).primal], [w8], [b]), want)


@torch.no_grad()
def test_the_field_refuses_them():
    _, m = pair(dense_inference="int8")
    batch = batch_of(20)
    with forward_ad.dual_level():
        f = batch["eigenfunctions"]
        with pytest.raises(RuntimeError):
            m({**batch, "eigenfunctions": forward_ad.make_dual(f, torch.ones_like(f))})
