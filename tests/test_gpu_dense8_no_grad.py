"""The checkpointed layer where no gradient is recorded keeps nothing, and gives the same results."""
import pytest
import torch

from test_gpu_dense8 import dense, leaves, make
from test_gpu_dense8_paths import batch_of, pair

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [None, "relu", "sigmoid"])
@pytest.mark.parametrize("rows", [100, 40000])
def test_nothing_is_made_under_no_grad(rows, act):
    """What a call takes: its output and the workspace of its products, no 8-bit rows and no mask."""
    from inf_hip import lib
    d = dense()
    n, k = 96, 1024
    xs, ws, bs, _ = leaves(rows, n, (k,), torch.float32, 1)

    def call():
        return d.linear([(xs[0], 0, 0)], ws, bs, act, checkpoint="int8")

    want = call().detach()
    with torch.no_grad():
        call()
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        base = torch.cuda.memory_stats()["requested_bytes.all.current"]  # as asked for, without the allocator's rounding
        y = call()
        torch.cuda.synchronize()
        peak = torch.cuda.memory_stats()["requested_bytes.all.peak"] - base
    work = lib.inf_linear_ckpt_workspace_bytes(rows, n, k, 0, 0)
    assert torch.equal(y, want) and not y.requires_grad
    assert peak == rows * n * 4 + work


def test_field_and_rows_made_before():
    _, m = pair(dense_checkpoints="int8")
    batch = batch_of(500)
    want = m(batch).detach()
    with torch.no_grad():
        assert torch.equal(m(batch), want)
    # rows given, with gradients recorded or not; then a gradient as always
    d = dense()
    x = make(64, 48, torch.float32, 9)
    r, w = d.quantize_rows(x), make(32, 48, torch.float32, 1).requires_grad_()
    y = d.linear([(x, 0, 0)], [w], [], "relu", checkpoint=[r])
    with torch.no_grad():
        assert torch.equal(d.linear([(x, 0, 0)], [w], [], "relu", checkpoint=[r]), y)
    dy = make(64, 32, torch.float32, 2)
    z = d.linear([(x, 0, 0)], [w], [], "relu", checkpoint="int8")
    assert torch.equal(torch.autograd.grad(y, w, dy)[0], torch.autograd.grad(z, w, dy)[0])
