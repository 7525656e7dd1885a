"""linear(..., checkpoint="int8", products="fp32"): the layer without a checkpoint, bit for bit, but for dW.

dW = dz^T (s q) from the same dz; its bound is that of test_gpu_dense8."""
import pytest
import torch

from test_gpu_dense8 import U32, dense, leaves, make, near, rows64
from test_gpu_dense8_paths import batch_of, pair

pytestmark = pytest.mark.gpu

ACTS = [None, "relu", "sigmoid"]


def dz64(y, dy, act):
    y, dy = y.detach().cpu().double(), dy.cpu().double()
    return dy * (y > 0) if act == "relu" else dy * y * (1 - y) if act == "sigmoid" else dy


def check_dw(got, x, y, dy, act):
    q, s = rows64(x.detach())
    v, dz = q * s[:, None], dz64(y, dy, act)
    # dz of a sigmoid: three roundings of dy y (1 - y)
    near(got, (dz.t() @ v, (3 * len(dz) + 12) * U32 * (dz.abs().t() @ v.abs())))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,widths", [(0, 40, (30,)), (1, 1, (1,)), (3, 33, (31,)), (65, 64, (63,)), (300, 256, (1023,)),
                                           (129, 257, (100, 40)), (5000, 3, (256,)), (33000, 65, (20,))])
def test_all_but_dw_bit_for_bit(rows, n, widths, dtype, act):
    d = dense()
    xs, ws, bs, dy = leaves(rows, n, widths, dtype, rows + n)
    segments = [(x, i, 0) for i, x in enumerate(xs)]
    plain = d.linear(segments, ws, bs, act)
    kept = d.linear(segments, ws, bs, act, checkpoint="int8", products="fp32")
    assert torch.equal(plain, kept)
    m = len(widths)
    want = torch.autograd.grad(plain, [*xs, *ws, *bs], dy)
    got = torch.autograd.grad(kept, [*xs, *ws, *bs], dy)
    for a, b in zip(want[:m] + want[2 * m:], got[:m] + got[2 * m:]):
        assert a.dtype == b.dtype and torch.equal(a, b)
    for x, g in zip(xs, got[m:2 * m]):
        if rows:
            check_dw(g, x, kept, dy, act)
        else:
            assert (g == 0).all()
    with torch.no_grad():
        assert torch.equal(d.linear(segments, ws, bs, act, checkpoint="int8", products="fp32"), plain)


def test_layouts_and_parts():
    """Column ranges of one weight, columns that no segment takes, strided and repeated inputs, gradients of some inputs
    only, rows made before, fewer biases than segments."""
    d = dense()
    g = torch.Generator().manual_seed(6)
    W = (torch.randn((40, 120), generator=g) * 0.1).cuda().requires_grad_()
    b = torch.randn(40, generator=g).cuda().requires_grad_()
    a, c = make(90, 50, torch.float32, 1, 0.3).requires_grad_(), make(90, 30, torch.float32, 2, 0.3).requires_grad_()
    dy = torch.randn((90, 40), generator=g).cuda()
    segments = [(a, 0, 0), (c, 0, 70)]
    for act in ACTS:
        for kept in ("int8", [d.quantize_rows(a), "int8"]):
            y = d.linear(segments, [W], [b], act, checkpoint=kept, products="fp32")
            plain = d.linear(segments, [W], [b], act)
            assert torch.equal(y, plain)
            want = torch.autograd.grad(plain, [a, c, W, b], dy)
            got = torch.autograd.grad(y, [a, c, W, b], dy)
            assert all(torch.equal(got[i], want[i]) for i in (0, 1, 3))
            check_dw(got[2][:, :50], a, y, dy, act)
            check_dw(got[2][:, 70:100], c, y, dy, act)
            assert (got[2][:, 50:70] == 0).all() and (got[2][:, 100:] == 0).all()
            y = d.linear(segments, [W.detach()], [b], act, checkpoint=kept, products="fp32")
            assert torch.equal(torch.autograd.grad(y, c, dy)[0], want[1])
    base, Wt = make(90, 101, torch.float32, 3, 0.3), (torch.randn((50, 40), generator=g) * 0.1).cuda()
    for x in (base[:, 1:51], base[7:8, :50].expand(90, 50), base[:, ::2][:, :50], base.t()[:90, :50]):
        w = Wt.t().detach().requires_grad_()
        y, plain = (d.linear([(x, 0, 0)], [w], [b.detach()], "sigmoid", **kw)
                    for kw in ({"checkpoint": "int8", "products": "fp32"}, {}))
        assert torch.equal(y, plain)
        check_dw(torch.autograd.grad(y.sum(), w)[0], x, y, torch.ones_like(y), "sigmoid")


def test_what_is_kept():
    """8 bits a value of x and one a ReLU output, as with the layer's own products."""
    d = dense()
    rows, k, n = 8192, 1024, 256
    x, w = make(rows, k, torch.float32), torch.randn((n, k)).cuda().requires_grad_()

    def held():
        base = torch.cuda.memory_stats()["requested_bytes.all.current"]
        y = d.linear([(x.clone(), 0, 0)], [w], [], "relu", checkpoint="int8", products="fp32")
        return torch.cuda.memory_stats()["requested_bytes.all.current"] - base, y

    bytes_, y = held()
    assert bytes_ == rows * n * 4 + rows * k + 128 + rows * 4 + rows * n // 8
    with pytest.raises(RuntimeError):  # second derivatives are refused
        torch.autograd.grad(torch.autograd.grad(y.sum(), w, create_graph=True)[0].sum(), w)
    for bad in ("bf16", 32, True):
        with pytest.raises(ValueError, match="products"):
            d.linear([(x, 0, 0)], [w], [], None, checkpoint="int8", products=bad)
    assert torch.equal(d.linear([(x, 0, 0)], [w], [], None, products="fp32"), d.linear([(x, 0, 0)], [w], [], None))


def test_field():
    """A training step: outputs and bias gradients are the fp32 field's, bit for bit."""
    a, b = pair(dense_checkpoints="int8", dense_products="fp32")
    batch = batch_of(700)
    target = torch.rand((700, 3), generator=torch.Generator().manual_seed(1)).cuda()
    for m in (a, b):
        (m(batch) - target).square().mean().backward()
    assert torch.equal(a(batch), b(batch))
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        if name.endswith("bias"):
            assert torch.equal(p.grad, q.grad), name
        else:
            assert float((p.grad - q.grad).norm() / p.grad.norm()) < 1e-2, name


def test_concat_layer():
    from layers import LinearWithConcatAndActivation
    torch.manual_seed(0)
    layer = LinearWithConcatAndActivation(48, 20, 40).cuda()
    x, y = make(64, 48, torch.float32, 1), make(64, 20, torch.float32, 2)
    want = layer(x, y)
    layer.checkpoint, layer.products = "int8", "fp32"
    assert torch.equal(layer(x, y), want)


def test_graph_replay_and_streams():
    d = dense()
    xs, ws, bs, dy = leaves(700, 70, (96,), torch.float32, 2)

    def step(x, dy, act):
        x = x.detach().requires_grad_()
        y = d.linear([(x, 0, 0)], ws, bs, act, checkpoint="int8", products="fp32")
        return [y.detach(), *torch.autograd.grad(y, [x, *ws, *bs], dy)]

    eager = step(xs[0], dy, "relu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(xs[0], dy, "relu")
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    sx, sdy, graph = xs[0].detach().clone(), dy.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx, sdy, "relu") + step(sx, sdy, "sigmoid")
    for i in range(3):
        sx.copy_(make(700, 96, torch.float32, 50 + i))
        sdy.copy_(torch.randn((700, 70), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        want = step(sx, sdy, "relu") + step(sx, sdy, "sigmoid")
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.parametrize("kw", [{}, {"products": "fp32"}])
@pytest.mark.parametrize("n,k,taken", [(1 << 21, 1, False), (1, 1 << 21, False), ((1 << 21) - 63, 1, False),
                                       ((1 << 21) - 64, 1, True), ((1 << 21) - 255, 1, True), (1, (1 << 21) - 64, True)])
def test_weights_too_large_are_refused_by_the_forward(n, k, taken, kw):
    """n k is counted with one side rounded up to 256 and the other to 64: of one column, 2^21 - 64 rows are the most."""
    d = dense()
    x, w = torch.ones((1, k), device="cuda"), torch.ones((n, k), device="cuda", requires_grad=True)

    def call():
        return d.linear([(x, 0, 0)], [w], [], "relu", checkpoint="int8", **kw)

    if not taken:
        with pytest.raises(RuntimeError, match="too large"):
            call()
        return
    y = call()
    assert (y == k).all() and (torch.autograd.grad(y.sum(), w)[0] == 1).all()
