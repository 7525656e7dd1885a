"""The 8-bit dense layers on more rows than one launch can hold (2^32 threads, up to 256 of them a row): the
results are those of calls on pieces of the rows, bit for bit (the forms taken here do not depend on the
number of rows).  Inputs are windows of one long vector, a value apart, where that saves memory."""
import pytest
import torch

from test_gpu_dense8 import dense, layer64, near, weight8

pytestmark = pytest.mark.gpu

ROWS = (1 << 26) + 13  # 64 threads a row pass 2^32
PIECE = 1 << 22


@pytest.fixture(autouse=True)
def memory_back():
    yield
    torch.cuda.empty_cache()


def windows(rows, k, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randn(rows + k, generator=g, device="cuda") * torch.rand(rows + k, generator=g, device="cuda") ** 4
    return v.to(dtype).as_strided((rows, k), (1, 1))


def pieces(rows):
    return [slice(r, min(r + PIECE, rows)) for r in range(0, rows, PIECE)]


def test_rows8_quantised():
    d = dense()
    x = windows(ROWS, 257)
    r = d.quantize_rows(x)
    for p in pieces(ROWS):
        want = d.quantize_rows(x[p])
        assert torch.equal(r.q[p], want.q) and torch.equal(r.scale[p], want.scale)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows8_restored(dtype):
    d = dense()
    r = d.Rows8(ROWS, 65, "cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for p in pieces(ROWS):
        r.q[p] = torch.randint(-127, 128, r.q[p].shape, generator=g, device="cuda", dtype=torch.int8)
    r.scale.copy_(torch.rand(ROWS, generator=g, device="cuda"))
    x = r.restore(dtype)
    for p in pieces(ROWS):
        assert torch.equal(x[p], (r.q[p].float() * r.scale[p, None]).to(dtype))


def test_checkpointed_layer_forward_and_weight_gradient():
    """dy has some rows only, the last ones among them: dW is their sum."""
    d = dense()
    n, k = 3, 257
    g = torch.Generator(device="cuda").manual_seed(2)
    x, w = windows(ROWS, k, seed=3), torch.randn((n, k), generator=g, device="cuda").requires_grad_()
    y = d.linear([(x, 0, 0)], [w], [], None, checkpoint="int8")
    for p in pieces(ROWS):
        assert torch.equal(y[p], d.linear([(x[p], 0, 0)], [w.detach()], [], None, checkpoint="int8"))
    some = torch.cat([torch.arange(0, ROWS, 1 << 17, device="cuda"), torch.arange(ROWS - 200, ROWS, device="cuda")])
    dy = torch.zeros((ROWS, n), device="cuda")
    dy[some] = torch.randn((len(some), n), generator=g, device="cuda")
    # zeros add nothing, so that the bound of the rows alone holds; row 2^26 is in both ranges and counts once
    once = some.unique()
    assert len(once) == len(some) - 1
    near(torch.autograd.grad(y, w, dy)[0], layer64([x[once]], [w], [], None, dy[once])["dw"][0])


@pytest.mark.parametrize("act", ["relu", "sigmoid"])
def test_checkpointed_layer_dx(act):
    d = dense()
    n, k = 65, 2
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((ROWS, k), generator=g, device="cuda").requires_grad_()
    w = torch.randn((n, k), generator=g, device="cuda")
    dy = windows(ROWS, n, seed=5)
    dx = torch.autograd.grad(d.linear([(x, 0, 0)], [w], [], act, checkpoint="int8"), x, dy)[0]
    for p in pieces(ROWS):
        xp = x.detach()[p].clone().requires_grad_()
        y = d.linear([(xp, 0, 0)], [w], [], act, checkpoint="int8")
        assert torch.equal(dx[p], torch.autograd.grad(y, xp, dy[p])[0])


@pytest.mark.parametrize("n,k", [(40, 24), (20, 300), (3, 24), (300, 24)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8])
def test_linear8(n, k, dtype):
    """The forms for many rows, a turn of each more than once; rows from and into 8 bits."""
    d = dense()
    rows = (1 << 24) + 777
    x = windows(rows, k, torch.float32 if dtype == torch.int8 else dtype, seed=6)
    if dtype == torch.int8:
        x = d.quantize_rows(x)
    qw, sw = weight8(n, k, 1)
    w, b = d.pack_weight8(qw.cuda(), sw.cuda()), torch.randn(n, device="cuda")
    for act, out in (("relu", torch.int8), (None, torch.bfloat16)):
        y = d.linear8([x], [w], [b], act, out=out)
        for p in pieces(rows):
            if dtype == torch.int8:
                part = d.Rows8(p.stop - p.start, k, "cuda")
                part.q.copy_(x.q[p])
                part.scale.copy_(x.scale[p])
            else:
                part = x[p]
            want = d.linear8([part], [w], [b], act, out=out)
            if out == torch.int8:
                assert torch.equal(y.q[p], want.q) and torch.equal(y.scale[p], want.scale)
            else:
                assert torch.equal(y[p], want)
