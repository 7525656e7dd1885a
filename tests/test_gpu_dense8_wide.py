"""The widest tiles of the 8-bit dense layers, and rows that are not finite in the form that holds the weight in LDS.

Tiles of 256 x 256 are taken from 256 of them on (a tile for each CU); 256 x 128 for an 8-bit result of 65 to 128
columns.  Tolerances as in test_gpu_dense8."""
import pytest
import torch

from test_gpu_dense8 import EPS, dense, layer64, leaves, make, near, oracle_linear8, relu_safe, weight8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [None, "relu", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", [(65300, 130, 33), (16400, 1000, 70), (65281, 256, 31)])
def test_checkpointed_layer(rows, n, k, dtype, act):
    """Forward tiles of 256 x 256; with n = 130 the rows of y do not start on 16 bytes."""
    xs, ws, bs, dy = leaves(rows, n, (k,), dtype, n)
    if act == "relu":
        dy = relu_safe(xs, ws, bs, dy)
    y = dense().linear([(xs[0], 0, 0)], ws, bs, act, checkpoint="int8")
    dx, dw, db = torch.autograd.grad(y, [xs[0], ws[0], bs[0]], dy)
    want = layer64(xs, ws, bs, act, dy)
    near(y, want["y"])
    near(dx, want["dx"][0], dtype)
    near(dw, want["dw"][0])
    near(db, want["db"])


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("rows,n,k", [(4100, 4090, 1030), (65300, 200, 1100), (65300, 100, 1100), (65300, 200, 300)])
def test_linear8(rows, n, k, dtype, out):
    d = dense()
    x = make(rows, k, torch.float32 if dtype == torch.int8 else dtype, rows)
    qw, sw = weight8(n, k, k)
    w = d.pack_weight8(qw.cuda(), sw.cuda())
    b = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    for act in (None, "relu", "sigmoid"):
        y = d.linear8([d.quantize_rows(x) if dtype == torch.int8 else x], [w], [b], act, out=out)
        want, err = oracle_linear8([x], [(qw, sw)], [b], act)
        got = y.cpu().double()
        assert ((got - want).abs() <= err + (EPS[out] if out != torch.float32 else 0) * (want.abs() + err)).all()


@pytest.mark.parametrize("rows,n,k", [(65300, 200, 300), (65300, 256, 1100), (65300, 100, 300), (65300, 128, 1100)])
def test_linear8_rows_out_are_the_rows_of_the_result(rows, n, k):
    d = dense()
    x = make(rows, k, torch.float32, 11)
    qw, sw = weight8(n, k, 4)
    w, b = d.pack_weight8(qw.cuda(), sw.cuda()), torch.randn(n).cuda()
    r = d.quantize_rows(x)
    add = d.pack_weight8(qw[:, :20].contiguous().cuda(), sw.cuda())
    for act in (None, "relu"):
        for xs, ws in (([r], [w]), ([x], [w]), ([x[:, :20], r], [add, w])):
            y = d.linear8(xs, ws, [b], act)
            got = d.linear8(xs, ws, [b], act, out=torch.int8)
            want = d.quantize_rows(y)
            assert torch.equal(got.q, want.q) and torch.equal(got.scale, want.scale)


@pytest.mark.parametrize("act", [None, "relu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("rows,n,k", [(16400, 33, 64), (16400, 256, 256), (16390, 100, 130), (20000, 130, 3)])
def test_linear8_bad_rows_with_the_weight_in_lds(rows, n, k, dtype, act):
    """NaN in the bad rows alone; weights whose scale is an infinity or a NaN: inf 0 and inf - inf are NaN (of negative
    sign, and stay NaN under a ReLU), an infinity stays one or, negative, becomes zero, as for the same call on few rows."""
    d = dense()
    x = make(rows, k, torch.float32 if dtype == torch.int8 else dtype, rows)
    at = torch.tensor([0, 5, 17, 4000, rows - 1])
    for i, m in enumerate(at):
        x[m, (5 * i) % k] = (float("inf"), -float("inf"), float("nan"))[i % 3]
    x[7] = 0
    rx = d.quantize_rows(x) if dtype == torch.int8 else x
    if dtype == torch.int8:  # a NaN of the other sign
        rx.scale.view(torch.int32)[at[1].item()] = -1
    qw, sw = weight8(n, k, 2)
    b = torch.randn(n, generator=torch.Generator().manual_seed(3))
    others = torch.ones(rows, dtype=torch.bool)
    others[at] = False
    w = d.pack_weight8(qw.cuda(), sw.cuda())
    y = d.linear8([rx], [w], [b.cuda()], act)
    assert torch.isnan(y[at.cuda()]).all() and torch.isfinite(y[others.cuda()]).all()
    for out in (torch.bfloat16, torch.int8):
        z = d.linear8([rx], [w], [b.cuda()], act, out=out)
        bad = torch.isnan(z.scale if out == torch.int8 else z.float().sum(1)).cpu()
        assert torch.equal(bad, ~others)
    # scales and biases that are not finite
    sw[0], sw[1], sw[2] = float("inf"), float("nan"), 3e38
    b[3], b[4], b[0] = -float("inf"), float("nan"), -float("inf")
    w = d.pack_weight8(qw.cuda(), sw.cuda())
    y = d.linear8([rx], [w], [b.cuda()], act)
    some = torch.tensor([*range(16), *at, 7])
    if dtype == torch.int8:
        part = d.Rows8(len(some), k, "cuda")
        part.q.copy_(rx.q[some.cuda()])
        part.scale.copy_(rx.scale[some.cuda()])
    else:
        part = x[some.cuda()]
    few = torch.cat([d.linear8([p], [w], [b.cuda()], act) for p in ([part] if dtype == torch.int8 else part.split(8))])
    got = y[some.cuda()]
    differ = int(((got != few) & ~(torch.isnan(got) & torch.isnan(few))).sum())
    assert differ == 0
    assert torch.isnan(y[7, [0, 1, 4]]).all() and not torch.isnan(y[7, 2])
