"""The dense layers in 8 bits (csrc/rows8.hip, linear8.hip, ckpt.hip) against plain
implementations in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32, relative; U that of the output's type (bf16
2^-8 / 2 = 2^-9 of a value's own power of two, at most 2^-8 / 2 relative: finfo.eps / 2).
  rows in 8 bits: q equal; the scale has two roundings (1 / 127 and its product with the
    maximum): 2 u and u^2; a restored value, from the scale as it is, one: u or U.
  linear8: acc is exact, then fl(acc), fl(sx sw), their product, the bias, the sum over
    segments: |error| <= 5 u (sum_s |acc t| + |bias|) a segment, plus U |y| for the output;
    sx and sw have one rounding each, which the oracle takes over (it reads the scales).
    A ReLU does not enlarge an error; a sigmoid's slope is at most 1/4, and its exp, add
    and divide cost 4 u more.
  checkpointed layer: fp32 values enter the products as two fp16 pieces.  hi is off by half a step, 2^-11 of
    the value, lo by 2^-11 of that and at most half of it again (a value just above a power of two has the
    largest hi error, whose lo then lies in the upper half of its own power of two): 2^-23 a value.  lo lo, at
    most 2^-22, is left out.  A product is off by 2^-23 + 2^-23 + 2^-22 = 8 u, and its three parts are three
    additions of u each of the partial sums, whatever their order: |error| <= (3 K + 8) u sum |a b|.  Of a
    value far below its row's largest, which is scaled to 2^14 at least, lo is a multiple of 2^-24: off by
    2^-25, 2^-39 of the largest: another 2^-39 (max |a| sum |b| + sum |a| max |b|).  dW: one operand is exact,
    the other has one rounding (u) and three exact pieces: the first bound covers it."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def dense():
    import dense as d
    return d


def oracle_rows(x):
    """(q, max|x| / 127 in 64 bits): the nearest whole numbers by exact comparison."""
    v = x.detach().cpu().to(torch.float64).numpy()
    a = np.abs(v)
    top = a.max(1, keepdims=True)
    bad = ~np.isfinite(top)
    t = np.where((top == 0) | bad, 1.0, top)
    f = np.floor(np.where(bad, 0.0, a) * 127.0 / t)
    f = np.where(f * t > 127.0 * a, f - 1, f)
    f = np.where((f + 1) * t <= 127.0 * a, f + 1, f)
    two, half = 254.0 * a, (2 * f + 1) * t
    q = f + ((two > half) | ((two == half) & (f % 2 == 1)))
    q = np.where(bad, 0.0, q)
    return (np.sign(np.where(bad, 0.0, v)) * q).astype(np.int8), np.where(bad, np.nan, top)[:, 0] / 127.0


def make(rows, k, dtype, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, k), generator=g) * torch.exp(spread * torch.randn((rows, 1), generator=g))
    return x.to(dtype).cuda()


def check_rows(x, r):
    q, s = oracle_rows(x)
    assert torch.equal(r.q.cpu(), torch.from_numpy(q))
    got = r.scale.cpu().double().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(s))
    np.testing.assert_allclose(got, s, rtol=2 * U32 + U32 ** 2, atol=2.0 ** -150)


SHAPES = [(1, 1), (1, 3), (7, 3), (5, 15), (3, 16), (2, 17), (9, 63), (4, 64), (33, 65), (3, 127), (2, 256), (5, 255),
          (130, 257), (1, 1023), (6, 1024), (3, 1025), (2, 2047), (3, 4096), (2, 4100), (1, 9001), (1000, 8)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,k", SHAPES)
def test_rows8(rows, k, dtype):
    x = make(rows, k, dtype)
    r = dense().quantize_rows(x)
    check_rows(x, r)
    for t in (torch.float32, torch.bfloat16):
        v = r.restore(t)
        want = r.q.cpu().double() * r.scale.cpu().double()[:, None]
        assert v.dtype == t and v.shape == x.shape
        assert ((v.cpu().double() - want).abs() <= (EPS[t] + U32) * want.abs()).all()


def test_rows8_ties_extremes_and_empty_rows():
    """Values whose ratio is exactly a half, one step beside it, rows of zeros, denormals, the
    largest numbers, infinities and NaNs."""
    k = 300
    g = torch.Generator().manual_seed(3)
    rows = []
    for top in (127.0, 254.0, 1.0, 3.0, 1e-30, 1e-38, 1e-42, 3.4e38):
        n = torch.randint(-126, 126, (k,), generator=g).double()
        v = ((n + 0.5) * top / 127.0).float()  # a half, as near as fp32 has it
        v[::3] = torch.nextafter(v[::3], torch.full_like(v[::3], float("inf")))
        v[1::3] = torch.nextafter(v[1::3], torch.full_like(v[1::3], -float("inf")))
        v[-1] = top
        rows.append(v)
    rows.append(torch.zeros(k))
    for bad in (float("inf"), -float("inf"), float("nan")):
        v = torch.randn(k, generator=g)
        v[17] = bad
        rows.append(v)
    x = torch.stack(rows).cuda()
    r = dense().quantize_rows(x)
    check_rows(x, r)
    assert (r.q[:8].float().abs().amax(1) == 127).all() and (r.q[8:] == 0).all()
    v = r.restore()
    assert (v[8] == 0).all() and torch.isnan(v[9:]).all() and torch.isfinite(v[:8]).all()


def test_rows8_every_ratio_of_bf16():
    """All 128 significands over all, three exponents apart: every exact half of two bf16 values."""
    sig = (1 + torch.arange(128) / 128).to(torch.bfloat16)
    for scale in (1.0, 2.0 ** -110, 2.0 ** 120):
        rows = torch.stack([torch.cat([sig * 2.0 ** -e * scale for e in range(1, 9)] + [s[None] * scale])
                            for s in sig.to(torch.bfloat16)]).to(torch.bfloat16)
        rows[:, ::2] *= -1
        x = rows.cuda()
        check_rows(x, dense().quantize_rows(x))
        check_rows(x.float(), dense().quantize_rows(x.float()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows8_strides(dtype):
    """Column ranges at odd offsets, a row repeated with stride 0, columns, no rows."""
    d = dense()
    base = make(40, 101, dtype, 5)
    for x in (base[:, 1:], base[:, 3:90], base[::3, 7:8], base[5:6].expand(12, 101), base.t(), base[:, ::2],
              base[3:3], base[:0, :5]):
        r = d.quantize_rows(x)
        assert r.shape == x.shape
        if x.shape[0]:
            check_rows(x, r)
        assert r.restore(dtype).shape == x.shape


# ---- linear8 ------------------------------------------------------------------------

def act64(z, act):
    if act == "relu":
        return z.clamp_min(0)
    return torch.special.expit(z) if act == "sigmoid" else z


def rows64(x):
    r = x if not torch.is_tensor(x) else dense().quantize_rows(x)
    return r.q.cpu().double(), r.scale.cpu().double()


def oracle_linear8(xs, ws, bs, act):
    """(y, bound of the fp32 roundings) from the 8-bit rows as they are."""
    z, mag = 0.0, 0.0
    for i, (x, (qw, sw)) in enumerate(zip(xs, ws)):
        q, s = rows64(x)
        t = (q @ qw.double().t()) * s[:, None] * sw.double()[None, :]
        b = bs[i].cpu().double() if i < len(bs) else torch.zeros(qw.shape[0]).double()
        z = z + t + b
        mag = mag + t.abs() + b.abs()
    err = 5 * U32 * mag * len(xs)
    y = act64(z, act)
    if act == "sigmoid":
        err = err / 4 + 4 * U32 * y
    return y, err


def weight8(n, k, seed):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    return q, torch.rand(n, generator=g) * 0.01 + 1e-4


SIZES = [(1, 1, 1), (1, 3, 1024), (1, 256, 1024), (2, 17, 63), (5, 256, 1023), (15, 128, 64), (16, 100, 129),
         (17, 3, 256), (33, 130, 100), (64, 64, 4096), (65, 257, 300), (127, 96, 127), (128, 128, 128),
         (300, 256, 256), (257, 511, 193), (1000, 3, 16), (520, 1030, 65), (1, 4096, 2048), (8, 4097, 33),
         (16390, 256, 256), (16400, 100, 77), (17001, 129, 200), (16384, 255, 3), (16385, 64, 128),
         (32769, 256, 1023), (32790, 40, 300), (32770, 3, 513), (32831, 129, 512), (32768, 253, 769),
         (2049, 2040, 100), (4095, 1025, 260)]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_linear8(rows, n, k, dtype, out):
    d = dense()
    x = make(rows, k, torch.float32 if dtype == torch.int8 else dtype, rows + n)
    qw, sw = weight8(n, k, k)
    w = d.pack_weight8(qw.cuda(), sw.cuda())
    b = torch.randn(n, generator=torch.Generator().manual_seed(n)).cuda()
    act = [None, "relu", "sigmoid"][(rows + n + k) % 3]
    xin = d.quantize_rows(x) if dtype == torch.int8 else x
    y = d.linear8([xin], [w], [b], act, out=out)
    want, err = oracle_linear8([x], [(qw, sw)], [b], act)
    got = y.cpu().double()
    assert y.dtype == out and y.shape == (rows, n)
    assert ((got - want).abs() <= err + (EPS[out] if out != torch.float32 else 0) * (want.abs() + err)).all()


@pytest.mark.parametrize("rows,n,k", [(1, 1, 5), (1, 256, 1024), (3, 255, 64), (130, 256, 256), (700, 128, 100),
                                      (70, 64, 1023), (20, 3, 40), (65, 300, 30), (9, 1025, 17), (16390, 256, 255),
                                      (16400, 100, 128), (16411, 37, 64), (32769, 256, 1024),
                                      (32800, 70, 290), (33000, 3, 1000)])
def test_linear8_rows_out_are_the_rows_of_the_result(rows, n, k):
    """out=int8 is quantize_rows of the fp32 result, bit for bit, whichever kernel makes it."""
    d = dense()
    x = make(rows, k, torch.float32, 11)
    qw, sw = weight8(n, k, 4)
    w = d.pack_weight8(qw.cuda(), sw.cuda())
    b = torch.randn(n).cuda()
    for xin in (x, d.quantize_rows(x)):
        for act in (None, "relu"):
            y = d.linear8([xin], [w], [b], act)
            r = d.linear8([xin], [w], [b], act, out=torch.int8)
            want = d.quantize_rows(y)
            assert torch.equal(r.q, want.q) and torch.equal(r.scale, want.scale)


def test_linear8_each_form_gives_the_same_numbers():
    """A row's result does not depend on how many rows come with it, nor on who quantised it."""
    d = dense()
    for n, k, rows in ((256, 1024, 600), (100, 77, 16500), (3, 256, 600), (256, 200, 20000),
                       (200, 1023, 32900)):
        x = make(rows, k, torch.float32, 2)
        qw, sw = weight8(n, k, 1)
        w, b = d.pack_weight8(qw.cuda(), sw.cuda()), torch.randn(n).cuda()
        whole = d.linear8([x], [w], [b], "relu")
        r8 = d.quantize_rows(x)
        assert torch.equal(d.linear8([r8], [w], [b], "relu"), whole)
        for m in (1, 2, 16, 17, 64, 65, 300, 16390):
            assert torch.equal(d.linear8([x[:m]], [w], [b], "relu"), whole[:m])


def test_linear8_segments_and_bad_rows():
    """Two segments (the skip layer), fewer biases than segments, rows of zeros, rows that are
    not finite: NaN in that row alone."""
    d = dense()
    rows, n = 150, 96
    x0, x1 = make(rows, 64, torch.float32, 1), make(rows, 33, torch.bfloat16, 2)
    x0[3] = 0
    x1[3] = 0
    ws = [weight8(n, 64, 5), weight8(n, 33, 6)]
    w = [d.pack_weight8(q.cuda(), s.cuda()) for q, s in ws]
    b = [torch.randn(n).cuda(), torch.randn(n).cuda()]
    for bs in (b, b[:1], []):
        y = d.linear8([x0, x1], w, bs, "relu")
        want, err = oracle_linear8([x0, x1], ws, bs, "relu")
        assert ((y.cpu().double() - want).abs() <= err).all()
    x0[7, 5], x1[9, 0], x0[11, 1] = float("inf"), float("nan"), -float("inf")
    for out in (torch.float32, torch.bfloat16):
        bad = torch.isnan(d.linear8([x0, x1], w, b, "relu", out=out)).cpu()
        assert bad[[7, 9, 11]].all() and bad.sum() == 3 * n
    r = d.linear8([x0, x1], w, b, None, out=torch.int8)
    assert torch.isnan(r.scale.cpu()[[7, 9, 11]]).all() and int(torch.isnan(r.scale).sum()) == 3


@pytest.mark.parametrize("out", [torch.float32, torch.int8])
def test_linear8_long_rows_add_and_bad_rows(out):
    """Many long rows on top of another segment's result; a bad row and a zero row stay by themselves."""
    d = dense()
    rows, n = 32770, 90
    x0, x1 = make(rows, 31, torch.float32, 1), make(rows, 700, torch.bfloat16, 2)
    x0[3], x1[3] = 0, 0
    ws = [weight8(n, 31, 5), weight8(n, 700, 6)]
    w = [d.pack_weight8(q.cuda(), s.cuda()) for q, s in ws]
    b = [torch.randn(n).cuda()]
    y = d.linear8([x0, x1], w, b, "sigmoid")
    want, err = oracle_linear8([x0, x1], ws, b, "sigmoid")
    assert ((y.cpu().double() - want).abs() <= err).all()
    x1[9, 0], x1[rows - 1, 699] = float("nan"), -float("inf")
    r = d.linear8([x0, x1], w, b, "relu", out=out)
    bad = torch.isnan(r.scale if out == torch.int8 else r.sum(1)).cpu()
    assert bad[[9, rows - 1]].all() and int(bad.sum()) == 2


def test_linear8_largest_sum_and_strided_weight():
    """Sums of 2^17 products 127 x 127 stay in 32 bits; weights of any strides pack the same."""
    d = dense()
    k = 1 << 17
    x = torch.ones((2, k), device="cuda")
    q = torch.full((5, k), 127, dtype=torch.int8, device="cuda")
    s = torch.full((5,), 2.0 ** -10, device="cuda")
    y = d.linear8([x], [d.pack_weight8(q, s)], [])
    want = np.float32(k * 127.0 * 127.0) * (np.float32(1.0 / 127.0) * np.float32(2.0 ** -10))
    np.testing.assert_allclose(y.cpu().numpy(), want, rtol=4 * U32)
    qw, sw = weight8(40, 50, 9)
    x = make(20, 50, torch.float32)
    a = d.linear8([x], [d.pack_weight8(qw.cuda(), sw.cuda())], [])
    assert torch.equal(a, d.linear8([x], [d.pack_weight8(qw.cuda().t().contiguous().t(), sw.cuda())], []))
    W = make(30, 80, torch.float32)
    w = d.quantize_weight(W, 21, 50)
    r = d.quantize_rows(W[:, 21:71])
    assert torch.equal(d.linear8([x], [w], []), d.linear8([x], [d.pack_weight8(r.q, r.scale)], []))


def test_linear8_leaves_what_is_not_its_own():
    """Rows of one buffer behind the last row, and other columns, stay as they were."""
    d = dense()
    qw, sw = weight8(100, 90, 1)
    w = d.pack_weight8(qw.cuda(), sw.cuda())
    from inf_hip import DTYPE_F32, lib, check
    from inf_hip import runtime as rt
    x = make(70, 90, torch.float32)
    buf = torch.full((80, 128), 7.0, device="cuda")
    ws = torch.empty(int(lib.inf_linear_int_workspace_bytes(70, 100, 90, 0, 0)), dtype=torch.uint8, device="cuda")
    check(lib.inf_linear_int(70, 100, 90, rt.ptr(x), DTYPE_F32, 90, None, rt.ptr(w.packed), rt.ptr(w.scale), None, None,
                             0, 0, rt.ptr(buf), DTYPE_F32, 128, None, rt.ptr(ws), rt.stream_handle()))
    assert torch.equal(buf[:70, :100], d.linear8([x], [w], []))
    assert (buf[70:] == 7).all() and (buf[:, 100:] == 7).all()


# ---- the layer with 8-bit checkpoints -------------------------------------------------

def far_below(a, b):
    """2^-39 (max |a| sum |b| + sum |a| max |b|) for each row of a with each column of b."""
    a, b = a.abs(), b.abs()
    return 2.0 ** -39 * (a.amax(1)[:, None] * b.sum(0)[None] + a.sum(1)[:, None] * b.amax(0)[None])


def layer64(xs, ws, bs, act, dy, c0s=None):
    """Output, gradients and their worst-case fp32 bounds."""
    z, zm, ez, k_all = 0.0, 0.0, 0.0, 0
    x64 = [x.detach().cpu().double() for x in xs]
    w64 = [w.detach().cpu().double() for w in ws]
    for i, (x, w) in enumerate(zip(x64, w64)):
        b = bs[i].detach().cpu().double() if i < len(bs) else torch.zeros(w.shape[0]).double()
        z = z + x @ w.t() + b
        zm = zm + x.abs() @ w.abs().t() + b.abs()
        ez = ez + far_below(x, w.t())
        k_all += x.shape[1]
    dy = dy.cpu().double()
    y = act64(z, act)
    ey = (3 * k_all + 8) * U32 * zm + ez
    if act == "relu":
        dz, edz = dy * (z > 0), 0.0
    elif act == "sigmoid":
        dz = dy * y * (1 - y)
        ey = ey / 4 + 4 * U32 * y
        edz = dy.abs() * ey + 4 * U32 * dy.abs()  # |d(y (1 - y))| <= |dy|'s share, and its roundings
    else:
        dz, edz = dy, 0.0
    rows, n = dz.shape
    out = {"y": (y, ey), "dx": [], "dw": [], "db": (dz.sum(0), (rows + 8) * U32 * dz.abs().sum(0)
                                                     + (edz.sum(0) if act == "sigmoid" else 0))}
    for x, w in zip(xs, w64):
        e = (3 * n + 8) * U32 * (dz.abs() @ w.abs()) + far_below(dz, w) + (edz @ w.abs() if act == "sigmoid" else 0)
        out["dx"].append((dz @ w, e))
        q, s = rows64(x.detach())
        v = q * s[:, None]
        e = (3 * rows + 8) * U32 * (dz.abs().t() @ v.abs()) + (edz.t() @ v.abs() if act == "sigmoid" else 0)
        out["dw"].append((dz.t() @ v, e))
    return out


def near(got, want, dtype=torch.float32):
    w, e = want
    lim = e + (EPS[dtype] * (w.abs() + e) if dtype != torch.float32 else 0) + 1e-37
    d = (got.detach().cpu().double() - w).abs()
    assert (d <= lim).all(), float((d / lim).max())


def relu_safe(xs, ws, bs, dy):
    """dy with zeros where an output is so near zero that fp32 may see it on the other side."""
    z, zm = 0.0, 0.0
    for i, (x, w) in enumerate(zip(xs, ws)):
        x, w = x.detach().cpu().double(), w.detach().cpu().double()
        b = bs[i].detach().cpu().double() if i < len(bs) else torch.zeros(w.shape[0]).double()
        z, zm = z + x @ w.t() + b, zm + x.abs() @ w.abs().t() + b.abs()
    k = sum(x.shape[1] for x in xs)
    return torch.where((z.abs() <= (3 * k + 8) * U32 * zm).cuda(), torch.zeros_like(dy), dy)


def leaves(rows, n, widths, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    xs = [make(rows, k, dtype, seed + i, 0.5).requires_grad_() for i, k in enumerate(widths)]
    ws = [((torch.rand((n, k), generator=g) * 2 - 1) * (6 / (n + k)) ** 0.5).cuda().requires_grad_() for k in widths]
    bs = [(0.1 * torch.randn(n, generator=g)).cuda().requires_grad_() for _ in widths]
    dy = (torch.randn((rows, n), generator=g) * torch.exp(torch.randn((rows, 1), generator=g))).cuda()
    return xs, ws, bs, dy


LAYERS = [(1, 1, (1,)), (1, 3, (5,)), (2, 33, (31,)), (64, 64, (64,)), (100, 3, (256,)), (65, 130, (63,)),
          (300, 256, (1023,)), (512, 256, (256,)), (129, 257, (255,)), (1000, 128, (3,)), (257, 64, (100, 40)),
          (600, 256, (256, 1024)), (3000, 96, (64,)), (77, 512, (512,)),
          (32769, 256, (256,)), (32800, 66, (257, 300)), (33000, 130, (1,)), (32768, 200, (511,)),
          (16001, 257, (255,)), (8200, 300, (400,))]


@pytest.mark.parametrize("act", [None, "relu", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n,widths", LAYERS)
def test_checkpointed_layer(rows, n, widths, dtype, act):
    xs, ws, bs, dy = leaves(rows, n, widths, dtype, rows + n)
    if act == "relu":
        dy = relu_safe(xs, ws, bs, dy)
    y = dense().linear([(x, i, 0) for i, x in enumerate(xs)], ws, bs, act, checkpoint="int8")
    y.backward(dy)
    want = layer64(xs, ws, bs, act, dy)
    near(y, want["y"])
    for x, w in zip(xs, want["dx"]):
        assert x.grad.dtype == dtype
        near(x.grad, w, dtype)
    for p, w in zip(ws, want["dw"]):
        near(p.grad, w)
    for b in bs:
        near(b.grad, want["db"])
    assert len({b.grad.data_ptr() for b in bs}) == len(bs)


def test_checkpointed_layer_single_products():
    """Sums of one product, whose bound is the pieces' own: values with the largest low pieces."""
    d = dense()
    g = torch.Generator().manual_seed(4)

    def worst(n):  # 2^e (1 + m 2^-10 + 2^-11 +- a little): in the middle between two fp16 values
        m = torch.randint(0, 16, (n,), generator=g).double()
        off = torch.randint(-3, 4, (n,), generator=g).double() * 2.0 ** -22
        e = torch.randint(-20, 20, (n,), generator=g).double()
        return ((1 + m * 2.0 ** -10 + 2.0 ** -11 + off) * 2.0 ** e).float()

    x, w = worst(500)[:, None].cuda(), worst(300)[:, None].cuda()
    y = d.linear([(x, 0, 0)], [w], [], None, checkpoint="int8")
    near(y, layer64([x], [w], [], None, torch.zeros((500, 300)))["y"])
    w, dy = worst(700)[None, :].cuda(), worst(400)[:, None].cuda()  # dx of one output
    xs = torch.zeros((400, 700), device="cuda").requires_grad_()
    y = d.linear([(xs, 0, 0)], [w], [], None, checkpoint="int8")
    near(torch.autograd.grad(y, xs, dy)[0], layer64([xs], [w], [], None, dy)["dx"][0])
    # a small value next to a large one that meets a zero
    x = torch.stack([torch.full((60,), 1e3), torch.logspace(-8, 3, 60)], 1).cuda()
    w = torch.tensor([[0.0, 1.0], [0.0, 0.37], [1e-9, 1e-3]], device="cuda")
    y = d.linear([(x, 0, 0)], [w], [], None, checkpoint="int8")
    near(y, layer64([x], [w], [], None, torch.zeros((60, 3)))["y"])


def test_checkpointed_layer_matches_the_exact_one():
    """Against linear() without checkpoints: the same output and dx to fp32, dW within the
    8-bit rounding: |q s - x| <= s / 2, so |dW - dW'| <= |dz|^T s / 2, plus fp32's own."""
    d = dense()
    xs, ws, bs, dy = leaves(400, 128, (200,), torch.float32, 8)
    dy = relu_safe(xs, ws, bs, dy)
    ya = d.linear([(xs[0], 0, 0)], ws, bs, "relu")
    ga = torch.autograd.grad(ya, [*xs, *ws, *bs], dy)
    yb = d.linear([(xs[0], 0, 0)], ws, bs, "relu", checkpoint="int8")
    gb = torch.autograd.grad(yb, [*xs, *ws, *bs], dy)
    want = layer64(xs, ws, bs, "relu", dy)
    assert ((ya - yb).abs().cpu().double() <= 2 * want["y"][1]).all()
    assert ((ga[0] - gb[0]).abs().cpu().double() <= 2 * want["dx"][0][1]).all()
    s = d.quantize_rows(xs[0]).scale.cpu().double()
    dz = (dy * (ya > 0)).cpu().double().abs()
    lim = (dz.t() @ s)[:, None] / 2 * (1 + 1e-6) + 2 * want["dw"][0][1]
    assert ((ga[1] - gb[1]).abs().cpu().double() <= lim).all()


def test_checkpointed_layer_against_differences():
    """dx and db against central differences of the layer itself (sigmoid, smooth): a step h
    is off by h^2 |f'''| / 6 (|sigma'''| <= 1/8) and by 2 u |f| / h."""
    d = dense()
    xs, ws, bs, dy = leaves(6, 5, (7,), torch.float32, 4)
    y = d.linear([(xs[0], 0, 0)], ws, bs, "sigmoid", checkpoint="int8")
    gx, gb = torch.autograd.grad(y, [xs[0], bs[0]], dy)
    h = 2.0 ** -7

    def f(x, b):
        with torch.no_grad():
            return float((d.linear([(x, 0, 0)], [ws[0].detach()], [b], "sigmoid", checkpoint="int8").double()
                          * dy.double()).sum())

    big = float(ws[0].detach().abs().max())
    lim = float(dy.abs().sum()) * (h * h / 48 * max(1, big ** 3) + 16 * U32 / h)
    x, b = xs[0].detach(), bs[0].detach()
    for i, j in ((0, 0), (2, 3), (5, 6)):
        e = torch.zeros_like(x)
        e[i, j] = h
        assert abs((f(x + e, b) - f(x - e, b)) / (2 * h) - float(gx[i, j])) <= lim
    for j in range(5):
        e = torch.zeros_like(b)
        e[j] = h
        assert abs((f(x, b + e) - f(x, b - e)) / (2 * h) - float(gb[j])) <= lim


@pytest.mark.parametrize("rows", [70, 16400, 32771])
@pytest.mark.parametrize("k", [90, 300])
def test_wider_rows_of_results_stay(rows, k):
    """Results as columns of wider buffers, through the C entries: what is around them stays."""
    d = dense()
    from inf_hip import DTYPE_F32, DTYPE_I8, lib, check
    from inf_hip import runtime as rt
    n = 100
    x, qw_sw = make(rows, k, torch.float32, rows), weight8(n, k, 1)
    w = d.pack_weight8(qw_sw[0].cuda(), qw_sw[1].cuda())
    wf = (torch.randn((n, k), generator=torch.Generator().manual_seed(3)) * 0.1).cuda()

    def work(size):
        return torch.empty(max(int(size), 16), dtype=torch.uint8, device="cuda")

    buf = torch.full((rows + 3, 128), 7.0, device="cuda")
    ws = work(lib.inf_linear_int_workspace_bytes(rows, n, k, 0, 0))
    check(lib.inf_linear_int(rows, n, k, rt.ptr(x), DTYPE_F32, k, None, rt.ptr(w.packed), rt.ptr(w.scale), None, None,
                             0, 0, rt.ptr(buf), DTYPE_F32, 128, None, rt.ptr(ws), rt.stream_handle()))
    assert torch.equal(buf[:rows, :n], d.linear8([x], [w], []))
    assert (buf[rows:] == 7).all() and (buf[:, n:] == 7).all()
    q8, s8 = torch.full((rows + 3, 128), 9, dtype=torch.int8, device="cuda"), torch.full((rows + 3,), 7.0, device="cuda")
    ws = work(lib.inf_linear_int_workspace_bytes(rows, n, k, 0, 4))
    check(lib.inf_linear_int(rows, n, k, rt.ptr(x), DTYPE_F32, k, None, rt.ptr(w.packed), rt.ptr(w.scale), None, None,
                             0, 0, rt.ptr(q8), DTYPE_I8, 128, rt.ptr(s8), rt.ptr(ws), rt.stream_handle()))
    want = d.linear8([x], [w], [], out=torch.int8)
    assert torch.equal(q8[:rows, :n], want.q) and torch.equal(s8[:rows], want.scale)
    assert (q8[rows:] == 9).all() and (s8[rows:] == 7).all() and (q8[:, 112:] == 9).all()
    # the checkpointed layer: y, and dx into columns of a buffer of rows that do not start on 16 bytes
    buf.fill_(7)
    ws = work(lib.inf_linear_ckpt_workspace_bytes(rows, n, k, 0, 0))
    check(lib.inf_linear_ckpt_forward(rows, n, k, rt.ptr(x), DTYPE_F32, k, rt.ptr(wf), k, 1, None, None, 0, 0,
                                      rt.ptr(buf), 128, None, None, 0, None, rt.ptr(ws), rt.stream_handle()))
    assert torch.equal(buf[:rows, :n], d.linear([(x, 0, 0)], [wf], [], None, checkpoint="int8"))
    assert (buf[rows:] == 7).all() and (buf[:, n:] == 7).all()
    dy = make(rows, n, torch.float32, 5)
    wide = torch.full((rows + 3, k + 33), 7.0, device="cuda")
    ws = work(lib.inf_linear_ckpt_workspace_bytes(rows, n, k, 0, 1))
    check(lib.inf_linear_ckpt_backward(rows, n, k, rt.ptr(dy), n, 0, None, 0, None, None, 0, None, rt.ptr(wf), k, 1,
                                       rt.ptr(wide), DTYPE_F32, k + 33, None, 0, None, rt.ptr(ws), rt.stream_handle()))
    xg = x.clone().requires_grad_()
    y = d.linear([(xg, 0, 0)], [wf], [], None, checkpoint="int8")
    assert torch.equal(wide[:rows, :k], torch.autograd.grad(y, xg, dy)[0])
    assert (wide[rows:] == 7).all() and (wide[:, k:] == 7).all()


def test_checkpointed_layer_layouts():
    """One weight split by column ranges, columns no segment takes (gradient zero), strided and
    repeated inputs, a transposed weight, gradients of some inputs only, shared rows."""
    d = dense()
    g = torch.Generator().manual_seed(6)
    W = (torch.randn((40, 120), generator=g) * 0.1).cuda().requires_grad_()
    b = torch.randn(40, generator=g).cuda().requires_grad_()
    a, c = make(90, 50, torch.float32, 1, 0.3).requires_grad_(), make(90, 30, torch.float32, 2, 0.3).requires_grad_()
    dy = torch.randn((90, 40), generator=g).cuda()
    y = d.linear([(a, 0, 0), (c, 0, 70)], [W], [b], None, checkpoint="int8")
    y.backward(dy)
    parts = [W.detach()[:, :50], W.detach()[:, 70:100]]
    want = layer64([a, c], parts, [b], None, dy)
    near(y, want["y"])
    near(W.grad[:, :50], want["dw"][0])
    near(W.grad[:, 70:100], want["dw"][1])
    assert (W.grad[:, 50:70] == 0).all() and (W.grad[:, 100:] == 0).all()
    near(a.grad, want["dx"][0])
    near(c.grad, want["dx"][1])
    # strided, repeated, transposed; a gradient that is one number repeated
    base = make(90, 101, torch.float32, 3, 0.3)
    row = make(1, 50, torch.float32, 4).requires_grad_()
    Wt = (torch.randn((50, 40), generator=g) * 0.1).cuda()
    for x in (base[:, 1:51], base[::1, 51:101], row.expand(90, 50), base[:, ::2][:, :50], base.t()[:90, :50]):
        rows = x.shape[0]
        w = Wt.t().detach().requires_grad_()
        y = d.linear([(x, 0, 0)], [w], [b.detach()], "sigmoid", checkpoint="int8")
        y.sum().backward()
        want = layer64([x], [w], [b], "sigmoid", torch.ones((rows, 40)))
        near(y, want["y"])
        near(w.grad, want["dw"][0])
    total = sum(want_row for want_row in layer64([row.expand(90, 50)], [Wt.t()], [b], "sigmoid",
                                                 torch.ones((90, 40)))["dx"][0][0])
    np.testing.assert_allclose(row.grad[0].cpu().double().numpy(), total.numpy(), rtol=1e-4, atol=1e-4)
    # rows made once for two layers; nothing kept where no weight asks
    x = make(64, 48, torch.float32, 9)
    r = d.quantize_rows(x)
    w = (torch.randn((32, 48), generator=g) * 0.1).cuda().requires_grad_()
    y1 = d.linear([(x, 0, 0)], [w], [], None, checkpoint=[r])
    y2 = d.linear([(x, 0, 0)], [w], [], None, checkpoint="int8")
    assert torch.equal(y1, y2)
    dy = torch.randn((64, 32), generator=g).cuda()
    assert torch.equal(torch.autograd.grad(y1, w, dy)[0], torch.autograd.grad(y2, w, dy)[0])
    xg = x.clone().requires_grad_()
    y = d.linear([(xg, 0, 0)], [w.detach()], [], "relu", checkpoint="int8")
    y.backward(dy)
    assert xg.grad is not None


def test_rows_far_apart():
    """Rows that are millions of values apart, of x and of the gradient."""
    d = dense()
    wide = torch.zeros((5, (1 << 21) + 9), device="cuda")
    wide[:, 7:57] = make(5, 50, torch.float32, 1)
    x, w = wide[:, 7:57], torch.randn((20, 50), generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    near_x = x.contiguous()
    r, want = d.quantize_rows(x), d.quantize_rows(near_x)
    assert torch.equal(r.q, want.q) and torch.equal(r.scale, want.scale)
    w8 = d.quantize_weight(w)
    assert torch.equal(d.linear8([x], [w8], []), d.linear8([near_x], [w8], []))
    dy = torch.zeros((5, 1 << 21), device="cuda")[:, 3:23]
    dy.copy_(make(5, 20, torch.float32, 3))
    got = [d.linear([(v, 0, 0)], [w], [], None, checkpoint="int8") for v in (x, near_x)]
    assert torch.equal(*got)
    assert torch.equal(*[torch.autograd.grad(y, w, dy)[0] for y in got])


def test_checkpointed_layer_no_rows_and_bad_rows():
    d = dense()
    xs, ws, bs, dy = leaves(0, 40, (30,), torch.float32)
    y = d.linear([(xs[0], 0, 0)], ws, bs, "relu", checkpoint="int8")
    y.backward(dy)
    assert y.shape == (0, 40) and (ws[0].grad == 0).all() and (bs[0].grad == 0).all() and xs[0].grad.shape == (0, 30)
    xs, ws, bs, dy = leaves(200, 40, (30,), torch.float32, 3)
    x = xs[0].detach().clone()
    x[5, 3], x[9, 0], x[11] = float("nan"), float("inf"), 0
    for act in (None, "relu", "sigmoid"):
        y = d.linear([(x, 0, 0)], ws, bs, act, checkpoint="int8")
        fine = torch.isfinite(y).all(1).cpu()
        assert not fine[5] and fine.sum() >= 198
        if act is None:
            assert not fine[9]
    # gradients of some size next to none at all, in the same call
    dy = dy * torch.logspace(-30, 20, 200).cuda()[:, None]
    want = layer64(xs, ws, bs, None, dy)
    y = d.linear([(xs[0], 0, 0)], ws, bs, None, checkpoint="int8")
    y.backward(dy)
    near(xs[0].grad, want["dx"][0])
    near(ws[0].grad, want["dw"][0])
    near(bs[0].grad, want["db"])


def test_checkpointed_layer_keeps_a_quarter():
    """What lives between forward and backward: 8 bits a value of x and one a ReLU output."""
    d = dense()
    rows, k, n = 8192, 1024, 256
    x, w = make(rows, k, torch.float32), torch.randn((n, k)).cuda().requires_grad_()
    held = {}
    for kept in (None, "int8"):
        y = d.linear([(x.clone(), 0, 0)], [w], [], "relu", checkpoint=kept)
        y.sum().backward()  # first use of everything
        w.grad = None
        torch.cuda.synchronize()
        del y
        base = torch.cuda.memory_allocated()
        y = d.linear([(x.clone(), 0, 0)], [w], [], "relu", checkpoint=kept)
        torch.cuda.synchronize()
        held[kept] = torch.cuda.memory_allocated() - base - rows * n * 4
    assert held["int8"] <= rows * (k + 4) + rows * n // 8 + 4096
    assert held[None] >= rows * k * 4


def test_refusals():
    d = dense()
    x, w = make(8, 16, torch.float32), torch.randn((4, 16)).cuda()
    b = torch.zeros(4).cuda()
    w8 = d.quantize_weight(w)
    for bad in (x[0], x.half(), x.double(), x[:, :0], x.int()):
        with pytest.raises(ValueError):
            d.quantize_rows(bad)
    with pytest.raises(RuntimeError, match="HIP"):
        d.quantize_rows(x.cpu())
    with pytest.raises(ValueError):
        d.quantize_rows(x).restore(torch.float16)
    for args in (([x[:, :15]], [w8], []), ([x], [w8, w8], []), ([], [], []), ([x], [w8], [b, b]), ([x], [w8], [b[:3]]),
                 ([x], [w8], [b.double()]), ([x, x[:4]], [w8, w8], []), ([x.half()], [w8], [])):
        with pytest.raises(ValueError):
            d.linear8(*args)
    with pytest.raises(ValueError):
        d.linear8([x], [w8], [], out=torch.float16)
    with pytest.raises(KeyError):
        d.linear8([x], [w8], [], "tanh")
    with pytest.raises(RuntimeError, match="gradient"):
        d.linear8([x.clone().requires_grad_()], [w8], [])
    with pytest.raises(RuntimeError, match="gradient"):
        d.linear8([x], [w8], [b.clone().requires_grad_()])
    with pytest.raises(RuntimeError, match="HIP"):
        d.linear8([x.cpu()], [w8], [])
    for q, s in ((w, b), (w8.packed.view(-1)[:16], b), (torch.zeros((4, 16), dtype=torch.int8).cuda(), b[:3])):
        with pytest.raises(ValueError):
            d.pack_weight8(q, s)
    with pytest.raises(ValueError):
        d.quantize_weight(w, 10, 10)
    r = d.quantize_rows(x)
    for kw in ({"checkpoint": "int4"}, {"checkpoint": []}, {"checkpoint": [d.quantize_rows(x[:4])]}):
        with pytest.raises(ValueError):
            d.linear([(x, 0, 0)], [w], [b], None, **kw)
    for seg, ws, bs in (([(x, 0, 1)], [w], [b]), ([(x, 0, 0)], [w.double()], [b]), ([(x, 0, 0)], [w], [b[:3]]),
                        ([(x, 0, 0), (x, 0, 0)], [w], [b]), ([(x, 0, 0)], [w, w], [b]), ([(x, 0, -1)], [w], [b]),
                        ([(x, 0, 0), (x[:4], 1, 0)], [w, w], [b])):
        with pytest.raises(ValueError):
            d.linear(seg, ws, bs, None, checkpoint="int8")
    # second derivatives are refused, not wrong
    wg = w.clone().requires_grad_()
    y = d.linear([(x, 0, 0)], [wg], [b], None, checkpoint="int8")
    g = torch.autograd.grad(y.sum(), wg, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()
    assert r.shape == (8, 16)


def test_streams_and_graph_replay():
    """On another stream than the tensors' own, and a captured training step and render layer
    replayed with new inputs, each replay equal to the eager result bit for bit."""
    d = dense()
    xs, ws, bs, dy = leaves(700, 128, (96,), torch.float32, 2)
    w8 = d.quantize_weight(ws[0])

    def step(x, dy):
        x = x.detach().requires_grad_()
        y = d.linear([(x, 0, 0)], ws, bs, "relu", checkpoint="int8")
        g = torch.autograd.grad(y, [x, *ws, *bs], dy)
        r = d.linear8([x.detach()], [w8], [bs[0].detach()], "relu", out=torch.int8)
        return [y.detach(), *g, r.q, r.scale, d.linear8([x.detach()[:1]], [w8], [bs[0].detach()])]

    eager = step(xs[0], dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(xs[0], dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    sx, sdy = xs[0].detach().clone(), dy.clone()
    graphs = []
    for _ in range(2):  # two graphs alive at once: neither may use the other's memory
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(sx, sdy)
        graphs.append((g, out))
    for i in range(4):
        sx.copy_(make(700, 96, torch.float32, 50 + i))
        sdy.copy_(torch.randn((700, 128), generator=torch.Generator().manual_seed(i)))
        for g, _ in graphs:
            g.replay()
        want = step(sx, sdy)
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_two_streams_at_once():
    """Calls of every form on two streams, neither waiting for the other, as one after the other."""
    d = dense()
    sets = []
    for i, (rows, n, k) in enumerate(((33000, 200, 300), (20000, 256, 256), (5, 64, 700), (9000, 300, 400))):
        xs, ws, bs, dy = leaves(rows, n, (k,), torch.float32, i)
        sets.append((xs[0], ws[0], bs[0], dy, d.quantize_weight(ws[0])))

    def calls(s):
        x, w, b, dy, w8 = s
        y = d.linear([(x, 0, 0)], [w], [b], "sigmoid", checkpoint="int8")
        g = torch.autograd.grad(y, [x, w, b], dy)
        with torch.no_grad():
            r = d.linear8([x], [w8], [b], "relu", out=torch.int8)
            return [y.detach(), *g, r.q, r.scale, d.linear8([r], [d.quantize_weight(w.t())], [])]

    want = [calls(s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    got = {}
    for i in range(len(sets)):
        for j, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i, j] = calls(sets[(i + j) % len(sets)])
    torch.cuda.synchronize()
    for (i, j), out in got.items():
        assert all(torch.equal(a, b) for a, b in zip(out, want[(i + j) % len(sets)]))


def test_graph_replay_of_many_rows():
    """The forms for many rows, captured and replayed with the program's own calls in between."""
    d = dense()
    rows, n, k = 33000, 130, 300
    xs, ws, bs, dy = leaves(rows, n, (k,), torch.bfloat16, 4)
    w8, v8 = d.quantize_weight(ws[0]), d.quantize_weight(torch.randn((n, n), device="cuda"))

    def step(x):
        x = x.detach().requires_grad_()
        y = d.linear([(x, 0, 0)], ws, bs, "sigmoid", checkpoint="int8")
        g = torch.autograd.grad(y, [x, *ws, *bs], dy)
        with torch.no_grad():
            h = d.linear8([x], [w8], [], "relu", out=torch.int8)
            return [y.detach(), *g, h.q, h.scale, d.linear8([h], [v8], [], out=torch.bfloat16)]

    sx = xs[0].detach().clone()
    step(sx)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sx)
    for i in range(3):
        sx.copy_(make(rows, k, torch.bfloat16, 60 + i))
        graph.replay()
        want = step(sx)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_more_values_than_32_bits_count():
    """Inputs of more than 2^31 values: the last rows are as they are alone (the checkpointed layer's, whose
    forms for few and many rows sum in other orders, as in 64 bits), and the weight's gradient is exact.  x holds whole numbers up to 127 of 1 / 128, the largest in every row, so that q is they and s
    is 1 / 128; one row in 257 has a gradient, of whole numbers up to 2: no sum passes 2^24."""
    d = dense()
    rows, k, n = (1 << 21) + 4099, 1031, 40
    tail = slice(rows - 300, rows)
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((rows, k), dtype=torch.bfloat16, device="cuda")
    for part in x.split(1 << 18):
        part.copy_(torch.randint(-127, 128, part.shape, generator=g, device="cuda", dtype=torch.int8)).div_(128)
    x[:, 0] = 127 / 128
    assert x.numel() > 1 << 31
    r, want = d.quantize_rows(x), d.quantize_rows(x[tail])
    assert (r.scale == 1 / 128).all()
    assert torch.equal(r.q[tail], want.q) and torch.equal(r.restore(torch.bfloat16)[tail], x[tail])
    qw, sw = weight8(n, k, 1)
    w8 = d.pack_weight8(qw.cuda(), sw.cuda())
    for xin, x_tail in ((x, x[tail]), (r, want)):
        assert torch.equal(d.linear8([xin], [w8], [], "relu")[tail], d.linear8([x_tail], [w8], [], "relu"))
    c8 = d.pack_weight8(qw[:, :1000].contiguous().cuda(), sw.cuda())  # the form for up to 1024 values
    assert torch.equal(d.linear8([x[:, :1000]], [c8], [])[tail], d.linear8([x[tail, :1000]], [c8], []))
    del r, xin
    some = torch.arange(rows - 1, -1, -257, device="cuda")
    for cols in (n, 66):  # (66: the form that holds whole rows of dz)
        w = (torch.randn((cols, k), generator=torch.Generator().manual_seed(cols)) * 0.1).cuda().requires_grad_()
        dy = torch.zeros((rows, cols), device="cuda")
        dy[some] = torch.randint(-2, 3, (len(some), cols), generator=g, device="cuda").float()
        xg = x.detach().requires_grad_()
        y = d.linear([(xg, 0, 0)], [w], [], None, checkpoint="int8")
        dx, dw = torch.autograd.grad(y, [xg, w], dy)
        want = layer64([x[tail]], [w], [], None, dy[tail])
        near(y[tail], want["y"])
        near(dx[tail], want["dx"][0], torch.bfloat16)
        assert torch.equal(dw.cpu().double(), dy[some].cpu().double().t() @ x[some].cpu().double())
        del y, dx, xg, dy


def test_repeats_are_equal():
    """No result depends on the order in which the device finishes."""
    d = dense()
    xs, ws, bs, dy = leaves(40000, 200, (300,), torch.float32, 2)
    first = None
    w8 = d.quantize_weight(ws[0])
    for _ in range(3):
        y = d.linear([(xs[0], 0, 0)], ws, bs, "relu", checkpoint="int8")
        got = [y.detach(), *torch.autograd.grad(y, [*xs, *ws, *bs], dy)]
        r = d.linear8([xs[0].detach()], [w8], [], out=torch.int8)
        got += [r.q, r.scale]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))
