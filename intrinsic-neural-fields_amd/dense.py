"""Autograd over the generic fp32 dense-layer kernels (csrc/dense.hip) for the layers the
fused plan does not cover: the view-dependent texture field (reference model.py:115-191)
-- a TextureField ending in a ReLU bottleneck, plus the two-layer directional MLP.

`linear(segments, bias, act)` computes act(sum_s x_s @ W_s[:, c_s:c_s + K_s]^T + sum bias)
in one output buffer: a plain nn.Linear (one segment), LinearWithConcatAndActivation
(layers.py:60-62: two weights, two biases) or a Linear over a concatenated input
(model.py:186-191: one weight split by column ranges) without materialising the concat.
Every product, activation, gradient and bias sum runs in libinf_hip.so; torch only
allocates.

In 8 bits (csrc/quant.hpp: whole numbers q and one scale s a row, x ~ s q):
`linear(..., checkpoint="int8")` keeps the inputs in 8 bits between forward and backward
(a quarter of the memory; ReLU's outputs as one bit each), with products in 16-bit pieces or, at
products="fp32", as without; `linear8` multiplies 8-bit rows
with 8-bit weights for rendering, and `quantize_rows` / `Rows8.restore` are the rows
themselves.

A training step of these layers that is captured into a HIP graph captures its forward too:
autograd ties a leaf's gradient accumulation to the stream of its first live graph, so no
eager graph of the same parameters may be alive while a backward pass is captured.
"""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

ACT = {None: 0, "relu": 1, "sigmoid": 2}


_runtime = None


def _rt():
    global _runtime
    if _runtime is None:
        from inf_hip import runtime  # raises if the HIP library is missing: no fallback
        _runtime = runtime
    return _runtime


def _gemm(M, N, K, A, sam, sak, B, sbn, sbk, bias, act, beta, C, ldc):
    rt = _rt()
    from inf_hip import lib
    rt.check(lib.inf_dense_gemm(M, N, K, rt.ptr(A), sam, sak, rt.ptr(B), sbn, sbk, rt.ptr(bias), act, float(beta),
                                rt.ptr(C), ldc, rt.stream_handle()), "dense_gemm")


def _products(spec, act, xs, ws, bs, y):
    """y = act(sum_s x_s W_s[:, c_s:]^T + sum bias), in fp32."""
    rows, n = y.shape
    for s, (wi, c0) in enumerate(spec):
        x, W = xs[s], ws[wi]
        _gemm(rows, n, x.shape[1], x, x.stride(0), x.stride(1), W[:, c0:], W.stride(0), W.stride(1),
              bs[s] if s < len(bs) else None, act if s == len(spec) - 1 else 0, 0.0 if s == 0 else 1.0, y, n)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, spec, act, *tensors):
        # spec: per segment (weight index, column offset); tensors: xs..., weights..., biases...
        nseg = len(spec)
        nw = max(w for w, _ in spec) + 1
        xs, ws, bs = tensors[:nseg], tensors[nseg:nseg + nw], tensors[nseg + nw:]
        B = xs[0].shape[0]
        N = ws[0].shape[0]
        y = torch.empty((B, N), dtype=torch.float32, device=xs[0].device)
        _products(spec, act, xs, ws, bs, y)
        ctx.spec, ctx.act, ctx.nw, ctx.nb = spec, act, nw, len(bs)
        ctx.save_for_backward(*xs, *ws, y)
        return y

    @staticmethod
    def backward(ctx, dy):
        rt = _rt()
        from inf_hip import lib
        spec, act, nw, nb = ctx.spec, ctx.act, ctx.nw, ctx.nb
        saved = ctx.saved_tensors
        nseg = len(spec)
        xs, ws, y = saved[:nseg], saved[nseg:nseg + nw], saved[-1]
        dy = dy.contiguous().to(torch.float32)
        B, N = y.shape
        if act:
            dz = torch.empty_like(y)
            rt.check(lib.inf_dense_act_bwd(y.numel(), rt.ptr(y), rt.ptr(dy), act, rt.ptr(dz), rt.stream_handle()),
                     "dense_act_bwd")
        else:
            dz = dy
        needs = ctx.needs_input_grad[2:]
        dxs = [None] * nseg
        dws = [None] * nw
        for s, (wi, c0) in enumerate(spec):
            x, W = xs[s], ws[wi]
            K = x.shape[1]
            if needs[s]:
                dx = torch.empty((B, K), dtype=torch.float32, device=y.device)
                # dx[b][k] = sum_n dz[b][n] W[n][c0 + k]
                _gemm(B, K, N, dz, N, 1, W[:, c0:], W.stride(1), W.stride(0), None, 0, 0.0, dx, K)
                dxs[s] = dx
            if needs[nseg + wi]:
                if dws[wi] is None:
                    dws[wi] = torch.empty(W.shape, dtype=torch.float32, device=y.device)
                g = dws[wi]
                # dW[n][c0 + k] = sum_b dz[b][n] x[b][k]
                _gemm(N, K, B, dz, 1, N, x, x.stride(1), x.stride(0), None, 0, 0.0, g[:, c0:], g.stride(0))
        dbs = []
        for i in range(nb):
            if needs[nseg + nw + i]:
                db = torch.empty(N, dtype=torch.float32, device=y.device)
                rt.check(lib.inf_colsum(B, N, rt.ptr(dz), N, rt.ptr(db), 0, rt.stream_handle()), "colsum")
                dbs.append(db)
            else:
                dbs.append(None)
        return (None, None, *dxs, *dws, *dbs)


def linear(segments, weights, biases, act=None, checkpoint=None, products=None):
    """segments: [(x_s, weight index, column offset)]; weights / biases: lists of tensors.

    checkpoint="int8": x_s (fp32, or bf16 taken as it is) is kept in 8 bits for the backward,
    where dW_s = dz^T (s q)_s; the output, dx_s and the bias gradients do not depend on it.
    A list names it for each segment: "int8", or the `Rows8` of that x_s where several layers
    read the same tensor.  Its products are not quite fp32's: a value counts to 2^-23 of itself, or
    to 2^-39 of the largest of its row (of x and dz; of W, its row forward, its column for dx) where
    that is more, a product to 2^-21; a term of dW to 2^-24 of itself, or to 2^-126 where that is
    more; their sums are fp32, in another order; a row of x with an infinity or a NaN gives NaN,
    and one whose largest value is below 2^-143 counts as zeros.  products="fp32" leaves all but dW
    as it is without a checkpoint, bit for bit, and takes the time of those products.  A weight has
    less than 2^29 values (rows and columns counted in 256s).  (As with every layer here: a
    backward is captured into a graph only while no eager graph of the same leaves is alive.)"""
    for t in [x for x, _, _ in segments] + list(weights) + list(biases):
        if not t.is_cuda:
            raise RuntimeError("the dense layers run on the HIP device only; there is no CPU fallback")
    if products not in (None, "fp32"):
        raise ValueError(f'products are "fp32" or, with a checkpoint, its own (None), not {products!r}')
    spec = tuple((wi, c0) for _, wi, c0 in segments)
    if checkpoint is not None:
        return _linear_ckpt(segments, spec, weights, biases, ACT[act], checkpoint, products)
    xs = [x.to(torch.float32) for x, _, _ in segments]
    return _Linear.apply(spec, ACT[act], *xs, *weights, *biases)


# ---- 8 bits -------------------------------------------------------------------------
# (These calls are short: addresses go to the library as plain numbers, and each allocation
# counts.)

_ON_CURRENT = contextlib.nullcontext()


def _on(device):
    """The device of the tensors as the current one, for launches on its current stream."""
    return _ON_CURRENT if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _at(t):
    return None if t is None else t.data_ptr()


def _round_up(n, m):
    return (n + m - 1) // m * m


def _rows_of(x, what):
    """x as rows whose values are next to each other (any distance between rows)."""
    if x.dim() != 2 or x.shape[1] < 1:
        raise ValueError(f"{what} must be a matrix [rows, k] with k >= 1, got {list(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"{what} must be fp32 or bf16, got {x.dtype}")
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _near(x):
    """x with rows less than 2^21 values apart, as the checkpointed layer's products take them."""
    # (of one row or none contiguous() is x itself, whatever the distance)
    return x if x.stride(0) < 1 << 21 else x.clone(memory_format=torch.contiguous_format)


def _has_tangent(x):
    """x is a dual tensor: forward-mode differentiation (also under no_grad) asks for its derivative."""
    return forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None


class Rows8:
    """The rows of a matrix in 8 bits: `q` int8 [rows, k] (rows start on 16 bytes) and
    `scale` fp32 [rows], standing for scale[:, None] * q.  Made by quantize_rows and linear8."""

    __slots__ = ("q", "scale")

    def __init__(self, rows, k, device):
        ld = _round_up(k, 16)
        # 128 bytes behind the last row: a product may read past it (include/inf_hip.h)
        self.q = torch.empty(rows * ld + 128, dtype=torch.int8, device=device).as_strided((rows, k), (ld, 1))
        self.scale = torch.empty(rows, dtype=torch.float32, device=device)

    @property
    def shape(self):
        return self.q.shape

    @property
    def device(self):
        return self.q.device

    def restore(self, dtype=torch.float32):
        """scale * q, rounded to fp32; bf16: that rounded again."""
        rt = _rt()
        if dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"8-bit rows are restored to fp32 or bf16, not {dtype}")
        q = self.q
        rows, k = q.shape
        out = torch.empty((rows, k), dtype=dtype, device=q.device)
        with _on(q.device):
            rt.check(rt.lib.inf_restore_rows(q.data_ptr(), q.stride(0), self.scale.data_ptr(), rows, k, out.data_ptr(),
                                             rt.dtype_code(out), k, _stream(q.device)), "restore_rows")
        return out


def quantize_rows(x):
    """x [rows, k] fp32 / bf16 in 8 bits: scale = fl(max|x| fl(1 / 127)) of each row, q the whole
    number nearest to 127 x / max|x| (the ratio itself; ties to even).  Rows of zeros have scale 0 (so have rows whose
    largest value is below 2^-143); a row with an infinity or a NaN has scale NaN, and whatever
    is made of it is NaN.  No gradient: x counts as detached, and a dual tensor of forward-mode
    differentiation is refused."""
    rt = _rt()
    rt.require_hip(x)
    if _has_tangent(x):
        raise RuntimeError("8-bit rows have no derivative: quantize_rows takes no dual tensor")
    x = _rows_of(x.detach(), "x")
    rows, k = x.shape
    r = Rows8(rows, k, x.device)
    with _on(x.device):
        rt.check(rt.lib.inf_quantize_rows(x.data_ptr(), rt.dtype_code(x), rows, k, x.stride(0), r.q.data_ptr(),
                                          r.q.stride(0), r.scale.data_ptr(), _stream(x.device)), "quantize_rows")
    return r


class Weight8:
    """A weight [n, k] in 8 bits with one scale a row, laid out for linear8 (`packed`)."""

    __slots__ = ("packed", "scale", "n", "k")

    def __init__(self, packed, scale, n, k):
        self.packed, self.scale, self.n, self.k = packed, scale, n, k


def pack_weight8(q, scale):
    """8-bit weights q int8 [n, k] (any strides) with scales fp32 [n], laid out for linear8."""
    rt = _rt()
    rt.require_hip(q, scale)
    if q.dim() != 2 or q.dtype != torch.int8 or min(q.shape) < 1:
        raise ValueError("an 8-bit weight is an int8 matrix [n, k]")
    n, k = q.shape
    if scale.shape != (n,) or scale.dtype != torch.float32 or scale.device != q.device:
        raise ValueError("an 8-bit weight has one fp32 scale a row, on its device")
    packed = torch.empty(int(rt.lib.inf_packed_weight_bytes(n, k)), dtype=torch.int8, device=q.device)
    with _on(q.device):
        rt.check(rt.lib.inf_pack_weight(q.data_ptr(), q.stride(0), q.stride(1), n, k, packed.data_ptr(),
                                        _stream(q.device)), "pack_weight")
    return Weight8(packed, scale.clone(), n, k)


def quantize_weight(W, col0=0, cols=None):
    """W[:, col0:col0 + cols] (fp32 / bf16) in 8 bits, laid out for linear8."""
    cols = W.shape[1] - col0 if cols is None else cols
    if col0 < 0 or cols < 1 or col0 + cols > W.shape[1]:
        raise ValueError(f"columns {col0}..{col0 + cols} of a weight with {W.shape[1]}")
    r = quantize_rows(W[:, col0:col0 + cols])
    return pack_weight8(r.q, r.scale)


def linear8(xs, weights, biases, act=None, out=torch.float32):
    """act(sum_s x_s W_s^T + sum bias) with the rows of x_s and W_s in 8 bits: the sums of their
    products are exact, and scales, bias and the sum over s are one fp32 rounding each.

    xs: for each segment a matrix fp32 / bf16 (put into 8 bits on the way) or a Rows8;
    weights: a Weight8 each; biases: fp32 [n], one for each of the first segments.
    out: torch.float32, torch.bfloat16 (the fp32 result rounded again), or torch.int8 for a Rows8
    of the fp32 result.
    For rendering: it has no gradient, and refuses inputs that ask for one, in forward mode too."""
    rt = _rt()
    i8 = rt.DTYPE_I8
    code = i8 if out is torch.int8 else rt.DTYPE_F32 if out is torch.float32 else \
        rt.DTYPE_BF16 if out is torch.bfloat16 else None
    if code is None:
        raise ValueError(f"linear8 gives fp32, bf16 or int8 rows, not {out}")
    if len(xs) < 1 or len(xs) != len(weights) or len(biases) > len(xs):
        raise ValueError("linear8 takes one weight and at most one bias for each segment")
    rows, n, device = xs[0].shape[0], weights[0].n, xs[0].device
    acc, last, lib, a = None, len(xs) - 1, rt.lib, ACT[act]
    recorded, dual = torch.is_grad_enabled(), forward_ad._current_level >= 0
    if device.type != "cuda":
        rt.require_hip(xs[0].q if isinstance(xs[0], Rows8) else xs[0])
    with _on(device):
        for s, (x, w) in enumerate(zip(xs, weights)):
            if isinstance(x, Rows8):
                q, scale, xc = x.q, x.scale.data_ptr(), i8
            else:
                if (recorded and x.requires_grad) or (dual and _has_tangent(x)):
                    raise RuntimeError("linear8 has no gradient: call it under torch.no_grad(), or train with linear")
                q, scale = _rows_of(x, "x"), None
                xc = rt.dtype_code(q)
            if q.shape[0] != rows or q.shape[1] != w.k or w.n != n:
                raise ValueError(f"segment {s}: x {list(q.shape)} and weight [{w.n}, {w.k}] do not fit [{rows}, {n}]")
            b = biases[s] if s < len(biases) else None
            if b is not None and (b.shape != (n,) or b.dtype != torch.float32 or not b.is_contiguous()):
                raise ValueError("a bias is a contiguous fp32 [n] tensor")
            if b is not None and ((recorded and b.requires_grad) or (dual and _has_tangent(b))):
                raise RuntimeError("linear8 has no gradient: call it under torch.no_grad(), or train with linear")
            if q.device != device or w.packed.device != device or (b is not None and b.device != device):
                raise ValueError("linear8 takes its tensors on one device")
            oc = code if s == last else rt.DTYPE_F32
            if oc == i8:
                y = Rows8(rows, n, device)
                op, ldo, osc = y.q.data_ptr(), y.q.stride(0), y.scale.data_ptr()
            else:
                y = torch.empty((rows, n), dtype=out if s == last else torch.float32, device=device)
                op, ldo, osc = y.data_ptr(), n, None
            to = a if s == last else 0
            nws = lib.inf_linear_int_call_workspace_bytes(rows, n, w.k, xc, oc, to, acc is not None)
            ws = torch.empty(nws, dtype=torch.uint8, device=device) if nws else None
            rt.check(lib.inf_linear_int(rows, n, w.k, q.data_ptr(), xc, q.stride(0), scale, w.packed.data_ptr(),
                                        w.scale.data_ptr(), _at(b), _at(acc), n, to, op, oc, ldo,
                                        osc, _at(ws), _stream(device)), "linear_int")
            acc = y
    return y


def _workspace(lib, rows, n, widths, backward, device):
    """One for all segments of a layer: their launches follow each other."""
    need = max([lib.inf_linear_ckpt_workspace_bytes(rows, n, k, 0, backward) for k in widths])
    return torch.empty(need, dtype=torch.uint8, device=device)


class _LinearCkpt(torch.autograd.Function):
    @staticmethod
    def forward(ctx, spec, act, kept, recorded, *tensors):
        # spec and tensors as _Linear; kept: per segment the Rows8 of x, or None to make them;
        # recorded: whether gradients are (needs_input_grad says what the tensors ask for, also
        # under no_grad; in here nothing is ever recorded)
        rt = _rt()
        lib = rt.lib
        nseg = len(spec)
        nb = len(tensors) - nseg
        nw = max(w for w, _ in spec) + 1
        nb -= nw
        needs = ctx.needs_input_grad if recorded else (False,) * (4 + len(tensors))
        W0 = tensors[nseg]
        rows, n, device = tensors[0].shape[0], W0.shape[0], W0.device
        # one allocation for what is kept: each segment's q and scale, then the mask
        at, places = 0, []
        for s, (wi, _) in enumerate(spec):
            make = needs[4 + nseg + wi] and kept[s] is None
            places.append(at if make else None)
            if make:
                at += _round_up(rows * _round_up(tensors[s].shape[1], 16) + 128, 256) + _round_up(rows * 4, 256)
        mask_at = at if act == 1 and any(needs) else None
        if mask_at is not None:
            at += rows * ((n + 31) // 32) * 4
        with _on(device):
            st = _stream(device)
            y = torch.empty((rows, n), dtype=torch.float32, device=device)
            yp = y.data_ptr()
            held = torch.empty(at, dtype=torch.uint8, device=device) if at else None
            base = held.data_ptr() if at else 0
            work = _workspace(lib, rows, n, [x.shape[1] for x in tensors[:nseg]], 0, device)
            for s, (wi, c0) in enumerate(spec):
                x, W = tensors[s], tensors[nseg + wi]
                k, last, own = x.shape[1], s == nseg - 1, kept[s]
                ldq = _round_up(k, 16)
                q = scale = None
                if places[s] is not None:
                    q = base + places[s]
                    scale = q + _round_up(rows * ldq + 128, 256)
                elif own is not None:
                    scale = own.scale.data_ptr()
                xc = rt.dtype_code(x)
                rt.check(lib.inf_linear_ckpt_forward(
                    rows, n, k, x.data_ptr(), xc, x.stride(0), W.data_ptr() + 4 * c0 * W.stride(1), W.stride(0),
                    W.stride(1), tensors[nseg + nw + s].data_ptr() if s < nb else None, yp if s else None, n,
                    act if last else 0, yp, n, base + mask_at if last and mask_at is not None else None, q, ldq, scale,
                    work.data_ptr(), st), "linear_ckpt_forward")
        if not recorded:
            return y
        ctx.layer = (spec, act, nw, nb, rows, n, places, mask_at, [t.shape[1] for t in tensors[:nseg]],
                     [t.dtype for t in tensors[:nseg]])
        save = [held, y if act == 2 else None, *tensors[nseg:nseg + nw]]
        for own in kept:
            if own is not None:
                save += [own.q, own.scale]
        ctx.kept = [own is not None for own in kept]
        ctx.save_for_backward(*save)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rt = _rt()
        lib = rt.lib
        spec, act, nw, nb, rows, n, places, mask_at, widths, dtypes = ctx.layer
        nseg = len(spec)
        saved = ctx.saved_tensors
        held, y, ws = saved[0], saved[1], saved[2:2 + nw]
        own = iter(saved[2 + nw:])
        needs = ctx.needs_input_grad
        if dy.dtype != torch.float32:
            dy = dy.to(torch.float32)
        if dy.stride(1) != 1 or dy.stride(0) < n:
            dy = dy.contiguous()
        dy = _near(dy)
        device = dy.device
        base = held.data_ptr() if held is not None else 0
        grads = [None] * (4 + nseg + nw + nb)
        with _on(device):
            st = _stream(device)
            work = _workspace(lib, rows, n, widths, 1, device)
            for s, (wi, c0) in enumerate(spec):
                W, k = ws[wi], widths[s]
                ldq = _round_up(k, 16)
                q = scale = None
                if places[s] is not None:
                    q = base + places[s]
                    scale = q + _round_up(rows * ldq + 128, 256)
                elif ctx.kept[s]:
                    qt, st_ = next(own), next(own)
                    q, scale, ldq = qt.data_ptr(), st_.data_ptr(), qt.stride(0)
                dx = dw = db = None
                if needs[4 + s]:
                    grads[4 + s] = dx = torch.empty((rows, k), dtype=dtypes[s], device=device)
                if needs[4 + nseg + wi]:
                    if grads[4 + nseg + wi] is None:
                        grads[4 + nseg + wi] = _weight_gradient(spec, widths, wi, W)
                    dw = grads[4 + nseg + wi].data_ptr() + 4 * c0
                if s < nb and needs[4 + nseg + nw + s]:
                    grads[4 + nseg + nw + s] = db = torch.empty(n, dtype=torch.float32, device=device)
                if dx is None and dw is None and db is None:
                    continue
                xc = rt.dtype_code(dx) if dx is not None else rt.DTYPE_F32
                rt.check(lib.inf_linear_ckpt_backward(
                    rows, n, k, dy.data_ptr(), dy.stride(0), act, _at(y), n,
                    base + mask_at if mask_at is not None else None, q, ldq, scale,
                    W.data_ptr() + 4 * c0 * W.stride(1), W.stride(0), W.stride(1), _at(dx), xc, k, dw, W.shape[1],
                    _at(db), work.data_ptr(), st), "linear_ckpt_backward")
        return tuple(grads)


class _LinearKept(torch.autograd.Function):
    """_Linear's products, with the inputs kept in 8 bits and a ReLU's output as bits for the backward."""

    @staticmethod
    def forward(ctx, spec, act, kept, recorded, *tensors):
        # as _LinearCkpt; x fp32
        rt = _rt()
        lib = rt.lib
        nseg = len(spec)
        nw = max(w for w, _ in spec) + 1
        xs, ws, bs = tensors[:nseg], tensors[nseg:nseg + nw], tensors[nseg + nw:]
        needs = ctx.needs_input_grad
        rows, n, device = xs[0].shape[0], ws[0].shape[0], xs[0].device
        with _on(device):
            y = torch.empty((rows, n), dtype=torch.float32, device=device)
            _products(spec, act, xs, ws, bs, y)
            if not recorded:
                return y
            kept = [(r or quantize_rows(x)) if needs[4 + nseg + wi] else None for r, x, (wi, _) in zip(kept, xs, spec)]
            out = y if act == 2 else None
            if act == 1 and any(needs):
                out = torch.empty((rows, (n + 31) // 32), dtype=torch.int32, device=device)
                rt.check(lib.inf_relu_mask(rows, n, y.data_ptr(), n, out.data_ptr(), _stream(device)), "relu_mask")
        ctx.layer = (spec, act, nw, len(bs), rows, n, [x.shape[1] for x in xs], [r is not None for r in kept])
        ctx.save_for_backward(out, *ws, *[t for r in kept if r is not None for t in (r.q, r.scale)])
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        rt = _rt()
        lib = rt.lib
        spec, act, nw, nb, rows, n, widths, has_rows = ctx.layer
        nseg = len(spec)
        out, ws = ctx.saved_tensors[0], ctx.saved_tensors[1:1 + nw]
        rows8 = iter(ctx.saved_tensors[1 + nw:])
        needs = ctx.needs_input_grad
        dy = dy.to(torch.float32).contiguous()
        device = dy.device
        grads = [None] * (4 + nseg + nw + nb)
        with _on(device):
            st = _stream(device)
            dz = dy if act == 0 else torch.empty_like(dy)
            if act == 1:
                rt.check(lib.inf_relu_mask_bwd(rows, n, dy.data_ptr(), n, out.data_ptr(), dz.data_ptr(), n, st),
                         "relu_mask_bwd")
            elif act == 2:
                rt.check(lib.inf_dense_act_bwd(dz.numel(), out.data_ptr(), dy.data_ptr(), act, dz.data_ptr(), st),
                         "dense_act_bwd")
            work = _workspace(lib, rows, n, widths, 1, device) if any(has_rows) else None
            for s, (wi, c0) in enumerate(spec):
                W, k = ws[wi], widths[s]
                if needs[4 + s]:
                    grads[4 + s] = dx = torch.empty((rows, k), dtype=torch.float32, device=device)
                    _gemm(rows, k, n, dz, n, 1, W[:, c0:], W.stride(1), W.stride(0), None, 0, 0.0, dx, k)
                if has_rows[s]:
                    q, scale = next(rows8), next(rows8)
                    if grads[4 + nseg + wi] is None:
                        grads[4 + nseg + wi] = _weight_gradient(spec, widths, wi, W)
                    dw = grads[4 + nseg + wi].data_ptr() + 4 * c0
                    rt.check(lib.inf_linear_ckpt_backward(
                        rows, n, k, dz.data_ptr(), n, 0, None, n, None, q.data_ptr(), q.stride(0), scale.data_ptr(), None,
                        0, 0, None, rt.DTYPE_F32, k, dw, W.shape[1], None, work.data_ptr(), st), "linear_ckpt_backward")
                if s < nb and needs[4 + nseg + nw + s]:
                    grads[4 + nseg + nw + s] = db = torch.empty(n, dtype=torch.float32, device=device)
                    rt.check(lib.inf_colsum(rows, n, dz.data_ptr(), n, db.data_ptr(), 0, st), "colsum")
        return tuple(grads)


def _weight_gradient(spec, widths, wi, W):
    """For the segments' columns of W to be written; zeros where no segment takes some of them."""
    covered = sum(k for (wj, _), k in zip(spec, widths) if wj == wi) == W.shape[1]
    return (torch.empty if covered else torch.zeros)(W.shape, dtype=torch.float32, device=W.device)


def _linear_ckpt(segments, spec, weights, biases, act, checkpoint, products):
    kept = [checkpoint] * len(segments) if isinstance(checkpoint, str) else list(checkpoint)
    if len(kept) != len(segments) or any(not isinstance(c, Rows8) and c != "int8" for c in kept):
        raise ValueError('checkpoint is "int8", or for each segment "int8" or the Rows8 of its input')
    if not segments or not weights or len(biases) > len(segments):
        raise ValueError("linear takes at least one segment and at most one bias for each")
    if max(w for w, _ in spec) + 1 != len(weights) or min(w for w, _ in spec) < 0:
        raise ValueError("every weight belongs to a segment")
    xs = [_near(_rows_of(x if x.dtype in (torch.float32, torch.bfloat16) else x.to(torch.float32), "x"))
          for x, _, _ in segments]
    rows, device = xs[0].shape[0], xs[0].device
    n = weights[0].shape[0]
    for W in weights:
        if W.dim() != 2 or W.dtype != torch.float32 or W.shape[0] != n or n < 1:
            raise ValueError("weights are fp32 matrices with the same number of rows")
    for b in biases:
        if b.shape != (n,) or b.dtype != torch.float32 or not b.is_contiguous():
            raise ValueError("a bias is a contiguous fp32 [n] tensor")
    taken = []
    for (wi, c0), x, c in zip(spec, xs, kept):
        k = x.shape[1]
        if x.shape[0] != rows or c0 < 0 or c0 + k > weights[wi].shape[1]:
            raise ValueError(f"x {list(x.shape)} at column {c0} does not fit weight {list(weights[wi].shape)}")
        if any(wi == w and c0 < b and a < c0 + k for w, a, b in taken):
            raise ValueError("segments of one weight take separate columns")
        taken.append((wi, c0, c0 + k))
        if c != "int8" and (c.shape != x.shape or c.device != device):
            raise ValueError(f"checkpoint {list(c.shape)} is not of x {list(x.shape)}")
    for t in (*xs, *weights, *biases):
        if t.device != device:
            raise ValueError("linear takes its tensors on one device")
    layer = _LinearCkpt
    if products == "fp32":
        for x in xs:  # what dW's product takes (include/inf_hip.h), before the backward finds out
            k = x.shape[1]
            if max(_round_up(n, 256) * _round_up(k, 64), _round_up(k, 256) * _round_up(n, 64)) >= 1 << 29:
                raise RuntimeError(f"linear with a checkpoint: a weight of {n} x {k} is too large")
        layer, xs = _LinearKept, [x.to(torch.float32) for x in xs]
    return layer.apply(spec, act, tuple(None if isinstance(c, str) else c for c in kept), torch.is_grad_enabled(),
                       *xs, *weights, *biases)


def view_angles(unit_dirs, face_idxs, face_normals):
    """model.py:164-169: acos(cos_sim(-dirs, normals[face])), [B]."""
    rt = _rt()
    from inf_hip import lib
    d = unit_dirs.to(torch.float32).contiguous()
    f = face_idxs.to(torch.int64).contiguous()
    nrm = face_normals.to(torch.float32).contiguous()
    out = torch.empty(d.shape[0], dtype=torch.float32, device=d.device)
    rt.check(lib.inf_view_angle(d.shape[0], rt.ptr(d), rt.ptr(f), rt.ptr(nrm), nrm.shape[0], rt.ptr(out),
                                rt.stream_handle()), "view_angle")
    return out


def ff_encode(x, bands, include_input):
    """FourierFeatEnc.forward (layers.py:21-25) for inputs of any width d: [.., 2dk (+d)]."""
    rt = _rt()
    from inf_hip import lib
    lead, d = x.shape[:-1], x.shape[-1]
    xf = x.reshape(-1, d).to(torch.float32).contiguous()
    k = bands.shape[0]
    w = 2 * d * k + (d if include_input else 0)
    out = torch.empty((xf.shape[0], w), dtype=torch.float32, device=xf.device)
    b = bands.to(torch.float32).contiguous()
    rt.check(lib.inf_ff_encode(xf.shape[0], d, rt.ptr(xf), rt.ptr(b), k, int(include_input), rt.ptr(out), w,
                               rt.stream_handle()), "ff_encode")
    return out.view(*lead, w)


def adam_step(p, grad, exp_avg, exp_avg_sq, step, lr, beta1, beta2, eps):
    rt = _rt()
    from inf_hip import lib
    for t in (p, grad, exp_avg, exp_avg_sq):
        if not (t.is_cuda and t.is_contiguous() and t.dtype == torch.float32):
            raise RuntimeError("HIP Adam needs contiguous fp32 device tensors")
    rt.check(lib.inf_adam_dense(p.numel(), rt.ptr(p), rt.ptr(grad), rt.ptr(exp_avg), rt.ptr(exp_avg_sq), int(step),
                                float(lr), float(beta1), float(beta2), float(eps), rt.stream_handle()), "adam_dense")
