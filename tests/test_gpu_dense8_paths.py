"""The 8-bit dense layers as the view-dependent field uses them: a training step with 8-bit
checkpoints and a render on 8-bit rows and weights, against the field without them and against
the same layers written out in 64 bits."""
import types

import numpy as np
import pytest
import torch

from test_dense8_cpu import field
from test_gpu_dense8 import U32, oracle_rows, rows64

pytestmark = pytest.mark.gpu


def batch_of(rows, seed=0):
    g = torch.Generator().manual_seed(seed)
    d = torch.randn((rows, 3), generator=g)
    return {"eigenfunctions": torch.randn((rows, 32), generator=g).cuda(),
            "unit_ray_dirs": (d / d.norm(dim=1, keepdim=True)).cuda(),
            "hit_face_idxs": torch.zeros(rows, dtype=torch.int64).cuda()}


def pair(**kernels):
    torch.manual_seed(0)
    a = field().cuda()
    torch.manual_seed(0)
    return a, field(**kernels).cuda()


def test_training_step_with_checkpoints():
    """Outputs and the gradients that do not go through the kept rows: fp32 (a ReLU next to its
    border may fall either way, so the gradients are compared as a whole).  Weight gradients:
    a row's relative rounding is at most 1 / 254 of its largest value, so a gradient is off by
    less than 1 / 100 of its own size here."""
    a, b = pair(dense_checkpoints="int8")
    batch = batch_of(700)
    target = torch.rand((700, 3), generator=torch.Generator().manual_seed(1)).cuda()
    for m in (a, b):
        (m(batch) - target).square().mean().backward()
    assert float((a(batch) - b(batch)).detach().abs().max()) <= 64 * U32 * 8
    for (name, p), q in zip(a.named_parameters(), b.parameters()):
        err = float((p.grad - q.grad).norm() / p.grad.norm())
        assert err < (1e-4 if name.endswith("bias") else 1e-2), (name, err)


def test_no_gradient_no_difference_in_training():
    """dense_inference is for calls without gradients only."""
    a, b = pair(dense_inference="int8")
    batch = batch_of(300)
    ya, yb = a(batch), b(batch)
    assert torch.equal(ya, yb)
    ga = torch.autograd.grad(ya.sum(), list(a.parameters()))
    gb = torch.autograd.grad(yb.sum(), list(b.parameters()))
    assert all(torch.equal(x, y) for x, y in zip(ga, gb))


@torch.no_grad()
def layers64(m, batch):
    """The 8-bit forward in 64 bits but for the fp32 roundings that the definition names."""
    import dense

    def put(z):  # fp32 rows into 8 bits
        q, _ = oracle_rows(z)
        s = z.abs().amax(1).float() * torch.tensor(1.0 / 127.0, dtype=torch.float32)
        return torch.from_numpy(q).double(), s

    def lin(xs, ws, bs, act):
        z = None
        for i, ((q, s), w) in enumerate(zip(xs, ws)):
            qw, sw = rows64(w.detach())
            t = (q @ qw.t()).float() * (s[:, None] * sw.float()[None, :])
            t = t + (bs[i].detach().cpu() if i < len(bs) else 0)
            z = t if z is None else t + z
        return torch.relu(z) if act == "relu" else 1 / (1 + torch.exp(-z))

    x = put(batch["eigenfunctions"].cpu())
    h = x
    for i, layer in enumerate(m.spatial_mlp.layers):
        if i == m.spatial_mlp.skip_layer_idx:
            h = put(lin([h, x], [layer.Lx.weight, layer.Ly.weight], [layer.Lx.bias, layer.Ly.bias], "relu"))
        else:
            h = put(lin([h], [layer[0].weight], [layer[0].bias], "relu"))
    view = put(m._get_embedded_view_dir(batch).cpu())
    l0, l2 = m.directional_mlp[0], m.directional_mlp[2]
    c = m.bottleneck_vec_dim
    h = put(lin([h, view], [l0.weight[:, :c], l0.weight[:, c:]], [l0.bias], "relu"))
    return lin([h], [l2.weight], [l2.bias], "sigmoid")


def test_render_layers():
    a, b = pair(dense_inference="int8")
    batch = batch_of(900)
    with torch.no_grad():
        ya, yb = a(batch), b(batch)
        with b.weights_laid_out():
            assert torch.equal(b(batch), yb) and torch.equal(b({k: v[:1] for k, v in batch.items()}), yb[:1])
        assert b._weights8 is None
    # the layers' own roundings: equal but for the last sigmoid's few steps
    assert float((yb.cpu() - layers64(b, batch)).abs().max()) <= 8 * U32
    assert 0 < float((ya - yb).abs().max()) < 0.05  # and near the fp32 field's colours
    # new weights are seen at once
    with torch.no_grad():
        b.directional_mlp[2].bias.add_(1.0)
        assert float((b(batch) - yb).abs().min()) > 0


def test_renderer_uses_them():
    import mesh as MS
    from oracle import raycast_oracle as R
    from renderer import Renderer
    V, F = R.icosphere(2)
    tri = V[F]
    n = np.cross(tri[:, 1] - tri[:, 0], tri[:, 2] - tri[:, 0])
    mesh = MS.TriMesh(V, F)
    mesh.face_normals = n / np.linalg.norm(n, axis=1, keepdims=True)
    a, b = pair(dense_inference="int8")
    E = torch.randn((V.shape[0], 32), generator=torch.Generator().manual_seed(2))
    cam = torch.tensor(np.concatenate([np.eye(3), [[0.0], [0.0], [-3.0]]], 1)).float()
    K = torch.tensor([[32.0, 0, 16], [0, 32.0, 16], [0, 0, 1]])
    img = [Renderer(m.eval(), mesh, eigenfunctions=E, H=32, W=32, device="cuda").render(cam, K) for m in (a, b)]
    assert 0 < np.abs(img[0] - img[1]).max() < 0.05
    vids, bary, hit, face, dirs = MS.cast_camera_rays(MS.get_ray_mesh_intersector(mesh), cam, K, None, H=32, W=32)
    from inf_hip import runtime
    feats = runtime.gather(E.cuda(), vids, bary)
    with torch.no_grad():
        pred = b({"eigenfunctions": feats, "unit_ray_dirs": dirs[hit], "hit_face_idxs": face})
    assert np.array_equal(img[1].reshape(-1, 3)[hit.cpu().numpy()], pred.cpu().numpy())


def test_concat_layer_with_checkpoints():
    from layers import LinearWithConcatAndActivation
    torch.manual_seed(0)
    layer = LinearWithConcatAndActivation(48, 20, 40).cuda()
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn((64, 48), generator=g).cuda(), torch.randn((64, 20), generator=g).cuda()
    out = layer(x, y)
    want = torch.autograd.grad(out.square().sum(), list(layer.parameters()))
    layer.checkpoint = "int8"
    got = layer(x, y)
    assert float((out - got).detach().abs().max()) <= 80 * U32 * float(out.detach().abs().max())
    for a, b in zip(want, torch.autograd.grad(got.square().sum(), list(layer.parameters()))):
        assert float((a - b).norm() / a.norm()) < 1e-2
