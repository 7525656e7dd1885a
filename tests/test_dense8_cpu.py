"""The 8-bit dense layers without a GPU: refusals of the C entries (before any launch), of
the Python entries on host tensors, and the configuration keys."""
import ctypes
import types

import numpy as np
import pytest
import torch

P = ctypes.c_void_p(4096)  # a pointer that is never followed: every call below is refused
ODD = ctypes.c_void_p(4100)


def refused(name, *args):
    import inf_hip
    assert getattr(inf_hip.lib, name)(*args) == -1, (name, args)
    assert b"invalid argument" in inf_hip.lib.inf_last_error()


def test_rows8_refusals():
    good = [P, 0, 4, 8, 8, P, 16, P, None]
    for i, v in ((0, None), (1, 2), (1, 4), (2, -1), (3, 0), (4, -8), (5, None), (5, ODD), (6, 8), (6, 24), (7, None)):
        refused("inf_quantize_rows", *[v if j == i else a for j, a in enumerate(good)])
    good = [P, 16, P, 4, 8, P, 0, 8, None]
    for i, v in ((0, None), (0, ODD), (1, 8), (1, 20), (2, None), (3, -1), (4, 0), (5, None), (6, 4), (7, 7)):
        refused("inf_restore_rows", *[v if j == i else a for j, a in enumerate(good)])
    good = [P, 8, 1, 4, 8, P, None]
    for i, v in ((0, None), (3, -1), (4, 0), (5, None), (5, ODD)):
        refused("inf_pack_weight", *[v if j == i else a for j, a in enumerate(good)])


def test_linear_int_refusals():
    # rows, n, k, x, dtype, ldx, x_scale, w, w_scale, bias, add, ldadd, act, out, dtype, ldo, out_scale, workspace, stream
    good = [4, 8, 16, P, 4, 16, P, P, P, None, None, 0, 0, P, 4, 16, P, P, None]
    for i, v in ((0, -1), (1, 0), (2, 0), (2, (1 << 17) + 1), (3, None), (3, ODD), (4, 2), (4, 5), (5, 8), (5, 24),
                 (6, None), (7, None), (7, ODD), (8, None), (12, 3), (12, -1), (13, None), (13, ODD), (14, 3), (15, 7),
                 (15, 24), (16, None), (17, None)):
        refused("inf_linear_int", *[v if j == i else a for j, a in enumerate(good)])
    refused("inf_linear_int", *[P if j == 10 else 7 if j == 11 else a for j, a in enumerate(good)])


def test_linear_ckpt_refusals():
    # rows, n, k, x, dtype, ldx, W, swn, swk, bias, add, ldadd, act, y, ldy, mask, q, ldq, scale, workspace, stream
    good = [4, 8, 16, P, 0, 16, P, 16, 1, None, None, 0, 1, P, 8, P, P, 16, P, P, None]
    for i, v in ((0, -1), (1, 0), (2, 0), (3, None), (4, 4), (4, 2), (5, -1), (6, None), (12, 3), (13, None), (14, 7),
                 (16, ODD), (17, 8), (17, 24), (18, None), (19, None)):
        refused("inf_linear_ckpt_forward", *[v if j == i else a for j, a in enumerate(good)])
    # rows, n, k, dy, lddy, act, y, ldy, mask, q, ldq, scale, W, swn, swk, dx, dtype, lddx, dW, lddw, db, workspace, stream
    good = [4, 8, 16, P, 8, 1, P, 8, P, P, 16, P, P, 16, 1, P, 0, 16, P, 16, P, P, None]
    for i, v in ((0, -1), (1, 0), (2, 0), (3, None), (4, -1), (5, 3), (8, None), (9, None), (9, ODD), (10, 8), (10, 24),
                 (11, None), (12, None), (16, 4), (17, 15), (19, 15), (21, None)):
        refused("inf_linear_ckpt_backward", *[v if j == i else a for j, a in enumerate(good)])
    sig = [2 if j == 5 else a for j, a in enumerate(good)]
    for i, v in ((6, None), (7, 7)):
        refused("inf_linear_ckpt_backward", *[v if j == i else a for j, a in enumerate(sig)])


def test_sizes():
    from inf_hip import lib
    assert lib.inf_packed_weight_bytes(3, 1) == 3 * 128 and lib.inf_packed_weight_bytes(3, 129) == 3 * 256
    assert lib.inf_packed_weight_bytes(3, 0) == -1 and lib.inf_linear_int_workspace_bytes(1, 0, 1, 0, 0) == -1
    assert lib.inf_linear_ckpt_workspace_bytes(1, 1, 0, 0, 1) == -1
    big = lib.inf_linear_int_workspace_bytes(1 << 22, 256, 4096, 0, 4)  # sizes past 32 bits
    assert big >= (1 << 22) * (4096 + 4)


def test_host_tensors_are_refused():
    import dense
    x = torch.zeros(4, 8)
    for call in (lambda: dense.quantize_rows(x), lambda: dense.quantize_weight(x),
                 lambda: dense.pack_weight8(x.to(torch.int8), torch.zeros(4)),
                 lambda: dense.linear([(x, 0, 0)], [x], [], None, checkpoint="int8")):
        with pytest.raises(RuntimeError, match="HIP"):
            call()


def field(**kernels):
    import model as M
    cfg = {"k": 32, "num_layers": 4, "mlp_hidden_dim": 64, "skip_layer_idx": 2, "kernels": kernels,
           "view_dependence": {"bottleneck_vec_dim": 16, "in_dim_view_dir": 3, "include_view_dir": True,
                               "embed_size": 4, "directional_hidden_dim": 32, "strategy": "extrinsic"}}
    return M.make_model(cfg, mesh=types.SimpleNamespace(face_normals=np.eye(3)))


def test_configuration():
    import model as M
    m = field()
    assert m.dense_inference is None and m.spatial_mlp.dense_checkpoints is None
    m = field(dense_checkpoints="int8", dense_inference="int8")
    assert m.dense_inference == "int8" and m.spatial_mlp.dense_checkpoints == "int8"
    for bad in ({"dense_checkpoints": "int4"}, {"dense_inference": True}):
        with pytest.raises(ValueError, match="int8"):
            field(**bad)
    with pytest.raises(ValueError, match="view-dependent"):
        M.make_model({"k": 32, "num_layers": 4, "mlp_hidden_dim": 64, "skip_layer_idx": 2,
                      "kernels": {"dense_inference": "int8"}})
