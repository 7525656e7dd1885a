"""The choice of the checkpointed layers' products, without a GPU: keys, refusals of the Python and C entries."""
import pytest
import torch

from test_dense8_cpu import ODD, P, field, refused


def test_configuration():
    m = field(dense_checkpoints="int8", dense_products="fp32")
    assert m.spatial_mlp.dense_products == "fp32" and m.spatial_mlp.dense_checkpoints == "int8"
    assert field(dense_checkpoints="int8").spatial_mlp.dense_products is None
    for bad in ({"dense_products": "fp32"}, {"dense_checkpoints": "int8", "dense_products": "bf16"}):
        with pytest.raises(ValueError, match="products"):
            field(**bad)
    import model as M
    with pytest.raises(ValueError, match="view-dependent"):
        M.make_model({"k": 32, "num_layers": 4, "mlp_hidden_dim": 64, "skip_layer_idx": 2,
                      "kernels": {"dense_products": "fp32"}})


def test_entries():
    import dense
    x = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="HIP"):
        dense.linear([(x, 0, 0)], [x], [], None, checkpoint="int8", products="fp32")
    good = [4, 8, P, 8, ODD, None]
    for i, v in ((0, -1), (0, 1 << 31), (1, 0), (2, None), (3, 7), (4, None)):
        refused("inf_relu_mask", *[v if j == i else a for j, a in enumerate(good)])
    good = [4, 8, P, 8, ODD, P, 8, None]
    for i, v in ((0, -1), (0, 1 << 31), (1, 0), (2, None), (3, -1), (4, None), (5, None), (6, 7)):
        refused("inf_relu_mask_bwd", *[v if j == i else a for j, a in enumerate(good)])
