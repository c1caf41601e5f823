"""Gradients of graphs whose tensors have several readers: a relu Dense that feeds a narrow Dense and a residual
stream, a gate or a norm as well (host path, against float64 autograd)."""
import pytest

from pyspark_tf_gke_amd import nn
from pyspark_tf_gke_amd.nn import engine as E
from pyspark_tf_gke_amd.nn import layers as L
from test_block_layers_cpu import agree, data, fp32_host  # noqa: F401


def built(inp, out):
    m = nn.Model(inp, out)
    m.build(device="cpu")
    m.compile(optimizer=nn.optimizers.SGD(0.0), loss="mse")
    return m


JOINS = {
    "add": lambda h, y: nn.Add(name="j")([h, y]),
    "add norm": lambda h, y: nn.RMSNormalization(name="n")(nn.Add(name="j")([h, y])),
    "add scaled": lambda h, y: nn.Add(name="j")([h, nn.Rescaling(0.7, name="s")(y)]),
    "branch": lambda h, y: nn.Multiply(name="j")([h, y]),
    "gate": lambda h, y: nn.Multiply(name="j")([y, h]),
    "layer norm beside": lambda h, y: nn.Add(name="j")([nn.LayerNormalization(name="n")(h), y]),
    "dropped": lambda h, y: nn.Add(name="j")([nn.Dropout(0.3, name="d")(h), y]),
}


@pytest.mark.parametrize("join", sorted(JOINS))
@pytest.mark.parametrize("width,narrow", [(64, 64), (16, 16), (128, 128), (64, 24)])
def test_relu_dense_with_two_readers(fp32_host, join, width, narrow):  # noqa: F811
    """h = relu(Dense) is read by Dense(narrow) and by the join: the mask of h applies to both gradients."""
    L.reset_name_counters()
    inp = nn.Input(shape=(24,))
    h = nn.Dense(width, activation="relu", name="h")(inp)
    y = nn.Dense(narrow, name="y")(h)
    if narrow != width:
        y = nn.Dense(width, name="z")(y)
    m = built(inp, nn.Dense(2, name="head")(JOINS[join](h, y)))
    # fp32 against float64: a few hundred roundings, most of them in sums of up to 128
    agree(m, *data(10, 24), 1, 2e-5)


def test_narrow_chain_still_hands_the_mask_over(fp32_host):  # noqa: F811
    """With one reader the narrow Dense applies the mask in its own pass."""
    L.reset_name_counters()
    inp = nn.Input(shape=(24,))
    h = nn.Dense(64, activation="relu", name="h")(inp)
    m = built(inp, nn.Dense(2, name="head")(h))
    ops = [op.inner for op in m.ops]
    assert all(isinstance(op, E.DenseOp) for op in ops) and ops[0].grad_masked_by_next and ops[1].mask_for_prev
    agree(m, *data(10, 24), 1, 2e-5)


