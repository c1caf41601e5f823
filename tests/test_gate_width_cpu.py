"""A row of gates wider than the kernels' rows is refused when the model is built; a gate of the branch's shape is not."""
import pytest

from pyspark_tf_gke_amd import nn


def test_wide_gate_rows_are_refused():
    a, g = nn.Input(shape=(2, 8200)).output, nn.Input(shape=(8200,)).output
    with pytest.raises(NotImplementedError, match="8192"):
        nn.Multiply()([a, g])
    assert nn.Multiply()([a, nn.Input(shape=(2, 8200)).output]).shape == (2, 8200)
    assert nn.Multiply()([g, nn.Input(shape=(8200,)).output]).shape == (8200,)
    assert nn.Multiply()([nn.Input(shape=(2, 8192)).output, nn.Input(shape=(8192,)).output]).shape == (2, 8192)
