"""A single layer's ``quantize``: the model is for inference from then on, as after its own."""
import numpy as np
import pytest

from test_block_layers_cpu import quantizable


def test_one_quantized_layer_refuses_what_would_leave_its_codes_behind(tmp_path):
    from pyspark_tf_gke_amd.utils.checkpoint import save_checkpoint

    m, x = quantizable()
    w = m.get_weights()
    assert not m.quantized
    m.layers[[l.name for l in m.layers].index("b0a")].quantize("int4", block_size=64)
    assert m.quantized
    y = np.zeros((12, 3), np.float32)
    for c in (lambda: m.set_weights(w), lambda: m.train_on_batch(x, y), lambda: save_checkpoint(m, str(tmp_path), 0),
              lambda: m.trainable_variables[0].assign(np.zeros(1))):
        with pytest.raises(RuntimeError, match="quantized"):
            c()
    assert np.isfinite(m.predict(x)).all()
