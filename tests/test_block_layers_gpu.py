"""Dropout, row norms, gates, residual scales and 4-bit Dense layers together, as a model trains on them and
answers with them, on the GPU."""
import numpy as np
import pytest
import torch

import block_oracle as BO
from pyspark_tf_gke_amd import nn
from pyspark_tf_gke_amd.models import build_cnn_model, build_deep_model
from pyspark_tf_gke_amd.nn import norm_ops as NO
from test_block_layers_cpu import data, engine_grads, tower, wide_model

pytestmark = pytest.mark.gpu

# bf16 activations and weights: about 50 roundings of 2**-9 (rms) on a path through the tower and back, at
# random, are 1.4 %; ReLU masks that flip near zero come on top.  A parameter's gradient is a sum over the samples
# that may cancel: with each term off by a share e at random, the sum of terms t_i is off by
# e * sqrt(sum t_i**2) in the mean square, however small the sum itself is
OUT_TOL, GRAD_TOL = 0.02, 0.06


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("norm", [nn.RMSNormalization, nn.LayerNormalization])
def test_tower_gradients(hip_built, gate, norm):
    m = tower(width=256, inputs=64, blocks=3, gate=gate, norm=norm, device="cuda")
    x, y = data(200, 64)
    for step in (1, 2):
        out, g = engine_grads(m, x, y)
        spread = {}
        want, _, ref = BO.run(m, x, y, step, spread=spread)
        assert float((out - want).norm() / want.norm()) < OUT_TOL
        for name, r in ref.items():
            assert float((g[name] - r).norm() / (r.norm() + spread[name].norm())) < GRAD_TOL, name


def test_training_step_captured_and_eager_agree(hip_built):
    """The whole step with dropout in a captured graph: masks advance with every replay, so the
    captured run's weights follow the eager run's."""
    x, y = data(64, 64)
    weights = []
    for jit in (False, True):
        m = tower(width=256, inputs=64, rate=0.3, device="cuda")
        m.compile(optimizer=nn.optimizers.SGD(0.05), loss="mse", jit_compile=jit)
        for _ in range(6):
            m.fit(x, y, batch_size=64, epochs=1, shuffle=False, verbose=0)
        assert NO.drop_state(m.ops).get() == 6
        weights.append(m.get_weights())
    for a, b in zip(*weights):
        # the same kernels on the same numbers; only the split-K sums of the Dense layers add in another order
        assert np.abs(a - b).max() <= 2e-2 * max(np.abs(a).max(), 1e-3)


def test_train_then_answer_from_4_bits(hip_built, tmp_path):
    m = tower(width=256, inputs=64, rate=0.1, device="cuda")
    m.compile(optimizer=nn.optimizers.Adam(1e-3), loss="mse")
    x, y = data(128, 64)
    m.fit(x, y, batch_size=32, epochs=2, verbose=0)
    m.quantize("int4", block_size=64)
    ref, _, _ = BO.run(m, x, y, 0, training=False)  # float64 on the values the codes stand for
    for n in (1, 5, 128):
        got = m.predict(x[:n])
        assert np.linalg.norm(got - ref[:n].numpy()) < OUT_TOL * np.linalg.norm(ref[:n].numpy())
    m.save(str(tmp_path / "q.keras"))
    m2 = nn.load_model(str(tmp_path / "q.keras"), device="cuda")
    np.testing.assert_array_equal(m2.predict(x), m.predict(x))
    with pytest.raises(RuntimeError):
        m.train_on_batch(x, y)


def test_image_regressor_with_dropout_and_4_bit_head(hip_built):
    m = build_cnn_model((64, 80, 3), flat=True, summary=False, device="cuda", dropout=0.25)
    x = np.random.default_rng(0).random((8, 64, 80, 3), dtype=np.float32)
    y = np.random.default_rng(1).random((8, 2), dtype=np.float32)
    for _ in range(2):
        assert np.isfinite(m.train_on_batch(x, y)[0])
    before = m.predict(x)
    m.quantize("int4")
    dense = [l for l in m.layers if getattr(l, "int4", None) is not None]
    assert len(dense) == 1 and dense[0].units == 2048
    after = m.predict(x)
    assert np.isfinite(after).all() and np.linalg.norm(after - before) < 0.2 * np.linalg.norm(before) + 0.05


def test_mlp_with_dropout(hip_built):
    m = build_deep_model(3, 5, device="cuda", dropout=0.3)
    r = np.random.default_rng(0)
    x, y = r.standard_normal((96, 3)).astype(np.float32), r.integers(0, 5, 96)
    m.fit(x, y, batch_size=32, epochs=2, verbose=0)
    assert NO.drop_state(m.ops).get() == 6 and np.isfinite(m.predict(x)).all()


_ = torch


@pytest.mark.parametrize("width", [8200, 16384])
def test_wide_rows_without_a_norm(hip_built, width):
    m = wide_model(width, device="cuda")
    x, y = data(37, 24)
    for step in (1, 2):
        out, g = engine_grads(m, x, y)
        spread = {}
        want, _, ref = BO.run(m, x, y, step, spread=spread)
        assert float((out - want).norm() / want.norm()) < OUT_TOL
        for name, r in ref.items():
            assert float((g[name] - r).norm() / (r.norm() + spread[name].norm())) < GRAD_TOL, name


def test_fp32_gradients_of_wide_rows_add(hip_built):
    from pyspark_tf_gke_amd.nn.functional import _add_into

    for dt in (torch.float32, torch.bfloat16):
        a, b = torch.randn(5, 20480, device="cuda"), torch.randn(5, 20480, device="cuda").to(dt)
        want = a + b.float()
        _add_into(a, b)
        assert torch.equal(a, want)
