"""Dropout, LayerNormalization, RMSNormalization, LayerScale, Multiply, Rescaling and Dense.quantize through
Sequential, the functional Model, save / load, checkpoints and refusals (host path)."""
import numpy as np
import pytest
import torch

import block_oracle as BO
from pyspark_tf_gke_amd import nn
from pyspark_tf_gke_amd.nn import layers as L
from pyspark_tf_gke_amd.nn import norm_ops as NO
from pyspark_tf_gke_amd.ops import dropout as D


@pytest.fixture
def fp32_host():
    from pyspark_tf_gke_amd.nn import engine

    old = engine.host_fp32()
    engine.host_fp32(True)
    yield
    engine.host_fp32(old)


def tower(width=72, blocks=2, rate=0.2, norm=nn.RMSNormalization, device="cpu", gate=False, inputs=24, outputs=2):
    """Residual Dense tower: every boundary is post-norm, gate, residual scale, dropout, Add, pre-norm."""
    L.reset_name_counters()
    inp = nn.Input(shape=(inputs,))
    h = nn.Dense(width, activation="relu", name="stem")(inp)
    g = nn.Dense(width, name="cond")(inp) if gate else None
    u = norm(name="n0")(h)
    for i in range(blocks):
        y = nn.Dense(width, activation="relu", name=f"b{i}a")(u)
        y = nn.Dense(width, name=f"b{i}b")(y)
        y = nn.LayerNormalization(name=f"b{i}post")(y)
        y = nn.Multiply(name=f"b{i}gate")([y, g]) if gate else nn.LayerScale(0.5, name=f"b{i}scale")(y)
        y = nn.Rescaling(0.7, name=f"b{i}res")(y)
        y = nn.Dropout(rate, name=f"b{i}drop")(y)
        h = nn.Add(name=f"b{i}add")([h, y])
        u = norm(name=f"b{i}pre")(h)
    m = nn.Model(inp, nn.Dense(outputs, name="head")(u))
    m.build(device=device)
    m.compile(optimizer=nn.optimizers.SGD(0.0), loss="mse")
    return m


def engine_grads(m, x, y):
    m.store.flat_grad.fill_(7.0)  # whole gradients are written, the others zeroed
    m.store.grad_clean = False
    m.store.zero_grad()
    xb, yb = m._prep_batch(x, y)
    out = m._run_forward(xb, True)
    m._run_backward(m._loss_grad(out, yb, m._stats_buf()))
    return out.detach().float().cpu(), {p.name: p.grad.detach().float().cpu().clone() for p in m.store.params}


def agree(m, x, y, step, tol):
    out, g = engine_grads(m, x, y)
    want, _, ref = BO.run(m, x, y, step)
    assert float((out - want).norm() / want.norm()) < tol
    for name, r in ref.items():
        assert float((g[name] - r).norm()) <= tol * float(r.norm()) + 1e-7, name


def data(n, k, out=2, seed=0):
    r = np.random.default_rng(seed)
    return r.standard_normal((n, k)).astype(np.float32), r.standard_normal((n, out)).astype(np.float32)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("norm", [nn.RMSNormalization, nn.LayerNormalization])
def test_tower_fuses_and_matches_autograd(fp32_host, gate, norm):
    m = tower(gate=gate, norm=norm)
    nodes = [op for op in m.ops if isinstance(op, NO.BlockNode)]
    assert len(nodes) == 3 and [len(n.outputs) for n in nodes] == [1, 2, 1]  # the last stream is only normalised
    x, y = data(10, 24)
    for step in (1, 2, 3):
        # fp32 against float64: a few hundred roundings, most of them in sums of 72
        agree(m, x, y, step, 2e-5)


def test_pieces_in_sequential(fp32_host):
    L.reset_name_counters()
    m = nn.Sequential([nn.Input(shape=(24,)), nn.LayerNormalization(), nn.Dense(80, activation="relu"), nn.Dropout(0.4),
                       nn.RMSNormalization(), nn.Rescaling(0.5), nn.Dropout(0.25, seed=11), nn.Dense(72),
                       nn.LayerScale(0.3), nn.Dense(2)])
    m.build(device="cpu")
    m.compile(optimizer=nn.optimizers.SGD(0.0), loss="mse")
    x, y = data(9, 24)
    agree(m, x, y, 1, 2e-5)
    agree(m, x, y, 2, 2e-5)
    ref, _, _ = BO.run(m, x, y, 0, training=False)
    np.testing.assert_allclose(m.predict(x), ref.numpy(), rtol=2e-5, atol=2e-5)
    assert NO.drop_state(m.ops).get() == 2  # inference draws nothing


@pytest.mark.parametrize("noise", [None, (None, 1, 1, None), (None, 1, 1, 1), (1, None, None, None)])
def test_image_model_with_channel_dropout(fp32_host, noise):
    L.reset_name_counters()
    inp = nn.Input(shape=(8, 6, 4))
    a = nn.Conv2D(16, 3, padding="same", name="c0")(inp)
    y = nn.LayerNormalization(name="n")(a)
    y = nn.Conv2D(16, 1, name="c1")(y)
    y = nn.Dropout(0.5, noise_shape=noise, name="d")(y)
    y = nn.Add(name="add")([a, y])
    y = nn.GlobalAveragePooling2D(name="gap")(y)
    m = nn.Model(inp, nn.Dense(2, name="head")(y))
    m.build(device="cpu")
    m.compile(optimizer=nn.optimizers.SGD(0.0), loss="mse")
    r = np.random.default_rng(0)
    agree(m, r.standard_normal((5, 8, 6, 4)).astype(np.float32), r.standard_normal((5, 2)).astype(np.float32), 1, 2e-5)


def test_gate_per_sample_and_same_tensor_twice(fp32_host):
    L.reset_name_counters()
    inp = nn.Input(shape=(4, 4, 4))
    a = nn.Conv2D(8, 3, padding="same", name="c0")(inp)
    g = nn.Dense(8, name="g")(nn.GlobalAveragePooling2D(name="gap0")(a))
    y = nn.Multiply(name="m")([a, g])  # one gate row for a sample's 16 pixels
    y = nn.Multiply(name="sq")([y, y])
    y = nn.Add(name="dbl")([y, y])
    m = nn.Model(inp, nn.Dense(2, name="head")(nn.GlobalAveragePooling2D(name="gap")(y)))
    m.build(device="cpu")
    m.compile(optimizer=nn.optimizers.SGD(0.0), loss="mse")
    r = np.random.default_rng(0)
    agree(m, r.standard_normal((5, 4, 4, 4)).astype(np.float32), r.standard_normal((5, 2)).astype(np.float32), 1, 2e-5)


def test_post_norm_add_without_stream(fp32_host):
    """u = norm(res + x) whose sum nobody else reads, and an Add whose branch is a plain Dense."""
    L.reset_name_counters()
    inp = nn.Input(shape=(24,))
    h = nn.Dense(72, name="a")(inp)
    y = nn.Dense(72, name="b")(h)
    u = nn.LayerNormalization(name="n", center=False)(nn.Add(name="s")([h, y]))
    m = nn.Model(inp, nn.Dense(2, name="head")(u))
    m.build(device="cpu")
    m.compile(optimizer=nn.optimizers.SGD(0.0), loss="mse")
    node = [op for op in m.ops if isinstance(op, NO.BlockNode)]
    assert len(node) == 1 and not node[0].op.want_h
    agree(m, *data(7, 24), 1, 2e-5)


def test_training_learns_and_masks_change():
    m = tower(rate=0.1)
    m.compile(optimizer=nn.optimizers.Adam(1e-2), loss="mse")
    x, y = data(64, 24)
    m.fit(x, y, batch_size=32, epochs=2, verbose=0)
    assert NO.drop_state(m.ops).get() == 4
    p = m.predict(x)
    assert np.isfinite(p).all() and np.array_equal(p, m.predict(x))


def test_save_load_export(tmp_path):
    m = tower(gate=True)
    x, _ = data(6, 24)
    want = m.predict(x)
    m.save(str(tmp_path / "m.keras"))
    m2 = nn.load_model(str(tmp_path / "m.keras"), device="cpu")
    np.testing.assert_array_equal(m2.predict(x), want)
    assert [l.get_config() for l in m2.layers] == [l.get_config() for l in m.layers]
    m.export(str(tmp_path / "sm"))
    np.testing.assert_array_equal(nn.saved_model.load(str(tmp_path / "sm"), device="cpu").model.predict(x), want)


def test_checkpoint_resumes_the_masks(tmp_path):
    from pyspark_tf_gke_amd.utils.checkpoint import load_checkpoint, save_checkpoint

    x, y = data(32, 24)

    def fresh():
        m = tower(rate=0.5)
        m.compile(optimizer=nn.optimizers.Adam(1e-2), loss="mse")
        return m

    a = fresh()
    for _ in range(3):
        a.train_on_batch(x, y)
    save_checkpoint(a, str(tmp_path), 0)
    b = fresh()
    load_checkpoint(b, str(tmp_path))
    assert NO.drop_state(b.ops).get() == 3
    for m in (a, b):
        m.train_on_batch(x, y)
    assert all(np.array_equal(p, q) for p, q in zip(a.get_weights(), b.get_weights()))


# ------------------------------------------------------------------------------------------ int4
def quantizable(device="cpu"):
    m = tower(width=128, inputs=64, outputs=3, device=device)
    return m, data(12, 64, 3)[0]


def test_quantize_runs_on_the_codes(fp32_host):
    m, x = quantizable()
    before = m.predict(x)
    m.quantize("int4", block_size=64)
    names = [l.name for l in m.layers if getattr(l, "int4", None) is not None]
    assert names == ["stem", "b0a", "b0b", "b1a", "b1b"]  # the narrow head stays as it was
    got = m.predict(x)
    # the codes' values in float64 through the oracle: the model now computes with exactly these
    ref, _, _ = BO.run(m, x, np.zeros((12, 3)), 0, training=False)
    # bf16 roundings: none (host fp32); fp32 sums only
    np.testing.assert_allclose(got, ref.numpy(), rtol=5e-5, atol=5e-5)
    # 4 bits: a step is 2/15 of a group's range, the model stays close to itself
    assert np.linalg.norm(got - before) < 0.5 * np.linalg.norm(before)


@pytest.mark.parametrize("zero", [False, True])
def test_quantized_save_load_export(tmp_path, zero):
    m, x = quantizable()
    m.quantize("int4", block_size=32, zero_point=zero)
    want = m.predict(x)
    path = tmp_path / "q.keras"
    m.save(str(path))
    m2 = nn.load_model(str(path), device="cpu")
    assert m2.quantized
    np.testing.assert_array_equal(m2.predict(x), want)
    assert all(np.array_equal(a, b) for a, b in zip(m.get_weights(), m2.get_weights()))
    m2.export(str(tmp_path / "sm"))
    m3 = nn.saved_model.load(str(tmp_path / "sm"), device="cpu").model
    assert m3.quantized
    np.testing.assert_array_equal(m3.predict(x), want)
    plain, _ = quantizable()
    plain.save(str(tmp_path / "p.keras"))
    assert path.stat().st_size < 0.3 * (tmp_path / "p.keras").stat().st_size


def test_quantized_model_refuses_training(tmp_path):
    from pyspark_tf_gke_amd.utils.checkpoint import load_checkpoint, save_checkpoint

    m, x = quantizable()
    save_checkpoint(m, str(tmp_path / "ck"), 0)
    w = m.get_weights()
    m.quantize("int4", block_size=64)
    y = np.zeros((12, 3), np.float32)
    m.evaluate(x, y, verbose=0)
    calls = [lambda: m.train_on_batch(x, y), lambda: m.fit(x, y, verbose=0), lambda: m(x, training=True),
             lambda: m.set_weights(w), lambda: m.trainable_variables[0].assign(np.zeros(1)),
             lambda: save_checkpoint(m, str(tmp_path / "c2"), 0), lambda: load_checkpoint(m, str(tmp_path / "ck"))]
    for c in calls:
        with pytest.raises(RuntimeError):
            c()
    with pytest.raises(ValueError):
        m.quantize("int4")
    with pytest.raises(NotImplementedError):
        quantizable()[0].quantize("int8")
    with pytest.raises(ValueError):
        quantizable()[0].quantize("int4", block_size=48)
    with pytest.raises(ValueError):  # no layer divides into groups of 128 inputs
        tower(width=72).quantize("int4")


def test_layer_refusals():
    for f in (lambda: nn.Dropout(1.5), lambda: nn.Dropout(-0.1), lambda: nn.LayerNormalization(epsilon=0.0),
              lambda: nn.RMSNormalization(epsilon=-1.0)):
        with pytest.raises(ValueError):
            f()
    for f in (lambda: nn.LayerNormalization(axis=1), lambda: nn.Rescaling(2.0, offset=1.0)):
        with pytest.raises(NotImplementedError):
            f()
    a, b = nn.Input(shape=(4, 4, 8)).output, nn.Input(shape=(4, 4, 6)).output
    with pytest.raises(ValueError):
        nn.Multiply()([a, b])
    with pytest.raises(ValueError):
        nn.Dropout(0.5, noise_shape=(None, 3, 1, None))(a)
    with pytest.raises(NotImplementedError):
        nn.Dropout(0.5, noise_shape=(None, 1, 4, 1))(a)


def test_ranks_draw_different_masks():
    l = nn.Dropout(0.5, seed=3)
    s = [D.mix_seed(l.seed_value(), r) for r in range(8)]
    assert len(set(s)) == 8
    k = [D.keep_mask((4096,), 0.5, v, 1) for v in s[:2]]
    assert 0.4 < float((k[0] == k[1]).float().mean()) < 0.6


_ = torch


def test_model_checker_answers_from_4_bits(tmp_path):
    """`test-model.py --quantize int4` (a 4-bit model file is taken as it is)."""
    import os
    import subprocess
    import sys

    from PIL import Image

    from pyspark_tf_gke_amd.models import tf_models

    m = tf_models.build_cnn_model((256, 320, 3), flat=False, summary=False, device="cpu")
    assert [l.units for l in m.layers if isinstance(l, L.Dense)] == [128, 2]
    m.quantize("int4", block_size=64)
    path = str(tmp_path / "m.keras")
    m.save(path)
    imgs = tmp_path / "images"
    imgs.mkdir()
    Image.fromarray(np.zeros((256, 320, 3), np.uint8)).save(imgs / "a.png")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "workloads", "raw-tf", "test-model.py"), "--model-dir",
                        str(tmp_path), "--model", path, "--images", str(imgs), "--device", "cpu", "--quantize", "int4"],
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "predicted (x=" in r.stdout, r.stderr[-2000:]


def wide_model(width, device="cpu"):
    """Residual scales, dropout and a gate of the branch's shape over rows wider than the kernels' 8192."""
    L.reset_name_counters()
    inp = nn.Input(shape=(24,))
    h = nn.Dense(width, name="stem")(inp)
    g = nn.Dense(width, name="cond")(inp)
    y = nn.Dropout(0.2, name="drop")(nn.Rescaling(0.5, name="half")(nn.Multiply(name="gate")([h, g])))
    m = nn.Model(inp, nn.Dense(2, name="head")(nn.Add(name="sum")([h, y])))
    m.build(device=device)
    m.compile(optimizer=nn.optimizers.SGD(0.0), loss="mse")
    return m


@pytest.mark.parametrize("width", [8200, 16384])
def test_wide_rows_without_a_norm(fp32_host, width):
    m = wide_model(width)
    assert any(isinstance(op, NO.BlockNode) and op.op.drop is not None and op.op.res for op in m.ops)
    agree(m, *data(3, 24), 1, 5e-5)


def test_norms_refuse_wide_rows():
    wide = nn.Input(shape=(8200,)).output
    for layer in (nn.LayerNormalization(), nn.RMSNormalization(), nn.LayerScale()):
        with pytest.raises(NotImplementedError, match="8192"):
            layer(wide)
    with pytest.raises(NotImplementedError, match="8192"):
        nn.Sequential([nn.Input(shape=(8200,)), nn.LayerNormalization(), nn.Dense(2)]).build(device="cpu")


def test_fp32_gradients_of_wide_rows_add():
    from pyspark_tf_gke_amd.nn.functional import _add_into

    a, b = torch.randn(3, 9001), torch.randn(3, 9001)
    want = a + b
    _add_into(a, b)
    assert torch.equal(a, want)
