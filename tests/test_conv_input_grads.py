"""Layers in front of convolutions whose input channels are padded (1, 3, 5, 6 or 12 of them): the gradient that
the convolution hands back has the channels of its input.  Host path against float64 autograd, and on the GPU."""
import numpy as np
import pytest
import torch

import block_oracle as BO
from pyspark_tf_gke_amd import nn
from pyspark_tf_gke_amd.nn import layers as L
from test_block_layers_cpu import agree, engine_grads, fp32_host  # noqa: F401


def compiled(m, device="cpu"):
    m.build(device=device)
    m.compile(optimizer=nn.optimizers.SGD(0.0), loss="mse")
    return m


def images(n, shape, seed=0):
    r = np.random.default_rng(seed)
    return r.standard_normal((n, *shape)).astype(np.float32), r.standard_normal((n, 2)).astype(np.float32)


FRONT = {
    "rescaling": lambda: [nn.Rescaling(0.5, name="f")],
    "layer norm": lambda: [nn.LayerNormalization(name="f")],
    "rms norm": lambda: [nn.RMSNormalization(name="f")],
    "layer scale": lambda: [nn.LayerScale(0.5, name="f")],
    "dropout": lambda: [nn.Dropout(0.3, name="f")],
    "dropout by channel, rescaling": lambda: [nn.Dropout(0.3, noise_shape=(None, 1, 1, None), name="f"),
                                              nn.Rescaling(0.5, name="g")],
    "rescaling, layer norm": lambda: [nn.Rescaling(0.5, name="g"), nn.LayerNormalization(name="f")],
}


def front_model(front, channels, device="cpu", units=16):
    L.reset_name_counters()
    return compiled(nn.Sequential([nn.Input(shape=(8, 6, channels)), *FRONT[front](),
                                   nn.Conv2D(units, 3, padding="same", name="c"), nn.GlobalAveragePooling2D(name="p"),
                                   nn.Dense(2, name="head")]), device)


# a layer norm over one channel is its offset, 0: the relative error of the output would be 0 / 0
@pytest.mark.parametrize("front,channels", [(f, c) for f in sorted(FRONT) for c in (1, 3, 4, 5, 12)
                                            if c > 1 or "layer norm" not in f])
def test_layer_in_front_of_a_convolution(fp32_host, front, channels):  # noqa: F811
    m = front_model(front, channels)
    # fp32 against float64: sums of up to 48 pixels x 9 x 16 terms, a few hundred roundings
    agree(m, *images(5, (8, 6, channels)), 1, 2e-5)


@pytest.mark.parametrize("filters", [3, 5, 6])
def test_layers_between_convolutions(fp32_host, filters):  # noqa: F811
    L.reset_name_counters()
    m = compiled(nn.Sequential([nn.Input(shape=(8, 6, 3)), nn.Conv2D(filters, 3, padding="same", name="c0"),
                                nn.LayerNormalization(name="n"), nn.Dropout(0.3, name="d"), nn.Rescaling(0.7, name="r"),
                                nn.Conv2D(8, 3, padding="same", name="c1"), nn.GlobalAveragePooling2D(name="p"),
                                nn.Dense(2, name="head")]))
    agree(m, *images(5, (8, 6, 3)), 1, 2e-5)
    inp = nn.Input(shape=(8, 6, 3))
    a = nn.Conv2D(filters, 3, padding="same", name="a")(inp)
    y = nn.Conv2D(filters, 3, padding="same", name="b")(nn.Dropout(0.4, name="d")(a))
    y = nn.Add(name="s")([a, nn.Multiply(name="m")([y, a])])
    y = nn.GlobalAveragePooling2D(name="p")(nn.Conv2D(8, 1, name="c")(y))
    agree(compiled(nn.Model(inp, nn.Dense(2, name="head")(y))), *images(5, (8, 6, 3)), 1, 2e-5)


@pytest.mark.parametrize("functional", [False, True])
def test_rescaled_images_into_a_strided_convolution(functional):
    """No gradient is wanted in front of the first weights: a strided convolution has none to give."""
    L.reset_name_counters()
    ls = [nn.Rescaling(1 / 255, name="f"), nn.Dropout(0.1, name="d"),
          nn.Conv2D(16, 3, strides=2, padding="same", name="c"), nn.GlobalAveragePooling2D(name="p"),
          nn.Dense(2, name="head")]
    if functional:
        inp = t = nn.Input(shape=(8, 6, 3))
        for l in ls:
            t = l(t)
        m = compiled(nn.Model(inp, t))
    else:
        m = compiled(nn.Sequential([nn.Input(shape=(8, 6, 3)), *ls]))
    x = np.random.default_rng(0).integers(0, 256, (5, 8, 6, 3), dtype=np.uint8)
    out, g = engine_grads(m, x, np.ones((5, 2), np.float32))
    assert all(bool(torch.isfinite(v).all()) and bool(v.any()) for v in g.values())


@pytest.mark.gpu
@pytest.mark.parametrize("front", sorted(FRONT))
@pytest.mark.parametrize("channels", [3, 4])
def test_layer_in_front_of_a_convolution_on_the_gpu(hip_built, front, channels):
    m = front_model(front, channels, "cuda")
    x, y = images(32, (8, 6, channels))
    for step in (1, 2):
        out, g = engine_grads(m, x, y)
        want, _, ref = BO.run(m, x, y, step)
        # bf16 activations, weights and gradients: fewer than 10 roundings of at most 2**-8 one after another on
        # a path through the model, so 4 % were they all of one sign; 16 filters' gradients add them at random
        assert float((out - want).norm() / want.norm()) < 0.04
        for name, r in ref.items():
            assert float((g[name] - r).norm()) < 0.04 * float(r.norm()) + 1e-6, name


@pytest.mark.gpu
def test_images_rescaled_in_front_train_on_the_gpu(hip_built):
    """uint8 images through Rescaling(1 / 255) into the first convolution of an image regressor."""
    L.reset_name_counters()
    m = nn.Sequential([nn.Input(shape=(32, 40, 3)), nn.Rescaling(1 / 255), nn.Conv2D(8, 5, padding="same"), nn.PReLU(),
                       nn.MaxPooling2D(), nn.Conv2D(16, 5, padding="same"), nn.PReLU(), nn.MaxPooling2D(),
                       nn.GlobalAveragePooling2D(), nn.Dense(2)])
    m.build(device="cuda")
    m.compile(optimizer=nn.optimizers.Adam(1e-3), loss="mse")
    r = np.random.default_rng(0)
    x, y = r.integers(0, 256, (16, 32, 40, 3), dtype=np.uint8), r.random((16, 2), dtype=np.float32)
    before = m.get_weights()
    for _ in range(2):
        assert np.isfinite(m.train_on_batch(x, y)[0])
    assert all(np.abs(a - b).max() > 0 for a, b in zip(before, m.get_weights()))


@pytest.mark.gpu
@pytest.mark.parametrize("functional", [False, True])
def test_first_convolution_takes_its_own_path_behind_a_rescaling(hip_built, functional):
    """Halving is exact in bf16: the model with a Rescaling(0.5) is the one without it on halved images."""

    def model(front):
        L.reset_name_counters()
        ls = [*front, nn.Conv2D(8, 5, padding="same", name="c0"), nn.PReLU(name="p0"), nn.MaxPooling2D(name="m0"),
              nn.Conv2D(16, 5, padding="same", name="c1"), nn.PReLU(name="p1"), nn.MaxPooling2D(name="m1"),
              nn.GlobalAveragePooling2D(name="gap"), nn.Dense(2, name="head")]
        if not functional:
            return compiled(nn.Sequential([nn.Input(shape=(32, 40, 3)), *ls]), "cuda")
        inp = t = nn.Input(shape=(32, 40, 3))
        for l in ls:
            t = l(t)
        return compiled(nn.Model(inp, t), "cuda")

    x, y = images(16, (32, 40, 3))
    a, ga = engine_grads(model([nn.Rescaling(0.5, name="r")]), x, y)
    b, gb = engine_grads(model([]), 0.5 * x, y)
    assert torch.equal(a, b)
    # the same kernels on the same numbers: only the order of fp32 sums over workgroups may differ, by at most
    # 16 * 32 * 40 terms * 2**-24 = 1.3e-3 of their magnitudes, which may cancel to some share of themselves
    for k in ga:
        assert float((ga[k] - gb[k]).norm()) <= 1e-2 * float(gb[k].norm()), k
