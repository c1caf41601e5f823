"""Residual scales, gates, dropout and joins without a norm over tensors of any shape (ops.norm.flat_fwd / flat_bwd), a
part of a larger tensor's mask (Drop.first), and models of odd batches and odd widths above the kernels' rows."""
import pytest
import torch

import norm_oracle as NO
from pyspark_tf_gke_amd.nn import engine as E
from pyspark_tf_gke_amd.nn import layers as L
from pyspark_tf_gke_amd.nn import norm_ops as NP
from pyspark_tf_gke_amd.ops import dropout as D
from pyspark_tf_gke_amd.ops import norm as N
from test_block_layers_cpu import agree, data, fp32_host, wide_model  # noqa: F401

SHAPES = [(1,), (7,), (5, 11), (1023,), (1, 1024), (1025,), (3, 4, 513), (3, 9001)]
DROP = (0.3, 0xABCDEF0123456789, 77)
DTYPES = [torch.bfloat16, torch.float32]


def tensors(shape, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(shape, generator=g).to(dtype).to(dev) for _ in range(4)]


def check_flat(shape, dtype, dev, gated, drop):
    x, res, gate, dh = tensors(shape, dtype, dev)
    gate = gate if gated else None
    kw = dict(gate=gate, scale=0.7, drop=None if drop is None else D.Drop(*drop))
    h, dx, dres, dgate = (torch.full_like(x, 7.0) for _ in range(4))
    assert N.flat_fwd(x, res=res, h=h, **kw) is h
    N.flat_bwd(x, dh=dh, dx=dx, dres=dres, dgate=dgate if gated else None, **kw)
    row = lambda t: None if t is None else t.reshape(1, -1)  # noqa: E731
    want = NO.run(row(x), row(res), None, row(gate), 0.7, drop, None, None, row(dh))
    for name, t in (("h", h), ("dx", dx), ("dres", dres)) + ((("dgate", dgate),) if gated else ()):
        NO.check(name, row(t), want[name], 1)
    # over the stream, as a gradient is added to what is there
    N.flat_fwd(x, res=res, h=res, **kw)
    assert torch.equal(res, h)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated,drop", [(False, None), (True, DROP)])
@pytest.mark.parametrize("shape", SHAPES)
def test_flat(dtype, gated, drop, shape):
    check_flat(shape, dtype, "cpu", gated, drop)


def check_part(dev, C, first, dtype=torch.float32):
    """Rows from mask index ``first`` on are those of a larger tensor that begins at 0."""
    lead = torch.randn(first, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    x, res, _, dh = tensors((6, C), dtype, dev)
    whole = torch.cat([lead, x.reshape(-1)])
    h, want = torch.empty_like(x), torch.empty_like(whole)
    D.dropout_fwd(whole, DROP[0], DROP[1], DROP[2], want)
    drop = D.Drop(*DROP, first)
    N.block_norm_fwd(x, drop=drop, h=h)
    assert torch.equal(h.reshape(-1), want[first:])
    dx = torch.empty_like(x)
    N.block_norm_bwd(x, None, drop=drop, dh=dh, dx=dx)
    assert torch.equal(dx == 0, (want[first:] == 0).view(6, C))


@pytest.mark.parametrize("first", [0, 8, 5, 1027])
@pytest.mark.parametrize("C", [8, 21])
def test_mask_from_an_index_on(C, first):
    check_part("cpu", C, first)


def test_refusals():
    x = torch.randn(4, 6)
    ok = dict(res=x.clone(), h=torch.empty_like(x))
    N.flat_fwd(x, **ok)
    for kw in (dict(ok, res=torch.randn(4, 5)), dict(ok, h=torch.empty(3, 6)), dict(ok, gate=torch.randn(6)),
               dict(ok, res=torch.randn(6, 4).t()), dict(ok, drop=D.Drop(0.5, 1, 0, -8))):
        with pytest.raises(ValueError):
            N.flat_fwd(x, **kw)
    with pytest.raises(ValueError):
        N.flat_fwd(torch.randn(6, 4).t(), **ok)
    g = x.clone()
    for kw in (dict(dh=torch.randn(4, 5), dx=x.clone()), dict(dh=x.clone()), dict(dh=None, dx=x.clone()),
               dict(dh=x.clone(), dgate=x.clone()), dict(dh=x.clone(), gate=g, dx=g),
               dict(dh=x.clone(), gate=g, dgate=g), dict(dh=g, dx=g, dres=g)):
        with pytest.raises(ValueError):
            N.flat_bwd(x, **kw)
    e = torch.empty(0, 6)
    N.flat_fwd(e, h=torch.empty(0, 6))
    N.flat_bwd(e, dh=e, dx=torch.empty(0, 6))


@pytest.mark.parametrize("batch,width", [(3, 8201), (1, 10001)])
def test_odd_wide_rows(fp32_host, batch, width):  # noqa: F811
    agree(wide_model(width), *data(batch, 24), 1, 5e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gated,drop", [(False, None), (True, DROP)])
@pytest.mark.parametrize("shape", SHAPES + [(37, 8201), (1, 300, 1027), (5, 20480)])
def test_flat_on_the_gpu(hip_built, dtype, gated, drop, shape):
    check_flat(shape, dtype, "cuda", gated, drop)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("first", [0, 8, 5, 1027, 8192])
@pytest.mark.parametrize("C", [3, 8, 21, 520, 1027])
def test_mask_from_an_index_on_the_gpu(hip_built, dtype, C, first):
    check_part("cuda", C, first, dtype)


def check_block_op(shape, dtype, dev):
    """A block op over rows that are wider than the kernels' and odd."""
    layer = L.Dropout(DROP[0], seed=DROP[1])
    op = NP.BlockOp("wide", gate_input=True, scale=0.7, drop=layer, res=True)
    NP.bind_drop_state([op])
    x, res, gate, dh = tensors(shape, dtype, dev)
    ws = E.Workspace()
    seed = D.mix_seed(DROP[1], 0)
    row = lambda t: t.reshape(1, -1)  # noqa: E731
    for step in (1, 2):
        h, = op.forward([x, gate, res], ws, True)
        dx, dgate, dres = op.backward([dh], ws)
        want = NO.run(row(x), row(res), None, row(gate), 0.7, (DROP[0], seed, step), None, None, row(dh))
        for name, t in (("h", h), ("dx", dx), ("dres", dres), ("dgate", dgate)):
            assert t.shape == x.shape
            NO.check(name, row(t), want[name], 1)


@pytest.mark.parametrize("shape", [(3, 8201), (2, 3, 8219)])
def test_odd_wide_block_op(shape):
    check_block_op(shape, torch.float32, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(37, 8201), (3, 10001), (5, 3, 8219)])
def test_odd_wide_block_op_on_the_gpu(hip_built, dtype, shape):
    check_block_op(shape, dtype, "cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(37, 8201), (1,), (3, 341)])
def test_gradients_of_odd_sizes_add(hip_built, shape):
    from pyspark_tf_gke_amd.nn.functional import _add_into

    for dt in (torch.float32, torch.bfloat16):
        a, b = torch.randn(shape, device="cuda"), torch.randn(shape, device="cuda").to(dt)
        want = a + b.float()
        _add_into(a, b)
        assert torch.equal(a, want)
