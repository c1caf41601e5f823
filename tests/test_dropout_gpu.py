import numpy as np
import pytest
import torch

import rng_oracle as O
from pyspark_tf_gke_amd.ops import dropout as D

pytestmark = pytest.mark.gpu
SEED, STEP = 0x0123456789ABCDEF, (3 << 35) + 17
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8}  # one rounding, relative


def _check(x, out, rate, noise=None, seed=SEED, step=STEP):
    shape = tuple(x.shape)
    full = tuple(s if v is None else v for v, s in zip(noise, shape)) if noise else shape
    keep = O.keep(O.shared_index(shape, full), rate, seed, step)
    want = np.where(keep, x.double().cpu().numpy() * O.scale(rate), 0.0)
    # the scale 65536 / (65536 - thr) is no fp32 number: fl(x * fl(s)) = x * s * (1 + d1) * (1 + d2) with
    # |d| <= 2**-24 each, then the output type's half step for bf16
    rtol = 2 * 2.0**-24 + (HALF[x.dtype] if x.dtype != torch.float32 else 0)
    np.testing.assert_allclose(out.double().cpu().numpy(), want, rtol=rtol * 1.001, atol=0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2047, 2048, 2049, 300_001])
@pytest.mark.parametrize("rate", [0.0, 0.1, 0.5, 1.0])
def test_elementwise(hip_built, dtype, n, rate):
    x = torch.randn(n, device="cuda", generator=torch.Generator("cuda").manual_seed(n)).to(dtype)
    out = torch.full_like(x, 7.0)
    D.dropout_fwd(x, rate, SEED, STEP, out)
    _check(x, out, rate)
    back = torch.full_like(x, 7.0)
    D.dropout_bwd(x, rate, SEED, torch.tensor([STEP], device="cuda"), back)
    assert torch.equal(out, back)
    D.dropout_fwd(x, rate, SEED, STEP, x)  # in place
    assert torch.equal(out, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("off", [1, 3])
def test_unaligned_views(hip_built, dtype, off):
    x = torch.randn(1000 + off, device="cuda").to(dtype)[off:]
    buf = torch.full((1000 + 2 * off,), 7.0, device="cuda", dtype=dtype)
    out = buf[off:off + 1000]
    D.dropout_fwd(x, 0.4, SEED, STEP, out)
    _check(x, out, 0.4)
    assert (buf[:off] == 7).all() and (buf[off + 1000:] == 7).all()  # nothing beside it is written


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,noise", [((5, 12, 16), (5, 1, 16)), ((5, 12, 16), (1, 1, 16)), ((5, 12, 16), (5, 1, 1)),
                                         ((5, 12, 16), (1, 12, 16)), ((5, 7, 3), (5, 1, 3)), ((5, 7, 3), (5, 1, 1)),
                                         ((9, 3, 13), (9, 1, 13)), ((3, 4, 5, 8), (None, 1, 1, None)),
                                         ((1000, 1), (1000, 1)), ((2, 2, 1), (2, 1, 1)), ((1, 9, 1), (1, 1, 1)),
                                         ((64, 100, 24), (64, 1, 24))])
def test_shared_entries(hip_built, dtype, shape, noise):
    x = torch.randn(shape, device="cuda").to(dtype)
    out = torch.full_like(x, 7.0)
    D.dropout_fwd(x, 0.35, SEED, STEP, out, noise)
    _check(x, out, 0.35, noise)


def test_empty_nan_and_other_stream(hip_built):
    e = torch.empty(0, 4, device="cuda")
    D.dropout_fwd(e, 0.5, 1, 0, torch.empty_like(e))
    x = torch.full((4096,), float("inf"), device="cuda")
    out = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        D.dropout_fwd(x, 0.5, 3, 0, out)
    s.synchronize()
    keep = O.keep(np.arange(4096), 0.5, 3, 0)
    o = out.cpu().numpy()
    assert np.isinf(o[keep]).all() and (o[~keep] == 0).all()


def test_graph_draws_a_new_mask_each_replay(hip_built):
    x = torch.randn(5000, device="cuda")
    out, back = torch.empty_like(x), torch.empty_like(x)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    g = torch.cuda.CUDAGraph()
    D.drop_advance(step)
    D.dropout_fwd(x, 0.5, SEED, step, out)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        D.drop_advance(step)
        D.dropout_fwd(x, 0.5, SEED, step, out)
        D.dropout_bwd(x, 0.5, SEED, step, back)
    for k in range(2, 6):
        g.replay()
        torch.cuda.synchronize()
        assert int(step) == k and torch.equal(out, back)
        _check(x, out, 0.5, step=k)
        torch.randn(100, device="cuda").sum().item()


def test_more_elements_than_32_bits(hip_built):
    """2^32 + 24 elements: both offsets and mask indices pass 32 bits."""
    n = (1 << 32) + 24
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    D.dropout_fwd(x, 0.5, SEED, STEP, x)
    for lo in (0, (1 << 31) - 40, n - 1000):
        got = x[lo:lo + 1000].float().cpu().numpy()
        keep = O.keep(np.arange(lo, min(n, lo + 1000)), 0.5, SEED, STEP)
        assert np.array_equal(got, np.where(keep, 2.0, 0.0))
    del x
    y = torch.ones(2, (1 << 31) + 16, 1, device="cuda", dtype=torch.bfloat16)
    D.dropout_fwd(y, 0.5, 5, 1, y, (2, 1, 1))
    keep = O.keep(np.arange(2), 0.5, 5, 1)
    for k in range(2):
        assert float(y[k, 0]) == float(y[k, -1]) == (2.0 if keep[k] else 0.0)


def test_refusals(hip_built):
    x = torch.zeros(64, device="cuda")
    with pytest.raises(ValueError):
        D.dropout_fwd(x, 0.5, 1, 0, torch.empty(64))
    with pytest.raises(ValueError):
        D.dropout_fwd(x, 0.5, 1, torch.zeros(1, dtype=torch.int64), torch.empty_like(x))
    with pytest.raises(ValueError):
        D.dropout_fwd(x[:32], 0.5, 1, 0, x[16:48])
