import pytest
import torch

from pyspark_tf_gke_amd.ops import quant as Q


def codes_for(N, K, group, zero, seed=0, dev="cpu", pow2=True):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, (N, K), generator=g)
    codes = (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8)
    if pow2:
        scale = torch.pow(2.0, torch.randint(-3, 2, (N, K // group), generator=g).float()).to(torch.bfloat16)
    else:
        scale = (torch.rand(N, K // group, generator=g) * 0.02 + 0.01).to(torch.bfloat16)
    z = torch.randint(0, 16, (N, K // group), generator=g).to(torch.uint8) if zero else None
    return codes.to(dev), scale.to(dev), None if z is None else z.to(dev), q


def dense64(codes, scale, zero, group):
    """The weight matrix in float64, from its definition."""
    N, K = codes.shape[0], codes.shape[1] * 2
    w = torch.empty(N, K, dtype=torch.float64)
    for k in range(K):
        q = (codes[:, k // 2].long() >> (4 * (k % 2))) & 15
        z = zero[:, k // group].long() if zero is not None else 8
        w[:, k] = (q - z).double() * scale[:, k // group].double()
    return w


@pytest.mark.parametrize("N,K,group", [(1, 32, 32), (16, 128, 128), (17, 160, 32), (33, 320, 64), (5, 384, 128)])
@pytest.mark.parametrize("zero", [False, True])
def test_layout_round_trip_and_product(N, K, group, zero):
    codes, scale, z, _ = codes_for(N, K, group, zero)
    w = Q.int4_layout(codes, scale, z, group)
    assert w.tiles.is_contiguous() and w.scale.is_contiguous()
    c2, s2, z2 = Q.int4_codes(w)
    assert torch.equal(c2, codes) and torch.equal(s2, scale) and (z is None or torch.equal(z2, z))
    w64 = dense64(codes, scale, z, group)
    assert torch.equal(Q.int4_dequantize(w).double(), w64)
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-3, 4, (3, K), generator=g).to(torch.bfloat16)
    b = torch.randint(-3, 4, (N,), generator=g).float()
    out = torch.empty(3, N)
    Q.int4_dense_fwd(x, w, b, "relu", out)
    assert torch.equal(out.double(), torch.relu(x.double() @ w64.t() + b.double()))  # exact in fp32


def test_tile_layout_by_hand():
    """One weight at a time lands in its lane, dword and nibble."""
    for n, k in ((0, 0), (3, 1), (15, 127), (7, 66), (2, 37)):
        q = torch.zeros(16, 128, dtype=torch.long)
        q[n, k] = 15
        codes = (q[:, 0::2] | (q[:, 1::2] << 4)).to(torch.uint8)
        w = Q.int4_layout(codes, torch.ones(16, 1, dtype=torch.bfloat16), None, 128)
        lane, dword, e = (k // 8 % 4) * 16 + n, k // 32, k % 8
        b = w.tiles[0, 0, lane].view(4, 4)[dword].tolist()
        word = sum(v << (8 * j) for j, v in enumerate(b))
        word = ((word >> 3) | (word << 29)) & 0xFFFFFFFF
        assert word == 15 << (4 * (e // 2 + 4 * (e % 2)))
        assert int(w.tiles.long().sum()) == sum(b)


@pytest.mark.parametrize("zero", [False, True])
def test_quantize_error(zero):
    """Every weight comes back within half a step of its group (and half a bf16 step of the scale
    for values at the rounded-up scale's edge)."""
    g = torch.Generator().manual_seed(3)
    w = torch.randn(24, 256, generator=g) * torch.rand(24, 1, generator=g)
    w[3] = 0
    w[4, :64] = w[4, :64].abs()
    codes, scale, z = Q.int4_quantize(w, 64, zero)
    back = Q.int4_dequantize(Q.int4_layout(codes, scale, z, 64))
    step = scale.float().repeat_interleave(64, 1)
    # a zero point is rounded too: half a step more where a range ends off the grid
    assert ((back - w).abs() <= step * (1.0 if zero else 0.5) * (1 + 2**-20)).all()
    assert not back[3].any()
    # laid-out weights quantise to themselves
    if not zero:
        s = 0.125
        q = torch.randint(-7, 8, (8, 128), generator=g).float()
        q[:, 0] = 7
        c, sc, _ = Q.int4_quantize(q * s, 128)
        assert torch.equal(Q.int4_dequantize(Q.int4_layout(c, sc, None, 128)), q * s)


def test_refusals():
    codes, scale, _, _ = codes_for(4, 128, 64, False)
    w = Q.int4_layout(codes, scale, None, 64)
    x, out = torch.zeros(2, 128, dtype=torch.bfloat16), torch.empty(2, 4)
    Q.int4_dense_fwd(x, w, None, None, out)
    for call, exc in [
        (lambda: Q.int4_quantize(torch.zeros(4, 100), 64), ValueError),
        (lambda: Q.int4_quantize(torch.zeros(4, 96), 48), ValueError),
        (lambda: Q.int4_quantize(torch.zeros(4)), ValueError),
        (lambda: Q.int4_quantize(torch.full((4, 64), float("nan")), 64), ValueError),
        (lambda: Q.int4_layout(codes, scale, None, 128), ValueError),
        (lambda: Q.int4_layout(codes, scale.float(), None, 64), ValueError),
        (lambda: Q.int4_layout(codes.int(), scale, None, 64), TypeError),
        (lambda: Q.int4_layout(codes, scale, torch.full((4, 2), 16, dtype=torch.uint8), 64), ValueError),
        (lambda: Q.int4_dense_fwd(x[:, :64], w, None, None, out), ValueError),
        (lambda: Q.int4_dense_fwd(x, w, None, "softmax", out), ValueError),
        (lambda: Q.int4_dense_fwd(x, w, None, None, torch.empty(2, 5)), ValueError),
        (lambda: Q.int4_dense_fwd(x, w, None, None, torch.empty(2, 4, dtype=torch.float16)), TypeError),
        (lambda: Q.int4_dense_fwd(x, w, torch.zeros(5), None, out), ValueError),
        (lambda: Q.int4_dense_fwd(x, w._replace(n=20), None, None, torch.empty(2, 20)), ValueError),
        (lambda: Q.int4_dense_fwd(x, w._replace(scale=w.scale[:, :, :8]), None, None, out), ValueError),
        (lambda: Q.int4_dense_fwd(x, w._replace(group=32), None, None, out), ValueError),
    ]:
        with pytest.raises(exc):
            call()


def test_layout_of_views():
    """Codes that are a slice of something, at any byte, lay out like a copy of their own."""
    codes, scale, z, _ = codes_for(20, 256, 64, True)
    want = Q.int4_layout(codes, scale, z, 64)
    flat = torch.zeros(20 * 128 + 3, dtype=torch.uint8)
    flat[3:] = codes.reshape(-1)
    wide = torch.zeros(20, 140, dtype=torch.uint8)
    wide[:, 5:133] = codes
    for v in (flat[3:].view(20, 128), wide[:, 5:133]):
        got = Q.int4_layout(v, scale, z, 64)
        assert torch.equal(got.tiles, want.tiles) and got.tiles.is_contiguous()
    codes16, scale16, _, _ = codes_for(16, 128, 128, False)  # a full tile: nothing to pad
    w = Q.int4_layout(codes16, scale16, None, 128)
    assert torch.equal(Q.int4_codes(w)[0], codes16)
    codes16.fill_(0)
    assert Q.int4_codes(w)[0].any()  # a copy, not a view
