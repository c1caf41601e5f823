import numpy as np
import pytest
import torch

import rng_oracle as O
from pyspark_tf_gke_amd.ops import dropout as D


def test_generator_known_answers():
    """The published known answers of Philox4x32-10."""
    kat = [((0,) * 4, (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
           ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
           ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
            (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]
    for ctr, key, want in kat:
        assert tuple(O.philox(np.array([ctr], np.uint64), key)[0]) == want
        blk = (ctr[1] << 32) | ctr[0]
        p = D._pieces(torch.tensor([blk - (1 << 64) if blk >> 63 else blk]), (ctr[3] << 32) | ctr[2],
                      (key[1] << 32) | key[0])[0].tolist()
        assert tuple(p[2 * j] | (p[2 * j + 1] << 16) for j in range(4)) == want


@pytest.mark.parametrize("shape,noise", [((7,), None), ((3, 5), None), ((4, 6, 5), (4, 1, 5)), ((4, 6, 5), (4, 1, 1)),
                                         ((4, 6, 5), (1, 6, 5)), ((4, 6, 5), (1, 1, 1)), ((2, 3, 4, 8), (2, 1, 1, 8)),
                                         ((2, 3, 4, 8), (None, 1, 1, None)), ((0, 4), None), ((1,), None)])
@pytest.mark.parametrize("rate", [0.0, 0.3, 1.0])
def test_matches_definition(shape, noise, rate):
    seed, step = 0xFEDCBA9876543210, (5 << 33) + 9
    x = torch.randn(shape)
    out = torch.empty_like(x)
    D.dropout_fwd(x, rate, seed, step, out, noise)
    full = tuple(s if v is None else v for v, s in zip(noise, shape)) if noise else shape
    keep = O.keep(O.shared_index(shape, full), rate, seed, step)
    want = np.where(keep, x.double().numpy() * O.scale(rate), 0.0)
    # fl(x * fl(s)): the scale and the product are each rounded to fp32
    np.testing.assert_allclose(out.numpy(), want, rtol=2.002 * 2.0**-24, atol=0)
    back = torch.empty_like(x)
    D.dropout_bwd(x, rate, seed, torch.tensor([step]), back, noise)
    assert torch.equal(out, back)


def test_nan_is_dropped():
    x = torch.full((64,), float("nan"))
    out = torch.empty_like(x)
    D.dropout_fwd(x, 0.5, 3, 0, out)
    keep = O.keep(np.arange(64), 0.5, 3, 0)
    assert np.array_equal(np.isnan(out.numpy()), keep) and (out.numpy()[~keep] == 0).all()


def test_refusals():
    x = torch.zeros(4, 6, 5)
    o = torch.empty_like(x)
    for rate in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            D.dropout_fwd(x, rate, 1, 0, o)
    with pytest.raises(ValueError):
        D.dropout_fwd(x, 0.5, 1, 0, o, (4, 2, 5))
    with pytest.raises(ValueError):
        D.dropout_fwd(x, 0.5, 1, 0, o, (4, 1))
    with pytest.raises(NotImplementedError):
        D.dropout_fwd(x, 0.5, 1, 0, o, (1, 6, 1))
    with pytest.raises(TypeError):
        D.dropout_fwd(x.half(), 0.5, 1, 0, o.half())
    with pytest.raises(ValueError):
        D.dropout_fwd(x, 0.5, 1, 0, torch.empty(4, 6, 4))
    with pytest.raises(ValueError):
        D.dropout_fwd(x.transpose(0, 1), 0.5, 1, 0, o.transpose(0, 1))
    with pytest.raises(TypeError):
        D.dropout_fwd(x, 0.5, 1, torch.zeros(1), o)
    with pytest.raises(TypeError):
        D.drop_advance(torch.zeros(2, dtype=torch.int64))


def test_advance_and_seeds():
    s = torch.tensor([41])
    assert int(D.drop_advance(s)) == 42
    seeds = {D.mix_seed(a, b) for a in range(40) for b in range(40)}
    assert len(seeds) == 1600 and all(0 <= v < 2**64 for v in seeds)


def test_rate_statistics():
    """200 000 kept-or-dropped draws at 0.25: within 6 standard deviations of the mean."""
    n = 200_000
    k = int(D.keep_mask((n,), 0.25, 77, 3).sum())
    assert abs(k - 0.75 * n) < 6 * (n * 0.75 * 0.25) ** 0.5
    a, b = D.keep_mask((n,), 0.5, 77, 3), D.keep_mask((n,), 0.5, 77, 4)
    assert abs(int((a == b).sum()) - n / 2) < 6 * (n / 4) ** 0.5


def test_noise_dims_against_the_definition():
    """Every shape of 1 and 3 with three axes and every noise shape of None, 1 and 3: the mask entries
    that (outer, mid, inner) names are those of broadcasting, or the shape is refused."""
    import itertools

    for shape in itertools.product((1, 3), repeat=3):
        for noise in itertools.product((None, 1, 3), repeat=3):
            full = tuple(s if v is None else v for s, v in zip(shape, noise))
            if any(v not in (1, s) for v, s in zip(full, shape)):
                with pytest.raises(ValueError):
                    D.noise_dims(shape, noise)
                continue
            shared = [k for k in range(3) if full[k] == 1 and shape[k] == 3]
            if shared and any(full[k] == 3 for k in range(shared[0], shared[-1] + 1)):
                with pytest.raises(NotImplementedError):
                    D.noise_dims(shape, noise)
                continue
            outer, mid, inner = D.noise_dims(shape, noise)
            n = full[0] * full[1] * full[2]
            assert outer * mid * inner == shape[0] * shape[1] * shape[2]
            want = torch.arange(n).view(full).expand(shape).reshape(-1)
            if mid == 1:
                assert torch.equal(want, torch.arange(len(want)))
            else:
                got = torch.arange(outer * inner).view(outer, 1, inner).expand(outer, mid, inner).reshape(-1)
                assert torch.equal(got, want)
    assert D.noise_dims((4, 5), None) == (20, 1, 1) and D.noise_dims((0, 5), (1, None)) == (0, 1, 1)
