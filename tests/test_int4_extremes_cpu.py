"""4-bit weights of groups whose range leaves fp32, and of groups below the smallest normal number."""
import pytest
import torch

from pyspark_tf_gke_amd.ops import quant as Q


def worst(w, zero):
    """Largest error of each group, in steps of its scale."""
    codes, scale, z = Q.int4_quantize(w, 32, zero)
    d = Q.int4_dequantize(Q.int4_layout(codes, scale, z, 32))
    return (d.double() - w.double()).abs().view(w.shape[0], -1, 32).amax(2) / scale.double()


@pytest.mark.parametrize("zero", [False, True])
@pytest.mark.parametrize("size", [3.3e38, 1.0, 1e-30, 1e-38, 1e-39])
def test_every_range(zero, size):
    w = (torch.rand(4, 64, generator=torch.Generator().manual_seed(1)) * 2 - 1) * size
    w[:, ::32], w[:, 1::32], w[1, 5] = size, -size, 0.0
    # half a step, rounded in fp32 (and with a zero point that is rounded itself, another half); the scale is the
    # least bf16 number that covers the range, so nothing is clamped.  Subnormal weights are off by 2**-149 besides
    assert float(worst(w, zero).max()) < (1.01 if zero else 0.51)
    assert float(worst(w, zero).max()) > 0.1


def test_a_group_of_zeros_beside_a_group_of_subnormal_numbers():
    w = torch.zeros(1, 64)
    w[0, 32:] = 3e-40
    for zero in (False, True):
        codes, scale, z = Q.int4_quantize(w, 32, zero)
        d = Q.int4_dequantize(Q.int4_layout(codes, scale, z, 32))
        assert not d[0, :32].any() and float((d[0, 32:] - 3e-40).abs().max()) <= float(scale[0, 1])
