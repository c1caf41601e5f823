"""What None and 1 mean in a noise shape."""
import pytest
import torch

from pyspark_tf_gke_amd.ops import dropout as D


@pytest.mark.parametrize("named,noise", [((5, 1, 1, 8), (None, 1, 1, None)), ((5, 1, 1, 1), (None, 1, 1, 1)),
                                         ((1, 4, 3, 8), (1, None, None, None)), (None, (None, None, None, None))])
def test_none_is_the_inputs_own_size(named, noise):
    shape = (5, 4, 3, 8)
    a, b = (D.keep_mask(shape, 0.5, 3, 1, v) for v in (named, noise))
    assert torch.equal(a, b)
    one = tuple(v if v is not None else s for v, s in zip(noise, shape))  # the entries drawn
    assert torch.equal(a, a[tuple(slice(0, n) for n in one)].expand(shape))
