"""A Dropout layer's backward pass draws the mask of its forward pass, whatever shape the gradient comes in."""
import pytest
import torch

from pyspark_tf_gke_amd import nn
from pyspark_tf_gke_amd.nn import engine as E
from pyspark_tf_gke_amd.nn import norm_ops as NO


def dropped(noise):
    op = NO.DropoutOp(nn.Dropout(0.5, noise_shape=noise, seed=3))
    NO.bind_drop_state([op])
    ws = E.Workspace()
    y = op.forward(torch.ones(6, 4, 5, 8), ws, True)
    return op, ws, y


@pytest.mark.parametrize("noise", [None, (None, 1, 1, None), (None, 1, 1, 1)])
def test_flattened_gradient_takes_the_mask_of_the_forward_pass(noise):
    op, ws, y = dropped(noise)
    dx = op.backward(torch.ones(6, 160), ws)
    assert 0 < int((y == 0).sum()) < y.numel() and torch.equal(dx.reshape(y.shape), y)


@pytest.mark.parametrize("noise", [None, (None, 1, 1, None)])
def test_gradient_of_other_channels_is_refused(noise):
    op, ws, _ = dropped(noise)
    with pytest.raises(ValueError, match="gradient of shape"):
        op.backward(torch.ones(6, 4, 5, 16), ws)
