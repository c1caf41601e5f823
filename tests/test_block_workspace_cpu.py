"""Buffers of the block ops: the same ones every step, and no row statistics where no norm needs them."""
import pytest

from test_block_layers_cpu import data, engine_grads, tower, wide_model


@pytest.mark.parametrize("model,inputs", [(lambda: wide_model(8200), 24), (lambda: wide_model(96), 24), (tower, 24)])
def test_every_step_takes_the_same_buffers(model, inputs):
    m = model()
    x, y = data(3, inputs)
    engine_grads(m, x, y)
    first = {k: t.data_ptr() for k, t in m.ws.bufs.items()}
    held = dict(m.ws.bufs)  # so that no address is given out again
    engine_grads(m, x, y)
    assert {k: t.data_ptr() for k, t in m.ws.bufs.items()} == first and len(held) == len(first)


def test_no_statistics_without_a_norm():
    m = wide_model(96)
    engine_grads(m, *data(3, 24))
    assert not [k for k in m.ws.bufs if k.endswith("/stats")]
