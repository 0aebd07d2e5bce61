"""Prepared weights on the device: values after a change in place, and memory while another stream still reads it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cd(lib, cuda):
    import cudeep_b200
    return cudeep_b200


def test_values_after_a_change_in_place(cd):
    linear, grouped = cd.nn.LinearFp8(160, 40, bias=False), cd.nn.GroupedLinear(2, 160, 40)
    x = cd.Tensor.ones([4, 160])
    x16 = x.to(cd.DType.bfloat16)
    offsets = cd.Tensor.from_numpy(np.array([0, 1, 4], np.int32))
    dy = cd.Tensor.ones([4, 40]).to(cd.DType.bfloat16)
    for value in (0.5, 0.25, 2.0):
        for layer in (linear, grouped):
            layer._parameters["weight"].fill_(value)
        full = np.full((4, 40), 160 * value, np.float32)
        assert np.array_equal(linear(x).numpy(), full)
        assert np.array_equal(linear.forward_saved(x, "relu")[0].numpy(), full)
        assert np.array_equal(grouped(x16, offsets).numpy(), full)
        assert np.array_equal(grouped.backward(dy, x16, offsets)[0].numpy(), np.full((4, 160), 40 * value, np.float32))
    linear._parameters["weight"].zero_()
    assert not linear(x).numpy().any()
