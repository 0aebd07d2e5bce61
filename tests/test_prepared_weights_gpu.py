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


@pytest.mark.parametrize("kind", ["linear", "grouped"])
def test_layer_deleted_while_another_stream_still_reads_its_weight(cd, kind):
    """The products queued on the side stream lie behind others that take milliseconds; blocks of the sizes that the layer
    held are taken and overwritten on the default stream right after it is gone."""
    rng = np.random.default_rng(1)
    m, n, k = 64, 512, 640
    w = (rng.standard_normal((n, k)) / 20).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    xn = rng.standard_normal((m, k)).astype(np.float32)
    offsets = cd.Tensor.from_numpy(np.array([0, 20, m], np.int32))
    side = cd.Stream()
    busy = cd.Tensor.ones([4096, 4096])
    busy.set_stream(side)

    def run(delete):
        x = cd.Tensor.from_numpy(xn)
        if kind == "linear":
            layer = cd.nn.LinearFp8(k, n)
            layer.load_state_dict({"weight": w, "bias": b})
            layer.weight_fp8()
            call = lambda: layer(x)      # noqa: E731
        else:
            layer = cd.nn.GroupedLinear(2, k, n)
            layer.load_state_dict({"weight": np.stack([w, -w])})
            layer.weight_bf16()
            x = x.to(cd.DType.bfloat16)
            x.numpy()
            call = lambda: layer(x, offsets)      # noqa: E731
        x.set_stream(side)
        held = [busy.matmul(busy) for _ in range(8)]
        y = call()
        if delete:
            del call, layer
            fill = [cd.Tensor.ones(s) for s in ([n, k], [n], [2, n, k], [n, k // 4], [n, k], [4, 5]) for _ in range(3)]
            assert len(fill) == 18
        assert len(held) == 8
        return y.numpy()

    want = run(False)
    for _ in range(3):
        assert np.array_equal(run(True), want)
