"""The weights that LinearFp8 and GroupedLinear prepare: when they are made anew, and when their memory may be used again.  On the
CPU, with a library that does nothing but note the calls it gets."""
import gc
import itertools
import threading

import pytest


class FakeLib:
    """Every function succeeds; `calls` lists (name, arguments).  Allocations get numbers of their own."""

    def __init__(self):
        self.calls = []
        self.hooks = {}
        self.addresses = itertools.count(0x1000, 0x1000)

    def __getattr__(self, name):
        if not name.startswith("cudeep_b200_"):
            raise AttributeError(name)
        name = name[len("cudeep_b200_"):]

        def call(*args):
            if name == "pool_alloc_on_stream":
                args[2]._obj.value = next(self.addresses)
            self.calls.append((name, tuple(getattr(a, "value", a) for a in args)))
            if name in self.hooks:
                self.hooks[name]()
            return 0
        return call

    def count(self, name):
        return sum(c[0] == name for c in self.calls)

    def freed(self, address):
        """Position of the call that frees a block; None if there is none."""
        return next((i for i, (n, a) in enumerate(self.calls) if n == "pool_free_on_stream" and a[0] == address), None)


@pytest.fixture()
def fake(monkeypatch):
    from cudeep_b200 import _lib
    lib = FakeLib()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    return lib


@pytest.fixture()
def cd():
    import cudeep_b200
    return cudeep_b200


SIDE = 0x51DE


def layer_and_call(cd, kind):
    D = cd.DType
    if kind == "linear":
        layer = cd.nn.LinearFp8(128, 64)
        call = lambda x: layer(x)      # noqa: E731
        make, x = "quantize_fp8", cd.Tensor([4, 128])
        held = lambda: [layer.weight_fp8().data, layer.weight_fp8().scales]      # noqa: E731
        per_call = 1      # x is quantised too
    else:
        layer = cd.nn.GroupedLinear(2, 128, 64)
        offsets = cd.Tensor([3], D.int32)
        call = lambda x: layer(x, offsets)      # noqa: E731
        make, x = "cast", cd.Tensor([4, 128], D.bfloat16)
        held = lambda: [layer.weight_bf16()]      # noqa: E731
        per_call = 0
    return layer, call, make, x, held, per_call


@pytest.mark.parametrize("kind", ["linear", "grouped"])
def test_made_again_after_a_change_in_place(cd, fake, kind):
    layer, call, make, x, _, per_call = layer_and_call(cd, kind)
    call(x)
    call(x)
    assert fake.count(make) == 1 + 2 * per_call
    for change in (lambda w: w.fill_(0.5), lambda w: w.zero_(), lambda w: w.reshape([-1]).fill_(2.0)):
        before = fake.count(make)
        change(layer._parameters["weight"])
        call(x)
        call(x)
        assert fake.count(make) - before == 1 + 2 * per_call
    # Through the tensor that the parameter shares its memory with.
    own = cd.Tensor.zeros(layer._parameters["weight"].shape())
    layer.register_parameter("weight", own)
    call(x)
    before = fake.count(make)
    own.fill_(3.0)
    call(x)
    assert fake.count(make) - before == 1 + per_call


@pytest.mark.parametrize("how", ["refresh", "replace", "change", "delete", "delete_after_taking_it"])
@pytest.mark.parametrize("kind", ["linear", "grouped"])
def test_other_streams_are_waited_for_before_the_memory_goes_back(cd, fake, kind, how):
    layer, call, _, x, held, _ = layer_and_call(cd, kind)
    x.set_stream(SIDE)
    call(x)
    addresses = [t.data_ptr() for t in held()]
    assert addresses and all(fake.freed(a) is None for a in addresses)
    start = len(fake.calls)
    if how == "refresh":
        layer.refresh()
    elif how == "replace":
        layer.register_parameter("weight", cd.Tensor.zeros(layer._parameters["weight"].shape()))
        call(x)
    elif how == "change":
        layer._parameters["weight"].fill_(1.0)
        call(x)
    else:
        if how == "delete_after_taking_it":      # a caller still holds the prepared weight when the layer goes
            taken = held()
            del held, call, layer
            gc.collect()
            assert all(fake.freed(a) is None for a in addresses)
            del taken
        else:
            del held, call, layer
        gc.collect()
    for a in addresses:
        at = fake.freed(a)
        assert at is not None
        assert any(n == "device_synchronize" for n, _ in fake.calls[start:at])


@pytest.mark.parametrize("kind", ["linear", "grouped"])
def test_one_stream_is_not_waited_for(cd, fake, kind):
    layer, call, _, x, held, _ = layer_and_call(cd, kind)
    call(x)
    addresses = [t.data_ptr() for t in held()]
    layer.refresh()
    assert all(fake.freed(a) is not None for a in addresses) and fake.count("device_synchronize") == 0


def test_the_other_parameters_of_the_layer_too(cd, fake):
    """The bias of the product and the weight that the gradient takes are read on the caller's stream."""
    D = cd.DType
    layer, x, grad = cd.nn.LinearFp8(128, 64), cd.Tensor([4, 128]), cd.Tensor([4, 64], D.bfloat16)
    x.set_stream(SIDE)
    grad.set_stream(SIDE)
    layer.backward(grad, layer.forward_saved(x)[1])
    addresses = [p.data_ptr() for p in layer.parameters()]
    start = len(fake.calls)
    del layer
    gc.collect()
    for a in addresses:
        assert any(n == "device_synchronize" for n, _ in fake.calls[start:fake.freed(a)])


@pytest.mark.parametrize("kind", ["linear", "grouped"])
def test_refresh_while_another_thread_prepares(cd, fake, kind):
    """The other thread comes in while this one waits for the weight to be made (which lets go of the interpreter's lock)."""
    layer, call, _, x, held, _ = layer_and_call(cd, kind)
    others = []

    def come_in():
        if not others:
            others.append(threading.Thread(target=layer.refresh))
            others[0].start()
            others[0].join(0.5)      # it may have to wait for this thread

    fake.hooks["stream_synchronize"] = come_in
    call(x)                          # takes the prepared weight, whichever
    assert all(t is not None for t in held())
    others[0].join(10)
    assert not others[0].is_alive()


@pytest.mark.parametrize("kind", ["linear", "grouped"])
def test_a_weight_that_could_not_be_made_is_not_kept(cd, fake, kind):
    """An error while preparing it leaves nothing behind, and the next call prepares it again."""
    layer, call, make, x, held, _ = layer_and_call(cd, kind)

    def fail():
        raise RuntimeError("planted")

    fake.hooks["stream_synchronize"] = fail
    for _ in range(2):
        with pytest.raises(RuntimeError, match="planted"):
            call(x)
    del fake.hooks["stream_synchronize"]
    before = fake.count(make)
    call(x)
    assert fake.count(make) > before and all(t is not None for t in held())
