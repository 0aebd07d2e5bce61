"""Linear, Conv2d, the activation modules and Sequential: forward of the reference's
python/cuDeep/nn.py:36-189 on this library's kernels.

Same constructor arguments, parameter names ("weight", "bias"), state_dict keys and default
initialisation (randn weights, zero bias, nn.py:104-108,131-137) as the reference.  Differences,
all on the forward path:
  * Linear.forward is one fused kernel (W consumed as stored, bias in the epilogue) instead of
    transpose-copy + matmul + broadcast_add;
  * Sequential.forward folds an activation module that directly follows a Linear or Conv2d into
    that layer's epilogue (the unfused result is the same function applied as a separate pass).
Training (autograd, optimisers) is outside this library's scope.

Additions: LinearFp8, the same layer on 8-bit products, and GroupedLinear, one weight for each of several row groups
(experts); both give the gradients of their products.
"""
from __future__ import annotations

import threading
from typing import Optional

import numpy as np

from . import _lib, lowp
from .tensor import DType, Tensor, _epilogue_code, conv2d, linear

_ACTIVATIONS = (None, "relu", "gelu", "silu", "sigmoid")     # by epilogue code


class Parameter(Tensor):
    """A tensor a Module owns: shares the storage of the tensor it was made from (reference nn.py:20-30)."""

    def __init__(self, data: Tensor):
        super().__init__(data.shape(), data.dtype(), _storage=data._storage, _strides=data.strides())

    def __repr__(self):
        return "Parameter(shape={}, dtype={})".format(self.shape(), self.dtype())


class Module:
    """Container of parameters and sub-modules with the reference's public surface (nn.py:33-90):
    forward / __call__, register_parameter / register_module, parameters / named_parameters,
    train / eval / training, state_dict / load_state_dict.  Parameter names are dotted paths,
    a module's own parameters before those of its children, children in registration order.
    Every query is one depth-first walk (`_owned`)."""

    def __init__(self):
        self._parameters: dict[str, Parameter] = {}
        self._modules: dict[str, "Module"] = {}
        self._training = True

    # -- calling ------------------------------------------------------------------------------
    def forward(self, *args, **kwargs):
        raise NotImplementedError(f"{type(self).__name__} does not define forward()")

    def __call__(self, *args, **kwargs):
        return self.forward(*args, **kwargs)

    # -- registration ---------------------------------------------------------------------------
    def register_parameter(self, name: str, tensor) -> None:
        self._parameters[name] = tensor if isinstance(tensor, Parameter) else Parameter(tensor)

    def register_module(self, name: str, module: "Module") -> None:
        self._modules[name] = module

    # -- traversal ------------------------------------------------------------------------------
    def _owned(self, prefix: str = ""):
        """(dotted name, owning module, key) of every parameter below this module."""
        for key in self._parameters:
            yield prefix + key, self, key
        for child_name, child in self._modules.items():
            yield from child._owned(f"{prefix}{child_name}.")

    def named_parameters(self):
        for name, owner, key in self._owned():
            yield name, owner._parameters[key]

    def parameters(self) -> list:
        return [p for _, p in self.named_parameters()]

    # -- mode -----------------------------------------------------------------------------------
    def train(self, mode=True):
        stack = [self]
        while stack:
            module = stack.pop()
            module._training = mode
            stack.extend(module._modules.values())
        return self

    def eval(self):
        return self.train(False)

    @property
    def training(self):
        return self._training

    # -- state ----------------------------------------------------------------------------------
    def state_dict(self) -> dict:
        return {name: p.numpy() for name, p in self.named_parameters()}

    def load_state_dict(self, sd: dict):
        """Replaces every parameter named in `sd`; names this module does not have are ignored."""
        for name, owner, key in list(self._owned()):
            if name in sd:
                owner._parameters[key] = Parameter(Tensor.from_numpy(np.ascontiguousarray(sd[name])))


class Linear(Module):
    """y = x W^T + b  (reference nn.py:97-115)."""

    def __init__(self, in_features, out_features, bias=True, dtype=DType.float32):
        super().__init__()
        self.in_features = in_features
        self.out_features = out_features
        self.register_parameter("weight", Tensor.randn([out_features, in_features], dtype))
        if bias:
            self.register_parameter("bias", Tensor.zeros([out_features], dtype))

    def forward(self, x, activation=None):
        return linear(x, self._parameters["weight"], self._parameters.get("bias"), activation)


class _Prepared:
    """What a layer makes of its weight before it is used, kept until the parameter is replaced (load_state_dict) or changed in
    place through a Tensor (fill_, zero_, also of another Tensor of the same memory).  What the library cannot see, values
    written to the parameter's address, needs a call of the layer's refresh().  It is made on the parameter's stream and finished
    before any stream uses it; once other streams have, they are waited for before its memory goes back to the pool, whether the
    layer lets go of it last or a caller."""

    def __init__(self):
        self.lock = threading.Lock()      # making a value waits for the device, and other threads run meanwhile
        self.of = self.version = self.value = None

    def get(self, parameter, make, stream):
        with self.lock:
            if self.of is not parameter or self.version != parameter._storage.version:
                self.of = self.value = None
                self.version = parameter._storage.version
                value = make(parameter)
                _lib.check(_lib.load().cudeep_b200_stream_synchronize(parameter.stream))
                self.value, self.of = value, parameter
            value = self.value
        for t in (value.data, value.scales) if isinstance(value, lowp.Fp8Tensor) else (value,):
            _used_on(t, stream)
        return value

    def drop(self):
        with self.lock:
            self.of = self.version = self.value = None


def _handle(stream):
    return getattr(stream, "value", stream) or 0


def _used_on(t, stream):
    """t, which the layer holds and a kernel on `stream` reads: its memory outlives that, should the layer go first."""
    if t is not None and _handle(stream) != _handle(t.stream):
        t._storage.shared = True
    return t


class LinearFp8(Linear):
    """Linear on 8-bit products: x is quantised in blocks of 1 x 128 at each call, the weight once in blocks of 128 x 128.
    x is float32 or bfloat16 [rows, in_features]; the result has its type.  Parameters as Linear's, in float32."""

    def __init__(self, in_features, out_features, bias=True):
        super().__init__(in_features, out_features, bias)
        self._weight8 = _Prepared()

    def refresh(self) -> None:
        """After writing to the parameter's address: the next call takes its new values."""
        self._weight8.drop()

    def weight_fp8(self, stream=None) -> lowp.Fp8Tensor:
        """The weight as the products on `stream` take it."""
        return self._weight8.get(self._parameters["weight"], lambda w: lowp.quantize_fp8(w, tiles=True), stream)

    def _bias(self, stream):
        return _used_on(self._parameters.get("bias"), stream)

    def forward(self, x, activation=None):
        return lowp.linear_fp8(lowp.quantize_fp8(x), self.weight_fp8(x.stream), self._bias(x.stream), activation, x.dtype())

    def forward_saved(self, x, activation=None):
        """(y, saved) for `backward`: y as forward's, saved holds x and, with an activation, the pre-activation in 8 bits.
        Without an activation nothing but the codes that the product reads anyway is kept."""
        activation = _ACTIVATIONS[_epilogue_code(activation)]
        x8 = lowp.quantize_fp8(x)
        z = lowp.linear_fp8(x8, self.weight_fp8(x.stream), self._bias(x.stream), None, DType.float32 if activation else x.dtype())
        if activation is None:
            return z, (x8, None, None)
        y = getattr(z, activation)()
        return y.to(x.dtype()), (x8, lowp.quantize_fp8(z), activation)

    def backward(self, grad, saved):
        """(dx, dweight, dbias) in float32 for bfloat16 `grad` of y and what forward_saved kept; the product for dx takes the
        weight in bfloat16."""
        x8, z8, activation = saved
        weight = _used_on(self._parameters["weight"], grad.stream)._cast_on(DType.bfloat16, grad.stream)
        dx, dw, db = lowp.linear_backward_saved(grad, x8, weight, z8, activation, DType.float32)
        return dx.to(DType.float32), dw, (db if "bias" in self._parameters else None)


class GroupedLinear(Module):
    """y[r] = x[r] W[g]^T for the rows of each group g: the experts' products of a mixture of experts.  x is bfloat16
    [rows, in_features] with the rows of a group next to each other, offsets an int32 Tensor of groups + 1 row numbers.  The
    parameter is float32 [groups, out_features, in_features]; the products take it in bfloat16."""

    def __init__(self, groups, in_features, out_features):
        super().__init__()
        self.groups, self.in_features, self.out_features = groups, in_features, out_features
        self.register_parameter("weight", Tensor.randn([groups, out_features, in_features]))
        self._weight16 = _Prepared()

    def refresh(self) -> None:
        """After writing to the parameter's address: the next call takes its new values."""
        self._weight16.drop()

    def weight_bf16(self, stream=None) -> Tensor:
        """The weight as the products on `stream` take it."""
        return self._weight16.get(self._parameters["weight"], lambda w: w.to(DType.bfloat16), stream)

    def forward(self, x, offsets):
        return lowp.grouped_linear(x, self.weight_bf16(x.stream), offsets)

    def backward(self, grad, x, offsets):
        """(dx in bfloat16, dweight in float32)."""
        return lowp.grouped_linear_backward(grad, x, self.weight_bf16(x.stream), offsets)


class Conv2d(Module):
    """2-D convolution (reference nn.py:118-142)."""

    def __init__(self, in_channels, out_channels, kernel_size, stride=1, padding=0, bias=True,
                 dtype=DType.float32):
        super().__init__()
        if isinstance(kernel_size, int):
            kernel_size = (kernel_size, kernel_size)
        if isinstance(stride, int):
            stride = (stride, stride)
        if isinstance(padding, int):
            padding = (padding, padding)
        self.stride = stride
        self.padding = padding
        self.register_parameter(
            "weight", Tensor.randn([out_channels, in_channels, kernel_size[0], kernel_size[1]], dtype))
        if bias:
            self.register_parameter("bias", Tensor.zeros([out_channels], dtype))

    def forward(self, x, activation=None):
        return conv2d(x, self._parameters["weight"], self._parameters.get("bias"), self.stride, self.padding,
                      activation)


class _Activation(Module):
    name: Optional[str] = None

    def forward(self, x):
        return getattr(x, self.name)()


class ReLU(_Activation):
    name = "relu"


class GELU(_Activation):
    name = "gelu"


class SiLU(_Activation):
    name = "silu"


class Sigmoid(_Activation):
    name = "sigmoid"


class Sequential(Module):
    """Runs modules in order (reference nn.py:173-189), fusing Linear/Conv2d + activation pairs."""

    def __init__(self, *modules, fuse=True):
        super().__init__()
        self.fuse = fuse
        for i, m in enumerate(modules):
            self.register_module(str(i), m)

    def forward(self, x):
        mods = list(self._modules.values())
        i = 0
        while i < len(mods):
            m = mods[i]
            nxt = mods[i + 1] if i + 1 < len(mods) else None
            if (self.fuse and isinstance(m, (Linear, Conv2d)) and isinstance(nxt, _Activation)
                    and (x.dtype() == DType.float32 or isinstance(m, LinearFp8))):
                x = m.forward(x, activation=nxt.name)
                i += 2
            else:
                x = m(x)
                i += 1
        return x

    def __getitem__(self, idx):
        return list(self._modules.values())[idx]

    def __len__(self):
        return len(self._modules)
