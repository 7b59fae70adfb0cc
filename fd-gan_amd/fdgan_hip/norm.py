"""Layer norm on the HIP path: the norm for a network whose batch statistics must not enter (a critic trained image by image), beside
the BatchNorm that the planned networks fold into their convolutions.

    layer_norm(x, normalized_shape, weight, bias, eps)    torch.nn.functional.layer_norm's semantics, differentiable
    LayerNorm(normalized_shape, ...)                      torch.nn.LayerNorm's constructor, attributes and state_dict keys

x: fp32, fp16 or bf16 on the GPU; the result has its shape and type and is contiguous.  weight / bias: fp32 or x's type.  Statistics and
sums are fp32 whatever the types; every result is rounded once.  A row may lie in a wider buffer (the leading dimensions at one
pitch: a channel slice of a concatenation); any other layout is copied first.  Gradients can be taken once; forward-mode derivatives
(torch.autograd.forward_ad, torch.func.jvp) are refused."""
import numbers

import torch

from . import lib as L

_op = None


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """torch.nn.functional.layer_norm(x, normalized_shape, weight, bias, eps) on the HIP path.  ValueError for shapes that do not fit and a
    negative eps, TypeError for other types, RuntimeError off the GPU and for tensors with a forward-mode tangent (csrc/torch_ops.cpp)."""
    global _op
    if _op is None:
        _op = L.torch_ops().layer_norm.default
    return _op(x, normalized_shape if isinstance(normalized_shape, (tuple, list)) else (int(normalized_shape),), weight, bias, eps)


class LayerNorm(torch.nn.Module):
    """torch.nn.LayerNorm's constructor, attributes and state_dict keys over layer_norm."""

    def __init__(self, normalized_shape, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__()
        self.normalized_shape = (normalized_shape,) if isinstance(normalized_shape, numbers.Integral) else tuple(normalized_shape)
        self.eps, self.elementwise_affine = eps, elementwise_affine
        if elementwise_affine:
            self.weight = torch.nn.Parameter(torch.ones(self.normalized_shape, device=device, dtype=dtype))
        else:
            self.register_parameter("weight", None)
        if elementwise_affine and bias:
            self.bias = torch.nn.Parameter(torch.zeros(self.normalized_shape, device=device, dtype=dtype))
        else:
            self.register_parameter("bias", None)

    def reset_parameters(self):
        if self.weight is not None:
            torch.nn.init.ones_(self.weight)
        if self.bias is not None:
            torch.nn.init.zeros_(self.bias)

    def forward(self, x):
        return layer_norm(x, self.normalized_shape, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return "%s, eps=%s, elementwise_affine=%s" % (self.normalized_shape, self.eps, self.elementwise_affine)
