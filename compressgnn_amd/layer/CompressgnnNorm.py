"""Layer norm of node features, with the ReLU and the dropout that follow it between two layers of a model.

out = drop(relu((x - mean) / sqrt(variance + eps) * weight + bias)), mean and variance over the last dimension: one
kernel forward and one pass over the rows for all gradients, with a small sum of the parameters' parts behind it.  Nothing of the size of x
is kept for the gradient but x itself.  The reference's models take these operators from torch.

A norm of rows that a reconstruct layer copies from representatives is best taken before it, on the representatives
(layer/CompressgnnReconstruct.py): rows that are copies of each other are normalised alike.
"""
import _paths  # noqa: F401
import torch
from torch.autograd.function import once_differentiable

import compressgnn_runtime as _native
from CompressgnnDropout import Masks

_ACTIVATIONS = (None, 'relu')
_layer_norm = _native.layer_norm


class _Normed(torch.autograd.Function):
    """(x, weight, bias, eps, relu, p, seed, offset, counter) -> out: the step of _native.layer_norm, for what a native
    one does not take part in"""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, relu, p, seed, offset, counter):
        out, stats = _native.layer_norm_forward(x, weight, bias, eps, relu, p, seed, offset, counter)
        ctx.save_for_backward(x, stats, weight, bias, counter)
        ctx.call = (relu, p, seed, offset)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, stats, weight, bias, counter = ctx.saved_tensors
        dx, dweight, dbias = _native.layer_norm_backward(grad, x, stats, weight, bias, *ctx.call, counter)
        return dx, None if weight is None else dweight, None if bias is None else dbias, None, None, None, None, None, None


def norm_act_dropout(x, weight=None, bias=None, eps=1e-5, activation=None, p=0.0, seed=0, offset=0, counter=None):
    """drop(act(layer_norm(x))) over the last dimension of x; activation: None or 'relu'; p, seed, offset and counter as
    in CompressgnnDropout.dropout, and the same mask: dropout(act(layer_norm(x)), p, seed, offset, counter).
    weight, bias: vectors of x's type, or float32 beside 16-bit rows, or None."""
    if activation not in _ACTIVATIONS:
        raise ValueError("activation must be None or 'relu'")
    relu = activation is not None
    out = _layer_norm(x, weight, bias, eps, relu, p, seed, offset, counter)
    return _Normed.apply(x, weight, bias, eps, relu, p, seed, offset, counter) if out is None else out


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last dimension of x."""
    out = _layer_norm(x, weight, bias, eps)
    return norm_act_dropout(x, weight, bias, eps) if out is None else out


class Compressgnn_LayerNorm(Masks, torch.nn.Module):
    """Layer norm of `features` features, then the activation (None or 'relu'), then, in training, dropout with probability p."""

    def __init__(self, features, eps=1e-5, affine=True, activation=None, p=0.0, seed=None, dtype=None):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError("activation must be None or 'relu'")
        if not 0 <= p <= 1:
            raise ValueError("p has to lie in [0, 1], got %r" % (p,))
        self.features, self.eps, self.activation, self.p = features, eps, activation, p
        self.weight = torch.nn.Parameter(torch.ones(features, dtype=dtype)) if affine else None
        self.bias = torch.nn.Parameter(torch.zeros(features, dtype=dtype)) if affine else None
        self._init_masks(seed)

    def forward(self, x):
        if x.dim() == 0 or x.size(-1) != self.features:
            raise ValueError("rows of %d features expected, got %s" % (self.features, tuple(x.shape)))
        if self.training and self.p > 0:
            return norm_act_dropout(x, self.weight, self.bias, self.eps, self.activation, self.p, *self._next_mask(x))
        return norm_act_dropout(x, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self):
        return "%d, eps=%g, affine=%s, activation=%r, p=%g" % (self.features, self.eps, self.weight is not None, self.activation, self.p)
