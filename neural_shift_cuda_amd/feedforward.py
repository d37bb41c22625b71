"""Token operators of a block's second half, next to the attention of
``attention.py`` (extensions, no counterpart in the reference).

    layer_norm(x, weight=None, bias=None, *, residual=None, eps=1e-5)
                                                     -> y or (y, s)
    gated_linear(x, gate_weight, up_weight, *, activation="silu")  -> h

Tokens are rows: the last dimension is a token's width, and whatever stands
before it counts rows.  GPU tensors go through autograd nodes in C++
(host/block_calls.cpp) into the HIP library (fp16, bf16, fp32; sums, means and
activations in fp32); CPU tensors use the ``*_reference`` implementations (any
floating type), which are also exported.  A GPU tensor never falls back to them.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import ops
from .attention import _acc, _same, _traceable

_C = ops._C

ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")
_CODES = {name: code for code, name in enumerate(ACTIVATIONS, 1)}  # as in neural_shift_hip.h


# ---------------------------------------------------------------------------
# Argument handling
# ---------------------------------------------------------------------------

def _rows(t: torch.Tensor, name: str) -> None:
    if t.dim() < 1:
        raise ValueError(f"{name} must have a width, (..., width); got a scalar")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be floating point; got {t.dtype}")


def _check_layer_norm(x, weight, bias, residual, eps) -> None:
    _rows(x, "x")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _same(name, t, x)
            if tuple(t.shape) != (x.shape[-1],):
                raise ValueError(f"{name} must be ({x.shape[-1]},); got {tuple(t.shape)}")
    if residual is not None:
        _same("residual", residual, x)
        if residual.shape != x.shape:
            raise ValueError(f"residual must be {tuple(x.shape)}; got {tuple(residual.shape)}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"eps must be finite and not negative; got {eps}")


def _check_gated(x, gate_weight, up_weight, activation) -> None:
    _rows(x, "x")
    for name, t in (("gate_weight", gate_weight), ("up_weight", up_weight)):
        _same(name, t, x)
        if t.dim() != 2 or t.shape[1] != x.shape[-1] or t.shape != gate_weight.shape:
            raise ValueError(f"gate_weight and up_weight must both be (hidden, {x.shape[-1]}); got "
                             f"{tuple(gate_weight.shape)} and {tuple(up_weight.shape)}")
    if activation not in _CODES:
        raise ValueError(f"activation must be one of {', '.join(ACTIVATIONS)}; got {activation!r}")


# ---------------------------------------------------------------------------
# CPU reference implementations (pure PyTorch, differentiable)
# ---------------------------------------------------------------------------

def layer_norm_reference(x, weight=None, bias=None, *, residual=None, eps: float = 1e-5):
    """CPU reference for ``layer_norm``."""
    _check_layer_norm(x, weight, bias, residual, eps)
    s = x if residual is None else x + residual
    y = s.to(_acc(x))
    if x.shape[-1]:
        y = y - y.mean(-1, keepdim=True)
        y = y - y.mean(-1, keepdim=True)  # what the first sum's rounding left
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.to(y.dtype)
    if bias is not None:
        y = y + bias.to(y.dtype)
    y = y.to(x.dtype)
    return y if residual is None else (y, s)


def _activated(g: torch.Tensor, activation: str) -> torch.Tensor:
    if activation == "silu":
        return torch.nn.functional.silu(g)
    if activation == "gelu":
        return torch.nn.functional.gelu(g)
    if activation == "gelu_tanh":
        return torch.nn.functional.gelu(g, approximate="tanh")
    return torch.relu(g) if activation == "relu" else torch.sigmoid(g)


def gated_linear_reference(x, gate_weight, up_weight, *, activation: str = "silu") -> torch.Tensor:
    """CPU reference for ``gated_linear``."""
    _check_gated(x, gate_weight, up_weight, activation)
    y = x.to(_acc(x))
    g, u = (torch.nn.functional.linear(y, w.to(y.dtype)) for w in (gate_weight, up_weight))
    return (_activated(g, activation) * u).to(x.dtype)


# ---------------------------------------------------------------------------
# Public API
# ---------------------------------------------------------------------------

def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Layer norm over the last dimension, of x or of its sum with a residual stream:

        s = x + residual
        y = (s - mean(s)) / sqrt(var(s) + eps) * weight + bias

    x (..., width) of any strides, residual of its shape, weight and bias
    (width,) or None, all of one type.  The variance is that of the row (divided
    by width).  s is rounded to the type, and the norm is of what is returned.

    Returns y, or (y, s) with a residual, contiguous.  Differentiable in all of
    them (x and residual have the same gradient); the weights' gradients are
    summed in fp32 in a fixed order.  The GPU serves widths up to 2^30."""
    if not x.is_cuda:
        return layer_norm_reference(x, weight, bias, residual=residual, eps=eps)
    done = _C and _C.layer_norm_as_is(x, weight, bias, residual, eps)
    if done is None:
        return _traceable(_layer_norm, (x, weight, bias, residual), eps=eps)
    return done[0] if residual is None else done


def _layer_norm(x, weight, bias, residual, *, eps):
    _check_layer_norm(x, weight, bias, residual, eps)
    ops._require_cuda_ext("layer_norm")
    w, b = (t if t is None else t.contiguous() for t in (weight, bias))
    y, s = _C.layer_norm(x, w, b, residual, eps)
    return y if residual is None else (y, s)


def gated_linear(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, *,
                 activation: str = "silu") -> torch.Tensor:
    """The gated projections of a feed-forward, in front of its last one:

        h = act(x gate_weight^T) * (x up_weight^T)

    x (..., width), gate_weight and up_weight (hidden, width), as a linear
    layer's, all of one type and any strides (the halves of one matrix are read
    where they lie).  `activation`: "silu", "gelu", "gelu_tanh", "relu" or
    "sigmoid".

    Returns h (..., hidden), contiguous: products, activation and their product
    in fp32, rounded once.  Differentiable in all three; training keeps two factors for each
    of h (4.25 bytes in bf16, 6 in fp16, 8 in fp32), and the gradients of the two projections
    are rounded to the type, as operands of the products that give the inputs' gradients.  The
    GPU serves width and hidden up to 2^20; rows that do not start on 16 bytes are copied
    first.  In fp32 large products are summed from bf16 products of three parts, which leave
    out 4e-8 of a product on average, and below 2^-21 of it."""
    if not x.is_cuda:
        return gated_linear_reference(x, gate_weight, up_weight, activation=activation)
    code = _CODES.get(activation)
    done = _C and code and _C.gated_linear_as_is(x, gate_weight, up_weight, code)
    if done is not None:
        return done
    return _traceable(_gated_linear, (x, gate_weight, up_weight), activation=activation)


def _gated_linear(x, gate_weight, up_weight, *, activation):
    _check_gated(x, gate_weight, up_weight, activation)
    ops._require_cuda_ext("gated_linear")
    return _C.gated_linear(x, gate_weight, up_weight, _CODES[activation])


__all__ = ["layer_norm", "gated_linear", "layer_norm_reference", "gated_linear_reference"]
