"""Root-mean-square norm with the residual's addition, as it stands before every sub-layer of a Switch block.

    y = norm.rms_norm(x, weight, eps)                            # in x's type
    y, total = norm.rms_norm(x, weight, eps, residual)           # total = x + residual goes on, y is its norm
    (codes, scales), total = norm.rms_norm(x, weight, eps, residual, quantize=True)      # y in 8 bits, for qmoe_amd.mx8
    layer = norm.RMSNorm.from_norm(block.layer[0].layer_norm)

There is no backward pass.
"""
import ctypes

import torch
import torch.nn as nn

from . import _lib, mx8
from .mx4 import _entry, _quick, _rows, _TYPES
from .sub1_hip import _launch, _need


def rms_norm(x, weight, eps=1e-6, residual=None, quantize=False):
    """s / sqrt(mean(s^2) + eps) * weight over the last dimension, s = x or x + residual rounded to the residual's type.

    x [.., W] in bf16, fp16 or fp32; weight [W] and residual (like x) in x's type or fp32.  Sums in 64 bits, what
    follows in fp32, rounded at the end: to x's type, or with `quantize` to 8 bits, (codes, scales) as mx8.quantize.  With a
    residual returns (result, s).  Rows may be strided."""
    got = _quick('rms_norm', _entry('sub1_rms_norm'), x, weight, eps, residual, quantize)
    if got is not None:
        return got
    eps = float(eps)
    if not _lib.NORM_LEAST_EPS <= eps <= 1e30:
        raise ValueError('eps must be %g..1e30, got %g' % (_lib.NORM_LEAST_EPS, eps))
    rows, ldx = _rows(x, 'x')
    kind = _TYPES.get(x.dtype)
    if kind is None:
        raise TypeError('x must be bf16, fp16 or fp32, got %s' % x.dtype)
    count, width = rows.shape
    if count > _lib.NORM_MAX_ROWS:
        raise ValueError('rms_norm: %d rows, more than %d' % (count, _lib.NORM_MAX_ROWS))
    if isinstance(weight, torch.Tensor) and weight.dtype not in (x.dtype, torch.float32):
        raise TypeError("weight must be in x's type or fp32, got %s" % weight.dtype)
    weight = weight.resolve_neg() if isinstance(weight, torch.Tensor) else weight
    p_weight = _need(weight, getattr(weight, 'dtype', None), 'weight', x.device, width, 1)
    n = _lib.Norm(p_weight, eps, width, kind, kind, _TYPES[weight.dtype])
    p_residual, ldr, total, p_total = None, 0, None, None
    if residual is not None:
        r, ldr = _rows(residual, 'residual', x.device)
        if residual.shape != x.shape:
            raise ValueError('residual must be %s, got %s' % (tuple(x.shape), tuple(residual.shape)))
        if residual.dtype not in (x.dtype, torch.float32):
            raise TypeError("residual must be in x's type or fp32, got %s" % residual.dtype)
        n.residual_type = _TYPES[residual.dtype]
        total = torch.empty(x.shape, dtype=residual.dtype, device=x.device)
        p_residual, p_total = r.data_ptr(), total.data_ptr()
    if quantize:
        y = mx8._empty(x.shape[:-1], width, x.device)
        p_y = (None, 0, y[0].data_ptr(), y[1].data_ptr())
    else:
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        p_y = (y.data_ptr(), width, None, None)
    if count:
        _launch(x.device, _lib.load().sub1_rms_norm, ctypes.byref(n), rows.data_ptr(), ldx, p_residual, ldr, p_total, width,
                *p_y, count)
    return y if residual is None else (y, total)


class RMSNorm(nn.Module):
    """A Switch block's layer norm: weight [W] and eps; forward(x, residual) as rms_norm, in 8 bits where `quantize` says so."""

    def __init__(self, weight, eps=1e-6, quantize=False):
        super().__init__()
        if not isinstance(weight, torch.Tensor) or weight.dim() != 1 or weight.numel() < 1:
            raise ValueError('weight must be a tensor [width]')
        if weight.dtype not in _TYPES:
            raise TypeError('weight must be bf16, fp16 or fp32, got %s' % weight.dtype)
        if not _lib.NORM_LEAST_EPS <= float(eps) <= 1e30:
            raise ValueError('eps must be %g..1e30, got %g' % (_lib.NORM_LEAST_EPS, eps))
        self.eps, self.quantize = float(eps), bool(quantize)
        self.register_buffer('weight', weight.detach())

    @staticmethod
    def from_norm(layer, quantize=False):
        """The layer of a `SwitchTransformersLayerNorm`-shaped module (`weight`, `variance_epsilon`)."""
        return RMSNorm(layer.weight, layer.variance_epsilon, quantize)

    def forward(self, x, residual=None):
        return rms_norm(x, self._buffers['weight'], self.eps, residual, self.quantize)
