"""Microscaled 8-bit activations (OCP Microscaling Formats 1.0, MXFP8 with e4m3 elements) for the 4-bit
layers of qmoe_amd.mx4: finer than activations in 4 bits, and at the matrix cores' rate for 8 bits.

    codes, scales = mx8.quantize(x)                      # or norm.rms_norm(.., quantize=True)
    h = mx8.product(codes, scales, w_codes, w_scales, width, relu=True, quantize=True)
    y = mx8.product(*h, wo_codes, wo_scales, d_ff)
    mlp = mx8.Mx4DenseMLP(wi, wo)                        # the same two products, of Mx4Linear layers

A row of W values is ceil(W / 32) blocks of 32: 32 bytes of codes (e4m3, one a byte, values behind W zero)
and one byte of scale, 2^(byte - 127), 255 for a block that is no number.  There is no backward pass.
"""
import torch
import torch.nn as nn

from . import _lib, mx4
from .mx4 import _blocks, _entry, _quick, _rows, _TYPES
from .sub1_hip import _launch, _need

BLOCK = mx4.BLOCK


def _activations(codes, scales, width, name, device=None):
    """(address of codes, of scales) of activations in the format, looked over."""
    if not 1 <= width <= _lib.MX4_MAX_WIDTH:
        raise ValueError('width must be 1..%d, got %d' % (_lib.MX4_MAX_WIDTH, width))
    blocks = _blocks(width)
    p_codes = _need(codes, torch.uint8, name + ' codes', device)
    p_scales = _need(scales, torch.uint8, name + ' scales', codes.device)
    if codes.dim() < 1 or codes.shape[-1] != 32 * blocks or scales.shape != codes.shape[:-1] + (blocks,):
        raise ValueError('%s codes must be [.., %d] and scales [.., %d] for a width of %d, got %s and %s' % (
            name, 32 * blocks, blocks, width, tuple(codes.shape), tuple(scales.shape)))
    if p_codes % 16:
        raise ValueError('%s codes must lie on 16 bytes' % name)
    return p_codes, p_scales


def _empty(shape, width, device):
    blocks = _blocks(width)
    return (torch.empty(shape + (32 * blocks,), dtype=torch.uint8, device=device),
            torch.empty(shape + (blocks,), dtype=torch.uint8, device=device))


def quantize(x):
    """(codes uint8 [.., 32 * blocks], scales uint8 [.., blocks]) of x [.., W] in bf16, fp16 or fp32.  Per block of
    32: the scale is the smallest 2^e, e at least -127, under which the largest magnitude is at most 448; a value
    becomes the nearest e4m3 times 2^e.  A block with an infinity or a NaN is NaN.  Rows may be strided."""
    got = _quick('mx8_quantize', _entry('sub1_mx8_quantize'), x)
    if got is not None:
        return got
    rows, ld = _rows(x, 'x')
    kind = _TYPES.get(x.dtype)
    if kind is None:
        raise TypeError('x must be bf16, fp16 or fp32, got %s' % x.dtype)
    count, width = rows.shape
    codes, scales = _empty(x.shape[:-1], width, x.device)
    if count:
        _launch(x.device, _lib.load().sub1_mx8_quantize, rows.data_ptr(), kind, ld, count, width, codes.data_ptr(),
                scales.data_ptr())
    return codes, scales


def dequantize(codes, scales, width, dtype=torch.bfloat16):
    """[.., width]: what codes and scales stand for, rounded to dtype (in bf16 exact but below 2^-126)."""
    got = _quick('mx8_dequantize', _entry('sub1_mx8_dequantize'), codes, scales, width, dtype)
    if got is not None:
        return got
    kind = _TYPES.get(dtype)
    if kind is None:
        raise TypeError('dtype must be bf16, fp16 or fp32, got %s' % dtype)
    width = mx4._whole(width, 'width')
    p_codes, p_scales = _activations(codes, scales, width, 'the')
    out = torch.empty(codes.shape[:-1] + (width,), dtype=dtype, device=codes.device)
    if out.numel():
        _launch(out.device, _lib.load().sub1_mx8_dequantize, p_codes, p_scales, out.numel() // width, width,
                out.data_ptr(), kind, width)
    return out


def product(x_codes, x_scales, codes, scales, width, relu=False, quantize=False):
    """bf16 [.., H] = x W^T with x [.., W] in 8 bits and W [H, W] in 4 (mx4.quantize).  `relu`: what is below zero becomes
    zero; `quantize`: the result in 8 bits, (codes [.., 32 * blocks of H], scales), rounded once.

    Sums are coarser than fp32 for more than one token: of eight neighbouring products each the matrix cores cut off what is
    below a step of 2^-13, at most 2^-12, of the largest (one from 2^-7 of the largest on loses nothing); what is left is added in
    fp32.  One token's are fp32 sums, so that its last bits may be others than in a batch.  Sums in fp32 for any number of tokens,
    in 1.8 to 2.7 times the time: mx4.product(mx8.dequantize(x_codes, x_scales, width), codes, scales)."""
    got = _quick('mx8_product', _entry('sub1_mx8_product'), x_codes, x_scales, codes, scales, width, relu, quantize)
    if got is not None:
        return got
    width = mx4._whole(width, 'width')
    p_x, p_xs = _activations(x_codes, x_scales, width, 'x')
    p_codes, p_scales = mx4._matrix(codes, scales, width, 'the', x_codes.device)
    if codes.dim() != 2:
        raise ValueError('codes must be 2-D')
    height, shape, device = codes.shape[0], x_codes.shape[:-1], codes.device
    tokens = x_codes.numel() // x_codes.shape[-1]
    if tokens > _lib.MX4_MAX_TOKENS:
        raise ValueError('product: %d tokens, more than %d' % (tokens, _lib.MX4_MAX_TOKENS))
    if not 1 <= height <= _lib.MX4_MAX_WIDTH:
        raise ValueError('the matrix must have 1..%d rows, got %d' % (_lib.MX4_MAX_WIDTH, height))
    if quantize:
        out = _empty(shape, height, device)
        p_y = (None, 0, out[0].data_ptr(), out[1].data_ptr())
    else:
        out = torch.empty(shape + (height,), dtype=torch.bfloat16, device=device)
        p_y = (out.data_ptr(), height, None, None)
    if tokens:
        _launch(device, _lib.load().sub1_mx8_product, p_codes, p_scales, height, width, p_x, p_xs, int(bool(relu)), *p_y,
                tokens)
    return out


class Mx4DenseMLP(nn.Module):
    """The dense MLP of a Switch block, wo(relu(wi(x))), of two mx4.Mx4Linear layers, in 8-bit activations: from
    one product to the next they stay in 8 bits.  forward takes activations in 8 bits, (codes, scales) as
    norm.rms_norm(.., quantize=True) and norm.RMSNorm give them, or bf16 ones, which it brings there."""

    def __init__(self, wi, wo):
        super().__init__()
        for layer, name in ((wi, 'wi'), (wo, 'wo')):
            if not isinstance(layer, mx4.Mx4Linear):
                raise TypeError('%s must be an Mx4Linear' % name)
        if wo.width != wi.codes.shape[0]:
            raise ValueError('wo takes %d values, wi gives %d' % (wo.width, wi.codes.shape[0]))
        self.wi, self.wo = wi, wo

    @staticmethod
    def from_mlp(mlp):
        """The layer of a `SwitchTransformersDenseActDense`-shaped module on the GPU (dense `wi` and `wo`, ReLU in
        `act`), its matrices rounded to 4 bits."""
        act = getattr(mlp, 'act', None)
        if act is not None and not isinstance(act, nn.ReLU):
            raise ValueError('Mx4DenseMLP runs ReLU; this one has %r' % (act,))
        for linear in (mlp.wi, mlp.wo):
            if getattr(linear, 'bias', None) is not None:
                raise ValueError('Mx4DenseMLP runs layers without a bias')
        return Mx4DenseMLP(mx4.Mx4Linear.make(mlp.wi.weight), mx4.Mx4Linear.make(mlp.wo.weight))

    def forward(self, x):
        """x bf16 [.., width] or (codes, scales) of such -> bf16 [.., height of wo]"""
        wi, wo = self.wi, self.wo
        if isinstance(x, torch.Tensor):
            if x.dtype != torch.bfloat16:
                raise TypeError('x must be torch.bfloat16, got %s' % x.dtype)
            if x.shape[-1:] != (wi.width,):
                raise ValueError('x must be [.., %d], got %s' % (wi.width, tuple(x.shape)))
            x = quantize(x)
        elif not (isinstance(x, (tuple, list)) and len(x) == 2):
            raise TypeError('x must be a torch.Tensor or (codes, scales)')
        h = product(*x, wi.codes, wi.scales, wi.width, True, True)
        return product(*h, wo.codes, wo.scales, wo.width)
