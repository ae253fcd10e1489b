"""Microscaled 4-bit layers (OCP Microscaling Formats 1.0, MXFP4) beside the ternary ones: for the
dense layers around the experts and for experts that do not stand three values a row.

    codes, scales = mx4.quantize(w)            # any rows of bf16, fp16 or fp32, on the GPU
    w = mx4.dequantize(codes, scales, width)
    layer = mx4.Mx4Linear.make(w)              # as Sub1Linear: y = layer(x), x bf16 [T, width]
    mlp = mx4.Mx4SparseMLP.from_mlp(mlp)       # as FasterMLP, the router in the launch too

A row of W values is ceil(W / 32) blocks of 32: 16 bytes of codes (value 2i in the low half of byte
i; a sign over the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one byte of scale, 2^(byte - 127), 255
for a block that is no number.  There is no backward pass: results are not connected to what they
were computed from, as everywhere in this package.
"""
import ctypes

import torch
import torch.nn as nn

from . import _lib
from .sub1_hip import _launch, _need

BLOCK = 32
_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}      # SUB1_MX4_BF16 ..


_entries = {}


def _entry(name):
    """The address of a library's function, for the calls that go all the way in C++."""
    at = _entries.get(name)
    if at is None:
        at = _entries[name] = ctypes.cast(getattr(_lib.load(), name), ctypes.c_void_p).value
    return at


def _there():
    """(the current device, torch's current stream on it)"""
    device = torch._C._cuda_getDevice()
    return device, torch._C._cuda_getCurrentRawStream(device)


def _quick(name, *args):
    """The result of a call whose tensors are plainly in order and on the current device, made in C++;
    None for any other, which the caller then looks at itself, for its copies or its error."""
    if not torch.cuda.is_initialized():      # (nothing is on a GPU yet)
        return None
    got = getattr(_lib.tensor_args(), name)(*args, *_there())
    if type(got) is int:
        _lib.check(got)
    return got


def _whole(value, name):
    """value as int, of whatever type of number."""
    if int(value) != value:
        raise ValueError('%s must be a whole number, got %r' % (name, value))
    return int(value)


def _blocks(width):
    return (width + BLOCK - 1) // BLOCK


def _rows(x, name, device=None):
    """(x as a matrix whose rows lie together, itself where they do; its row stride)."""
    if not isinstance(x, torch.Tensor):
        raise TypeError('%s must be a torch.Tensor' % name)
    if not x.is_cuda:
        raise ValueError('%s must live on the GPU' % name)
    if device is not None and x.device != device:
        raise ValueError('%s is on %s, expected %s' % (name, x.device, device))
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError('%s must have a last dimension, got %s' % (name, tuple(x.shape)))
    if x.shape[-1] > _lib.MX4_MAX_WIDTH:
        raise ValueError('%s has rows of %d, more than %d' % (name, x.shape[-1], _lib.MX4_MAX_WIDTH))
    x = x.resolve_neg()
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.stride(1) != 1 and x.shape[1] > 1 or x.stride(0) < x.shape[1] and x.shape[0] > 1:
        x = x.contiguous()
    return x, max(x.stride(0), x.shape[1])


def quantize(x):
    """(codes uint8 [.., 16 * blocks], scales uint8 [.., blocks]) of x [.., W] in bf16, fp16 or
    fp32.  Per block of 32: the scale is 2^e, e = floor(log2 of the largest magnitude) - 2 and not
    below -127; a value becomes the nearest of the magnitudes times 2^e (of two the one with an even
    code; at most 6 * 2^e).  A block with an infinity or a NaN is NaN.  Rows may be strided."""
    got = _quick('mx4_quantize', _entry('sub1_mx4_quantize'), x)
    if got is not None:
        return got
    rows, ld = _rows(x, 'x')
    kind = _TYPES.get(x.dtype)
    if kind is None:
        raise TypeError('x must be bf16, fp16 or fp32, got %s' % x.dtype)
    count, width = rows.shape
    blocks = _blocks(width)
    codes = torch.empty(x.shape[:-1] + (16 * blocks,), dtype=torch.uint8, device=x.device)
    scales = torch.empty(x.shape[:-1] + (blocks,), dtype=torch.uint8, device=x.device)
    if count:
        _launch(x.device, _lib.load().sub1_mx4_quantize, rows.data_ptr(), kind, ld, count, width, codes.data_ptr(),
                scales.data_ptr())
    return codes, scales


def _matrix(codes, scales, width, name, device=None):
    """(address of codes, of scales) of a matrix in the format, looked over."""
    blocks = _blocks(width)
    if not 1 <= width <= _lib.MX4_MAX_WIDTH:
        raise ValueError('width must be 1..%d, got %d' % (_lib.MX4_MAX_WIDTH, width))
    p_codes = _need(codes, torch.uint8, name + ' codes', device)
    p_scales = _need(scales, torch.uint8, name + ' scales', codes.device)
    if codes.dim() < 1 or codes.shape[-1] != 16 * blocks or scales.shape != codes.shape[:-1] + (blocks,):
        raise ValueError('%s codes must be [.., %d] and scales [.., %d] for a width of %d, got %s and %s' % (
            name, 16 * blocks, blocks, width, tuple(codes.shape), tuple(scales.shape)))
    if p_codes % 16:
        raise ValueError('%s codes must lie on 16 bytes' % name)
    return p_codes, p_scales


def dequantize(codes, scales, width, dtype=torch.bfloat16):
    """[.., width]: what codes and scales stand for, rounded to dtype (exact in bf16 and fp32)."""
    got = _quick('mx4_dequantize', _entry('sub1_mx4_dequantize'), codes, scales, width, dtype)
    if got is not None:
        return got
    kind = _TYPES.get(dtype)
    if kind is None:
        raise TypeError('dtype must be bf16, fp16 or fp32, got %s' % dtype)
    p_codes, p_scales = _matrix(codes, scales, width, 'the')
    out = torch.empty(codes.shape[:-1] + (width,), dtype=dtype, device=codes.device)
    if out.numel():
        _launch(out.device, _lib.load().sub1_mx4_dequantize, p_codes, p_scales, out.numel() // width, width,
                out.data_ptr(), kind, width)
    return out


def _fewer_tokens(x, what):
    if x.shape[0] > _lib.MX4_MAX_TOKENS:
        raise ValueError('%s: %d tokens, more than %d' % (what, x.shape[0], _lib.MX4_MAX_TOKENS))


def product(x, codes, scales):
    """bf16 [.., H] = x W^T for x bf16 [.., W] and W [H, W] in the format; fp32 sums."""
    got = _quick('mx4_product', _entry('sub1_mx4_product'), None, x, codes, scales, 0)
    if got is not None:
        return got
    rows, ld = _rows(x, 'x')
    if x.dtype != torch.bfloat16:
        raise TypeError('x must be torch.bfloat16, got %s' % x.dtype)
    tokens, width = rows.shape
    p_codes, p_scales = _matrix(codes, scales, width, 'the', x.device)
    if codes.dim() != 2:
        raise ValueError('codes must be 2-D')
    _fewer_tokens(rows, 'product')
    height = codes.shape[0]
    y = torch.empty(x.shape[:-1] + (height,), dtype=torch.bfloat16, device=x.device)
    if y.numel():
        _launch(x.device, _lib.load().sub1_mx4_product, p_codes, p_scales, height, width, rows.data_ptr(), ld,
                y.data_ptr(), height, tokens)
    return y


def product_quantized(x_codes, x_scales, codes, scales, width):
    """bf16 [.., H] = x W^T with x [.., W] and W [H, W] both in the format; fp32 sums."""
    p_x, p_xs = _matrix(x_codes, x_scales, width, 'x', None)
    p_codes, p_scales = _matrix(codes, scales, width, 'the', x_codes.device)
    if codes.dim() != 2:
        raise ValueError('codes must be 2-D')
    tokens, height = x_scales.numel() // x_scales.shape[-1], codes.shape[0]
    if tokens > _lib.MX4_MAX_TOKENS:
        raise ValueError('product_quantized: %d tokens, more than %d' % (tokens, _lib.MX4_MAX_TOKENS))
    y = torch.empty(x_codes.shape[:-1] + (height,), dtype=torch.bfloat16, device=codes.device)
    if y.numel():
        _launch(codes.device, _lib.load().sub1_mx4_product_quantized, p_codes, p_scales, height, width, p_x, p_xs,
                y.data_ptr(), height, tokens)
    return y


class Mx4Linear(nn.Module):
    """A linear layer held in the format: buffers `codes` uint8 [H, 16 * blocks], `scales` uint8 [H,
    blocks] and, as in Sub1Linear, an empty bf16 `weight`.  forward(x) takes bf16 activations; with
    `quantize_activations` it brings them to the format first and multiplies in 4 bits."""

    def __init__(self, codes, scales, width, quantize_activations=False):
        super().__init__()
        if codes.dim() != 2 or codes.shape[0] < 1:
            raise ValueError('codes must be [height, 16 * blocks], got %s' % (tuple(codes.shape),))
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError('codes and scales must be torch.uint8')
        width = _whole(width, 'width')
        blocks = _blocks(width)
        if codes.shape[1] != 16 * blocks or tuple(scales.shape) != (codes.shape[0], blocks):
            raise ValueError('codes must be [H, %d] and scales [H, %d] for a width of %d, got %s and %s' % (
                16 * blocks, blocks, width, tuple(codes.shape), tuple(scales.shape)))
        self.width = width
        self.quantize_activations = bool(quantize_activations)
        self.register_buffer('codes', codes)
        self.register_buffer('scales', scales)
        self.register_buffer('weight', torch.zeros(0, dtype=torch.bfloat16, device=codes.device))

    @staticmethod
    def make(w, quantize_activations=False):
        """The layer of a dense matrix [H, W] on the GPU, rounded to the format."""
        if not isinstance(w, torch.Tensor) or w.dim() != 2:
            raise ValueError('w must be a matrix')
        codes, scales = quantize(w.detach())
        return Mx4Linear(codes, scales, w.shape[1], quantize_activations)

    def forward(self, x):
        """x bf16 [.., width] -> bf16 [.., height]"""
        buffers = self._buffers
        codes, scales = buffers['codes'], buffers['scales']
        if self.quantize_activations:
            got = _quick('mx4_product', _entry('sub1_mx4_product_quantized'), _entry('sub1_mx4_quantize'), x, codes, scales,
                         self.width)
        else:
            got = _quick('mx4_product', _entry('sub1_mx4_product'), None, x, codes, scales, self.width)
        if got is not None:
            return got
        if not isinstance(x, torch.Tensor):
            raise TypeError('x must be a torch.Tensor')
        if x.shape[-1:] != (self.width,):
            raise ValueError('x must be [.., %d], got %s' % (self.width, tuple(x.shape)))
        if not self.quantize_activations:
            return product(x, codes, scales)
        if x.dtype != torch.bfloat16:
            raise TypeError('x must be torch.bfloat16, got %s' % x.dtype)
        x_codes, x_scales = quantize(x)
        return product_quantized(x_codes, x_scales, codes, scales, self.width)


class Mx4SparseMLP(nn.Module):
    """The sparse MLP of a Switch block with its experts in the format, for the few tokens of a
    generating model: router, choice of experts, both products with ReLU between and the weighted sum
    in one call (what reference sub1.py:299-321 does around its experts).

    router  [E, d_model] in bf16 or fp32
    wi, wo  (codes, scales) of all experts' matrices: [E, d_ff, ..] of width d_model, [E, d_model, ..]
            of width d_ff
    top_k   experts a token (1 to 8); `normalize`: their shares add up to 1
    capacity  with one expert a token: how many tokens of a sequence (the last but one dimension of what
            forward gets) an expert takes; the others keep their input, times their share.  Sequences that are
            longer than it have at most 256 tokens
    router_outputs  whether forward returns (hidden, (logits, index)) or hidden alone

    Logits are summed in 64 bits and rounded to fp32; of equal ones the expert of the lower index comes
    first.  What goes from an expert's first product to its second is rounded to bf16, as between two layers
    of a bf16 model.  Batches of more than 256 tokens run in parts, each of which reads its experts anew."""

    def __init__(self, router, wi, wo, top_k=1, normalize=False, capacity=None, router_outputs=True):
        super().__init__()
        if router.dim() != 2 or router.dtype not in (torch.bfloat16, torch.float32):
            raise ValueError('router must be [experts, d_model] in bf16 or fp32')
        experts, d_model = router.shape
        if wi[0].dim() != 3 or wo[0].dim() != 3:
            raise ValueError("the experts' codes must be [experts, height, 16 * blocks]")
        d_ff = wi[0].shape[1]
        for (codes, scales), height, width, name in ((wi, d_ff, d_model, 'wi'), (wo, d_model, d_ff, 'wo')):
            want = (experts, height, 16 * _blocks(width)), (experts, height, _blocks(width))
            if (tuple(codes.shape), tuple(scales.shape)) != want:
                raise ValueError('%s must be codes %s and scales %s, got %s and %s' % (
                    (name,) + want + (tuple(codes.shape), tuple(scales.shape))))
            if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
                raise TypeError('%s must be torch.uint8' % name)
        top_k = _whole(top_k, 'top_k')
        if not 1 <= top_k <= min(experts, _lib.MX4_LAYER_TOP_K):
            raise ValueError('top_k must be 1..%d, got %d' % (min(experts, _lib.MX4_LAYER_TOP_K), top_k))
        if experts > _lib.MX4_LAYER_EXPERTS or max(d_model, d_ff) > _lib.MX4_MAX_WIDTH:
            raise ValueError('at most %d experts of %d' % (_lib.MX4_LAYER_EXPERTS, _lib.MX4_MAX_WIDTH))
        capacity = None if capacity is None else _whole(capacity, 'capacity')
        if capacity is not None and (top_k != 1 or capacity < 1):
            raise ValueError('a capacity is at least 1 and goes with one expert a token')
        self.experts, self.d_model, self.d_ff = experts, d_model, d_ff
        self.top_k, self.normalize, self.capacity = top_k, bool(normalize), capacity
        self.router_outputs = bool(router_outputs)
        for name, t in (('router', router), ('wi_codes', wi[0]), ('wi_scales', wi[1]), ('wo_codes', wo[0]),
                        ('wo_scales', wo[1])):
            self.register_buffer(name, t)

    @staticmethod
    def from_mlp(mlp, top_k=1, normalize=False, router_outputs=True):
        """The layer of a `SwitchTransformersSparseMLP`-shaped module on the GPU: `mlp.router` with a
        linear `classifier` (and `expert_capacity`, with one expert a token taken where there is one, for
        which forward refuses sequences of more than 256 tokens that are longer than it), `mlp.experts` (a
        ModuleDict of modules with dense `wi`/`wo`), whose matrices are rounded to the format."""
        experts = list(mlp.experts.values())
        for expert in experts:
            act = getattr(expert, 'act', None)
            if act is not None and not isinstance(act, nn.ReLU):
                raise ValueError('Mx4SparseMLP runs ReLU experts; this one has %r' % (act,))
        for linear in [mlp.router.classifier] + [l for e in experts for l in (e.wi, e.wo)]:
            if getattr(linear, 'bias', None) is not None:
                raise ValueError('Mx4SparseMLP runs layers without a bias')
        router = mlp.router.classifier.weight.detach()
        if router.dtype != torch.bfloat16:
            router = router.float()
        wi, wo = [[quantize(getattr(e, name).weight.detach()) for e in experts] for name in ('wi', 'wo')]
        stack = [tuple(torch.stack([m[i] for m in w]) for i in (0, 1)) for w in (wi, wo)]
        capacity = getattr(mlp.router, 'expert_capacity', None) if top_k == 1 else None
        return Mx4SparseMLP(router.contiguous(), stack[0], stack[1], top_k, normalize, capacity, router_outputs)

    def _parts(self, tokens, length):
        """(first, tokens) of each launch: whole sequences where their order counts."""
        most = _lib.MX4_LAYER_TOKENS
        if self.capacity is not None and length > self.capacity and tokens > most:
            if length > most:
                raise ValueError('a capacity is kept over sequences of at most %d tokens, got %d' % (most, length))
            most -= most % length
        return [(first, min(most, tokens - first)) for first in range(0, tokens, most)]

    def forward(self, hidden):
        """hidden bf16 [.., S, d_model] -> hidden bf16 like it, with `router_outputs` also (logits
        fp32 [.., S, E], index int64 [.., S, top_k])."""
        b = self._buffers
        got = _quick('mx4_layer', _entry('sub1_mx4_layer_forward'), _entry('sub1_mx4_layer_scratch_bytes'), hidden, b['router'],
                     b['wi_codes'], b['wi_scales'], b['wo_codes'], b['wo_scales'], self.top_k, int(self.normalize),
                     self.capacity or 0)      # (one past 2^30 goes the other way)
        if got is not None:
            return (got[0], got[1:]) if self.router_outputs else got[0]
        if not isinstance(hidden, torch.Tensor):
            raise TypeError('hidden must be a torch.Tensor')
        if hidden.dim() < 2 or hidden.shape[-1] != self.d_model:
            raise ValueError('hidden must be [.., S, %d], got %s' % (self.d_model, tuple(hidden.shape)))
        device, shape = self.router.device, hidden.shape
        x = hidden.contiguous().resolve_neg()
        p_x = _need(x, torch.bfloat16, 'hidden', device)
        if self.router.dtype not in (torch.bfloat16, torch.float32):
            raise TypeError('router must be bf16 or fp32, got %s' % self.router.dtype)
        length = shape[-2]
        capacity = self.capacity if self.capacity is not None and length > self.capacity else 0   # 0: all are taken
        p_wi = _matrix(self.wi_codes, self.wi_scales, self.d_model, 'wi', device)
        p_wo = _matrix(self.wo_codes, self.wo_scales, self.d_ff, 'wo', device)
        layer = _lib.Mx4Layer(_need(self.router, self.router.dtype, 'router', device), p_wi[0], p_wi[1], p_wo[0], p_wo[1],
                              self.experts, self.d_model, self.d_ff, self.top_k, _TYPES[self.router.dtype],
                              self.normalize, capacity)
        tokens = x.numel() // self.d_model
        y = torch.empty_like(x)
        logits = torch.empty(shape[:-1] + (self.experts,), dtype=torch.float32, device=device)
        index = torch.empty(shape[:-1] + (self.top_k,), dtype=torch.int64, device=device)
        lib = _lib.load()
        for first, count in self._parts(tokens, length):
            # of the call's own, from torch's allocator: two calls at once, on streams or in captured
            # graphs, never share it
            scratch = torch.empty(lib.sub1_mx4_layer_scratch_bytes(ctypes.byref(layer), count), dtype=torch.uint8,
                                  device=device)
            _launch(device, lib.sub1_mx4_layer_forward, ctypes.byref(layer), p_x + 2 * first * self.d_model, count,
                    length if capacity else 1, y.data_ptr() + 2 * first * self.d_model,
                    logits.data_ptr() + 4 * first * self.experts, index.data_ptr() + 8 * first * self.top_k,
                    scratch.data_ptr(), scratch.numel())
        if self.router_outputs:
            return y, (logits, index)
        return y
