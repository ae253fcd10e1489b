"""Which experts a token goes to, and the weighted sum of what they put out.

    shares, index = routing.route(logits, top_k=2, normalize=True)
    shares, index = routing.route(logits, 8, scores='sigmoid', bias=balance, groups=8, top_groups=4, group_mark=2)
    y = routing.combine(outputs, shares, residual)               # outputs [T, top_k, W]
    mlp = routing.RoutedMLP(classifier, experts, top_k=2)        # around a Sub1Experts

There is no backward pass.
"""
import ctypes

import torch
import torch.nn as nn

from . import _lib, sub1
from .mx4 import _entry, _quick, _rows, _TYPES, _whole
from .sub1_hip import _launch, _need

_SCORES = {'softmax': 0, 'sigmoid': 1}      # SUB1_ROUTE_SOFTMAX, _SIGMOID


def _plan(experts, top_k, scores, groups, top_groups, group_mark):
    """(top_k, groups, top_groups, group_mark) as whole numbers that go together."""
    top_k, groups, group_mark = _whole(top_k, 'top_k'), _whole(groups, 'groups'), _whole(group_mark, 'group_mark')
    top_groups = groups if top_groups is None else _whole(top_groups, 'top_groups')
    if scores not in _SCORES:
        raise ValueError("scores must be 'softmax' or 'sigmoid', got %r" % (scores,))
    if not 1 <= experts <= _lib.ROUTE_MAX_EXPERTS:
        raise ValueError('1..%d experts, got %d' % (_lib.ROUTE_MAX_EXPERTS, experts))
    if not 1 <= groups <= _lib.ROUTE_MAX_GROUPS or experts % groups:
        raise ValueError('groups must be 1..%d of one size, got %d of %d experts' % (_lib.ROUTE_MAX_GROUPS, groups, experts))
    if not 1 <= top_groups <= groups:
        raise ValueError('top_groups must be 1..%d, got %d' % (groups, top_groups))
    if group_mark not in (1, 2):
        raise ValueError('group_mark must be 1 or 2, got %d' % group_mark)
    most = min(experts // groups * top_groups, _lib.ROUTE_MAX_TOP_K)
    if not 1 <= top_k <= most:
        raise ValueError('top_k must be 1..%d, got %d' % (most, top_k))
    return top_k, groups, top_groups, group_mark


def route(logits, top_k, scores='softmax', bias=None, groups=1, top_groups=None, group_mark=1, normalize=False, scale=1.0,
          dtype=torch.int64):
    """(shares fp32 [.., top_k], index [.., top_k] of `dtype`, int64 or int32) by a router's logits [.., E].

    s = softmax(logits) or sigmoid(logits); c = s + bias (fp32 [E]; it decides, and is no part of the shares).  Of `groups`
    groups of experts that lie together the top_groups (default: all) with the largest marks are taken, a mark being the sum of
    a group's group_mark (1 or 2) largest c; of their experts the top_k with the largest c, the largest first.  shares = s at
    those, with `normalize` over their sum (unless that is zero), times `scale`.

    What decides is compared in 64 bits, without a bias in the order of the logits themselves; of equal ones the lower index
    comes first, what is no number last.  Experts masked by a logit of -inf score 0."""
    got = _quick('route', _entry('sub1_route'), logits, top_k, _SCORES.get(scores) if isinstance(scores, str) else None, bias,
                 groups, groups if top_groups is None else top_groups, group_mark, normalize, scale, dtype)
    if got is not None:
        return got
    rows, ld = _rows(logits, 'logits')
    kind = _TYPES.get(logits.dtype)
    if kind is None:
        raise TypeError('logits must be bf16, fp16 or fp32, got %s' % logits.dtype)
    if dtype not in (torch.int64, torch.int32):
        raise TypeError('dtype must be int64 or int32, got %s' % dtype)
    tokens, experts = rows.shape
    top_k, groups, top_groups, group_mark = _plan(experts, top_k, scores, groups, top_groups, group_mark)
    if tokens > _lib.ROUTE_MAX_TOKENS:
        raise ValueError('route: %d tokens, more than %d' % (tokens, _lib.ROUTE_MAX_TOKENS))
    scale = float(scale)
    if not abs(scale) <= 3.4e38:
        raise ValueError('scale must be a finite fp32, got %g' % scale)
    p_bias = None
    if bias is not None:
        bias = bias.resolve_neg() if isinstance(bias, torch.Tensor) else bias
        p_bias = _need(bias, torch.float32, 'bias', logits.device, experts, 1)
    r = _lib.Router(p_bias, experts, top_k, groups, top_groups, group_mark, _SCORES[scores], bool(normalize), scale)
    shares = torch.empty(logits.shape[:-1] + (top_k,), dtype=torch.float32, device=logits.device)
    index = torch.empty(logits.shape[:-1] + (top_k,), dtype=dtype, device=logits.device)
    if tokens:
        _launch(logits.device, _lib.load().sub1_route, ctypes.byref(r), rows.data_ptr(), kind, ld, tokens, shares.data_ptr(),
                index.data_ptr(), dtype.itemsize)
    return shares, index


def combine(outputs, shares, residual=None):
    """[.., W] = sum over k of shares[.., k] outputs[.., k, :], plus residual [.., W]: outputs [.., K, W] in bf16, fp16 or fp32,
    shares fp32 [.., K], residual and result in outputs' type; fp32 sums, in the order of k."""
    got = _quick('combine', _entry('sub1_combine'), outputs, shares, residual)
    if got is not None:
        return got
    if not isinstance(outputs, torch.Tensor):
        raise TypeError('outputs must be a torch.Tensor')
    if outputs.dtype not in _TYPES:
        raise TypeError('outputs must be bf16, fp16 or fp32, got %s' % outputs.dtype)
    if outputs.dim() < 2:
        raise ValueError('outputs must be [.., K, W], got %s' % (tuple(outputs.shape),))
    device, dtype = outputs.device, outputs.dtype
    top_k, width = outputs.shape[-2:]
    if not 1 <= top_k <= _lib.ROUTE_MAX_TOP_K or not 1 <= width <= _lib.MX4_MAX_WIDTH:
        raise ValueError('at most %d outputs a token of width 1..%d, got %d of %d' % (
            _lib.ROUTE_MAX_TOP_K, _lib.MX4_MAX_WIDTH, top_k, width))
    shape = outputs.shape[:-2]
    tokens = outputs.numel() // (top_k * width)
    if tokens > _lib.ROUTE_MAX_TOKENS:
        raise ValueError('combine: %d tokens, more than %d' % (tokens, _lib.ROUTE_MAX_TOKENS))
    outputs = outputs.contiguous().resolve_neg()
    p_outputs = _need(outputs, dtype, 'outputs')
    if not isinstance(shares, torch.Tensor):
        raise TypeError('shares must be a torch.Tensor')
    if shares.shape != shape + (top_k,):
        raise ValueError('shares must be %s, got %s' % (tuple(shape) + (top_k,), tuple(shares.shape)))
    shares = shares.contiguous().resolve_neg()
    p_shares = _need(shares, torch.float32, 'shares', device)
    p_residual = None
    if residual is not None:
        if not isinstance(residual, torch.Tensor):
            raise TypeError('residual must be a torch.Tensor')
        if residual.shape != shape + (width,):
            raise ValueError('residual must be %s, got %s' % (tuple(shape) + (width,), tuple(residual.shape)))
        residual = residual.contiguous().resolve_neg()
        p_residual = _need(residual, dtype, 'residual', device)
    y = torch.empty(shape + (width,), dtype=dtype, device=device)
    if tokens:
        _launch(device, _lib.load().sub1_combine, p_outputs, _TYPES[dtype], p_shares, p_residual, tokens, top_k, width,
                y.data_ptr())
    return y


class RoutedMLP(nn.Module):
    """A sparse MLP of compressed ternary experts with several experts a token: a router's logits, the choice, all pairs of
    token and expert through one expert launch, their weighted sum.  (FasterMLP is the Switch layer itself: one expert a
    token, by the wrapped module's router.)

    classifier  a module that gives logits [.., E] in bf16, fp16 or fp32 for hidden states [.., d_model]
    experts     sub1.Sub1Experts, E of them
    The other arguments as in route; `bias` becomes a buffer, which stays fp32 whatever type the module is brought to."""

    def __init__(self, classifier, experts, top_k=2, scores='softmax', bias=None, groups=1, top_groups=None, group_mark=1,
                 normalize=True, scale=1.0):
        super().__init__()
        if not isinstance(experts, sub1.Sub1Experts):
            raise TypeError('experts must be Sub1Experts')
        if not callable(classifier):
            raise TypeError('classifier must be a module')
        self.count = len(experts._wi) if experts._wi is not None else experts._prepared.experts
        self.top_k, self.groups, self.top_groups, self.group_mark = _plan(self.count, top_k, scores, groups, top_groups, group_mark)
        if bias is not None and (not isinstance(bias, torch.Tensor) or bias.dtype != torch.float32 or tuple(bias.shape) != (self.count,)):
            raise ValueError('bias must be fp32 [%d]' % self.count)
        self.scores, self.normalize, self.scale = scores, bool(normalize), float(scale)
        self.classifier, self.experts = classifier, experts
        self.register_buffer('bias', None if bias is None else bias.detach())

    def _apply(self, fn, *args, **kwargs):
        bias = self.bias
        super()._apply(fn, *args, **kwargs)
        if bias is not None and self.bias.dtype != torch.float32:
            self.bias = bias.to(self.bias.device)       # moved, with the values that it had
        return self

    def forward(self, hidden, residual=None):
        """hidden bf16 [.., d_model] -> (bf16 like it, residual added where there is one, shares [.., k], index [.., k])"""
        if not isinstance(hidden, torch.Tensor) or hidden.dtype != torch.bfloat16 or hidden.dim() < 1:
            raise TypeError('hidden must be bf16 [.., d_model]')
        if hidden.shape[-1] != self.experts._d_model:
            raise ValueError('hidden must be [.., %d], got %s' % (self.experts._d_model, tuple(hidden.shape)))
        logits = self.classifier(hidden)
        if logits.shape != hidden.shape[:-1] + (self.count,):
            raise ValueError('the classifier gives %s for %d experts' % (tuple(logits.shape), self.count))
        shares, index = route(logits, self.top_k, self.scores, self.bias, self.groups, self.top_groups, self.group_mark,
                              self.normalize, self.scale, torch.int32)
        pairs = hidden.reshape(-1, 1, hidden.shape[-1]).expand(-1, self.top_k, -1).reshape(-1, hidden.shape[-1])
        outputs = self.experts(pairs, index.reshape(-1))
        return combine(outputs.view(index.shape + hidden.shape[-1:]), shares, residual), shares, index
