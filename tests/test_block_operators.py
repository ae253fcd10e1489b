"""Operators around the experts on the CPU: what the entry points and the modules refuse, and the oracle against
itself."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

from oracle import block_oracle as bo
from qmoe_amd import _lib, mx4, mx8, norm, routing

ONE, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4097)       # never followed: checks come first
WIDE = _lib.MX4_MAX_WIDTH


def test_oracle_by_hand():
    x = np.zeros((1, 40))
    x[0, :8] = [448, -448, 449, 17, 19, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10]
    x[0, 32:35] = [1.75, 1.0625, -0.01]
    codes, scales = bo.quantize8(x)
    assert codes.shape == (1, 64) and scales.tolist() == [[128, 119]]          # 449 asks for the next scale
    got = bo.dequantize8(codes, scales, 40)
    assert got[0, :8].tolist() == [448, -448, 448, 17 - 1, 19 + 1, 0, 0, 2.0 ** -8]
    assert got[0, 32:34].tolist() == [1.75, 1.0]
    shares, index = bo.route(np.array([[0.0, 1, 1, np.nan, -np.inf]]), 5, 'sigmoid', None, 1, 1, 1, False, 1.0)
    assert index.tolist() == [[1, 2, 0, 4, 3]] and shares[0, 3] == 0
    shares, index = bo.route(np.array([[5.0, 0, 3, 3]]), 2, 'softmax', None, 2, 1, 2, True, 2.0)
    assert index.tolist() == [[0, 1]] and abs(shares.sum() - 2) < 1e-15


def test_header_constants_match_binding():
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include', 'sub1_hip.h')).read()
    for name, value in (('ROUTE_MAX_EXPERTS', _lib.ROUTE_MAX_EXPERTS), ('ROUTE_MAX_TOP_K', _lib.ROUTE_MAX_TOP_K),
                        ('ROUTE_SOFTMAX', 0), ('ROUTE_SIGMOID', 1)):
        assert int(re.search(r'#define SUB1_%s (\d+)' % name, text).group(1)) == value
    assert '#define SUB1_MX8_FORMS 13' in text and _lib.MX8_FORMS == 13
    assert '#define SUB1_NORM_MAX_ROWS (1 << 30)' in text and _lib.NORM_MAX_ROWS == 1 << 30
    assert '#define SUB1_ROUTE_MAX_TOKENS (1 << 24)' in text and _lib.ROUTE_MAX_TOKENS == 1 << 24
    assert '#define SUB1_NORM_LEAST_EPS 1e-30' in text and _lib.NORM_LEAST_EPS == 1e-30


@pytest.mark.parametrize('args,status', [
    ((None, 0, 8, 4, 8, ONE, ONE, None), -1), ((ONE, 0, 8, 4, 8, None, ONE, None), -1),
    ((ONE, 0, 8, 4, 8, ONE, None, None), -1), ((ONE, 3, 8, 4, 8, ONE, ONE, None), -2),
    ((ONE, -1, 8, 4, 8, ONE, ONE, None), -2), ((ONE, 0, 7, 4, 8, ONE, ONE, None), -2),
    ((ONE, 0, 8, 4, 0, ONE, ONE, None), -2), ((ONE, 0, 8, -1, 8, ONE, ONE, None), -2),
    ((ONE, 0, WIDE + 1, 4, WIDE + 1, ONE, ONE, None), -2), ((ODD, 0, 8, 4, 8, ONE, ONE, None), -3),
    ((ctypes.c_void_p(4098), 2, 8, 4, 8, ONE, ONE, None), -3), ((ONE, 0, 8, 4, 8, ctypes.c_void_p(4104), ONE, None), -3),
    ((None, 0, 8, 0, 8, None, None, None), 0)])
def test_quantize_and_back_refuse(args, status):
    lib = _lib.load()
    x, kind, ld, rows, width, codes, scales, stream = args
    assert lib.sub1_mx8_quantize(*args) == status
    assert lib.sub1_mx8_dequantize(codes, scales, rows, width, x, kind, ld, stream) == status
    if status:
        assert b'sub1_mx8_dequantize' in lib.sub1_last_error()


@pytest.mark.parametrize('change,status', [
    ({0: None}, -1), ({1: None}, -1), ({4: None}, -1), ({5: None}, -1), ({7: None}, -1), ({9: ONE}, -1),
    ({7: None, 9: ONE}, -1), ({7: None, 10: ONE}, -1), ({10: ONE}, -1), ({2: 0}, -2), ({3: 0}, -2), ({2: WIDE + 1}, -2), ({3: WIDE + 1}, -2),
    ({8: 47}, -2), ({11: -1}, -2), ({11: _lib.MX4_MAX_TOKENS + 1}, -2), ({0: ODD}, -3), ({4: ctypes.c_void_p(4104)}, -3), ({7: ODD}, -3),
    ({7: None, 9: ODD, 10: ONE}, -3), ({11: 0, 0: None, 4: None}, 0)])
def test_the_product_refuses(change, status):
    args = [ONE, ONE, 48, 64, ONE, ONE, 0, ONE, 48, None, None, 5, None]
    for at, value in change.items():
        args[at] = value
    assert _lib.load().sub1_mx8_product(*args) == status


def test_forms_that_are_not_there():
    for which in (-1, _lib.MX8_FORMS + 1):
        assert _lib.load().sub1_test_mx8_form(which) == -2
    assert _lib.load().sub1_test_mx8_form(0) == 0


def test_the_norm_refuses():
    lib = _lib.load()

    def call(fields=(), **change):
        f = dict(weight=4096, eps=1e-6, width=64, type=0, residual_type=0, weight_type=0)
        f.update(fields)
        a = dict(x=ONE, ldx=64, residual=ONE, ldr=64, total=ONE, ldt=64, y=ONE, ldy=64, codes=None, scales=None, rows=3)
        a.update(change)
        return lib.sub1_rms_norm(ctypes.byref(_lib.Norm(**f)), *a.values(), None)

    for fields, status in ((dict(weight=None), -1), (dict(weight=4097), -3), (dict(eps=0), -2), (dict(eps=-1.0), -2),
                           (dict(eps=float('nan')), -2), (dict(eps=float('inf')), -2), (dict(width=0), -2), (dict(width=WIDE + 1), -2), (dict(type=3), -2),
                           (dict(type=-1), -2), (dict(residual_type=1), -2), (dict(weight_type=1), -2), (dict(type=2), -2)):
        assert call(fields) == status, fields
    for change, status in ((dict(x=None), -1), (dict(residual=None), -1), (dict(total=None), -1), (dict(y=None), -1),
                           (dict(codes=ONE), -1), (dict(y=None, codes=ONE), -1), (dict(codes=ONE, scales=ONE), -1), (dict(ldx=63), -2),
                           (dict(ldr=63), -2), (dict(ldt=63), -2), (dict(ldy=63), -2), (dict(rows=-1), -2),
                           (dict(rows=_lib.NORM_MAX_ROWS + 1), -2), (dict(x=ODD), -3), (dict(residual=ODD), -3), (dict(total=ODD), -3),
                           (dict(y=ODD), -3), (dict(y=None, codes=ODD, scales=ONE), -3), (dict(rows=0, x=None), 0)):
        assert call(**change) == status, change
    assert lib.sub1_rms_norm(None, ONE, 64, None, 0, None, 0, ONE, 64, None, None, 1, None) == -1


def test_routing_refuses():
    lib = _lib.load()

    def call(fields=(), **change):
        f = dict(bias=4096, experts=64, top_k=4, groups=8, top_groups=2, group_mark=2, scores=1, normalize=1, scale=1.0)
        f.update(fields)
        a = dict(logits=ONE, type=2, ldl=64, tokens=3, shares=ONE, index=ONE, bytes=8)
        a.update(change)
        return lib.sub1_route(ctypes.byref(_lib.Router(**f)), *a.values(), None)

    for fields, status in ((dict(experts=0), -2), (dict(experts=_lib.ROUTE_MAX_EXPERTS + 8), -2), (dict(groups=0), -2),
                           (dict(groups=65, experts=130), -2), (dict(groups=7), -2), (dict(top_groups=0), -2), (dict(top_groups=9), -2),
                           (dict(group_mark=0), -2), (dict(group_mark=3), -2), (dict(top_k=0), -2), (dict(top_k=17), -2),
                           (dict(top_k=65, top_groups=8, experts=640), -2), (dict(scores=2), -2), (dict(scores=-1), -2),
                           (dict(scale=float('nan')), -2), (dict(scale=float('inf')), -2), (dict(bias=4098), -3)):
        assert call(fields, ldl=4096) == status, fields
    for change, status in ((dict(logits=None), -1), (dict(shares=None), -1), (dict(index=None), -1), (dict(type=3), -2), (dict(ldl=63), -2),
                           (dict(tokens=-1), -2), (dict(tokens=_lib.ROUTE_MAX_TOKENS + 1), -2), (dict(bytes=2), -2),
                           (dict(logits=ODD), -3), (dict(shares=ODD), -3), (dict(index=ctypes.c_void_p(4100)), -3), (dict(tokens=0, logits=None), 0)):
        assert call(**change) == status, change
    assert lib.sub1_route(None, ONE, 2, 64, 1, ONE, ONE, 8, None) == -1

    for change, status in ({0: None}, -1), ({2: None}, -1), ({7: None}, -1), ({1: 3}, -2), ({4: -1}, -2), ({4: _lib.ROUTE_MAX_TOKENS + 1}, -2), \
            ({5: 0}, -2), ({5: 65}, -2), ({6: 0}, -2), ({6: WIDE + 1}, -2), ({0: ODD}, -3), ({2: ODD}, -3), ({3: ODD}, -3), ({7: ODD}, -3), \
            ({4: 0, 0: None}, 0):
        args = [ONE, 0, ONE, ONE, 3, 2, 64, ONE, None]
        for at, value in change.items():
            args[at] = value
        assert lib.sub1_combine(*args) == status, change


def test_python_refuses_what_is_not_on_the_gpu_or_of_other_shapes():
    x, w = torch.zeros(2, 64).bfloat16(), torch.ones(64).bfloat16()
    codes8, codes4, scales = torch.zeros(2, 64, dtype=torch.uint8), torch.zeros(2, 32, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8)
    for call in (lambda: norm.rms_norm(x, w), lambda: mx8.quantize(x), lambda: mx8.dequantize(codes8, scales, 64),
                 lambda: mx8.product(codes8, scales, codes4, scales, 64), lambda: routing.route(x, 2),
                 lambda: routing.combine(torch.zeros(2, 3, 64).bfloat16(), torch.zeros(2, 3)),
                 lambda: mx8.dequantize(codes8, scales, 0), lambda: mx8.dequantize(codes8, scales, WIDE + 1), lambda: mx8.dequantize(codes8, scales, 64.5),
                 lambda: norm.rms_norm(x, w, 0.0), lambda: norm.rms_norm(x, w, float('nan')), lambda: routing.combine(x[0], x[0])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: norm.rms_norm(None, w), lambda: mx8.quantize([1.0]), lambda: routing.combine(None, None),
                 lambda: mx8.dequantize(codes8, scales, 64, torch.int8), lambda: routing.combine(codes8, scales),
                 lambda: mx8.product(None, scales, codes4, scales, 64)):
        with pytest.raises(TypeError):
            call()


def test_plans_that_do_not_go_together():
    for args in ((64, 4, 'softmin', 1, 1, 1), (0, 1, 'softmax', 1, 1, 1), (4097, 1, 'softmax', 1, 1, 1), (64, 0, 'softmax', 1, 1, 1),
                 (64, 65, 'softmax', 1, 1, 1), (64, 4, 'softmax', 7, 1, 1), (64, 4, 'softmax', 0, 1, 1), (130, 1, 'softmax', 65, 1, 1),
                 (64, 4, 'softmax', 8, 9, 1), (64, 4, 'softmax', 8, 0, 1), (64, 9, 'softmax', 8, 1, 1), (64, 4, 'softmax', 8, 2, 3),
                 (64, 4.5, 'softmax', 1, 1, 1), (200, 65, 'softmax', 1, 1, 1)):
        with pytest.raises(ValueError):
            routing._plan(*args)
    assert routing._plan(64, np.int64(4), 'sigmoid', 8.0, None, 2) == (4, 8, 8, 2)


def test_modules_refuse():
    layer = norm.RMSNorm(torch.ones(8), 1e-5)
    assert layer.eps == 1e-5 and dict(layer.named_buffers())['weight'].shape == (8,)
    for wrong, error in ((dict(weight=None), ValueError), (dict(weight=torch.ones(2, 2)), ValueError), (dict(weight=torch.ones(0)), ValueError),
                         (dict(weight=torch.ones(8).double()), TypeError), (dict(eps=0), ValueError)):
        with pytest.raises(error):
            norm.RMSNorm(**{**dict(weight=torch.ones(8)), **wrong})

    def linear(height, width):
        nb = -(-width // 32)
        return mx4.Mx4Linear(torch.zeros(height, 16 * nb, dtype=torch.uint8), torch.zeros(height, nb, dtype=torch.uint8), width)

    mlp = mx8.Mx4DenseMLP(linear(96, 64), linear(64, 96))
    with pytest.raises(ValueError):
        mx8.Mx4DenseMLP(linear(96, 64), linear(64, 64))
    with pytest.raises(TypeError):
        mx8.Mx4DenseMLP(torch.nn.Linear(64, 96), linear(64, 96))
    for wrong, error in ((torch.zeros(2, 64), TypeError), (torch.zeros(2, 65).bfloat16(), ValueError), (None, TypeError), ((1, 2, 3), TypeError),
                         (torch.zeros(2, 64).bfloat16(), ValueError)):          # (the last: not on a GPU)
        with pytest.raises(error):
            mlp(wrong)
    dense = torch.nn.Module()
    dense.wi, dense.wo, dense.act = torch.nn.Linear(64, 96, bias=False), torch.nn.Linear(96, 64, bias=False), torch.nn.GELU()
    with pytest.raises(ValueError, match='ReLU'):
        mx8.Mx4DenseMLP.from_mlp(dense)
    dense.act, dense.wi = torch.nn.ReLU(), torch.nn.Linear(64, 96)
    with pytest.raises(ValueError, match='bias'):
        mx8.Mx4DenseMLP.from_mlp(dense)
    with pytest.raises(TypeError):
        routing.RoutedMLP(torch.nn.Linear(64, 4), torch.nn.Linear(64, 64))
