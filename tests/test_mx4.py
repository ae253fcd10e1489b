"""Microscaled 4-bit operators on the CPU: what the entry points and the modules refuse, and the oracle
against itself."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import mx4_oracle as mo
from qmoe_amd import _lib, mx4

ONE, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4097)       # never followed: checks come first
WIDE = _lib.MX4_MAX_WIDTH


def test_oracle_by_hand():
    x = np.zeros((1, 40))
    x[0, :10] = [6, -6, 0.25, 0.75, -1.25, 1.75, 2.5, 3.5, 5, 0.2500001]
    x[0, 32:36] = [7.9, 8.1, -0.6, 1e-30]                     # the scale goes up at 8
    codes, scales = mo.quantize(x)
    assert codes.shape == (1, 32) and scales.tolist() == [[127, 128]]
    got = mo.dequantize(codes, scales, 40)
    assert got[0, :10].tolist() == [6, -6, 0, 1, -1, 2, 2, 4, 4, 0.5]
    assert got[0, 32:36].tolist() == [8, 8, -1, 0]
    assert mo.route(np.array([[1.0, 3, np.nan, 3, -np.inf]]), 5).tolist() == [[1, 3, 0, 4, 2]]


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
    assert lib.sub1_mx4_quantize(*args) == status
    assert lib.sub1_mx4_dequantize(codes, scales, rows, width, x, kind, ld, stream) == status
    if status:
        assert b'sub1_mx4_dequantize' in lib.sub1_last_error()


@pytest.mark.parametrize('change,status', [
    ({0: None}, -1), ({1: None}, -1), ({4: None}, -1), ({6: None}, -1), ({2: 0}, -2), ({3: 0}, -2), ({2: WIDE + 1}, -2),
    ({3: WIDE + 1}, -2), ({5: 63}, -2), ({7: 47}, -2), ({8: -1}, -2), ({8: _lib.MX4_MAX_TOKENS + 1}, -2), ({0: ODD}, -3),
    ({4: ODD}, -3), ({6: ODD}, -3), ({8: 0, 0: None, 4: None}, 0)])
def test_products_refuse(change, status):
    lib = _lib.load()
    args = [ONE, ONE, 48, 64, ONE, 64, ONE, 48, 5, None]
    for at, value in change.items():
        args[at] = value
    assert lib.sub1_mx4_product(*args) == status
    if 5 in change:
        return
    other = args[:5] + [ONE] + args[6:]
    assert lib.sub1_mx4_product_quantized(*other) == status


def test_the_layer_refuses():
    lib = _lib.load()

    def call(layer=(), args=()):
        fields = dict(router=4096, wi_codes=4096, wi_scales=4096, wo_codes=4096, wo_scales=4096, experts=4, d_model=64,
                      d_ff=96, top_k=1, router_type=2, normalize=0, capacity=0)
        fields.update(layer)
        l = _lib.Mx4Layer(**fields)
        a = dict(x=ONE, tokens=6, length=3, y=ONE, logits=ONE, index=ONE, scratch=ONE, scratch_bytes=1 << 30)
        a.update(args)
        return lib.sub1_mx4_layer_forward(ctypes.byref(l), *a.values(), None)

    for layer, status in (
            (dict(experts=0), -2), (dict(experts=_lib.MX4_LAYER_EXPERTS + 1), -2), (dict(d_model=0), -2), (dict(d_ff=0), -2),
            (dict(d_model=WIDE + 1), -2), (dict(d_ff=WIDE + 1), -2), (dict(top_k=0), -2), (dict(top_k=5), -2),
            (dict(experts=100, top_k=9), -2), (dict(router_type=1), -2), (dict(capacity=-1), -2),
            (dict(capacity=1, top_k=2), -2), (dict(router=None), -1), (dict(wi_codes=None), -1), (dict(wi_scales=None), -1),
            (dict(wo_codes=None), -1), (dict(wo_scales=None), -1), (dict(router=4098), -3), (dict(wi_codes=4104), -3),
            (dict(wo_codes=4104), -3)):
        assert call(layer) == status, layer
    for args, status in ((dict(tokens=-1), -2), (dict(tokens=_lib.MX4_LAYER_TOKENS + 1, length=1), -2), (dict(length=4), -2),
                         (dict(length=0), -2), (dict(x=None), -1), (dict(y=None), -1), (dict(logits=None), -1),
                         (dict(index=None), -1), (dict(scratch=None), -1), (dict(scratch_bytes=100), -2), (dict(x=ODD), -3),
                         (dict(index=ctypes.c_void_p(4100)), -3), (dict(scratch=ctypes.c_void_p(4096 + 16)), -3)):
        assert call(args=args) == status, args
    assert call(args=dict(tokens=0, x=None)) == 0
    assert lib.sub1_mx4_layer_forward(None, ONE, 1, 1, ONE, ONE, ONE, ONE, 1 << 30, None) == -1
    assert lib.sub1_mx4_layer_scratch_bytes(None, 1) == 0


def test_header_constants_match_binding():
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'include', 'sub1_hip.h')).read()
    for name, value in (('LAYER_TOKENS', _lib.MX4_LAYER_TOKENS), ('LAYER_TOP_K', _lib.MX4_LAYER_TOP_K), ('MAX_WIDTH', WIDE),
                        ('LAYER_EXPERTS', _lib.MX4_LAYER_EXPERTS), ('BF16', 0), ('FP16', 1), ('FP32', 2)):
        assert int(re.search(r'#define SUB1_MX4_%s (\d+)' % name, text).group(1)) == value


def test_modules_refuse_what_is_not_a_matrix_in_the_format():
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    assert dict(mx4.Mx4Linear(codes, scales, 33).named_buffers())['weight'].numel() == 0
    for c, s, width, error in ((codes, scales, 32, ValueError), (codes, scales, 65, ValueError), (codes[0], scales[0], 64, ValueError),
                               (codes, scales[:7], 64, ValueError), (codes.int(), scales, 64, TypeError)):
        with pytest.raises(error):
            mx4.Mx4Linear(c, s, width)
    for call in (lambda: mx4.quantize(torch.zeros(2, 32)), lambda: mx4.Mx4Linear.make(torch.zeros(2, 32)),
                 lambda: mx4.dequantize(codes, scales, 64), lambda: mx4.product(torch.zeros(2, 64).bfloat16(), codes, scales),
                 lambda: mx4.product_quantized(codes, scales, codes, scales, 64),
                 lambda: mx4.Mx4Linear(codes, scales, 64)(torch.zeros(2, 64).bfloat16()),
                 lambda: mx4.Mx4Linear(codes, scales, 64)(torch.zeros(2, 65).bfloat16())):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        mx4.quantize(None)
    with pytest.raises(TypeError):
        mx4.dequantize(codes, scales, 64, torch.int32)


@pytest.mark.parametrize('quantized', [False, True])
def test_a_layer_refuses_another_width_before_it_looks_further(quantized):
    layer = mx4.Mx4Linear(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8), 60, quantized)
    for wrong in (torch.zeros(2, 64).bfloat16(), torch.zeros(2, 33), torch.tensor(1.0)):
        with pytest.raises(ValueError, match='x must be \\[.., 60\\]'):
            layer(wrong)
    for wrong in (None, [0.0] * 60):
        with pytest.raises(TypeError):
            layer(wrong)
    with pytest.raises(ValueError, match='GPU'):
        layer(torch.zeros(2, 60).bfloat16())


def test_the_sparse_mlp_refuses():
    def stack(experts, height, width):
        nb = mo.blocks_of(width)
        return (torch.zeros(experts, height, 16 * nb, dtype=torch.uint8), torch.zeros(experts, height, nb, dtype=torch.uint8))

    router, wi, wo = torch.zeros(4, 64), stack(4, 96, 64), stack(4, 64, 96)
    layer = mx4.Mx4SparseMLP(router, wi, wo, capacity=3)
    for args, options in (((router[0], wi, wo), {}), ((router.half(), wi, wo), {}), ((router[:3], wi, wo), {}),
                          ((router, wo, wi), {}), ((router, wi, stack(4, 64, 97 + 32)), {}), ((router, wi, wo), dict(top_k=0)),
                          ((router, wi, wo), dict(top_k=5)), ((router, wi, wo), dict(top_k=2, capacity=1)),
                          ((router, wi, wo), dict(capacity=0)), ((router, (wi[0][0], wi[1][0]), wo), {})):
        with pytest.raises(ValueError):
            mx4.Mx4SparseMLP(*args, **options)
    with pytest.raises(TypeError):
        mx4.Mx4SparseMLP(router, (wi[0].int(), wi[1]), wo)
    with pytest.raises(TypeError):
        layer([1, 2])
    for hidden in (torch.zeros(64).bfloat16(), torch.zeros(2, 65).bfloat16(), torch.zeros(2, 64).bfloat16()):
        with pytest.raises(ValueError):
            layer(hidden)
    # parts of whole sequences, as long as they fit
    assert layer._parts(600, 100) == [(0, 200), (200, 200), (400, 200)]
    assert layer._parts(256, 256) == [(0, 256)] and layer._parts(0, 5) == []
    with pytest.raises(ValueError):
        layer._parts(514, 257)
    assert mx4.Mx4SparseMLP(router, wi, wo)._parts(600, 300) == [(0, 256), (256, 256), (512, 88)]


def test_numbers_that_are_not_whole_are_refused():
    codes, scales = torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    for width in (60, 60.0, np.int64(60), np.float32(60)):
        assert type(mx4.Mx4Linear(codes, scales, width).width) is int
    experts = torch.zeros(4, 64, 32, dtype=torch.uint8), torch.zeros(4, 64, 2, dtype=torch.uint8)
    layer = mx4.Mx4SparseMLP(torch.zeros(4, 64), experts, experts, np.int32(1), capacity=np.int64(3))
    assert type(layer.top_k) is int and type(layer.capacity) is int
    with pytest.raises(ValueError, match='width'):
        mx4.Mx4Linear(codes, scales, 60.5)
    for wrong in (dict(top_k=1.5), dict(capacity=2.5)):
        with pytest.raises(ValueError, match=list(wrong)[0]):
            mx4.Mx4SparseMLP(torch.zeros(4, 64), experts, experts, **wrong)


def test_a_module_with_other_experts_is_refused():
    import types

    def mlp(**change):
        parts = dict(act=torch.nn.ReLU(), bias=False)
        parts.update(change)
        expert = torch.nn.Module()
        expert.wi = torch.nn.Linear(64, 96, bias=parts['bias'])
        expert.wo = torch.nn.Linear(96, 64, bias=False)
        expert.act = parts['act']
        router = types.SimpleNamespace(classifier=torch.nn.Linear(64, 1, bias=False))
        return types.SimpleNamespace(router=router, experts={'expert_0': expert})

    for change in (dict(act=torch.nn.GELU()), dict(bias=True), {}):       # the last: its matrices are not on a GPU
        with pytest.raises(ValueError):
            mx4.Mx4SparseMLP.from_mlp(mlp(**change))
