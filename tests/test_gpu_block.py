"""The operators around the experts together, as a block's sub-layers use them, on other streams and in graphs."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as bo
from oracle import mx4_oracle as mo
from qmoe_amd import mx4, mx8, norm, quant, routing, sub1
from test_gpu_mx4 import gen, host, within

pytestmark = pytest.mark.gpu


def block(d_model, d_ff, experts, seed, top_k=2):
    """(norm into 8 bits, dense MLP, norm, routed MLP of ternary experts) and the dense router's weight"""
    g = gen(seed)

    def w(height, width):
        return (torch.randn((height, width), generator=g) / width ** 0.5).cuda()

    first = norm.RMSNorm((0.5 + torch.rand(d_model, generator=g)).bfloat16().cuda(), 1e-6, quantize=True)
    second = norm.RMSNorm((0.5 + torch.rand(d_model, generator=g)).cuda(), 1e-6)
    dense = mx8.Mx4DenseMLP(mx4.Mx4Linear.make(w(d_ff, d_model)), mx4.Mx4Linear.make(w(d_model, d_ff)))
    layers = [[sub1.Sub1Linear.make(quant.ternarize(w(*shape))) for _ in range(experts)] for shape in ((d_ff, d_model), (d_model, d_ff))]
    router = torch.nn.Linear(d_model, experts, bias=False).cuda()
    with torch.no_grad():
        router.weight.copy_(w(experts, d_model) * 2)
    stack = sub1.Sub1Experts(*layers)
    routed = routing.RoutedMLP(lambda h: router(h.float()).detach(), stack, top_k, scores='sigmoid', groups=4, top_groups=2, group_mark=2,
                               bias=0.05 * torch.randn(experts, generator=g).cuda())
    return first, dense, second, routed, layers


def through(parts, hidden, residual):
    first, dense, second, routed = parts
    x, stream = first(hidden, residual)
    y, stream = second(dense(x), stream)
    return routed(y, stream)


@pytest.mark.parametrize('d_model,d_ff,tokens', [(96, 160, 1), (128, 256, 5), (200, 330, 40), (768, 1500, 13)])
def test_a_block(d_model, d_ff, tokens):
    """A dense sub-layer and a sparse one, each step against the oracle on what the step before gave."""
    experts = 8
    *parts, layers = block(d_model, d_ff, experts, d_model)
    first, dense, second, routed = parts
    g = gen(tokens)
    hidden, residual = (torch.randn((tokens, d_model), generator=g).bfloat16().cuda() for _ in range(2))

    def rounded(v):
        return torch.from_numpy(v.astype(np.float32)).bfloat16().double().numpy()

    x, stream = first(hidden, residual)
    y, off, s = bo.rms_norm(host(hidden), host(first.weight), 1e-6, host(residual), rounded)
    assert np.array_equal(host(stream), s)
    bo.check_quantized(x[0].cpu().numpy(), x[1].cpu().numpy(), y, off)

    out = dense(x)
    h = mx8.product(*x, dense.wi.codes, dense.wi.scales, d_model, True, True)
    wi, wo = (mo.dequantize(l.codes.cpu().numpy(), l.scales.cpu().numpy(), l.width) for l in (dense.wi, dense.wo))
    value = bo.dequantize8(x[0].cpu().numpy(), x[1].cpu().numpy(), d_model)
    exact, off = bo.product8_bound_finely(value, wi)
    bo.check_quantized(h[0].cpu().numpy(), h[1].cpu().numpy(), np.maximum(exact, 0), off)
    value = bo.dequantize8(h[0].cpu().numpy(), h[1].cpu().numpy(), d_ff)
    within(out, *bo.to_bf16(*bo.product8_bound_finely(value, wo)))

    y, stream2 = second(out, stream)
    want, off, s = bo.rms_norm(host(out), host(second.weight), 1e-6, host(stream), rounded)
    assert np.array_equal(host(stream2), s)
    within(y, *bo.to_bf16(want, off))

    got, shares, index = routed(y, stream2)
    logits = routed.classifier(y)
    want, at = bo.route(host(logits), 2, 'sigmoid', host(routed.bias), 4, 2, 2, True, 1.0)
    assert np.array_equal(index.cpu().numpy(), at) and np.abs(host(shares) - want).max() <= 40 * 2.0 ** -23
    each = torch.stack([torch.cat([layers[1][e](torch.relu(layers[0][e](y[t:t + 1]))) for e in at[t]]) for t in range(tokens)])
    sums, off = bo.combine(host(each), host(shares), host(stream2))
    # the experts' launch and its single layers add in the same order
    within(got, *bo.to_bf16(sums, off))
    again, _, _ = through(parts, hidden, residual)
    assert torch.equal(again, got)
    assert through(parts, hidden[:0], residual[:0])[0].shape == (0, d_model)


def test_modules_take_other_shapes():
    *parts, _ = block(64, 96, 4, 1)
    first, dense, second, routed = parts
    hidden = torch.randn((2, 3, 64), generator=gen(1)).bfloat16().cuda()
    flat = hidden.view(6, 64)
    got, want = through(parts, hidden, hidden), through(parts, flat, flat)
    assert got[0].shape == (2, 3, 64) and torch.equal(got[0].view(6, 64), want[0])
    assert got[1].shape == got[2].shape == (2, 3, 2) and torch.equal(got[2].view(6, 2), want[2])
    assert torch.equal(dense(hidden), dense(mx8.quantize(hidden)))
    assert routed(hidden)[0].shape == (2, 3, 64)
    with pytest.raises(ValueError):
        routed(hidden[..., :63])
    with pytest.raises(TypeError):
        routed(hidden.float())
    module = torch.nn.Module()
    module.wi, module.wo, module.act = torch.nn.Linear(64, 96, bias=False).cuda(), torch.nn.Linear(96, 64, bias=False).cuda(), torch.nn.ReLU()
    made = mx8.Mx4DenseMLP.from_mlp(module)
    assert torch.equal(made.wi.codes, mx4.quantize(module.wi.weight.detach())[0]) and made(hidden).shape == hidden.shape


def calls(seed, tokens):
    """Every operator's call on inputs of its own, as a function that gives all results."""
    g = gen(seed)

    def t(*shape):
        return torch.randn(shape, generator=g).cuda()

    x, r, w = t(tokens, 500).bfloat16(), t(tokens, 500), t(500)
    codes, scales = mx4.quantize(t(700, 500) / 22)
    logits, bias = t(tokens, 96), 0.1 * t(96)
    outputs, shares = t(tokens, 3, 300).half(), t(tokens, 3)

    def run():
        x8, total = norm.rms_norm(x, w, 1e-6, r, True)
        h = mx8.product(*x8, codes, scales, 500, True, True)
        return [*x8, total, norm.rms_norm(x, w), mx8.product(*x8, codes, scales, 500), *h, mx8.dequantize(*h, 700), *mx8.quantize(x),
                *routing.route(logits, 5, 'sigmoid', bias, 8, 3, 2, True), *routing.route(logits, 2), routing.combine(outputs, shares)]
    return run


@pytest.mark.parametrize('tokens', [1, 7, 90, 700])
def test_graphs(tokens):
    """Two graphs in turn, replayed between eager calls on the same inputs."""
    runs = [calls(seed, tokens) for seed in (1, 2)]
    want = [run() for run in runs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for run in runs:
            run()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for run in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run())
        graphs.append(graph)
    for _ in range(3):
        for out in outs:
            for o in out:
                o.zero_()
        for graph in graphs:
            graph.replay()
        eager = [run() for run in runs]
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want[i], outs[i], eager[i]))


def test_streams():
    """Calls of two streams at once."""
    runs = [calls(seed, 200) for seed in (3, 4)]
    want = [run() for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(runs[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for out in got[i] for a, b in zip(out, want[i]))
