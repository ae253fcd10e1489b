"""Routing's forms: each is taken where it is meant to be, with numbers, ties and what is no number; how exact shares are."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as bo
from qmoe_amd import _lib, routing
from test_gpu_mx4 import gen, host
from test_gpu_norm import TYPES
from test_gpu_routing import check, check_many

pytestmark = pytest.mark.gpu

FOUR, ONE, EXACT = b'route_quick_kernel, 16 lanes a token', b'route_quick_kernel, 64 lanes a token', b'route_exact_kernel'
# (tokens, experts, groups, top_groups, top_k, form): 1, 2, 4, 8, 16 and 32 experts a lane of 16, to 64 of a lane of 64, more
FORMS = [(2501, 16, 1, 1, 4, FOUR), (2503, 12, 3, 2, 3, FOUR), (2502, 32, 1, 1, 12, FOUR), (2501, 24, 4, 3, 5, FOUR), (2601, 64, 1, 1, 2, FOUR),
         (2601, 60, 5, 2, 6, FOUR), (2507, 128, 1, 1, 1, FOUR), (2507, 100, 2, 1, 8, FOUR), (2510, 256, 8, 4, 8, FOUR), (2511, 250, 1, 1, 3, FOUR),
         (4097, 512, 1, 1, 12, FOUR), (4098, 300, 3, 2, 5, FOUR), (4099, 480, 4, 2, 6, FOUR), (4103, 512, 16, 7, 10, FOUR), (4101, 300, 1, 1, 2, FOUR),
         (2500, 16, 1, 1, 4, ONE), (4096, 512, 1, 1, 12, ONE), (4096, 480, 4, 2, 6, ONE), (2600, 64, 1, 1, 13, ONE), (33, 64, 1, 1, 56, ONE),
         (41, 128, 8, 4, 8, ONE), (39, 256, 1, 1, 30, ONE), (37, 512, 4, 1, 8, ONE), (35, 1024, 1, 1, 4, ONE), (4200, 1024, 4, 2, 4, ONE), (21, 2048, 2, 1, 8, ONE),
         (19, 4096, 1, 1, 8, ONE), (19, 4096, 64, 9, 8, ONE), (17, 100, 1, 1, 57, EXACT), (15, 4095, 3, 2, 5, EXACT), (2600, 100, 1, 1, 64, EXACT)]


def last():
    return _lib.load().sub1_last_kernel()


def scores_of(logits, scores):
    """In 64 bits.  (torch.softmax over more than 1024 values has exponentials of 32 bits on the GPU: off by 1.8e-6.)"""
    l = logits.double()
    if scores == 'sigmoid':
        return 1 / (1 + torch.exp(-l))
    s = torch.exp(l - l.amax(-1, keepdim=True))
    return s / s.sum(-1, keepdim=True)


def decided(logits, scores, bias, groups, top_groups):
    """[T]: whether the definition says which groups are taken: marks that are equal but for the order of their rounding (s1 + (s2 + b)
    and (s1 + b) + s2: a few steps of 2^-52 apart) go by the last bits of the exponentials.  Groups of the same logits and biases have
    marks of the same bits."""
    if top_groups == groups:
        return torch.ones(len(logits), dtype=torch.bool, device=logits.device)
    c = (scores_of(logits, scores) + bias.double()).view(len(logits), groups, -1)
    best, at = torch.sort(c, dim=-1, descending=True, stable=True)
    marks, order = torch.sort(best[..., :2].sum(-1), dim=-1, descending=True, stable=True)
    apart = marks[:, top_groups - 1] - marks[:, top_groups] > 2.0 ** -45
    pair = []
    for values in (logits.float(), bias.expand_as(logits)):
        two = values.view(len(logits), groups, -1).gather(-1, at[..., :2])
        two = two.gather(1, order[:, top_groups - 1:top_groups + 1, None].expand(-1, 2, two.shape[-1]))
        pair.append((two[:, 0] == two[:, 1]).all(-1))
    return apart | (pair[0] & pair[1])


@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('tokens,experts,groups,top_groups,top_k,form', FORMS)
def test_forms(tokens, experts, groups, top_groups, top_k, form, scores, name):
    g = gen(tokens + experts)
    logits = (2 * torch.randn((tokens, experts), generator=g) + torch.randn((1, experts), generator=g)).cuda()
    for bias in (None, 0.1 * torch.randn(experts, generator=g).cuda()):
        for group_mark in (1, 2):
            check_many(logits.to(TYPES[name]), top_k, scores, bias, groups, top_groups, group_mark, group_mark == 1)
            assert last() == form
        # many equal ones, rows of padding, many close ones
        coarse = (logits / 2).round()
        coarse[::5] = 0.5
        coarse, steps = coarse.to(TYPES[name]), None if bias is None else (4 * bias).round() / 4
        if steps is not None:
            coarse = coarse[decided(coarse, scores, steps, groups, top_groups)]
            coarse = coarse.repeat(-(-tokens // len(coarse)), 1)[:tokens]
        check_many(coarse, top_k, scores, steps, groups, top_groups, 2, True)
        assert last() == form
        check_many((1 + 1e-6 * logits).to(TYPES[name]), top_k, scores, None if bias is None else 1e-6 * bias, groups, top_groups, 1, True)


@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('tokens,experts,groups,top_groups,top_k,form', FORMS)
def test_masks_and_what_is_no_number(tokens, experts, groups, top_groups, top_k, form, scores):
    """Rows with masks, infinities and NaN give what the oracle gives, and so do their neighbours."""
    inf, nan = float('inf'), float('nan')
    logits = torch.randn((tokens, experts), generator=gen(tokens))
    odd = [1, 2, 3, 5, 6, 8, 9, 10, 12, tokens - 2, tokens - 1]
    for at, row in zip(odd, range(len(odd))):
        logits[at] = [torch.full((experts,), -inf), torch.where(torch.arange(experts) < 2, logits[at], -inf),
                      torch.where(torch.arange(experts) == experts // 2, nan, logits[at]), torch.full((experts,), nan),
                      torch.where(torch.arange(experts) == experts // 3, inf, logits[at]), torch.where(torch.arange(experts) % 3 == 0, -inf, logits[at]),
                      torch.where(torch.arange(experts) > 2, torch.finfo(torch.float32).min, logits[at]), torch.zeros(experts),
                      torch.where(torch.arange(experts) == 0, 800.0, torch.full((experts,), -800.0)),
                      torch.where(torch.arange(experts) == experts - 1, nan, logits[at]), torch.full((experts,), -inf)][row]
    some = sorted({0, 4, 7, 11, 13, tokens - 3, *odd})
    for bias in (None, 0.1 * torch.randn(experts, generator=gen(2)).cuda()):
        for group_mark in (1, 2):
            shares, index = routing.route(logits.cuda(), top_k, scores, bias, groups, top_groups, group_mark, True)
            assert last() == form
            want, at = bo.route(host(logits[some]), top_k, scores, None if bias is None else host(bias), groups, top_groups, group_mark, True, 1.0)
            assert np.array_equal(index[some].cpu().numpy(), at)
            got = host(shares[some])
            assert np.array_equal(np.isnan(got), np.isnan(want))
            close = np.abs(got - want) <= 2.0 ** -23 * np.abs(want) + 2.0 ** -149
            assert close[~np.isnan(want)].all()


@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('tokens,experts,top_k', [(5, 4096, 64), (700, 4096, 8), (4100, 512, 8), (2600, 64, 12), (300, 64, 40), (9, 200, 60), (1, 128, 1)])
def test_how_exact_shares_are(tokens, experts, top_k, name):
    """A share is rounded once, from 64 bits.  Those of a softmax have a sum of exponentials in 32 bits under them:
    each is off, relatively, by 2^-24 |x| for x's own rounding (x = its logit less the largest), as much for that of
    x log2(e), a quarter for the constant's, and by 2^-23 for the instruction; the sum is off by their mean by weight.
    Shares over their sum have it under both sides."""
    logits = (2.5 * torch.randn((tokens, experts), generator=gen(tokens + experts))).to(TYPES[name]).cuda()
    l = logits.double()
    for scores in ('softmax', 'sigmoid'):
        for normalize in (False, True):
            for scale in (1.0, 2.5):
                shares, index = routing.route(logits, top_k, scores, None, 1, None, 1, normalize, scale)
                s = scores_of(logits, scores)
                want = s.gather(1, index)
                if normalize:
                    want = want / want.sum(-1, keepdim=True)
                off = torch.zeros((tokens, 1), dtype=torch.float64, device='cuda')
                if scores == 'softmax' and not normalize:
                    off = ((2.25 * (l.amax(-1, keepdim=True) - l) + 2) * s).sum(-1, keepdim=True) * 2.0 ** -24
                want = scale * want
                assert bool(((shares - want).abs() <= (off * 1.001 + 2.0 ** -24 * 1.001) * want).all())
    assert float(off.max()) == 0        # (the last: sigmoid scores)
