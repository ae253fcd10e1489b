"""Routing against the oracle in 64 bits: indexes to the last, shares and weighted sums within derived bounds."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as bo
from qmoe_amd import _lib, routing
from test_gpu_mx4 import gen, host
from test_gpu_norm import TYPES, part

pytestmark = pytest.mark.gpu


def check(logits, top_k, scores='softmax', bias=None, groups=1, top_groups=None, group_mark=1, normalize=False, scale=1.0, dtype=torch.int64):
    shares, index = routing.route(logits, top_k, scores, bias, groups, top_groups, group_mark, normalize, scale, dtype)
    want, at = bo.route(host(logits), top_k, scores, None if bias is None else host(bias), groups, groups if top_groups is None else top_groups,
                        group_mark, normalize, scale)
    assert index.dtype == dtype and np.array_equal(index.cpu().numpy(), at)
    got = host(shares)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # an exponential, a sum over the experts, two quotients and a factor in fp32, the sum of the shares
    bound = (logits.shape[-1] + top_k + 16) * 2.0 ** -23 * np.abs(want) + 2.0 ** -126
    assert (np.abs(got - want) <= bound)[~np.isnan(want)].all()
    return shares, index


CASES = [  # experts, top_k, groups, top_groups
    (1, 1, 1, 1), (2, 2, 1, 1), (7, 3, 1, 1), (64, 1, 1, 1), (64, 64, 1, 1), (65, 8, 1, 1), (128, 1, 1, 1), (128, 2, 1, 1), (160, 6, 8, 3),
    (256, 8, 8, 4), (256, 8, 1, 1), (300, 5, 3, 2), (2048, 1, 1, 1), (2048, 2, 1, 1), (4096, 64, 1, 1), (4096, 8, 64, 5), (64, 7, 64, 9),
    (130, 4, 2, 1), (33, 3, 33, 20), (4095, 3, 63, 62), (512, 10, 16, 16), (1000, 4, 4, 1), (24, 2, 12, 1), (1500, 6, 1, 1), (1366 * 3, 7, 3, 2)]
CASES = [c for c in CASES if c[0] <= _lib.ROUTE_MAX_EXPERTS]


@pytest.mark.parametrize('experts,top_k,groups,top_groups', CASES)
@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('biased', [False, True])
def test_route(experts, top_k, groups, top_groups, scores, biased):
    g = gen(experts + top_k)
    bias = 0.1 * torch.randn(experts, generator=g).cuda() if biased else None
    for i, (name, tokens) in enumerate((('fp32', 1), ('bf16', 37), ('fp16', 5), ('fp32', 130))):
        logits = part((2 * torch.randn((tokens, experts), generator=g) + torch.randn((1, experts), generator=g)).to(TYPES[name]), i % 2 == 1)
        for group_mark in (1, 2):
            check(logits, top_k, scores, bias, groups, top_groups, group_mark, i % 2 == 0, (1.0, 2.5, -0.5, 1.0)[i], (torch.int64, torch.int32)[i % 2])


@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('experts,groups,top_groups', [(60, 1, 1), (60, 6, 2), (300, 1, 1), (300, 12, 5), (2100, 1, 1), (2100, 7, 3)])
def test_ties_masks_and_what_is_no_number(scores, experts, groups, top_groups):
    inf, nan = float('inf'), float('nan')
    logits = torch.randn((20, experts), generator=gen(experts))
    logits[0] = 0.5                                           # all equal
    logits[1] = logits[1].round()                             # many equal
    logits[2] = -inf                                          # nothing left
    logits[3, 2:] = -inf                                      # two left
    logits[4, experts - 3] = nan
    logits[5] = nan
    logits[6, 5] = inf
    logits[7, 3:] = torch.finfo(torch.float32).min            # masked by the lowest value
    logits[8] = torch.finfo(torch.float32).min
    logits[9] = 1e4 * logits[9]
    logits[10] = 0.0
    logits[10, ::2] = -0.0                                    # equal too
    logits[11, :] = 1e-3
    logits[11, 7] = 1e-3 * (1 + 2 ** -23)                     # a step of fp32 above
    logits[12, ::3] = -inf
    logits[13] = -800.0
    logits[14, 0], logits[14, 1:] = 800.0, -800.0
    for bias in (None, torch.zeros(experts).cuda(), torch.randn(experts, generator=gen(1)).cuda()):
        for group_mark in (1, 2):
            for normalize in (False, True):
                check(logits.cuda(), 4, scores, bias, groups, top_groups, group_mark, normalize)
                check(logits.bfloat16().cuda(), 8, scores, bias, groups, top_groups, group_mark, normalize)
    bias = torch.randn(experts, generator=gen(2))
    bias[3], bias[4], bias[5] = nan, inf, -inf
    check(logits.cuda(), 5, scores, bias.cuda(), groups, top_groups, 1, True)


@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
def test_scores_closer_than_fp32_can_tell(scores):
    """Biases that bring two experts' marks together to within their own rounding: 64 bits decide."""
    g = gen(11)
    logits = torch.randn((64, 96), generator=g)
    l = logits.double()
    s = torch.softmax(l, -1) if scores == 'softmax' else torch.sigmoid(l)
    for t in range(64):
        # this token's best two differ by a rounding of fp32
        bias = torch.full((96,), -2.0)
        a, b = torch.randperm(96, generator=g)[:2].tolist()
        bias[a] = 0.0
        bias[b] = (s[t, a] - s[t, b]).float()
        check(logits[t:t + 1].cuda(), 2, scores, bias.cuda())
        grouped = bias.clone()
        check(logits[t:t + 1].cuda(), 2, scores, grouped.cuda(), 8, 2, 2)


def check_many(logits, top_k, scores, bias, groups, top_groups, group_mark, normalize):
    """Many tokens at once, numbers alone: the same by sorts over all of them."""
    shares, index = routing.route(logits, top_k, scores, bias, groups, top_groups, group_mark, normalize)
    l = logits.double()
    s = torch.softmax(l, -1) if scores == 'softmax' else 1 / (1 + torch.exp(-l))
    c = s if bias is None else s + bias.double()
    key = l if bias is None else c
    if top_groups < groups:
        of = torch.sort((key if group_mark == 1 else c).view(len(l), groups, -1), -1, descending=True)[0][..., :group_mark].sum(-1)
        best = torch.sort(of, dim=-1, descending=True, stable=True)[1][:, :top_groups]
        kept = torch.zeros_like(of, dtype=torch.bool).scatter_(1, best, True).repeat_interleave(key.shape[1] // groups, 1)
        key = torch.where(kept, key, -float('inf'))
    at = torch.sort(key, dim=-1, descending=True, stable=True)[1][:, :top_k]
    assert torch.equal(index, at)
    want = s.gather(1, at)
    if normalize:
        want = want / want.sum(-1, keepdim=True)
    assert bool(((shares - want).abs() <= (logits.shape[-1] + top_k + 16) * 2.0 ** -23 * want + 2.0 ** -126).all())


@pytest.mark.parametrize('experts,top_k,groups,top_groups', CASES)
@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('biased', [False, True])
def test_route_many_tokens(experts, top_k, groups, top_groups, scores, biased):
    g = gen(experts + top_k + 1)
    bias = 0.1 * torch.randn(experts, generator=g).cuda() if biased else None
    for i, (name, tokens) in enumerate((('fp32', 3001), ('bf16', 2601), ('fp16', 1536))):
        logits = part((2 * torch.randn((tokens, experts), generator=g) + torch.randn((1, experts), generator=g)).to(TYPES[name]), i % 2 == 1)
        for group_mark in (1, 2):
            check_many(logits, top_k, scores, bias, groups, top_groups, group_mark, i % 2 == 0)
        # many equal ones, and many close ones
        check_many((logits.float() / 2).round().to(TYPES[name]), top_k, scores, bias, groups, top_groups, 2, True)
        check_many((1 + 1e-6 * logits.float()).to(TYPES[name]), top_k, scores, None if bias is None else 1e-6 * bias, groups, top_groups, 1, True)


@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('experts,groups,top_groups', [(60, 1, 1), (60, 6, 2), (256, 8, 4), (200, 1, 1), (480, 4, 2)])
def test_what_is_no_number_among_many_tokens(scores, experts, groups, top_groups):
    """Rows with masks and NaN give in a large call what they give in a small one, and their neighbours too."""
    inf, nan = float('inf'), float('nan')
    g = gen(experts)
    logits = torch.randn((2800, experts), generator=g)
    logits[3] = -inf
    logits[100, 2:] = -inf
    logits[101, 5] = nan
    logits[500] = nan
    logits[501, 7] = inf
    logits[900:904, ::3] = -inf
    logits[1200, 3:] = torch.finfo(torch.float32).min
    logits[1300] = 0.25
    logits[2799, -1] = nan
    rows = [0, 2, 3, 4, 99, 100, 101, 102, 500, 501, 502, 903, 1199, 1200, 1201, 1300, 1301, 2798, 2799]
    for bias in (None, 0.1 * torch.randn(experts, generator=g).cuda()):
        for group_mark in (1, 2):
            many = routing.route(logits.cuda(), 6, scores, bias, groups, top_groups, group_mark, True)
            few = check(logits[rows].cuda(), 6, scores, bias, groups, top_groups, group_mark, True)
            assert torch.equal(many[1][rows], few[1])
            assert torch.allclose(many[0][rows], few[0], rtol=1e-5, atol=1e-37, equal_nan=True)


@pytest.mark.parametrize('experts,top_k', [(12, 12), (12, 10), (24, 11), (9, 9)])
def test_equal_ones_beside_rows_with_fewer_numbers(experts, top_k):
    """Rows that share a wavefront: one has its last two equal where another has none left but what is no number."""
    logits = torch.randn((2601, experts), generator=gen(experts))
    logits[:, -2:] = -9.0
    for i in range(2):
        logits[i::4, :2].view(torch.int32)[:] = -1             # NaN with every bit set
    for dtype in (torch.float32, torch.bfloat16):
        l = logits.to(dtype)
        assert bool(l.isnan().any())
        _, index = routing.route(l.cuda(), top_k, 'sigmoid')
        _, want = bo.route(host(l), top_k, 'sigmoid', None, 1, 1, 1, False, 1.0)
        assert np.array_equal(index.cpu().numpy(), want)


@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
@pytest.mark.parametrize('experts,top_k,groups,top_groups', [(40, 3, 1, 1), (128, 1, 1, 1), (256, 8, 8, 4), (512, 12, 1, 1), (500, 7, 4, 2), (2048, 2, 1, 1), (4096, 20, 1, 1)])
@pytest.mark.parametrize('tokens', [70, 2604])
def test_many_equal_ones(tokens, experts, top_k, groups, top_groups, scores):
    """Rows of padding (all equal), coarse logits, such that differ in their last bits alone: equal ones by the lower index,
    others as they are, with no bias, one of zeros and one of few values."""
    g = gen(experts + tokens)
    logits = torch.randn((tokens, experts), generator=g)
    logits[::2] = 0
    logits[1::8] = (2 * logits[1::8]).round() / 2
    logits[3::8] = 1 + torch.randint(0, 3, logits[3::8].shape, generator=g) * 2.0 ** -23
    logits[5::16, experts // 3:] = -2.5
    logits = logits.cuda()
    for bias in (None, torch.zeros(experts).cuda(), torch.randint(0, 2, (experts,), generator=g).float().cuda() / 4):
        for group_mark in (1, 2):
            check_many(logits, top_k, scores, bias, groups, top_groups, group_mark, True)
    some = logits[:40].clone()
    some[7:, ::3] = -float('inf')                             # masked in part, and whole
    some[20:30] = -float('inf')
    some[31, 1:] = -float('inf')
    for bias in (None, torch.zeros(experts).cuda()):
        want = check(some, top_k, scores, bias, groups, top_groups, 2, True)
        got = routing.route(some.repeat(-(-tokens // 40), 1), top_k, scores, bias, groups, top_groups, 2, True)
        assert torch.equal(got[1], want[1].repeat(-(-tokens // 40), 1))
        assert torch.allclose(got[0], want[0].repeat(-(-tokens // 40), 1), rtol=1e-5, atol=0)


def test_shapes_of_routing():
    logits = torch.randn((3, 5, 40), generator=gen(3)).cuda()
    shares, index = routing.route(logits, 2)
    assert shares.shape == index.shape == (3, 5, 2)
    for other in (logits.transpose(0, 1).contiguous().transpose(0, 1), torch._neg_view(-logits), torch.stack((logits, logits), -1)[..., 0]):
        got = routing.route(other, 2)
        assert torch.equal(got[0], shares) and torch.equal(got[1], index)
    assert routing.route(logits[0, 0], 2)[1].shape == (2,)
    got = routing.route(logits[:0], 2, dtype=torch.int32)
    assert got[0].shape == (0, 5, 2) and got[1].dtype == torch.int32
    assert torch.equal(routing.route(logits, 2.0, normalize=1, scale=2)[0], routing.route(logits, 2, normalize=True, scale=2.0)[0])
    assert torch.equal(routing.route(logits[0, 0].expand(4, 40), 2)[1], index[0, 0].expand(4, 2))
    bias = torch.zeros(40, device='cuda')
    for wrong, error in ((dict(logits=logits.double()), TypeError), (dict(logits=logits[..., :0]), ValueError), (dict(top_k=0), ValueError),
                         (dict(top_k=41), ValueError), (dict(scores='tanh'), ValueError), (dict(scores=None), ValueError), (dict(groups=3), ValueError),
                         (dict(bias=bias[:39]), ValueError), (dict(bias=bias.double()), TypeError), (dict(bias=bias.cpu()), ValueError),
                         (dict(dtype=torch.int16), TypeError), (dict(scale=float('inf')), ValueError), (dict(top_k=1.5), ValueError),
                         (dict(bias=0.5), TypeError), (dict(scale=1e39), ValueError)):
        with pytest.raises(error):
            routing.route(**{**dict(logits=logits, top_k=2), **wrong})


def test_tokens_past_32_bits():
    tokens, experts = (1 << 21) + 3, 2048
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip('needs 30 GB')
    logits = torch.zeros((tokens, experts), dtype=torch.bfloat16, device='cuda')
    logits[-3:] = torch.randn((3, experts), generator=gen(1)).bfloat16().cuda()
    shares, index = routing.route(logits, 3)
    want, at = bo.route(host(logits[-4:]), 3, 'softmax', None, 1, 1, 1, False, 1.0)
    assert np.array_equal(index[-4:].cpu().numpy(), at) and np.allclose(host(shares[-4:]), want, rtol=1e-3)
    assert bool((index[:-3] == torch.arange(3, device='cuda')).all())


# -------------------------------------------------------------- the weighted sum ---

@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('tokens,top_k,width', [(1, 1, 1), (3, 2, 7), (13, 2, 1024), (5, 8, 1023), (700, 3, 100), (2, 64, 33), (1, 4, 65536), (300, 4, 2080),
                                                (9000, 2, 40)])
@pytest.mark.parametrize('residual', [False, True])
def test_combine(name, tokens, top_k, width, residual):
    g = gen(tokens + width)
    outputs = torch.randn((tokens, top_k, width), generator=g).to(TYPES[name]).cuda()
    shares = torch.randn((tokens, top_k), generator=g).cuda()
    r = (4 * torch.randn((tokens, width), generator=g)).to(TYPES[name]).cuda() if residual else None
    y, off = bo.combine(host(outputs), host(shares), None if r is None else host(r))
    got = routing.combine(outputs, shares, r)
    assert got.dtype == outputs.dtype and got.shape == (tokens, width)
    assert (np.abs(host(got) - y) <= off + bo.HALF[name] * (np.abs(y) + off) + bo.LEAST[name] / 2).all()


def test_what_combine_is_given():
    g = gen(4)
    outputs, shares = torch.randn((2, 3, 4, 50), generator=g).bfloat16().cuda(), torch.rand((2, 3, 4), generator=g).cuda()
    r = torch.randn((2, 3, 50), generator=g).bfloat16().cuda()
    y = routing.combine(outputs, shares, r)
    assert y.shape == (2, 3, 50)
    assert torch.equal(routing.combine(outputs.transpose(0, 1).contiguous().transpose(0, 1), shares.transpose(0, 1).contiguous().transpose(0, 1),
                                       r.transpose(0, 1).contiguous().transpose(0, 1)), y)
    assert torch.equal(routing.combine(torch._neg_view(-outputs), shares, torch._neg_view(-r)), y)
    assert routing.combine(outputs[0, 0], shares[0, 0]).shape == (50,)
    assert routing.combine(outputs[:0], shares[:0], r[:0]).shape == (0, 3, 50)
    bad = outputs.clone()
    bad[0, 0, 1, 3], bad[1, 2, 0, 4] = float('nan'), float('inf')
    got = routing.combine(bad, shares, r)
    assert bool(got[0, 0, 3].isnan()) and bool(got[1, 2, 4].isinf())
    got[0, 0, 3], got[1, 2, 4] = y[0, 0, 3], y[1, 2, 4]
    assert torch.equal(got, y)
    for wrong, error in ((dict(shares=shares[..., :3]), ValueError), (dict(shares=shares.double()), TypeError), (dict(shares=shares.cpu()), ValueError),
                         (dict(residual=r[..., :49]), ValueError), (dict(residual=r.float()), TypeError), (dict(outputs=outputs.double()), TypeError),
                         (dict(outputs=outputs[..., :0]), ValueError), (dict(outputs=outputs[:, :, :0], shares=shares[..., :0]), ValueError),
                         (dict(shares=None), TypeError), (dict(residual=1.0), TypeError)):
        with pytest.raises(error):
            routing.combine(**{**dict(outputs=outputs, shares=shares, residual=r), **wrong})


def test_combine_past_32_bits():
    tokens, top_k, width = 70000, 2, 32768
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip('needs 40 GB')
    outputs = torch.ones((tokens, top_k, width), dtype=torch.bfloat16, device='cuda')
    outputs[-1, 1] = 3
    shares = torch.full((tokens, top_k), 0.5, device='cuda')
    y = routing.combine(outputs, shares)
    assert bool((y[:-1] == 1).all()) and bool((y[-1] == 2).all())
