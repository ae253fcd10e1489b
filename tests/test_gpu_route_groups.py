"""Groups of experts whose marks are small sums of large scores and biases: 64 bits decide which are taken."""
import pytest
import torch

from qmoe_amd import _lib, routing
from test_gpu_mx4 import gen

pytestmark = pytest.mark.gpu


def by_sorting(logits, top_k, scores, bias, groups, top_groups):
    """index [T, top_k] by marks of two, from sorts in 64 bits"""
    l = logits.double()
    c = (torch.softmax(l, -1) if scores == 'softmax' else 1 / (1 + torch.exp(-l))) + bias.double()
    marks = torch.sort(c.view(len(l), groups, -1), -1, descending=True)[0][..., :2].sum(-1)
    best = torch.sort(marks, dim=-1, descending=True, stable=True)[1][:, :top_groups]
    kept = torch.zeros_like(marks, dtype=torch.bool).scatter_(1, best, True).repeat_interleave(l.shape[1] // groups, 1)
    return torch.sort(torch.where(kept, c, -float('inf')), dim=-1, descending=True, stable=True)[1][:, :top_k]


@pytest.mark.parametrize('experts,groups,top_groups,top_k,tokens,form', [
    (16, 8, 4, 2, 60000, b'16 lanes'), (16, 8, 4, 8, 2500, b'64 lanes'), (256, 8, 3, 6, 30000, b'16 lanes'), (64, 32, 9, 4, 60000, b'64 lanes'),
    (512, 8, 4, 13, 8000, b'64 lanes')])
@pytest.mark.parametrize('size', [100.0, 1e3, 1e5])
@pytest.mark.parametrize('scores', ['softmax', 'sigmoid'])
def test_marks_of_opposite_signs(experts, groups, top_groups, top_k, tokens, form, size, scores):
    """A group's best two have biases of +size and -size, its others less: a mark is near 1 where fp32 is off by size 2^-23."""
    g = gen(experts + tokens)
    logits = torch.randn((tokens, experts), generator=g).cuda()
    for some in (False, True):              # all of the groups, every other
        bias = torch.full((groups, experts // groups), -2 * size)
        for i in range(groups):
            at = torch.randperm(experts // groups, generator=g)[:2]
            bias[i, at] = torch.tensor([0.25, -0.25]) if some and i % 2 else torch.tensor([size, -size])
        bias = bias.flatten().cuda()
        _, index = routing.route(logits, top_k, scores, bias, groups, top_groups, 2)
        assert form in _lib.load().sub1_last_kernel()
        assert torch.equal(index, by_sorting(logits, top_k, scores, bias, groups, top_groups))


@pytest.mark.parametrize('form,tokens', [(b'64 lanes', 400), (b'16 lanes', 4000)])
def test_a_large_group_not_taken_beside_small_ones(form, tokens):
    """One group's mark is off by more than that of the last one taken, and lies next to it."""
    g = gen(7)
    logits = torch.randn((tokens, 16), generator=g).cuda()
    s = torch.sigmoid(logits.double())
    for size in (1e3, 3e4):
        bias = torch.zeros(16)
        bias[4], bias[5] = size, -size
        moved = logits.clone()              # group 2's mark that of group 6 and the smallest steps to both sides
        want = (s[:, 12] + s[:, 13] - s[:, 4]).clamp(1e-3, 1 - 1e-3) + 1e-7 * torch.randn(tokens, generator=g).cuda()
        moved[:, 5] = torch.log(want / (1 - want)).float()
        _, index = routing.route(moved, 3, 'sigmoid', bias.cuda(), 8, 4, 2)
        assert form in _lib.load().sub1_last_kernel()
        assert torch.equal(index, by_sorting(moved, 3, 'sigmoid', bias.cuda(), 8, 4))
