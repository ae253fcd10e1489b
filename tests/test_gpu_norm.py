"""The norm against the oracle in 64 bits, within the bounds that it derives."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import block_oracle as bo
from qmoe_amd import _lib, mx8, norm
from test_gpu_mx4 import gen, host

pytestmark = pytest.mark.gpu

TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def part(x, strided):
    """On the GPU; strided: as a part of wider rows, NaN around it"""
    if not strided:
        return x.cuda()
    whole = torch.full((x.shape[0], x.shape[1] + 7), float('nan'), dtype=x.dtype, device='cuda')
    whole[:, 3:3 + x.shape[1]] = x.cuda()
    return whole[:, 3:3 + x.shape[1]]


def check(x, weight, eps, residual, quantize, got, name):
    def rounded(v):      # to the residual's type, from the fp32 sum
        with np.errstate(over='ignore', invalid='ignore'):
            return torch.from_numpy(v.astype(np.float32)).to(residual.dtype).double().numpy()

    r = None if residual is None else host(residual)
    y, off, s = bo.rms_norm(host(x), host(weight), eps, r, rounded)
    if residual is not None:
        got, total = got
        assert total.dtype == residual.dtype and np.array_equal(host(total), s, equal_nan=True)
    if quantize:
        bo.check_quantized(got[0].cpu().numpy(), got[1].cpu().numpy(), y, off)
        return
    assert got.dtype == x.dtype and got.shape == x.shape
    got, fine = host(got), np.isfinite(y)
    assert np.array_equal(np.isnan(got), np.isnan(y))
    bound = off + bo.HALF[name] * (np.abs(y) + off) + bo.LEAST[name] / 2
    largest = float(torch.finfo(TYPES[name]).max)
    inside = fine & (np.abs(y) + bound <= largest)
    assert (np.abs(got - y)[inside] <= bound[inside]).all()
    outside = fine & (np.abs(y) - bound > largest * (1 + bo.HALF[name]))
    assert np.isinf(got[outside]).all()


WIDTHS = [1, 7, 8, 31, 33, 64, 100, 511, 512, 520, 768, 1023, 1024, 1500, 2048, 2080, 2500, 3600, 4096, 4100, 6143, 8192, 8200, 16384, 20000, 32768,
          33000, 65536]


@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('width', WIDTHS)
def test_norm(name, width):
    """All of the types, few rows and many, in every kernel."""
    g = gen(width)
    for rows in (1, 5, 600 if width <= 8192 else 3):
        x = (torch.randn((rows, width), generator=g) * torch.exp2(3 * torch.randn((1, width), generator=g))).clamp(-6e4, 6e4).to(TYPES[name])
        w = torch.randn((width,), generator=g)
        r = 3 * torch.randn((rows, width), generator=g)
        for weight in {TYPES[name], torch.float32}:
            for residual in (None, *{TYPES[name], torch.float32}):
                for quantize in (False, True):
                    strided = (width + rows + quantize) % 2 == 1
                    a = part(x, strided), w.to(weight).cuda(), 1e-6, None if residual is None else part(r.to(residual), not strided)
                    check(*a, quantize, norm.rms_norm(*a, quantize=quantize), name)


@pytest.mark.parametrize('rows', [3, 700])
@pytest.mark.parametrize('width', [96, 2080, 40000])
def test_rows_at_the_ends(rows, width):
    """Zeros, the smallest and the largest values, one value alone, infinities and NaN, each in its row."""
    if rows > 100 and width > 10000:
        rows = 20
    for name, dtype in TYPES.items():
        info = torch.finfo(dtype)
        x = torch.ones((max(rows, 10), width))
        x[0] = 0
        x[1] = info.smallest_normal / 4
        x[2] = info.max
        x[3, 1:] = 0
        x[4, 5], x[5, 6], x[6, 7] = float('inf'), float('nan'), -float('inf')
        x[7] *= info.max
        x[7, ::2] *= -0.5
        x[8, ::3] = info.smallest_normal
        x = x.to(dtype).cuda()
        w = (0.1 + torch.rand(width, generator=gen(1))).to(dtype).cuda()
        for eps in (1e-6, 1e-30, 2.0):
            for quantize in (False, True):
                check(x, w, eps, None, quantize, norm.rms_norm(x, w, eps, quantize=quantize), name)
        r = torch.full_like(x, info.max / 2)                  # sums past the type's range
        if name != 'fp32':
            check(x, w, 1e-6, r, False, norm.rms_norm(x, w, 1e-6, r), name)
        check(x, w, 1e-6, -r, False, norm.rms_norm(x, w, 1e-6, -r), name)


def test_shapes_and_copies():
    g = gen(1)
    x, w = torch.randn((3, 4, 70), generator=g).bfloat16().cuda(), torch.randn(70, generator=g).bfloat16().cuda()
    y = norm.rms_norm(x, w)
    assert y.shape == x.shape
    assert torch.equal(norm.rms_norm(x.view(12, 70), w).view_as(y), y)
    assert torch.equal(norm.rms_norm(x.transpose(0, 1).contiguous().transpose(0, 1), w), y)
    assert torch.equal(norm.rms_norm(x, torch.stack((w, w), -1)[:, 0].contiguous()), y)
    assert torch.equal(norm.rms_norm(torch._neg_view(-x), torch._neg_view(-w)), y)
    y1, total = norm.rms_norm(x, w, 1e-6, x.transpose(0, 1).contiguous().transpose(0, 1))
    assert torch.equal(total, x + x) and total.shape == x.shape and torch.equal(y1, norm.rms_norm(x + x, w))
    (codes, scales), total = norm.rms_norm(x, w, 1e-6, x.float(), True)
    assert codes.shape == (3, 4, 96) and scales.shape == (3, 4, 3) and total.dtype == torch.float32
    assert norm.rms_norm(x[0, 0], w).shape == (70,)
    for empty in (x[:0], x[:, :0]):
        assert norm.rms_norm(empty, w).shape == empty.shape
        (codes, scales), total = norm.rms_norm(empty, w, 1e-6, empty, quantize=True)
        assert codes.shape == empty.shape[:-1] + (96,) and total.shape == empty.shape
    assert torch.equal(norm.rms_norm(x, w, 1), norm.rms_norm(x, w, 1.0))
    layer = norm.RMSNorm(w, 1e-5).cuda()
    assert torch.equal(layer(x), norm.rms_norm(x, w, 1e-5)) and torch.equal(layer(x, x)[1], x + x)

    class Given:
        weight, variance_epsilon = torch.nn.Parameter(w), 1e-5
    assert torch.equal(norm.RMSNorm.from_norm(Given, True)(x)[0], norm.rms_norm(x, w, 1e-5, quantize=True)[0])
    for wrong, error in ((dict(weight=w[:69]), ValueError), (dict(weight=w.half()), TypeError), (dict(weight=w.cpu()), ValueError),
                         (dict(residual=x[:2]), ValueError), (dict(residual=x.half()), TypeError), (dict(residual=x.cpu()), ValueError),
                         (dict(x=x.double()), TypeError), (dict(eps=1e-31), ValueError), (dict(weight=None), TypeError)):
        with pytest.raises(error):
            norm.rms_norm(**{**dict(x=x, weight=w), **wrong})


def test_in_place_and_nothing_beside():
    """y over x and the total over the residual, in rows of a wider tensor."""
    lib, g = _lib.load(), gen(2)
    for rows, width in ((5, 100), (700, 1000), (3, 40000)):
        x, r = torch.randn((rows, width), generator=g).cuda(), torch.randn((rows, width), generator=g).cuda()
        w = torch.randn(width, generator=g).cuda()
        want, total = norm.rms_norm(x, w, 1e-6, r)
        bx, br = (torch.full((rows + 2, width + 6), 7.0, device='cuda') for _ in range(2))
        bx[1:-1, 2:-4], br[1:-1, 2:-4] = x, r
        n = _lib.Norm(w.data_ptr(), 1e-6, width, 2, 2, 2)
        px, pr = bx[1:, 2:].data_ptr(), br[1:, 2:].data_ptr()
        assert lib.sub1_rms_norm(ctypes.byref(n), px, width + 6, pr, width + 6, pr, width + 6, px, width + 6, None, None, rows,
                                 torch.cuda.current_stream().cuda_stream) == 0
        assert torch.equal(bx[1:-1, 2:-4], want) and torch.equal(br[1:-1, 2:-4], total)
        bx[1:-1, 2:-4], br[1:-1, 2:-4] = 7, 7
        assert bool((bx == 7).all()) and bool((br == 7).all())


def test_more_rows_than_a_launch():
    rows, width = (1 << 21) + 5, 1100
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip('needs 30 GB')
    x = torch.ones((rows, width), dtype=torch.bfloat16, device='cuda')
    x[(1 << 21) - 1:] = torch.randn((6, width), generator=gen(1)).bfloat16().cuda()
    w = torch.randn(width, generator=gen(2)).bfloat16().cuda()
    y, total = norm.rms_norm(x, w, 1e-6, x)
    want = norm.rms_norm(x[-6:].contiguous(), w, 1e-6, x[-6:].contiguous())
    assert torch.equal(y[-6:], want[0]) and torch.equal(total[-6:], want[1])
    assert torch.equal(y[:3], y[7:10]) and torch.equal(y[0], y[1 << 20])
    del y, total
    codes, scales = norm.rms_norm(x, w, quantize=True)
    want = norm.rms_norm(x[-6:].contiguous(), w, quantize=True)
    assert torch.equal(codes[-6:], want[0]) and torch.equal(scales[-6:], want[1])
