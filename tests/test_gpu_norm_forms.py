"""The norm's forms for many rows: each is taken where it is meant to be, and gives what the form for few rows gives."""
import ctypes

import pytest
import torch

from qmoe_amd import _lib, norm
from test_gpu_mx4 import gen
from test_gpu_norm import TYPES, check, part

pytestmark = pytest.mark.gpu

QUARTERS, WAVES, GROUPS, WIDE = (b'rms_norm_kernel, 16 lanes a row', b'rms_norm_kernel, a wavefront a row',
                                 b'rms_norm_kernel, a workgroup a row', b'rms_norm_wide_kernel, a workgroup a row')
# (width, rows, form for values of 16 bits, for such of 32): one to four eights a lane, two to eight, in the last workgroup one row
# more than a wavefront takes, or a wavefront's last row missing
FORMS = [(7, 2049, QUARTERS, QUARTERS), (128, 4098, QUARTERS, QUARTERS), (200, 2051, QUARTERS, QUARTERS), (384, 2055, QUARTERS, QUARTERS),
         (385, 5003, QUARTERS, QUARTERS), (511, 2050, QUARTERS, QUARTERS), (513, 4097, WAVES, WAVES), (1023, 4098, WAVES, WAVES),
         (1500, 4099, WAVES, WAVES), (2047, 4101, WAVES, WAVES), (2080, 4099, WAVES, GROUPS), (2600, 4097, WAVES, GROUPS), (3500, 4098, WAVES, GROUPS),
         (4096, 4103, WAVES, GROUPS), (4100, 4099, GROUPS, GROUPS), (16385, 40, GROUPS, GROUPS), (33000, 20, WIDE, WIDE), (2080, 4096, GROUPS, GROUPS),
         (512, 2048, GROUPS, GROUPS)]


def rows_of(name, rows, width, g):
    """Ordinary rows of growing size and, among them, zeros, the largest and smallest values, infinities and NaN"""
    info = torch.finfo(TYPES[name])
    x = torch.randn((rows, width), generator=g) * torch.exp2(torch.randn((rows, 1), generator=g))
    x[-3] = 0
    x[-6] = info.smallest_normal / 4
    x[-11] = info.max
    x[rows // 2, width // 2], x[rows // 2 + 2, width - 1], x[rows // 2 + 5, 0] = float('inf'), float('nan'), -float('inf')
    return x.to(TYPES[name])


def residuals(name):
    return [None, TYPES[name]] + [torch.float32] * (name != 'fp32')


def flat(got):
    return [t for one in (got if isinstance(got, tuple) else (got,)) for t in (one if isinstance(one, tuple) else (one,))]


@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('width,rows,narrow,wide', FORMS)
def test_forms(width, rows, narrow, wide, name):
    g = gen(width + rows)
    x, r, w = rows_of(name, rows, width, g), 3 * torch.randn((rows, width), generator=g), torch.randn((width,), generator=g)
    some = [0, 1, 2, 3, 4, 5, rows // 2 - 1, rows // 2, rows // 2 + 1, rows // 2 + 2, rows // 2 + 5] + list(range(rows - 13, rows))
    for k, residual in enumerate(residuals(name)):
        for quantize in (False, True):
            weight = w.to(torch.float32 if (width + k + quantize) % 2 else TYPES[name]).cuda()
            a = part(x, (rows + quantize) % 2 == 0), weight, 1e-6, None if residual is None else part(r.to(residual), (rows + quantize) % 2 == 1)
            got = norm.rms_norm(*a, quantize=quantize)
            assert _lib.load().sub1_last_kernel() == (wide if name == 'fp32' or residual == torch.float32 else narrow)
            pieces = []
            for at in range(0, rows, 1500):
                few = norm.rms_norm(a[0][at:at + 1500], weight, 1e-6, None if residual is None else a[3][at:at + 1500], quantize)
                assert _lib.load().sub1_last_kernel() in (GROUPS, WIDE)
                pieces.append(flat(few))
            for all_rows, of_few in zip(flat(got), zip(*pieces)):
                assert torch.equal(all_rows.contiguous().view(torch.uint8), torch.cat(of_few).contiguous().view(torch.uint8))
            picked = [t[some] for t in flat(got)]       # and against 64 bits
            y = tuple(picked[:2]) if quantize else picked[0]
            check(a[0][some], weight, 1e-6, None if residual is None else a[3][some], quantize,
                  y if residual is None else (y, picked[-1]), name)


@pytest.mark.parametrize('name', TYPES)
@pytest.mark.parametrize('width,rows', [(100, 2049), (250, 2050), (300, 2051), (500, 4099), (1000, 4097), (2041, 4098), (4100, 4099), (40001, 3)])
def test_in_place(width, rows, name):
    """y over x and the total over the residual, in rows of a wider tensor, nothing beside them."""
    lib, g, kind = _lib.load(), gen(width), {'bf16': 0, 'fp16': 1, 'fp32': 2}[name]
    x = torch.randn((rows, width), generator=g).to(TYPES[name]).cuda()
    w = torch.randn(width, generator=g).to(TYPES[name]).cuda()
    for rtype in residuals(name):
        r = None if rtype is None else torch.randn((rows, width), generator=g).to(rtype).cuda()
        want = flat(norm.rms_norm(x, w, 1e-6, r))
        bx = torch.full((rows + 2, width + 5), 7.0, dtype=x.dtype, device='cuda')
        bx[1:-1, 2:-3] = x
        px, br, pr, ld = bx[1:, 2:].data_ptr(), None, None, 0
        if r is not None:
            br = torch.full((rows + 2, width + 5), 7.0, dtype=rtype, device='cuda')
            br[1:-1, 2:-3] = r
            pr, ld = br[1:, 2:].data_ptr(), width + 5
        n = _lib.Norm(w.data_ptr(), 1e-6, width, kind, 2 if rtype == torch.float32 else kind, kind)
        assert lib.sub1_rms_norm(ctypes.byref(n), px, width + 5, pr, ld, pr, ld, px, width + 5, None, None, rows,
                                 torch.cuda.current_stream().cuda_stream) == 0
        assert lib.sub1_last_kernel() == (WIDE if width > 32768 else QUARTERS if width <= 512 else
                                          WAVES if width <= (2048 if torch.float32 in (rtype, TYPES[name]) else 4096) else GROUPS)
        for whole, of in zip((bx, br), want):
            assert torch.equal(whole[1:-1, 2:-3], of)
            whole[1:-1, 2:-3] = 7
            assert bool((whole == 7).all())
