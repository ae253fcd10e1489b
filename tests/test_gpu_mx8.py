"""8-bit activations against the oracle in 64 bits: codes, scales and expanded values to the bit, products with
4-bit matrices within the bounds that the oracle derives."""
import numpy as np
import pytest
import torch

from oracle import block_oracle as bo
from oracle import mx4_oracle as mo
from qmoe_amd import _lib, mx4, mx8
from test_gpu_mx4 import SHAPES, gen, host, matrix, within

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def activations(tokens, width, seed, spread=2):
    """(codes, scales) on the GPU and the values they stand for: any codes that are numbers, differing scales."""
    g = gen(seed)
    nb = mo.blocks_of(width)
    codes = torch.randint(0, 256, (tokens, 32 * nb), dtype=torch.uint8, generator=g)
    codes[(codes & 127) == 127] -= 1
    codes[:, width:] = 0                                      # values behind the width are zero
    scales = torch.randint(119 - spread, 119 + spread + 1, (tokens, nb), dtype=torch.int64, generator=g).to(torch.uint8)
    return codes.cuda(), scales.cuda(), bo.dequantize8(codes.numpy(), scales.numpy(), width)


# ------------------------------------------------------- to the format and back ---

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,width', [(1, 1), (3, 31), (1, 32), (5, 33), (2, 64), (7, 1023), (4, 2080), (300, 97)])
@pytest.mark.parametrize('strided', [False, True])
def test_quantize_to_the_bit(dtype, rows, width, strided):
    g = gen(rows * 1000 + width)
    x = torch.randn((rows, width), generator=g) * torch.exp2(4 * torch.randn((rows, width), generator=g))
    x = torch.where(torch.rand((rows, width), generator=g) < 0.3, (x * 4).round() / 4, x).clamp(-6e4, 6e4).to(dtype)
    given = x.cuda()
    if strided:
        whole = torch.full((rows, width + 9), float('nan'), dtype=dtype, device='cuda')
        whole[:, 2:2 + width] = given
        given = whole[:, 2:2 + width]
    codes, scales = mx8.quantize(given)
    want_codes, want_scales = bo.quantize8(host(x))
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    back = mx8.dequantize(codes, scales, width, dtype)
    assert torch.equal(back.cpu(), torch.from_numpy(bo.dequantize8(want_codes, want_scales, width)).to(dtype))


@pytest.mark.parametrize('dtype', TYPES)
def test_blocks_at_the_ends_of_the_range(dtype):
    info = torch.finfo(dtype)
    rows = [[0.0, -0.0], [info.smallest_normal, -info.smallest_normal / 4], [info.tiny * 3, 0.0], [info.max, -info.max / 2],
            [info.max, 1.0], [float('inf'), 1.0], [-float('inf'), 1.0], [float('nan'), 1.0], [1.0, 0.25], [1.0, -0.125]]
    for e in (-133, -130, -128, -127, -126, -125, -24, -14, 0, 1, 15, 125):
        rows += [[s * 2.0 ** e, 2.0 ** e / 3] for s in (1, 1.25, 1.5, 1.75, 1.7500001, 1.7578125, 1.8, 1.9, 5, 7, 7.9)]
    x = torch.zeros((len(rows), 96), dtype=dtype)
    for i, (a, b) in enumerate(rows):
        x[i, 32], x[i, 63] = a, b
        x[i, 1] = 1.5                                          # blocks beside it are as ever
    codes, scales = mx8.quantize(x.cuda())
    want_codes, want_scales = bo.quantize8(host(x))
    assert np.array_equal(scales.cpu().numpy(), want_scales) and np.array_equal(codes.cpu().numpy(), want_codes)


@pytest.mark.parametrize('dtype', TYPES)
def test_every_code_under_every_scale(dtype):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 8)
    got = mx8.dequantize(codes.cuda(), scales.cuda(), 256, dtype).cpu()
    with np.errstate(over='ignore', invalid='ignore'):
        want = torch.from_numpy(bo.dequantize8(codes.numpy(), scales.numpy(), 256).astype(np.float32)).to(dtype)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=1), want.nan_to_num(nan=1))


def test_shapes_and_rows_that_need_a_copy():
    x = torch.randn((3, 4, 70), generator=gen(5)).cuda()
    codes, scales = mx8.quantize(x)
    assert codes.shape == (3, 4, 96) and scales.shape == (3, 4, 3)
    assert mx8.dequantize(codes, scales, 70, torch.float32).shape == x.shape
    for other in (x.transpose(0, 1).contiguous().transpose(0, 1), torch.stack((x, x), -1)[..., 0], -torch._neg_view(x)):
        assert torch.equal(mx8.quantize(other)[0], codes) and torch.equal(mx8.quantize(other)[1], scales)
    assert torch.equal(mx8.quantize(torch._neg_view(x))[0], mx8.quantize(-x)[0])
    assert torch.equal(mx8.quantize(x[0, 0].expand(5, 70))[0], codes[0, 0].expand(5, 96))
    assert torch.equal(mx8.quantize(x[0, 0])[0], codes[0, 0])
    for empty in (x[:0], x[:, :0]):
        c, s = mx8.quantize(empty)
        assert c.shape == empty.shape[:2] + (96,) and mx8.dequantize(c, s, 70).shape == empty.shape
    with pytest.raises(TypeError):
        mx8.quantize(x.double())
    with pytest.raises(ValueError):
        mx8.quantize(x[..., :0])
    with pytest.raises(ValueError):
        mx8.dequantize(codes, scales, 97)


def test_more_blocks_than_one_launch_counts():
    """A row of one value is a block of four threads: 2^29 + 9 of them are more than one launch's 2^31, and
    the codes pass 2^34 bytes."""
    rows = (1 << 29) + 9
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB')
    x = torch.zeros((rows, 1), dtype=torch.bfloat16, device='cuda')
    at = torch.tensor([0, 1, 1 << 28, (1 << 29) - 1, 1 << 29, rows - 2, rows - 1], device='cuda')
    x[at, 0] = torch.arange(1, 8, device='cuda').bfloat16()
    codes, scales = mx8.quantize(x)
    want_codes, want_scales = bo.quantize8(host(x[at]))
    assert np.array_equal(codes[at].cpu().numpy(), want_codes) and np.array_equal(scales[at].cpu().numpy(), want_scales)
    back = mx8.dequantize(codes, scales, 1)
    assert np.array_equal(host(back[at]), bo.dequantize8(want_codes, want_scales, 1)) and int((back != 0).sum()) == 7


# ------------------------------------------------------------------- products ---

MORE = [(300, 225, 257), (130, 224, 300), (1300, 1000, 1030), (3500, 2080, 3600), (2048, 4096, 20), (4101, 515, 70), (4099, 300, 129),
        (1100, 999, 500), (37, 2081, 31), (1000, 225, 62), (513, 257, 90), (1025, 480, 130), (7, 250, 3), (8200, 97, 64), (33000, 256, 18),
        (500, 6144, 260), (31, 5000, 1), (32, 33, 1), (4000, 128, 1), (33, 1, 5), (2080, 6144, 600), (640, 320, 2500)]


def some(tokens):
    """A few tokens, the first and the last among them."""
    return sorted({0, tokens // 3, tokens - 1})


@pytest.mark.parametrize('height,width,tokens', SHAPES + MORE)
@pytest.mark.parametrize('relu', [False, True])
def test_product(height, width, tokens, relu):
    codes, scales, w = matrix(height, width, height + width, spread=3)
    x_codes, x_scales, x = activations(tokens, width, tokens + width)
    got = mx8.product(x_codes, x_scales, codes, scales, width, relu)
    assert not (relu and bool((got < 0).any()))
    for at, bounds in ((slice(None), bo.product8_bound), (some(tokens), bo.product8_bound_finely)):
        exact, bound = bo.to_bf16(*bounds(x[at], w))
        within(got[at], np.maximum(exact, 0) if relu else exact, bound)


@pytest.mark.parametrize('height,width,tokens', SHAPES + MORE)
def test_product_into_eight_bits(height, width, tokens):
    codes, scales, w = matrix(height, width, height + width, spread=3)
    x_codes, x_scales, x = activations(tokens, width, tokens + width)
    relu = bool((height + tokens) % 2)
    y_codes, y_scales = mx8.product(x_codes, x_scales, codes, scales, width, relu, True)
    for at, bounds in ((slice(None), bo.product8_bound), (some(tokens), bo.product8_bound_finely)):
        exact, off = bounds(x[at], w)
        bo.check_quantized(y_codes[at].cpu().numpy(), y_scales[at].cpu().numpy(), np.maximum(exact, 0) if relu else exact, off)


@pytest.fixture
def form():
    """Sets the form that products take, and back."""
    yield lambda which: _lib.check(_lib.load().sub1_test_mx8_form(which))
    _lib.check(_lib.load().sub1_test_mx8_form(0))


@pytest.mark.parametrize('which', range(1, _lib.MX8_FORMS + 1))
@pytest.mark.parametrize('height,width,tokens', [(300, 1000, 300), (33, 256, 2), (577, 2079, 515), (289, 225, 257), (96, 4500, 65), (2081, 640, 31),
                                                 (64, 1152, 128), (1100, 3201, 1030)])
def test_every_form(which, height, width, tokens, form):
    """Odd tiles, rows of a step, of fewer steps than there are groups that share them, and many."""
    codes, scales, w = matrix(height, width, height + width, spread=3)
    x_codes, x_scales, x = activations(tokens, width, tokens + width)
    exact, off = bo.product8_bound(x, w)
    fine = some(tokens)
    finely = bo.product8_bound_finely(x[fine], w)
    form(which)
    got = mx8.product(x_codes, x_scales, codes, scales, width)
    within(got, *bo.to_bf16(exact, off))
    within(got[fine], *bo.to_bf16(*finely))
    y_codes, y_scales = mx8.product(x_codes, x_scales, codes, scales, width, True, True)
    bo.check_quantized(y_codes.cpu().numpy(), y_scales.cpu().numpy(), np.maximum(exact, 0), off)
    bo.check_quantized(y_codes[fine].cpu().numpy(), y_scales[fine].cpu().numpy(), np.maximum(finely[0], 0), finely[1])
    x_scales[-1, -1], scales[height // 2, 0] = 255, 255       # no numbers in the last token and a row
    got = host(mx8.product(x_codes, x_scales, codes, scales, width))
    assert np.isnan(got[-1]).all() and np.isnan(got[:, height // 2]).all()
    assert np.isfinite(np.delete(got[:-1], height // 2, 1)).all()


@pytest.mark.parametrize('which', range(1, _lib.MX8_FORMS + 1))
@pytest.mark.parametrize('height,width,tokens', [(130, 1, 70), (33, 33, 2), (300, 96, 300), (70, 128, 31), (577, 129, 130), (289, 224, 257)])
def test_every_form_on_rows_of_few_blocks(which, height, width, tokens, form):
    """Fewer than eight: their scales are loaded one by one; some groups have no step at all."""
    codes, scales, w = matrix(height, width, height + width, spread=3)
    x_codes, x_scales, x = activations(tokens, width, tokens + width)
    exact, off = bo.product8_bound_finely(x, w)
    form(which)
    within(mx8.product(x_codes, x_scales, codes, scales, width), *bo.to_bf16(exact, off))
    y_codes, y_scales = mx8.product(x_codes, x_scales, codes, scales, width, True, True)
    bo.check_quantized(y_codes.cpu().numpy(), y_scales.cpu().numpy(), np.maximum(exact, 0), off)
    x_scales[-1, -1], scales[height // 2, -1] = 255, 255
    got = host(mx8.product(x_codes, x_scales, codes, scales, width))
    assert np.isnan(got[-1]).all() and np.isnan(got[:, height // 2]).all()
    assert np.isfinite(np.delete(got[:-1], height // 2, 1)).all()


@pytest.mark.parametrize('which', [0, 1, 2, 3, 4])
def test_the_most_tokens(which, form):
    """As many as a call takes, through a narrow matrix: the most tiles of tokens that a launch has."""
    tokens, height, width = _lib.MX4_MAX_TOKENS, 33, 40
    codes, scales, w = matrix(height, width, 1)
    x_codes, x_scales, x = activations(tokens, width, 2)
    form(which)
    got = mx8.product(x_codes, x_scales, codes, scales, width)
    at = [0, 15, 16, tokens // 2, tokens - 17, tokens - 16, tokens - 1]
    within(got[at], *bo.to_bf16(*bo.product8_bound_finely(x[at], w)))
    # two roundings of 2^-8 of a value each, and twice 5 eights' products cut off by 7 2^-14 of the eight's largest (0.0043 of it)
    form(0)
    for part in (slice(0, 3000), slice(tokens - 3000, tokens)):
        again = mx8.product(x_codes[part].contiguous(), x_scales[part].contiguous(), codes, scales, width)
        assert bool(((got[part].float() - again.float()).abs() <= 0.02 * again.float().abs().max()).all())


@pytest.mark.parametrize('which', range(1, _lib.MX8_FORMS + 1))
def test_sums_past_fp32(which, form):
    """Scales whose products fp32 does not hold: infinite, of the sum's sign."""
    codes, scales, w = matrix(70, 256, 5)
    codes &= 0x77
    codes |= 0x11                                             # no zeros, none negative
    x_codes = torch.full((70, 256), 0x38, dtype=torch.uint8, device='cuda')
    x_codes[1::2] |= 0x80
    x_scales, scales = torch.full((70, 8), 254, dtype=torch.uint8, device='cuda'), torch.full_like(scales, 254)
    form(which)
    got = mx8.product(x_codes, x_scales, codes, scales, 256)
    assert bool((got[0::2] == float('inf')).all()) and bool((got[1::2] == -float('inf')).all())
    assert bool((mx8.product(x_codes[:1], x_scales[:1], codes, scales, 256) == float('inf')).all())


@pytest.mark.parametrize('tokens', [1, 5, 16, 40, 130, 600])
@pytest.mark.parametrize('quantize', [False, True])
@pytest.mark.parametrize('relu', [False, True])
def test_what_is_no_number_stays_in_its_row(tokens, quantize, relu):
    height, width = 150, 333
    codes, scales, w = matrix(height, width, 7)
    x_codes, x_scales, x = activations(tokens, width, 8)
    x_codes[tokens - 1, width - 1] = 127                      # no number
    x_scales[tokens // 2, 3] = 255
    scales[5, 3] = 255
    scales[height - 1, mo.blocks_of(width) - 1] = 255
    got = mx8.product(x_codes, x_scales, codes, scales, width, relu, quantize)
    if quantize:
        got = mx8.dequantize(*got, height)
    got = host(got)
    gone = [5, height - 1]
    if quantize:                                              # with their blocks
        gone = [r for r in range(height) if r // 32 in (0, (height - 1) // 32)]
    for t in range(tokens):
        if t in (tokens - 1, tokens // 2):
            assert np.isnan(got[t]).all()
        else:
            assert np.isnan(got[t, gone]).all() and np.isfinite(np.delete(got[t], gone)).all()


@pytest.mark.parametrize('tokens', [1, 3, 70, 400])
def test_scales_far_from_one(tokens):
    """Scales whose product is ordinary, and whose single values fp32 holds barely or not in its normal range."""
    height, width = 200, 417
    codes, scales, w = matrix(height, width, 3, spread=1)
    x_codes, x_scales, x = activations(tokens, width, 4, spread=1)
    for by in (-100, 100):
        s, xs = scales.int() + by, x_scales.int() - by
        got = mx8.product(x_codes, xs.to(torch.uint8), codes, s.to(torch.uint8), width)
        within(got[:9], *bo.to_bf16(*bo.product8_bound_finely(x[:9], w)))


@pytest.mark.parametrize('height,width,tokens', [(50, 100, 3), (50, 100, 40), (333, 200, 300), (16, 64, 129), (45, 700, 1), (1000, 1056, 700)])
@pytest.mark.parametrize('quantize', [False, True])
def test_nothing_is_written_beside_the_result(height, width, tokens, quantize):
    codes, scales, w = matrix(height, width, 1)
    x_codes, x_scales, x = activations(tokens, width, 2)
    lib, nb = _lib.load(), mo.blocks_of(height)
    stream = torch.cuda.current_stream().cuda_stream
    args = (codes.data_ptr(), scales.data_ptr(), height, width, x_codes.data_ptr(), x_scales.data_ptr(), 0)
    if quantize:
        c = torch.full((tokens * 32 * nb + 64,), 0x5a, dtype=torch.uint8, device='cuda')
        s = torch.full((tokens * nb + 64,), 0x5a, dtype=torch.uint8, device='cuda')
        assert lib.sub1_mx8_product(*args, None, 0, c[32:].data_ptr(), s[32:].data_ptr(), tokens, stream) == 0
        want = mx8.product(x_codes, x_scales, codes, scales, width, False, True)
        for got, right in ((c, want[0]), (s, want[1])):
            assert bool((got[:32] == 0x5a).all()) and bool((got[-32:] == 0x5a).all())
            assert torch.equal(got[32:-32], right.flatten())
    else:
        y = torch.full((tokens + 2, height + 5), 7.0, dtype=torch.bfloat16, device='cuda')
        assert lib.sub1_mx8_product(*args, y[1:, 2:].data_ptr(), height + 5, None, None, tokens, stream) == 0
        assert torch.equal(y[1:-1, 2:-3], mx8.product(x_codes, x_scales, codes, scales, width))
        y[1:-1, 2:-3] = 7.0
        assert bool((y == 7).all())


def test_shapes_of_products():
    codes, scales, w = matrix(70, 96, 1)
    x_codes, x_scales, x = activations(12, 96, 2)
    want = mx8.product(x_codes, x_scales, codes, scales, 96)
    got = mx8.product(x_codes.view(3, 4, -1), x_scales.view(3, 4, -1), codes, scales, 96)
    assert got.shape == (3, 4, 70) and torch.equal(got.view(12, 70), want)
    assert mx8.product(x_codes[0], x_scales[0], codes, scales, 96).shape == (70,)
    assert mx8.product(x_codes[:0], x_scales[:0], codes, scales, 96).shape == (0, 70)
    c, s = mx8.product(x_codes[:0], x_scales[:0], codes, scales, 96, quantize=True)
    assert c.shape == (0, 96) and s.shape == (0, 3)
    assert torch.equal(mx8.product(x_codes, x_scales, codes, scales, 96.0, 1, 0), torch.relu(want))
    for wrong in ((x_codes, x_scales, codes, scales, 97), (x_codes, x_scales[:, :2], codes, scales, 96), (x_codes, x_scales, codes[None], scales[None], 96),
                  (x_codes, x_scales, codes.cpu(), scales, 96), (x_codes[:, 1:], x_scales, codes, scales, 96),
                  (x_codes.t().contiguous().t(), x_scales, codes, scales, 96)):
        with pytest.raises(ValueError):
            mx8.product(*wrong)
    with pytest.raises(TypeError):
        mx8.product(x_codes.int(), x_scales, codes, scales, 96)


def test_products_past_32_bits():
    """y of more than 2^32 bytes, and activations of more than 2^31."""
    tokens, height, width = 40000, 65536, 64
    if torch.cuda.mem_get_info()[0] < 30 << 30:
        pytest.skip('needs 30 GB')
    codes, scales, w = matrix(height, width, 1)
    x_codes, x_scales, x = activations(tokens, width, 2)
    got = mx8.product(x_codes, x_scales, codes, scales, width)
    for t in (0, 1, 20011, 32767, 32768, tokens - 1):
        within(got[t][None], *bo.to_bf16(*bo.product8_bound_finely(x[t][None], w)))
    got = mx8.product(x_codes, x_scales, codes, scales, width, True, True)
    for t in (0, 32768, tokens - 1):
        exact, off = bo.product8_bound_finely(x[t][None], w)
        bo.check_quantized(got[0][t][None].cpu().numpy(), got[1][t][None].cpu().numpy(), np.maximum(exact, 0), off)
    del got
    tokens, width = 34000, 65536
    codes, scales, w = matrix(40, width, 1)
    x_codes = torch.zeros((tokens, width), dtype=torch.uint8, device='cuda')
    x_scales = torch.full((tokens, width // 32), 119, dtype=torch.uint8, device='cuda')
    last_codes, last_scales, last = activations(2, width, 3)
    x_codes[-2:], x_scales[-2:] = last_codes, last_scales
    got = mx8.product(x_codes, x_scales, codes, scales, width)
    within(got[-2:], *bo.to_bf16(*bo.product8_bound_finely(last, w)))
    assert bool((got[:-2] == 0).all())
