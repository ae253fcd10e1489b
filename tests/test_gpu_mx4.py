"""Microscaled 4-bit operators against the oracle in 64 bits: codes, scales and expanded values to the bit,
products and the sparse MLP within the bounds that the oracle derives (half a step of bf16 where a
value is rounded to it, half steps of fp32 along a sum)."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import mx4_oracle as mo
from qmoe_amd import _lib, mx4

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def host(t):
    return t.detach().cpu().double().numpy()


def matrix(height, width, seed, spread=0):
    """(codes, scales) on the GPU and the values they stand for: any codes, scales around 1 / sqrt(width)."""
    g = gen(seed)
    nb = mo.blocks_of(width)
    codes = torch.randint(0, 256, (height, 16 * nb), dtype=torch.uint8, generator=g)
    behind = torch.arange(32 * nb) >= width                   # values behind the width are zero
    keep = torch.where(behind[0::2], 0, 15) | torch.where(behind[1::2], 0, 240)
    codes &= keep.to(torch.uint8)
    middle = 127 - 2 - int(np.log2(width) / 2)
    scales = torch.randint(middle - spread, middle + spread + 1, (height, nb), dtype=torch.int64, generator=g).to(torch.uint8)
    return codes.cuda(), scales.cuda(), mo.dequantize(codes.numpy(), scales.numpy(), width)


def activations(tokens, width, seed, strided=False):
    """bf16; strided: a part of wider rows, NaN around it"""
    x = torch.randn((tokens, width), generator=gen(seed)).bfloat16()
    if not strided:
        return x.cuda()
    whole = torch.full((tokens, width + 7), float('nan'), dtype=torch.bfloat16)
    whole[:, 3:3 + width] = x
    return whole.cuda()[:, 3:3 + width]


def within(got, exact, bound):
    got = host(got)
    assert got.shape == exact.shape
    nan = np.isnan(exact)
    assert np.array_equal(np.isnan(got), nan)
    off = np.abs(np.where(nan, 0, got) - np.where(nan, 0, exact)) - np.where(nan, 0, bound)
    assert (off <= 0).all(), 'off by %g beyond its bound at %s' % (off.max(), np.unravel_index(off.argmax(), off.shape))


# ------------------------------------------------------- to the format and back ---

@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows,width', [(1, 1), (3, 31), (1, 32), (5, 33), (2, 64), (7, 1023), (4, 2080), (300, 97)])
@pytest.mark.parametrize('strided', [False, True])
def test_quantize_to_the_bit(dtype, rows, width, strided):
    g = gen(rows * 1000 + width)
    x = torch.randn((rows, width), generator=g) * torch.exp2(4 * torch.randn((rows, width), generator=g))
    x = torch.where(torch.rand((rows, width), generator=g) < 0.3, (x * 4).round() / 4, x).clamp(-6e4, 6e4).to(dtype)
    if strided:
        whole = torch.full((rows, width + 9), float('nan'), dtype=dtype, device='cuda')
        whole[:, 2:2 + width] = x.cuda()
        codes, scales = mx4.quantize(whole[:, 2:2 + width])
    else:
        codes, scales = mx4.quantize(x.cuda())
    want_codes, want_scales = mo.quantize(host(x))
    assert np.array_equal(scales.cpu().numpy(), want_scales)
    assert np.array_equal(codes.cpu().numpy(), want_codes)
    back = mx4.dequantize(codes, scales, width, dtype)
    want = torch.from_numpy(mo.dequantize(want_codes, want_scales, width)).to(dtype)
    assert torch.equal(back.cpu(), want)


@pytest.mark.parametrize('dtype', TYPES)
def test_blocks_at_the_ends_of_the_range(dtype):
    info = torch.finfo(dtype)
    rows = [[0.0, -0.0], [info.smallest_normal, -info.smallest_normal / 4], [info.tiny * 3, 0.0], [info.max, -info.max / 2],
            [info.max, 1.0], [float('inf'), 1.0], [-float('inf'), 1.0], [float('nan'), 1.0], [1.0, 0.25], [1.0, -0.125]]
    for e in (-133, -130, -128, -127, -126, -125, -24, -14, 0, 1, 15, 125):
        rows += [[s * 2.0 ** e, 2.0 ** e / 3] for s in (1, 1.25, 1.5, 1.75, 1.9, 5, 7, 7.9)]
    x = torch.zeros((len(rows), 96), dtype=dtype)
    for i, (a, b) in enumerate(rows):
        x[i, 32], x[i, 63] = a, b
        x[i, 1] = 1.5                                          # blocks beside it are as ever
    codes, scales = mx4.quantize(x.cuda())
    want_codes, want_scales = mo.quantize(host(x))
    assert np.array_equal(scales.cpu().numpy(), want_scales) and np.array_equal(codes.cpu().numpy(), want_codes)


@pytest.mark.parametrize('dtype', TYPES)
def test_every_code_under_every_scale(dtype):
    codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 16)
    got = mx4.dequantize(codes.cuda(), scales.cuda(), 512, dtype).cpu()
    with np.errstate(over='ignore', invalid='ignore'):
        want = torch.from_numpy(mo.dequantize(codes.numpy(), scales.numpy(), 512)).to(dtype)
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(nan=1), want.nan_to_num(nan=1))


def test_shapes_and_rows_that_need_a_copy():
    x = torch.randn((3, 4, 70), generator=gen(5)).cuda()
    codes, scales = mx4.quantize(x)
    assert codes.shape == (3, 4, 48) and scales.shape == (3, 4, 3)
    back = mx4.dequantize(codes, scales, 70, torch.float32)
    assert back.shape == x.shape
    for other in (x.transpose(0, 1).contiguous().transpose(0, 1), torch.stack((x, x), -1)[..., 0]):
        assert torch.equal(mx4.quantize(other)[0], codes) and torch.equal(mx4.quantize(other)[1], scales)
    row = x[0, 0].expand(5, 70)                                # the same row five times
    assert torch.equal(mx4.quantize(row)[0], codes[0, 0].expand(5, 48))
    assert torch.equal(mx4.quantize(x[0, 0])[0], codes[0, 0])
    for empty in (x[:0], x[:, :0]):
        codes, scales = mx4.quantize(empty)
        assert codes.shape == empty.shape[:2] + (48,)
        assert mx4.dequantize(codes, scales, 70).shape == empty.shape
    with pytest.raises(TypeError):
        mx4.quantize(x.double())
    with pytest.raises(ValueError):
        mx4.quantize(x[..., :0])
    with pytest.raises(ValueError):
        mx4.dequantize(codes, scales, 97)


def test_more_blocks_than_one_launch_counts():
    """A row of one value is a block of four threads: 2^29 + 9 of them are more than one launch's 2^31, and
    the codes pass 2^32 bytes."""
    rows = (1 << 29) + 9
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip('needs 40 GB')
    x = torch.zeros((rows, 1), dtype=torch.bfloat16, device='cuda')
    at = torch.tensor([0, 1, 1 << 28, (1 << 29) - 1, 1 << 29, rows - 2, rows - 1], device='cuda')
    x[at, 0] = torch.arange(1, 8, device='cuda').bfloat16()
    codes, scales = mx4.quantize(x)
    want_codes, want_scales = mo.quantize(host(x[at]))
    assert np.array_equal(codes[at].cpu().numpy(), want_codes) and np.array_equal(scales[at].cpu().numpy(), want_scales)
    back = mx4.dequantize(codes, scales, 1)
    assert np.array_equal(host(back[at]), mo.dequantize(want_codes, want_scales, 1)) and int((back != 0).sum()) == 7


# ------------------------------------------------------------------- products ---

SHAPES = [(1, 1, 1), (16, 32, 1), (17, 33, 2), (3, 127, 16), (48, 129, 17), (100, 1000, 33), (65, 2080, 64), (130, 160, 65),
          (257, 96, 200), (200, 3001, 13), (300, 515, 300), (40, 64, 70), (40, 63, 70), (4100, 96, 30), (1000, 1056, 700), (77, 2049, 1), (9, 6144, 1), (2081, 100, 1),
          (3000, 416, 1100), (2050, 2080, 2100), (4100, 515, 40), (2600, 1000, 150), (4099, 225, 66), (2100, 96, 200),
          (8200, 64, 33), (2801, 2080, 100), (333, 2079, 15), (70, 1100, 29), (4081, 1024, 17), (100, 97, 140),
          (8300, 70, 35), (3000, 417, 1100)]


@pytest.mark.parametrize('height,width,tokens', SHAPES)
@pytest.mark.parametrize('strided', [False, True])
def test_product(height, width, tokens, strided):
    codes, scales, w = matrix(height, width, height + width, spread=3)
    x = activations(tokens, width, tokens + width, strided)
    within(mx4.product(x, codes, scales), *mo.product_bound(host(x), w))


@pytest.mark.parametrize('height,width,tokens', SHAPES + [(300, 225, 257), (130, 224, 300), (1300, 1000, 1030), (3500, 2080, 3600),
                                                          (2048, 4096, 20), (4101, 515, 70), (4099, 300, 129), (1100, 999, 500),
                                                          (37, 2081, 31), (1000, 225, 62), (513, 257, 90), (1025, 480, 130), (7, 250, 3),
                                                          (8200, 97, 64), (33000, 256, 18)])
def test_product_of_two_in_the_format(height, width, tokens):
    codes, scales, w = matrix(height, width, height + width, spread=3)
    x_codes, x_scales, x = matrix(tokens, width, tokens + width, spread=2)
    got = mx4.product_quantized(x_codes, x_scales, codes, scales, width)
    within(got, *mo.product_bound(x, w))


@pytest.mark.parametrize('tokens', [1, 5, 16, 40, 130, 600])
@pytest.mark.parametrize('quantized', [False, True])
def test_what_is_no_number_stays_in_its_row(tokens, quantized):
    height, width = 150, 333
    codes, scales, w = matrix(height, width, 7)
    x = activations(tokens, width, 8)
    x[tokens // 2, 100] = float('inf')
    x[tokens - 1, width - 1] = float('nan')
    scales[5, 3] = 255
    scales[height - 1, mo.blocks_of(width) - 1] = 255
    layer = mx4.Mx4Linear(codes, scales, width, quantize_activations=quantized)
    got = host(layer(x))
    for t in range(tokens):
        if t == tokens - 1 or (quantized and t == tokens // 2):
            assert np.isnan(got[t]).all()
            continue
        assert np.isnan(got[t, [5, height - 1]]).all()
        rest = np.delete(got[t], [5, height - 1])
        assert (~np.isfinite(rest)).all() if t == tokens // 2 else np.isfinite(rest).all()


@pytest.mark.parametrize('height,width,tokens', [(50, 100, 3), (50, 100, 40), (333, 200, 300), (16, 64, 129)])
@pytest.mark.parametrize('quantized', [False, True])
def test_nothing_is_written_beside_y(height, width, tokens, quantized):
    """Through the C entry, which takes a row stride for y."""
    lib = _lib.load()
    codes, scales, w = matrix(height, width, 9)
    ldy = height + 5
    whole = torch.full((tokens + 2, ldy), 7.0, dtype=torch.bfloat16, device='cuda')
    at = whole.data_ptr() + 2 * ldy
    stream = torch.cuda.current_stream().cuda_stream
    x = activations(tokens, width, 10)
    if quantized:
        c, s = mx4.quantize(x)
        x = mx4.dequantize(c, s, width)
        _lib.check(lib.sub1_mx4_product_quantized(codes.data_ptr(), scales.data_ptr(), height, width, c.data_ptr(), s.data_ptr(),
                                                  at, ldy, tokens, stream))
    else:
        _lib.check(lib.sub1_mx4_product(codes.data_ptr(), scales.data_ptr(), height, width, x.data_ptr(), width, at, ldy, tokens,
                                        stream))
    within(whole[1:-1, :height], *mo.product_bound(host(x), w))
    assert (whole[0] == 7).all() and (whole[-1] == 7).all() and (whole[1:-1, height:] == 7).all()


def test_the_forms_of_the_product():
    """Which kernel a call takes, at the sizes where the choice turns."""
    lib = _lib.load()
    for tokens, height, width, strided, name in (
            (1, 700, 128, False, b'mx4_one_kernel'), (1, 300, 65536, False, b'mx4_one_kernel'), (2, 700, 128, True, b'mx4_few_kernel'),
            (16, 700, 992, False, b'mx4_few_kernel'), (16, 700, 993, True, b'mx4_few_lines_kernel'), (32, 4097, 128, False, b'mx4_few_kernel'),
            (32, 4096, 128, False, b'mx4_few_lines_kernel'), (33, 2720, 128, True, b'mx4_few_lines_kernel'), (33, 2721, 128, False, b'mx4_many_direct_kernel'),
            (33, 700, 63, False, b'mx4_few_kernel'), (33, 8192, 128, True, b'mx4_few_lines_kernel'), (33, 8193, 128, True, b'mx4_many_kernel')):
        codes, scales, w = matrix(height, width, tokens)
        x = activations(tokens, width, tokens + 1, strided)
        y = mx4.product(x, codes, scales)
        assert lib.sub1_last_kernel() == name
        within(y, *mo.product_bound(host(x), w))
    for tokens, height, width, name in (
            (64, 300, 256, b'mx4_both_few_kernel'), (256, 1024, 256, b'mx4_both_few_kernel'), (65, 4128, 256, b'mx4_both_kernel<2, 1>'), (257, 300, 224, b'mx4_both_few_kernel'),
            (1000, 2100, 256, b'mx4_both_kernel<2, 2>'), (2817, 3841, 256, b'mx4_both_kernel<4, 2>')):
        codes, scales, w = matrix(height, width, tokens)
        x_codes, x_scales, x = matrix(tokens, width, tokens + 1)
        y = mx4.product_quantized(x_codes, x_scales, codes, scales, width)
        assert lib.sub1_last_kernel() == name
        within(y, *mo.product_bound(x, w))


@pytest.mark.parametrize('height,width,tokens', [(2048, 130, 2048), (2176, 2081, 2049)])
def test_whole_tiles_of_unaligned_activations(height, width, tokens):
    """A tile's sums lie in LDS at a pitch wider than its rows; the last tokens' are the ones that need its room."""
    codes, scales, w = matrix(height, width, 17, spread=3)
    x = activations(tokens, width, 18, strided=True)
    for _ in range(2):
        y = mx4.product(x, codes, scales)
        assert _lib.load().sub1_last_kernel() == b'mx4_many_kernel'
        within(y, *mo.product_bound(host(x), w))


def test_a_few_tokens_get_the_same_bits_whatever_tokens_they_come_with():
    codes, scales, _ = matrix(200, 1000, 11)
    x = activations(32, 1000, 12)
    want = mx4.product(x, codes, scales)
    for some in (slice(0, 2), slice(3, 8), slice(9, 30), slice(30, 32)):
        assert torch.equal(mx4.product(x[some], codes, scales), want[some])


@pytest.mark.parametrize('tokens', [1, 5, 40, 300])
@pytest.mark.parametrize('scale', [1, 20, 120, 200, 240])
def test_scales_far_from_one(tokens, scale):
    """As large and as small as a bf16 result and its fp32 sum have room for."""
    codes, scales, _ = matrix(70, 300, 15)
    scales.fill_(scale)
    w = mo.dequantize(codes.cpu().numpy(), scales.cpu().numpy(), 300)
    x = activations(tokens, 300, 16) * (2.0 ** 12 if scale < 10 else 1)
    within(mx4.product(x, codes, scales), *mo.product_bound(host(x), w))
    c, s = mx4.quantize(x)
    within(mx4.product_quantized(c, s, codes, scales, 300), *mo.product_bound(host(mx4.dequantize(c, s, 300)), w))


def test_linear_layers():
    w = torch.randn((70, 100), generator=gen(13)).cuda()
    x = activations(12, 100, 14).view(3, 4, 100)
    for quantized in (False, True):
        layer = mx4.Mx4Linear.make(w, quantize_activations=quantized)
        codes, scales = mo.quantize(host(w))
        assert np.array_equal(layer.codes.cpu().numpy(), codes) and np.array_equal(layer.scales.cpu().numpy(), scales)
        flat = host(x).reshape(12, 100)
        if quantized:
            flat = mo.dequantize(*mo.quantize(flat), 100)
        exact, bound = mo.product_bound(flat, mo.dequantize(codes, scales, 100))
        y = layer(x)
        assert y.shape == (3, 4, 70)
        within(y.reshape(12, 70), exact, bound)
        assert layer(x[:0]).shape == (0, 4, 70)
        again = mx4.Mx4Linear(torch.zeros_like(layer.codes), torch.zeros_like(layer.scales), 100, quantized)
        again.load_state_dict(layer.state_dict())
        assert torch.equal(again(x), y)
        for wrong, error in ((x.float(), TypeError), (x[..., :99], ValueError), (x.cpu(), ValueError)):
            with pytest.raises(error):
                layer(wrong)


@pytest.mark.parametrize('quantized', [False, True])
def test_another_width_of_as_many_blocks_runs_nothing(quantized):
    codes, scales, _ = matrix(50, 60, 41)
    layer = mx4.Mx4Linear(codes, scales, 60, quantize_activations=quantized)
    lib = _lib.load()
    mx4.product(activations(1, 60, 42), codes, scales)
    before = lib.sub1_last_kernel()
    assert before == b'mx4_one_kernel'
    for width in (64, 33):
        with pytest.raises(ValueError, match='x must be'):
            layer(activations(5, width, 43))
        assert lib.sub1_last_kernel() == before
    for wrong, error in ((None, TypeError), ([1.0] * 60, TypeError), (torch.zeros((), device='cuda').bfloat16(), ValueError)):
        with pytest.raises(error):
            layer(wrong)


@pytest.mark.parametrize('height,width,tokens,strided', [
    (300, 65536, 1, False), (300, 65535, 1, True), (300, 40000, 1, False), (40, 32769, 1, True), (300, 6144, 1, False),
    (4097, 1024, 1, False), (50, 65536, 5, False), (50, 65535, 13, True), (700, 993, 16, True), (4100, 900, 31, False),
    (2721, 2081, 33, True), (130, 65536, 70, False), (130, 65533, 90, True), (1000, 3008, 300, False), (2048, 130, 2048, True),
    (2048, 2080, 2050, False)])
@pytest.mark.parametrize('quantized', [False, True])
def test_sums_that_are_exact(height, width, tokens, strided, quantized):
    """Activations of a few whole numbers under one scale: fp32 adds them up exactly in any order, so y is the
    exact value, rounded once.  A value left out shows, at whatever width."""
    codes, scales, w = matrix(height, width, 90)
    x = torch.randint(-3, 4, (tokens, width), generator=gen(91)).bfloat16()
    x[:, [0, -1]] = 3.0
    unit = np.abs(w[w != 0]).min()
    assert (host(x[:1].abs()) @ np.abs(w).T).max() / unit < 2 ** 24 and (3 * np.abs(w).sum(-1)).max() / unit < 2 ** 24
    want = torch.from_numpy(host(x) @ w.T).float().bfloat16()         # (exact in fp32)
    if strided:
        whole = torch.full((tokens, width + 7), float('nan'), dtype=torch.bfloat16)
        whole[:, 3:3 + width] = x
        x = whole.cuda()[:, 3:3 + width]
    layer = mx4.Mx4Linear(codes, scales, width, quantize_activations=quantized)
    assert torch.equal(layer(x.cuda()).cpu(), want)


@pytest.mark.parametrize('width', [900, 993, 2080, 2081])
def test_both_forms_for_a_few_tokens_sum_alike(width):
    """From the row's length alone: a token's bits are the same with 31 others, fifteen or one."""
    lib = _lib.load()
    codes, scales, _ = matrix(4112, width, 95, spread=3)
    x = activations(32, width, 96)
    want = mx4.product(x, codes, scales)
    assert lib.sub1_last_kernel() == b'mx4_few_kernel'
    for some in (slice(0, 16), slice(16, 32), slice(30, 32)):
        assert torch.equal(mx4.product(x[some], codes, scales), want[some])
        assert lib.sub1_last_kernel() == (b'mx4_few_kernel' if width < 993 else b'mx4_few_lines_kernel')
    assert torch.equal(mx4.product(x, codes[:2000], scales[:2000]), want[:, :2000])
    assert lib.sub1_last_kernel() == b'mx4_few_lines_kernel'


# ----------------------------------------------------------------- the sparse MLP ---

def experts(count, d_model, d_ff, seed):
    """wi, wo as the layer takes them and as float64"""
    wi, wo = matrix(count * d_ff, d_model, seed, 1), matrix(count * d_model, d_ff, seed + 1, 1)
    shaped = [tuple(t.view(count, -1, t.shape[-1]) for t in m[:2]) for m in (wi, wo)]
    return shaped[0], shaped[1], wi[2].reshape(count, d_ff, d_model), wo[2].reshape(count, d_model, d_ff)


def against_the_oracle(layer, hidden, wi, wo):
    y, (logits, index) = layer(hidden)
    length = hidden.shape[-2]
    x = host(hidden).reshape(-1, hidden.shape[-1])
    exact, bound, want_logits, want_index = mo.sparse_mlp(x, host(layer.router), wi, wo, layer.top_k, layer.normalize,
                                                          layer.capacity, length)
    assert y.shape == hidden.shape and y.dtype == torch.bfloat16
    assert index.shape == hidden.shape[:-1] + (layer.top_k,) and logits.shape == hidden.shape[:-1] + (layer.experts,)
    assert np.array_equal(index.cpu().numpy().reshape(want_index.shape), want_index)
    got = logits.cpu().numpy().reshape(want_logits.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want_logits))
    # sums in 64 bits, rounded once: at most the neighbour where the sum lies between two
    assert (np.abs(np.nan_to_num(got) - np.nan_to_num(want_logits)) <= 2.0 ** -23 * np.abs(np.nan_to_num(want_logits))).all()
    within(y.reshape(-1, y.shape[-1]), exact, bound)
    return y, logits, index


CONFIGS = [
    # experts, d_model, d_ff, sequences, length, top_k, normalize, capacity, router
    (1, 1, 1, 1, 1, 1, False, None, torch.float32),
    (4, 64, 96, 1, 1, 1, False, None, torch.float32),
    (5, 33, 127, 2, 3, 2, True, None, torch.bfloat16),
    (7, 130, 250, 3, 7, 1, False, 2, torch.float32),
    (8, 100, 200, 1, 64, 8, True, None, torch.bfloat16),
    (3, 128, 64, 16, 16, 2, False, None, torch.float32),
    (2, 96, 160, 5, 40, 1, False, 11, torch.bfloat16),
    (200, 40, 70, 9, 7, 3, False, None, torch.float32),
    (4096, 24, 32, 1, 17, 1, False, None, torch.bfloat16),
    (64, 2080, 65, 1, 2, 1, False, None, torch.float32),
    (6, 70, 1300, 300, 1, 2, True, None, torch.float32),       # in two parts
    (2, 100, 90, 4, 8, 1, False, 3, torch.float32),            # grouped, with a capacity
    (2, 100, 90, 1, 40, 1, False, None, torch.bfloat16),       # and without
    (4, 97, 300, 8, 7, 4, True, None, torch.float32),
    (300, 600, 520, 3, 9, 2, True, None, torch.float32),       # more experts than a workgroup looks through by itself
    (300, 72, 2100, 2, 9, 1, False, 1, torch.bfloat16),
    (16, 1030, 700, 1, 30, 1, False, None, torch.float32),     # rows of half a wavefront, eight of them
    (40, 500, 4200, 1, 1, 1, False, None, torch.float32),
    (6, 70, 130, 6, 100, 1, False, 20, torch.float32),         # in three, of whole sequences
]


@pytest.mark.parametrize('config', CONFIGS)
def test_sparse_mlp(config):
    count, d_model, d_ff, sequences, length, top_k, normalize, capacity, dtype = config
    wi, wo, dense_wi, dense_wo = experts(count, d_model, d_ff, 20)
    router = (torch.randn((count, d_model), generator=gen(21)) / d_model ** 0.5).to(dtype).cuda()
    layer = mx4.Mx4SparseMLP(router, wi, wo, top_k, normalize, capacity)
    hidden = activations(sequences * length, d_model, 22).view(sequences, length, d_model)
    y, _, _ = against_the_oracle(layer, hidden, dense_wi, dense_wo)
    layer.router_outputs = False
    assert torch.equal(layer(hidden), y)
    assert torch.equal(layer(hidden.transpose(0, 1).contiguous().transpose(0, 1)), y)


def test_the_forms_of_the_sparse_mlp():
    lib = _lib.load()
    wi, wo, _, _ = experts(4, 64, 96, 30)
    router = torch.randn((4, 64), generator=gen(31)).cuda()
    for top_k, tokens, capacity, name in ((1, 12, None, b'mx4_one_wo_kernel'), (1, 13, None, b'mx4_wo_kernel'), (2, 6, None, b'mx4_one_wo_kernel'),
                                          (2, 7, None, b'mx4_wo_kernel'), (1, 12, 2, b'mx4_one_wo_kernel'), (1, 13, 2, b'mx4_wo_kernel')):
        mx4.Mx4SparseMLP(router, wi, wo, top_k, capacity=capacity)(activations(tokens, 64, 32))
        assert lib.sub1_last_kernel() == name


def test_equal_logits_and_tokens_that_are_no_numbers():
    wi, wo, dense_wi, dense_wo = experts(6, 64, 96, 30)
    router = torch.randn((6, 64), generator=gen(31))
    router[4] = router[1]
    router[5] = router[1]
    router[0] = 0
    hidden = activations(9, 64, 32).view(1, 9, 64)
    hidden[0, 2] = 0                                           # all logits are equal
    hidden[0, 5, 3] = float('nan')
    hidden[0, 7, 9] = float('inf')
    for top_k, capacity in ((1, 2), (3, None), (6, None)):
        layer = mx4.Mx4SparseMLP(router.cuda(), wi, wo, top_k, False, capacity)
        y, logits, index = layer(hidden)[0], *layer(hidden)[1]
        want = mo.route(logits[0].cpu().numpy(), top_k)
        assert np.array_equal(index[0].cpu().numpy(), want)
        assert want[2].tolist() == list(range(top_k)) and want[5].tolist() == list(range(top_k))
        assert y[0, 5].isnan().all() and y[0, 7].isnan().all()
        fine = [0, 1, 2, 3, 4, 6, 8]
        clean = hidden.clone()
        clean[0, [5, 7]] = 0.0 if capacity is None else hidden[0, [0, 0]]
        if capacity is None:
            against_the_oracle(layer, clean, dense_wi, dense_wo)
            assert torch.equal(layer(clean)[0][0, fine], y[0, fine])


@pytest.mark.parametrize('count', [2, 16, 300])
@pytest.mark.parametrize('sign', [0, -0x8000])
def test_tokens_that_are_no_numbers_beyond_a_capacity(count, sign):
    """all of them go to the expert of the lowest index; those that it takes and those that keep their input are NaN"""
    hidden = torch.full((2, 12, 64), 0x7fc0 + sign, dtype=torch.int16, device='cuda').view(torch.bfloat16)
    wi, wo, _, _ = experts(count, 64, 96, 33)
    layer = mx4.Mx4SparseMLP(torch.randn((count, 64), generator=gen(34)).cuda(), wi, wo, capacity=3)
    hidden[:, 4] = 0.5
    for _ in range(2):
        stale = torch.ones_like(hidden)
        del stale
        y, (logits, index) = layer(hidden)
        nan = torch.ones(2, 12, dtype=torch.bool, device='cuda')
        nan[:, 4] = False
        assert torch.equal(y.isnan().all(-1), nan) and torch.equal(y.isnan().any(-1), nan)
        assert (index[nan] == 0).all()


@pytest.mark.parametrize('capacity', [300, 2 ** 32 + 1])
def test_a_capacity_that_no_sequence_reaches(capacity):
    wi, wo, _, _ = experts(3, 64, 96, 35)
    router = torch.randn((3, 64), generator=gen(36)).cuda()
    layer = mx4.Mx4SparseMLP(router, wi, wo, capacity=capacity)
    free = mx4.Mx4SparseMLP(router, wi, wo)
    for length in (8, 300):
        hidden = activations(2 * length, 64, 37).view(2, length, 64)
        assert torch.equal(layer(hidden)[0], free(hidden)[0])
    with pytest.raises(ValueError):
        mx4.Mx4SparseMLP(router, wi, wo, capacity=299)(hidden)


def launches(call):
    """How many nodes the call's launches make in a captured graph, which is not run."""
    call()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    count = ctypes.c_size_t()
    assert _lib.load().hipGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(count)) == 0
    return count.value


@pytest.mark.parametrize('shape,free_launches', [((1, 1), 3), ((2, 3), 3), ((5, 4), 3), ((9, 5), 4)])
def test_a_capacity_that_cannot_bind_takes_no_launch(shape, free_launches):
    """Sequences no longer than the capacity: launches and bits of a layer without one.  The choice among a
    sequence's tokens is a launch of its own in the form for a token at a time, and part of the plan in the other."""
    wi, wo, dense_wi, dense_wo = experts(8, 64, 96, 38)
    router = torch.randn((8, 64), generator=gen(39)).cuda()
    hidden = activations(shape[0] * shape[1], 64, 40).view(shape + (64,))
    free = mx4.Mx4SparseMLP(router, wi, wo, router_outputs=False)
    assert launches(lambda: free(hidden)) == free_launches
    for capacity in (shape[1], 64):
        layer = mx4.Mx4SparseMLP(router, wi, wo, capacity=capacity, router_outputs=False)
        assert launches(lambda: layer(hidden)) == free_launches
        assert torch.equal(layer(hidden), free(hidden))
    if shape[1] > 1:
        layer = mx4.Mx4SparseMLP(router, wi, wo, capacity=shape[1] - 1)
        assert launches(lambda: layer(hidden)) == 4
        against_the_oracle(layer, hidden, dense_wi, dense_wo)


@pytest.mark.parametrize('d_model,d_ff,tokens,capacity', [
    (64, 40000, 1, None), (64, 65536, 3, None), (64, 65535, 6, 2), (40000, 64, 1, None), (65536, 96, 6, None), (65535, 70, 5, 1),
    (64, 40000, 20, None), (40000, 64, 20, None), (64, 65536, 20, 7)])
def test_wide_experts_exactly(d_model, d_ff, tokens, capacity):
    """Rows that need more LDS than a launch has without asking, in numbers whose sums are exact: tokens go to
    the two experts in turn with a share of one, h is small."""
    wi, wo = matrix(2 * d_ff, d_model, 92), matrix(2 * d_model, d_ff, 93)
    wi[0][:, 0] &= 0xf0                                       # the first value chooses the expert and does nothing else
    dense_wi, dense_wo = wi[2].reshape(2, d_ff, d_model), wo[2].reshape(2, d_model, d_ff)
    dense_wi[:, :, 0] = 0
    shaped = [tuple(t.view(2, -1, t.shape[-1]) for t in m[:2]) for m in (wi, wo)]
    router = torch.zeros((2, d_model))
    router[0, 0], router[1, 0] = 4, -4
    x = torch.zeros((tokens, d_model))
    at = torch.randint(1, d_model - 1, (tokens, 2), generator=gen(94))
    x.scatter_(1, at, 1.0)
    x[:, -1] = -1
    x[:, 0] = 64.0 * (1 - 2 * (torch.arange(tokens) % 2))
    layer = mx4.Mx4SparseMLP(router.cuda(), *shaped, capacity=capacity)
    y, (logits, index) = layer(x.bfloat16().cuda().view(1, tokens, d_model))
    assert index.flatten().tolist() == [t % 2 for t in range(tokens)]
    for t in range(tokens):
        if capacity is not None and t // 2 >= capacity:
            want = x[t].numpy().astype(np.float64)
        else:
            h = host(torch.from_numpy(np.maximum(dense_wi[t % 2] @ x[t].double().numpy(), 0)).float().bfloat16())
            unit = np.abs(dense_wo[dense_wo != 0]).min() * np.abs(h[h != 0]).min()
            assert (np.abs(dense_wo[t % 2]) @ h).max() / unit < 2 ** 24
            want = dense_wo[t % 2] @ h
        assert torch.equal(y[0, t].cpu(), torch.from_numpy(want).float().bfloat16()), t


@pytest.mark.parametrize('capacity', [1, 2, 3])
@pytest.mark.parametrize('count', [6, 2])
def test_a_capacity_beside_tokens_that_are_no_numbers(capacity, count):
    """They take places of the experts that they go to; the others' results are the oracle's."""
    wi, wo, dense_wi, dense_wo = experts(count, 64, 96, 30)
    router = torch.randn((count, 64), generator=gen(31))
    hidden = activations(18, 64, 32).view(2, 9, 64)
    hidden[0, 2] = 0
    hidden[:, 5, 3] = float('nan')
    hidden[1, 7, 9] = float('inf')
    y, _, _ = against_the_oracle(mx4.Mx4SparseMLP(router.cuda(), wi, wo, capacity=capacity), hidden, dense_wi, dense_wo)
    nan = torch.zeros(2, 9, dtype=torch.bool)
    nan[:, 5] = nan[1, 7] = True
    assert torch.equal(y.isnan().all(-1).cpu(), nan) and torch.equal(y.isnan().any(-1).cpu(), nan)


def test_all_tokens_to_one_expert():
    wi, wo, dense_wi, dense_wo = experts(5, 100, 90, 40)
    router = torch.zeros((5, 100))
    router[3] = 1.0
    hidden = activations(70, 100, 41).abs().view(2, 35, 100)
    for capacity in (None, 1, 16, 17, 35):
        layer = mx4.Mx4SparseMLP(router.cuda(), wi, wo, 1, False, capacity)
        _, _, index = against_the_oracle(layer, hidden, dense_wi, dense_wo)
        assert (index == 3).all()


def test_a_token_gets_the_same_bits_in_every_batch():
    wi, wo, _, _ = experts(16, 200, 300, 50)
    router = torch.randn((16, 200), generator=gen(51)).cuda()
    layer = mx4.Mx4SparseMLP(router, wi, wo, 2, True, router_outputs=False)
    hidden = activations(256, 200, 52)
    want = layer(hidden)
    for some in (slice(0, 70), slice(7, 120), slice(100, 228)):
        assert torch.equal(layer(hidden[some]), want[some])


def test_on_two_streams_and_in_two_graphs():
    """Two layers' calls on streams of their own at once, and two graphs captured on one stream and
    replayed on two, between eager calls: every result that of the eager call."""
    layers, inputs, wants = [], [], []
    for i in range(2):
        wi, wo, _, _ = experts(12, 150, 170, 60 + i)
        router = torch.randn((12, 150), generator=gen(62 + i)).cuda()
        layers.append(mx4.Mx4SparseMLP(router, wi, wo, 1 + i))
        inputs.append(activations(40, 150, 64 + i))
        wants.append(layers[i](inputs[i]))
    linear = mx4.Mx4Linear(*matrix(90, 150, 66)[:2], 150, quantize_activations=True)
    wide = mx4.Mx4Linear(*matrix(20, 40000, 67)[:2], 40000)     # more LDS than a launch has without asking
    wide_x = activations(1, 40000, 68)
    wide_want = wide(wide_x)
    linear_want = [linear(x) for x in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def same(got, i):
        return torch.equal(got[0], wants[i][0]) and torch.equal(got[1][0], wants[i][1][0]) and torch.equal(got[1][1], wants[i][1][1])

    results = []
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                results.append((i, layers[i](inputs[i])))
    torch.cuda.synchronize()
    assert all(same(got, i) for i, got in results)
    # one layer on both streams at once
    results = []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(layers[0](inputs[0]))
    torch.cuda.synchronize()
    assert all(same(got, 0) for got in results)
    graphs, outputs = [], []
    static = [x.clone() for x in inputs]
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append((layers[i](static[i]), linear(static[i]), wide(wide_x)))
        graphs.append(graph)
    for turn in range(4):
        for (y, (logits, index)), z, u in outputs:
            for t in (y, logits, index, z, u):
                t.zero_()
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
        if turn % 2:
            assert same(layers[0](inputs[0]), 0)
        torch.cuda.synchronize()
        for i in range(2):
            assert same(outputs[i][0], i) and torch.equal(outputs[i][1], linear_want[i])
            assert torch.equal(outputs[i][2], wide_want)


def test_a_dense_switch_layer_brought_to_the_format():
    """From the module of the installed transformers: its router, its capacity, its experts rounded to the
    format, against that module with the rounded weights, in fp32."""
    pytest.importorskip('transformers')
    from transformers.models.switch_transformers import modeling_switch_transformers as hf
    cfg = hf.SwitchTransformersConfig(d_model=64, d_ff=160, num_experts=6, expert_capacity=4, num_layers=2,
                                      num_sparse_encoder_layers=1, num_heads=2, d_kv=16, vocab_size=64,
                                      router_jitter_noise=0.0, dense_act_fn='relu', dropout_rate=0.0)
    torch.manual_seed(5)
    dense = hf.SwitchTransformersSparseMLP(cfg).eval().cuda()
    for p in dense.parameters():
        torch.nn.init.normal_(p, std=0.2)
    layer = mx4.Mx4SparseMLP.from_mlp(dense, router_outputs=False)
    assert layer.capacity == 4
    hidden = activations(22, 64, 70).view(2, 11, 64)
    wi, wo = [np.stack([mo.dequantize(*mo.quantize(host(getattr(e, n).weight)), getattr(e, n).weight.shape[1])
                        for e in dense.experts.values()]) for n in ('wi', 'wo')]
    exact, bound, _, index = mo.sparse_mlp(host(hidden).reshape(22, 64), host(dense.router.classifier.weight), wi, wo, 1, False, 4, 11)
    assert max(np.bincount(index[:11, 0])) > 4                # some tokens keep their input
    within(layer(hidden).view(22, 64), exact, bound)


def test_values_that_torch_keeps_with_the_other_sign():
    """A conjugate's imaginary part is a view whose values torch negates when they are read."""
    parts = torch.view_as_complex(torch.randn((40, 3, 2), generator=gen(44)).cuda()).conj().imag
    for x in (parts[:, :1], parts, torch._neg_view(parts.contiguous())):
        assert x.is_neg()
        codes, scales = mx4.quantize(x)
        want_codes, want_scales = mo.quantize(host(x))
        assert np.array_equal(codes.cpu().numpy(), want_codes) and np.array_equal(scales.cpu().numpy(), want_scales)
    codes, scales, w = matrix(70, 100, 45)
    x = torch._neg_view(activations(9, 100, 46))
    within(mx4.product(x, codes, scales), *mo.product_bound(host(x), w))
    wi, wo, dense_wi, dense_wo = experts(4, 100, 96, 47)
    layer = mx4.Mx4SparseMLP(torch.randn((4, 100), generator=gen(48)).cuda(), wi, wo)
    against_the_oracle(layer, x, dense_wi, dense_wo)


@pytest.mark.parametrize('kind', [int, np.int64, np.int32, float])
def test_whole_numbers_of_any_type(kind):
    codes, scales, w = matrix(50, 60, 41)
    x = activations(5, 60, 42)
    for quantized in (False, True):
        layer = mx4.Mx4Linear(codes, scales, kind(60), quantized)
        assert type(layer.width) is int
        flat = mo.dequantize(*mo.quantize(host(x)), 60) if quantized else host(x)
        within(layer(x), *mo.product_bound(flat, w))
    wi, wo, dense_wi, dense_wo = experts(4, 64, 96, 49)
    router = torch.randn((4, 64), generator=gen(50)).cuda()
    hidden = activations(300, 64, 51).view(50, 6, 64)          # in two parts, and in one
    for some in (hidden, hidden[:2]):
        against_the_oracle(mx4.Mx4SparseMLP(router, wi, wo, kind(1), False, kind(2)), some, dense_wi, dense_wo)
        against_the_oracle(mx4.Mx4SparseMLP(router, wi, wo, kind(2)), some, dense_wi, dense_wo)


def test_quantised_layers_in_a_row_as_a_block_runs_them():
    """A 4-bit projection, the sparse MLP on its result, a 4-bit projection with 4-bit activations."""
    g = gen(80)
    first = mx4.Mx4Linear.make(torch.randn((96, 72), generator=g).cuda() / 8)
    wi, wo, dense_wi, dense_wo = experts(5, 96, 130, 81)
    mlp = mx4.Mx4SparseMLP(torch.randn((5, 96), generator=g).cuda(), wi, wo, 2, True, router_outputs=False)
    last = mx4.Mx4Linear.make(torch.randn((40, 96), generator=g).cuda() / 10, quantize_activations=True)
    x = activations(9, 72, 82)
    a = first(x)
    b = mlp(a)
    c = last(b)
    values = [mo.dequantize(l.codes.cpu().numpy(), l.scales.cpu().numpy(), l.width) for l in (first, last)]
    within(a, *mo.product_bound(host(x), values[0]))
    exact, bound, _, _ = mo.sparse_mlp(host(a), host(mlp.router), dense_wi, dense_wo, 2, True, 0, 9)
    within(b, exact, bound)
    within(c, *mo.product_bound(mo.dequantize(*mo.quantize(host(b)), 96), values[1]))
