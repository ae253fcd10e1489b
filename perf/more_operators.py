"""The operators around the experts and the 4-bit layers of a block, as measurable cases.

Four paths:

  norm      root-mean-square norm of rows, the residual's addition before it, the result
            in the input's type or in 8 bits (blocks of 32 values in e4m3 with a power
            of two each)
  product   activations in those 8 bits times a matrix in microscaled 4-bit floats, ReLU
            and 8 bits of the result in the same call where the next layer wants them
  route     which experts a token goes to and with what shares, from the router's logits
  combine   the weighted sum of a token's experts' outputs, the residual added

Widths are those of the Switch shapes of qmoe_amd.synthetic.SHAPES (d_model 768 to 2080, d_ff to 6144)
and odd ones between them.  Values in 8 bits are returned as what they stand for.

`own` chooses who computes: the elementary operations below, or the package.
"""
import math

import torch

own = False

DEVICE = 'cuda:0'
BLOCK = 32
EPS = 1e-6
LARGE, C2048 = (1024, 4096), (2080, 6144)      # (d_model, d_ff)
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def listed():
    return [
        # generation, batch 1: the norm before a 4-bit layer that takes 8 bits
        dict(name='norm_one_token', kind='norm', rows=1, width=2080, dtype='bf16', residual='same', weight='same',
             quantize=True, strided=False),
        # a part of each row of a wider tensor, odd sizes, the first norm of a model
        dict(name='norm_ragged', kind='norm', rows=61, width=1023, dtype='fp16', residual='', weight='fp32',
             quantize=False, strided=True),
        # encoding 32 sequences of 512 tokens
        dict(name='norm_sequences', kind='norm', rows=16384, width=2080, dtype='bf16', residual='same', weight='same',
             quantize=True, strided=False),
        # generation, batch 1: one token through the largest wo
        dict(name='product_one_token', kind='product', tokens=1, height=2080, width=6144, relu=False, quantize=False),
        # a batch that generates together through the largest wi, on its way to wo
        dict(name='product_batch', kind='product', tokens=61, height=6144, width=2080, relu=True, quantize=True),
        # some sequences through a matrix of odd sizes
        dict(name='product_ragged', kind='product', tokens=333, height=3001, width=1023, relu=False, quantize=False),
        # encoding sixteen sequences of 512 tokens, the largest wo
        dict(name='product_sequences', kind='product', tokens=8192, height=2080, width=6144, relu=False, quantize=False),
        # generation, batch 1: the Switch router's choice
        dict(name='route_one_token', kind='route', tokens=1, experts=128, top_k=1, scores='softmax', bias=False,
             groups=1, top_groups=1, group_mark=1, normalize=False, dtype='fp32', strided=False),
        # a batch over the largest layer's experts, two each, logits in bf16 and part of a wider tensor
        dict(name='route_many_experts', kind='route', tokens=333, experts=2048, top_k=2, scores='softmax', bias=False,
             groups=1, top_groups=1, group_mark=1, normalize=True, dtype='bf16', strided=True),
        # encoding: balanced by a bias, in groups, eight experts each
        dict(name='route_groups', kind='route', tokens=8192, experts=256, top_k=8, scores='sigmoid', bias=True,
             groups=8, top_groups=4, group_mark=2, normalize=True, dtype='fp32', strided=False),
        # a small, odd batch, two experts a token
        dict(name='combine_few', kind='combine', tokens=13, top_k=2, width=1024, dtype='bf16', residual=True),
        # encoding, four experts a token
        dict(name='combine_sequences', kind='combine', tokens=8192, top_k=4, width=2080, dtype='bf16', residual=True),
    ]


def draw(rng):
    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kind = rng.choice(['norm', 'product', 'product', 'route', 'combine'])
    if kind == 'norm':
        width = log(1, 6144) if rng.random() < 0.5 else rng.choice([768, 1024, 2080])
        rows = log(1, max(1, min(16384, 16384 * 2080 // (2 * width))))
        dtype = rng.choice(sorted(TYPES))
        return dict(kind=kind, rows=rows, width=width, dtype=dtype, residual=rng.choice(['', 'same', 'same', 'fp32']),
                    weight=rng.choice(['same', 'fp32']), quantize=rng.random() < 0.5, strided=rng.random() < 0.3)
    if kind == 'product':
        pair = rng.choice([LARGE, C2048]) if rng.random() < 0.4 else (rng.randint(500, 2080), rng.randint(2000, 6144))
        height, width = rng.choice([pair, pair[::-1]])
        return dict(kind=kind, tokens=log(1, 8192), height=height, width=width, relu=rng.random() < 0.5,
                    quantize=rng.random() < 0.5)
    if kind == 'route':
        groups = rng.choice([1, 1, 2, 4, 8])
        top_groups = rng.randint(1, groups)
        size = log(max(2, 8 // top_groups), 2048 // groups)
        experts = groups * size
        return dict(kind=kind, tokens=log(1, max(1, min(8192, 8192 * 256 // experts))), experts=experts,
                    top_k=rng.choice([k for k in (1, 2, 4, 8) if k <= size * top_groups]),
                    scores=rng.choice(['softmax', 'sigmoid']), bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
                    group_mark=rng.choice([1, 2]), normalize=rng.random() < 0.5, dtype=rng.choice(['bf16', 'fp32']),
                    strided=rng.random() < 0.3)
    return dict(kind=kind, tokens=log(1, 8192), top_k=rng.choice([1, 2, 3, 4]), width=rng.randint(500, 2080),
                dtype=rng.choice(['bf16', 'bf16', 'fp16']), residual=rng.random() < 0.5)


# ------------------------------------------------------------- preparing ---

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _normal(shape, g):
    return torch.randn(shape, generator=g, device=DEVICE)


def _part(x, strided):
    """x [rows, width], as a part of wider rows where strided"""
    if not strided:
        return x
    whole = torch.full((x.shape[0], x.shape[1] + 37), 7.0, dtype=x.dtype, device=x.device)
    whole[:, 5:5 + x.shape[1]] = x
    return whole[:, 5:5 + x.shape[1]]


def _matrix4(height, width, g):
    """(codes uint8 [height, 16 nb], scales uint8 [height, nb]) of a matrix of about normal weights, N(0, 1 / width):
    two codes a byte over the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6, the largest of a block 4 or 6, its scale a power
    of two."""
    blocks = -(-width // BLOCK)
    v = torch.zeros((height, blocks * BLOCK), device=DEVICE)
    v[:, :width] = _normal((height, width), g) / width ** 0.5
    v = v.view(height, blocks, BLOCK)
    power = torch.floor(torch.log2(v.abs().amax(-1, keepdim=True))) - 2
    code = torch.bucketize(v.abs() * torch.exp2(-power),
                           torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEVICE)).to(torch.uint8)
    code |= 8 * (v < 0).to(torch.uint8)
    codes = (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-2)
    return codes, (power.squeeze(-1) + 127).to(torch.uint8)


def prepare(case, seed):
    g = _generator(1000 * seed + 29)
    state = dict(case)
    kind = case['kind']
    if kind == 'norm':
        rows, width, dtype = case['rows'], case['width'], TYPES[case['dtype']]
        # hidden states: some channels much larger than the others
        channels = torch.exp2(2 * _normal((1, width), g)).clamp(max=64)
        state['x'] = _part((_normal((rows, width), g) * channels).to(dtype), case['strided'])
        if case['residual']:
            r = _normal((rows, width), g) * channels * 4
            state['r'] = _part(r.to(dtype if case['residual'] == 'same' else torch.float32), case['strided'])
        state['w'] = (0.2 + 0.1 * _normal((width,), g)).to(dtype if case['weight'] == 'same' else torch.float32)
    elif kind == 'product':
        # activations behind a norm, blocks of differing sizes
        x = _normal((case['tokens'], case['width']), g) * torch.exp2(2 * _normal((1, case['width']), g)).clamp(max=64)
        state['x'] = _stored8(x)
        state['w'] = _matrix4(case['height'], case['width'], g)
    elif kind == 'route':
        # logits of a router that prefers some experts
        logits = 2 * _normal((case['tokens'], case['experts']), g) + _normal((1, case['experts']), g)
        state['logits'] = _part(logits.to(TYPES[case['dtype']]), case['strided'])
        state['b'] = 0.1 * _normal((case['experts'],), g) if case['bias'] else None
    else:
        dtype = TYPES[case['dtype']]
        state['outputs'] = _normal((case['tokens'], case['top_k'], case['width']), g).to(dtype)
        state['shares'] = torch.softmax(_normal((case['tokens'], case['top_k']), g), dim=-1)
        state['r'] = (4 * _normal((case['tokens'], case['width']), g)).to(dtype) if case['residual'] else None
    return state


# --------------------------------------------------------------- running ---

def run(state):
    with torch.no_grad():
        return _RUN[own, state['kind']](state)


def _own_norm(s):
    from qmoe_amd import mx8, norm
    y = norm.rms_norm(s['x'], s['w'], EPS, s.get('r'), quantize=s['quantize'])
    y, total = y if 'r' in s else (y, None)
    if s['quantize']:
        y = mx8.dequantize(*y, s['width'])
    return y, total


def _own_product(s):
    from qmoe_amd import mx8
    y = mx8.product(*s['x'], *s['w'], s['width'], relu=s['relu'], quantize=s['quantize'])
    return mx8.dequantize(*y, s['height']) if s['quantize'] else y


def _own_route(s):
    from qmoe_amd import routing
    return routing.route(s['logits'], s['top_k'], scores=s['scores'], bias=s['b'], groups=s['groups'],
                         top_groups=s['top_groups'], group_mark=s['group_mark'], normalize=s['normalize'])


def _own_combine(s):
    from qmoe_amd import routing
    return routing.combine(s['outputs'], s['shares'], s['r'])


def _power(exponent):
    """2^exponent as fp32, exactly, for -126 to 127 and int32"""
    return ((exponent + 127) << 23).view(torch.float32)


def _blocks(x):
    """fp32 [.., nb, 32], zeros behind the last value"""
    return torch.nn.functional.pad(x.float(), (0, -x.shape[-1] % BLOCK)).unflatten(-1, (-1, BLOCK))


def _exponents(v):
    """int32 [.., nb, 1]: the least e with all of a block at most 448 2^e (e4m3's largest), not below -119, far from
    what these cases hold"""
    bits = v.abs().amax(-1, keepdim=True).view(torch.int32)
    return ((bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000).int()).clamp(min=-119)


def _stored8(x):
    """(codes uint8 [.., 32 nb], scales uint8 [.., nb])"""
    v = _blocks(x)
    e = _exponents(v)
    codes = (v * _power(-e)).to(torch.float8_e4m3fn).view(torch.uint8).flatten(-2)
    return codes, (e + 127).to(torch.uint8).squeeze(-1)


def _plain_norm(s):
    x, r = s['x'], s.get('r')
    total = None if r is None else (x.float() + r.float()).to(r.dtype)
    v = (x if r is None else total).float()
    y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * s['w'].float()
    return (_values8(y) if s['quantize'] else y.to(x.dtype)), total


def _values8(y):
    """bf16: what y is in 8 bits (exact, an e4m3 has three bits behind its leading one)"""
    v = _blocks(y)
    scale = _power(_exponents(v))
    kept = (v * (1 / scale)).to(torch.float8_e4m3fn).float() * scale
    return kept.flatten(-2)[..., :y.shape[-1]].bfloat16()


def _plain_product(s):
    (x, xs), (w, ws) = s['x'], s['w']
    x = (x.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, BLOCK)) * _power(xs.int() - 127)[..., None]).flatten(-2)
    code = torch.stack((w & 15, w >> 4), dim=-1).flatten(-2)
    m = (code & 7).float()
    m = 0.5 * m + 0.5 * (m - 4).clamp(min=0) + (m - 6).clamp(min=0)
    w = torch.where(code >= 8, -m, m).unflatten(-1, (-1, BLOCK))
    w = (w * _power(ws.int() - 127)[..., None]).flatten(-2)
    y = x @ w.t()
    if s['relu']:
        y = y.clamp(min=0)
    return _values8(y) if s['quantize'] else y.bfloat16()


def _plain_route(s):
    # in 64 bits: which of two close scores is larger decides
    logits = s['logits'].double()
    if s['scores'] == 'softmax':
        scores = torch.exp(logits - logits.amax(-1, keepdim=True))
        scores = scores / scores.sum(-1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-logits))
    marks = scores if s['b'] is None else scores + s['b'].double()
    if s['groups'] > 1:
        grouped = marks.unflatten(-1, (s['groups'], -1))
        of_group = torch.sort(grouped, dim=-1, descending=True)[0][..., :s['group_mark']].sum(-1)
        best = torch.sort(of_group, dim=-1, descending=True, stable=True)[1][..., :s['top_groups']]
        kept = torch.zeros_like(of_group, dtype=torch.bool).scatter_(-1, best, True)
        marks = torch.where(kept[..., None], grouped, -math.inf).flatten(-2)
    index = torch.sort(marks, dim=-1, descending=True, stable=True)[1][..., :s['top_k']]
    shares = torch.gather(scores, -1, index)
    if s['normalize']:
        shares = shares / shares.sum(-1, keepdim=True)
    return shares.float(), index


def _plain_combine(s):
    y = (s['shares'][..., None] * s['outputs'].float()).sum(-2)
    if s['r'] is not None:
        y = y + s['r'].float()
    return y.to(s['outputs'].dtype)


_RUN = {(True, 'norm'): _own_norm, (True, 'product'): _own_product, (True, 'route'): _own_route,
        (True, 'combine'): _own_combine, (False, 'norm'): _plain_norm, (False, 'product'): _plain_product,
        (False, 'route'): _plain_route, (False, 'combine'): _plain_combine}


# --------------------------------------------- what it needs, and the truth ---

def work(case):
    kind = case['kind']
    if kind == 'norm':
        n, size = case['rows'] * case['width'], TYPES[case['dtype']].itemsize
        r = {'': 0, 'same': size, 'fp32': 4}[case['residual']]
        w = size if case['weight'] == 'same' else 4
        stored = case['rows'] * -(-case['width'] // BLOCK) * 33
        # 8 bits: written, read back and written as values
        return dict(bytes=n * (size + 2 * r) + w * case['width'] + (2 * stored + 2 * n if case['quantize'] else n * size),
                    flops=0)
    if kind == 'product':
        t, h, w = case['tokens'], case['height'], case['width']
        blocks, out = -(-w // BLOCK), -(-h // BLOCK)
        y = 2 * t * out * 33 + 2 * t * h if case['quantize'] else 2 * t * h
        return dict(bytes=h * blocks * 17 + t * blocks * 33 + y, flops=2 * t * h * w)
    if kind == 'route':
        t, e = case['tokens'], case['experts']
        return dict(bytes=t * e * TYPES[case['dtype']].itemsize + (4 * e if case['bias'] else 0) + 12 * t * case['top_k'],
                    flops=0)
    t, size = case['tokens'], TYPES[case['dtype']].itemsize
    rows = case['top_k'] + 1 + (1 if case['residual'] else 0)
    return dict(bytes=t * (rows * case['width'] * size + 4 * case['top_k']), flops=0)


_GRID4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _grid8():
    """The magnitudes of e4m3 in order: 127 of them, by exponent field and mantissa."""
    low = [m / 8 * 2.0 ** -6 for m in range(8)]
    return low + [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)]


def _scales64(bytes_):
    table = torch.tensor([math.ldexp(1.0, i - 127) for i in range(255)] + [math.nan], dtype=torch.float64, device=bytes_.device)
    return table[bytes_.long()]


def _nearest8(y):
    """float64 in, float64 out: each block of 32 in 8 bits under the smallest power of two that reaches its largest."""
    shape = y.shape
    v = torch.nn.functional.pad(y, (0, -shape[-1] % BLOCK)).reshape(shape[0], -1, BLOCK)
    largest = v.abs().max(-1, keepdim=True)[0]
    m, above = torch.frexp(largest)                         # largest = m 2^above, 1/2 <= m < 1; 448 = 7/8 2^9
    scale = _scales64(((above - 9 + (m > 0.875)).clamp(min=-119) + 127).clamp(0, 254))
    grid = torch.tensor(_grid8(), dtype=torch.float64, device=y.device)
    scaled = v.abs() / scale
    middle = (grid[1:] + grid[:-1]) / 2
    at = torch.bucketize(scaled, middle)                    # on the middle: the lower
    on = torch.bucketize(scaled, middle, right=True) > at   # where the even one counts
    at = torch.where(on & (at % 2 == 1), at + 1, at)
    return (torch.sign(v) * grid[at] * scale).reshape(shape[0], -1)[:, :shape[-1]]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case['kind']
    if kind == 'norm':
        x, total = s['x'].double(), None
        if 'r' in s:
            total = x + s['r'].double()
            x = total.to(s['r'].dtype).double()             # what the norm is given is what is written
        y = x / torch.sqrt(torch.square(x).sum(-1, keepdim=True) / case['width'] + EPS) * s['w'].double()
        return (torch.cat([_nearest8(part) for part in y.split(2048)]) if case['quantize'] else y), total
    if kind == 'product':
        codes, scales = s['x']
        grid = torch.tensor(_grid8() + [math.nan], dtype=torch.float64, device=codes.device)
        x = torch.cat((grid, -grid))[codes.long()] * _scales64(scales).repeat_interleave(BLOCK, -1)
        codes, scales = s['w']
        grid = torch.tensor(_GRID4 + tuple(-v for v in _GRID4), dtype=torch.float64, device=codes.device)
        w = grid[torch.stack((codes % 16, codes // 16), -1).reshape(codes.shape[0], -1).long()]
        w = w * _scales64(scales).repeat_interleave(BLOCK, -1)
        y = torch.matmul(x, w.transpose(0, 1))
        y = torch.relu(y) if case['relu'] else y
        return torch.cat([_nearest8(part) for part in y.split(2048)]) if case['quantize'] else y
    if kind == 'route':
        logits = s['logits'].to(torch.float64)
        scores = torch.softmax(logits, -1) if case['scores'] == 'softmax' else torch.sigmoid(logits)
        c = scores + (0 if s['b'] is None else s['b'].to(torch.float64))
        left = torch.ones_like(c, dtype=torch.bool)
        if case['groups'] > 1:
            size = case['experts'] // case['groups']
            best = c.view(-1, case['groups'], size).topk(min(size, case['group_mark']), -1)[0].sum(-1)
            taken = torch.argsort(-best, dim=-1, stable=True)[:, :case['top_groups']]
            left = (taken[:, :, None] == torch.arange(case['experts'], device=c.device) // size).any(1)
        index = torch.argsort(torch.where(left, -c, math.inf), dim=-1, stable=True)[:, :case['top_k']]
        shares = scores.gather(1, index)
        return (shares / shares.sum(1, keepdim=True) if case['normalize'] else shares), index.contiguous()
    y = torch.matmul(s['shares'].double()[:, None], s['outputs'].double())[:, 0]
    return y if s['r'] is None else y + s['r'].double()
