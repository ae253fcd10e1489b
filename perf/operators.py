"""The operators on microscaled 4-bit floats, as measurable cases.

The format: blocks of 32 values along the last dimension, each value one of
0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, each block with a power of two as its scale.
Four paths:

  quantize   values to the format and back
  product    activations (bf16) times a matrix held in the format
  product4   the same, the activations quantised in the call too
  moe        a whole mixture-of-experts layer for a few tokens: router, choice of
             experts, their two products with ReLU between, weighted sum

Matrix sizes are the larger Switch shapes of qmoe_amd.synthetic.SHAPES (wi is [d_ff,
d_model], wo [d_model, d_ff]) and odd ones between them, weights N(0, 1 / width),
activations N(0, 1).

`own` chooses who computes: the elementary operations below, or the package.
"""
import math

import torch

own = False

DEVICE = 'cuda:0'
BLOCK = 32
LARGE, C2048 = (1024, 4096), (2080, 6144)      # (d_model, d_ff)
TYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def listed():
    return [
        # generation: the activations of one token on their way into a 4-bit product
        dict(name='quantize_one_row', kind='quantize', rows=1, width=2080, dtype='bf16', strided=False),
        # a part of each row of a wider tensor, odd sizes
        dict(name='quantize_ragged', kind='quantize', rows=61, width=1023, dtype='fp16', strided=True),
        # storing: 24 matrices of a layer at once
        dict(name='quantize_weights', kind='quantize', rows=24576, width=4096, dtype='bf16', strided=False),
        # generation, batch 1: one token through the largest wo
        dict(name='product_one_token', kind='product', tokens=1, height=2080, width=6144, strided=False),
        # a small, odd batch through a matrix of odd sizes
        dict(name='product_few_ragged', kind='product', tokens=13, height=3001, width=1023, strided=True),
        # one sequence of the length the projections are timed with
        dict(name='product_sequence', kind='product', tokens=568, height=4096, width=1024, strided=False),
        # a long one through the largest wi
        dict(name='product_long', kind='product', tokens=2272, height=6144, width=2080, strided=False),
        # a batch that generates together, activations in 4 bits too
        dict(name='product4_batch', kind='product4', tokens=61, height=2080, width=6144, strided=False),
        # encoding sixteen sequences of 512 tokens
        dict(name='product4_sequences', kind='product4', tokens=8192, height=6144, width=2080, strided=False),
        # generation, batch 1: one token through a slice of the largest layer
        dict(name='moe_one_token', kind='moe', d_model=2080, d_ff=6144, experts=64, sequences=1, length=1,
             top_k=1, normalize=False, capacity=0, router='fp32'),
        # a small, odd batch, two experts a token
        dict(name='moe_few_tokens', kind='moe', d_model=1024, d_ff=4096, experts=128, sequences=13, length=1,
             top_k=2, normalize=True, capacity=0, router='bf16'),
        # four short sequences through a Switch layer of odd sizes, at most two tokens of a
        # sequence to an expert
        dict(name='moe_sequences', kind='moe', d_model=1000, d_ff=2501, experts=32, sequences=4, length=16,
             top_k=1, normalize=False, capacity=2, router='fp32'),
    ]


def draw(rng):
    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    def sides():
        if rng.random() < 0.4:
            pair = rng.choice([LARGE, C2048])
        else:
            pair = rng.randint(500, 2080), rng.randint(2000, 6144)
        return pair

    kind = rng.choice(['quantize', 'product', 'product', 'product4', 'moe', 'moe'])
    if kind == 'quantize':
        width = log(1, 6144)
        rows = log(1, max(1, min(24576, 24576 * 4096 // width)))
        return dict(kind=kind, rows=rows, width=width, dtype=rng.choice(sorted(TYPES)),
                    strided=rng.random() < 0.3)
    d_model, d_ff = sides()
    if kind != 'moe':
        height, width = rng.choice([(d_ff, d_model), (d_model, d_ff)])
        return dict(kind=kind, tokens=log(1, 2272 if kind == 'product' else 8192), height=height, width=width,
                    strided=rng.random() < 0.3)
    experts = log(4, max(4, min(256, 2 ** 30 // (2 * d_model * d_ff))))
    sequences, length = log(1, 16), log(1, 8)
    top_k = rng.choice([1, 1, 2, 4])
    # no more work than thirteen tokens through two experts each, sixty-four through one of odd sizes
    most = max(1, 26 * 2 * 1024 * 4096 // (2 * d_model * d_ff))
    while sequences * length * top_k > most:
        if top_k > 1:
            top_k //= 2
        elif length > 1:
            length -= 1
        else:
            sequences -= 1
    return dict(kind=kind, d_model=d_model, d_ff=d_ff, experts=experts, sequences=sequences, length=length,
                top_k=top_k, normalize=top_k > 1 and rng.random() < 0.5,
                capacity=rng.choice([0, 1, 3]) if top_k == 1 else 0, router=rng.choice(['bf16', 'fp32']))


# ---------------------------------------------------- the format, plainly ---

def _quantize(x):
    """(magnitudes with sign as fp32 [.., nb, 32], exponents int32 [.., nb, 1], whether finite) of x [.., W]."""
    width = x.shape[-1]
    blocks = (width + BLOCK - 1) // BLOCK
    v = torch.zeros(x.shape[:-1] + (blocks * BLOCK,), dtype=torch.float32, device=x.device)
    v[..., :width] = x
    v = v.view(x.shape[:-1] + (blocks, BLOCK))
    largest = v.abs().amax(dim=-1, keepdim=True)
    # floor(log2): the exponent field; below the normal numbers anything small does, as -127 is the least
    exponent = ((largest.view(torch.int32) >> 23) - 127 - 2).clamp(min=-127)
    fine = torch.isfinite(largest)
    scaled = torch.where(fine, v, torch.zeros_like(v)) * _power(-exponent)
    a = scaled.abs()
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float())
    q += (a > 2.5).float() + (a >= 3.5).float() + 2 * (a > 5).float()
    return torch.where(scaled < 0, -q, q), exponent, fine


def _power(exponent):
    """2^exponent as fp32, exactly, for -127 to 127."""
    half = torch.div(exponent, 2, rounding_mode='floor')
    return ((half + 127) << 23).view(torch.float32) * ((exponent - half + 127) << 23).view(torch.float32)


def _store(x):
    """(codes uint8 [.., 16 nb], scales uint8 [.., nb]): the low half of byte i holds value 2 i."""
    q, exponent, fine = _quantize(x)
    a = q.abs()
    code = (2 * a - (a - 2).clamp(min=0) - 0.5 * (a - 4).clamp(min=0)).to(torch.uint8)      # 0 .. 7
    code += 8 * (q < 0).to(torch.uint8)
    codes = (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-2)
    scales = torch.where(fine, exponent + 127, torch.full_like(exponent, 255)).to(torch.uint8)
    return codes, scales.squeeze(-1)


def _load(codes, scales, width):
    """fp32 [.., W]"""
    code = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    m = (code & 7).float()
    value = 0.5 * m + 0.5 * (m - 4).clamp(min=0) + (m - 6).clamp(min=0)
    value = torch.where(code >= 8, -value, value)
    scale = _power(scales.to(torch.int32) - 127)
    return (value.view(scales.shape + (BLOCK,)) * scale[..., None]).flatten(-2)[..., :width]


# ------------------------------------------------------------- preparing ---

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _rows(rows, width, dtype, strided, g):
    """[rows, width], a part of wider rows where strided"""
    if not strided:
        return torch.randn((rows, width), generator=g, device=DEVICE).to(dtype)
    whole = torch.randn((rows, width + 37), generator=g, device=DEVICE).to(dtype)
    return whole[:, 5:5 + width]


def _matrices(count, height, width, g):
    """(codes [count, height, 16 nb], scales [count, height, nb]) of normal weights"""
    parts = []
    step = max(1, (1 << 26) // (height * width))
    for first in range(0, count, step):
        w = torch.randn((min(step, count - first), height, width), generator=g, device=DEVICE)
        parts.append(_store(w / width ** 0.5))
    return torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])


def prepare(case, seed):
    g = _generator(1000 * seed + 17)
    kind = case['kind']
    if kind == 'quantize':
        x = _rows(case['rows'], case['width'], TYPES[case['dtype']], case['strided'], g)
        # blocks of very different sizes, as outlying channels make them
        x *= torch.exp2(4 * torch.randn((1, case['width']), generator=g, device=DEVICE)).to(x.dtype).clamp(max=64)
        return dict(kind=kind, x=x, width=case['width'])
    if kind in ('product', 'product4'):
        codes, scales = _matrices(1, case['height'], case['width'], g)
        state = dict(kind=kind, codes=codes[0], scales=scales[0], width=case['width'],
                     x=_rows(case['tokens'], case['width'], torch.bfloat16, case['strided'], g))
        if own:
            from qmoe_amd import mx4
            state['layer'] = mx4.Mx4Linear(state['codes'], state['scales'], case['width'],
                                           quantize_activations=kind == 'product4')
        return state
    d_model, d_ff, experts = case['d_model'], case['d_ff'], case['experts']
    router = torch.randn((experts, d_model), generator=g, device=DEVICE) / d_model ** 0.5
    state = dict(kind=kind, d_model=d_model, d_ff=d_ff, top_k=case['top_k'], normalize=case['normalize'],
                 capacity=case['capacity'], router=router.to(TYPES[case['router']]),
                 wi=_matrices(experts, d_ff, d_model, g), wo=_matrices(experts, d_model, d_ff, g))
    hidden = torch.randn((case['sequences'], case['length'], d_model), generator=g, device=DEVICE)
    state['hidden'] = hidden.bfloat16()
    if own:
        from qmoe_amd import mx4
        state['layer'] = mx4.Mx4SparseMLP(state['router'], state['wi'], state['wo'], top_k=case['top_k'],
                                          normalize=case['normalize'], capacity=case['capacity'] or None)
    return state


# --------------------------------------------------------------- running ---

def run(state):
    with torch.no_grad():
        if own:
            return _run_own(state)
        return _run_plain(state)


def _run_own(state):
    from qmoe_amd import mx4
    if state['kind'] == 'quantize':
        codes, scales = mx4.quantize(state['x'])
        return mx4.dequantize(codes, scales, state['width'], state['x'].dtype)
    if state['kind'] == 'moe':
        hidden, (logits, index) = state['layer'](state['hidden'])
        return hidden, logits, index
    return state['layer'](state['x'])


def _values(x):
    """fp32: what the format keeps of x"""
    q, exponent, fine = _quantize(x)
    value = torch.where(fine, q * _power(exponent), torch.full_like(q, math.nan))
    return value.flatten(-2)[..., :x.shape[-1]]


def _run_plain(state):
    kind = state['kind']
    if kind == 'quantize':
        return _values(state['x']).to(state['x'].dtype)
    if kind in ('product', 'product4'):
        x = state['x'].float() if kind == 'product' else _values(state['x'])
        return (x @ _load(state['codes'], state['scales'], state['width']).t()).bfloat16()
    return _moe_plain(state)


def _moe_plain(state):
    hidden, top_k = state['hidden'], state['top_k']
    x = hidden.flatten(0, 1)
    # in 64 bits: which of two close logits is larger decides
    logits = (x.double() @ state['router'].double().t()).float()
    left, chosen = logits.clone(), []
    for _ in range(top_k):
        best = left.amax(dim=-1, keepdim=True)
        first = (left == best).int().argmax(dim=-1, keepdim=True)       # the lowest index of equals
        chosen.append(first)
        left.scatter_(-1, first, -math.inf)
    index = torch.cat(chosen, dim=-1)
    shifted = torch.exp(logits - logits.amax(dim=-1, keepdim=True))
    p = torch.gather(shifted / shifted.sum(dim=-1, keepdim=True), -1, index)
    if state['normalize']:
        p = p / p.sum(dim=-1, keepdim=True)
    expert = index.flatten()
    pair_x = x.float().repeat_interleave(top_k, dim=0)
    out = torch.empty((expert.numel(), state['d_model']), dtype=torch.float32, device=x.device)
    for first in range(0, expert.numel(), 4):
        which = slice(first, first + 4)
        e = expert[which]
        wi = _load(state['wi'][0][e], state['wi'][1][e], state['d_model'])
        h = (wi * pair_x[which, None]).sum(dim=-1).clamp(min=0)
        del wi
        wo = _load(state['wo'][0][e], state['wo'][1][e], state['d_ff'])
        out[which] = (wo * h[:, None]).sum(dim=-1)
        del wo
    if state['capacity']:
        of = index.view(hidden.shape[:2])
        rank = ((of[:, :, None] == of[:, None, :]).int().tril()).sum(dim=-1)       # its place among its expert's
        out = torch.where(rank.view(-1, 1) > state['capacity'], x.float(), out)
    y = (p[:, :, None] * out.view(-1, top_k, state['d_model'])).sum(dim=1)
    return y.bfloat16().view(hidden.shape), logits.view(hidden.shape[:2] + (-1,)), index.view(hidden.shape[:2] + (-1,))


# --------------------------------------------- what it needs, and the truth ---

def _stored(height, width):
    return height * ((width + BLOCK - 1) // BLOCK) * 17


def work(case):
    kind = case['kind']
    if kind == 'quantize':
        n, size = case['rows'] * case['width'], TYPES[case['dtype']].itemsize
        # written and read back
        return dict(bytes=2 * n * size + 2 * _stored(case['rows'], case['width']), flops=0)
    if kind in ('product', 'product4'):
        t, h, w = case['tokens'], case['height'], case['width']
        return dict(bytes=_stored(h, w) + 2 * t * (h + w), flops=2 * t * h * w)
    d_model, d_ff, experts = case['d_model'], case['d_ff'], case['experts']
    tokens = case['sequences'] * case['length']
    pairs = tokens * case['top_k']
    # the experts that some token goes to, on average, are read once each
    hit = experts * (1 - (1 - case['top_k'] / experts) ** tokens)
    expert = _stored(d_ff, d_model) + _stored(d_model, d_ff)
    bytes_ = hit * expert + experts * d_model * TYPES[case['router']].itemsize
    bytes_ += tokens * (4 * d_model + 4 * experts + 8 * case['top_k'])
    return dict(bytes=bytes_, flops=4 * pairs * d_model * d_ff + 2 * tokens * experts * d_model)


_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _scaled(x, power):
    """float64 x 2^power for powers of -127 to 128, exactly (torch's ldexp goes through a 32-bit pow)"""
    table = torch.tensor([2.0 ** p for p in range(-127, 129)], dtype=torch.float64, device=x.device)
    return x * table[power.long() + 127]


def _nearest(x):
    """float64: x in the format, by the nearest of its values (of two the one with an even code)."""
    width = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -width % BLOCK)).unflatten(-1, (-1, BLOCK))
    largest = x.abs().amax(-1, keepdim=True)
    _, above = torch.frexp(largest)                         # largest = m 2^above, 1/2 <= m < 1
    power = torch.where(largest > 0, above - 1 - 2, torch.full_like(above, -127)).clamp(-127, 127)
    scaled = _scaled(x, -power)
    grid = torch.tensor(_GRID, dtype=torch.float64, device=x.device)
    at = torch.bucketize(scaled.abs(), (grid[1:] + grid[:-1]) / 2)          # below or at the middle: the lower
    middle = torch.zeros_like(scaled, dtype=torch.bool)
    for low in (1, 3, 5):                                   # an odd code gives way
        middle |= scaled.abs() == (_GRID[low] + _GRID[low + 1]) / 2
    at += middle.long()
    value = _scaled(torch.copysign(grid[at], scaled), power)
    return torch.where(torch.isfinite(largest), value, math.nan).flatten(-2)[..., :width]


def _expanded(codes, scales, width):
    """float64 by table"""
    table = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float64, device=codes.device)
    value = torch.empty(codes.shape + (2,), dtype=torch.float64, device=codes.device)
    value[..., 0] = table[(codes % 16).long()]
    value[..., 1] = table[(codes // 16).long()]
    value = value.flatten(-2).unflatten(-1, (-1, BLOCK))
    return _scaled(value, scales[..., None].to(torch.int32) - 127).flatten(-2)[..., :width]


def exact(case, seed):
    state = prepare(case, seed)
    kind = case['kind']
    if kind == 'quantize':
        return torch.cat([_nearest(part) for part in state['x'].split(2048)])
    if kind in ('product', 'product4'):
        x = state['x'].double() if kind == 'product' else _nearest(state['x'])
        return torch.matmul(x, _expanded(state['codes'], state['scales'], case['width']).transpose(0, 1))
    hidden = state['hidden'].double()
    logits = torch.einsum('bsd,ed->bse', hidden, state['router'].double())
    order = torch.argsort(logits.float(), dim=-1, descending=True, stable=True)
    index = order[..., :case['top_k']].contiguous()
    p = torch.softmax(logits, dim=-1).gather(-1, index)
    if case['normalize']:
        p = p / p.sum(-1, keepdim=True)
    y = torch.zeros_like(hidden)
    for b in range(case['sequences']):
        taken = {}
        for s in range(case['length']):
            for j in range(case['top_k']):
                e = int(index[b, s, j])
                taken[e] = taken.get(e, 0) + 1
                if case['capacity'] and taken[e] > case['capacity']:
                    out = hidden[b, s]
                else:
                    wi = _expanded(state['wi'][0][e], state['wi'][1][e], case['d_model'])
                    wo = _expanded(state['wo'][0][e], state['wo'][1][e], case['d_ff'])
                    out = torch.mv(wo, torch.relu(torch.mv(wi, hidden[b, s])))
                y[b, s] += p[b, s, j] * out
    return y, logits, index
