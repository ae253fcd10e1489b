"""Microscaled 4-bit operators in 64 bits, from their definition: test infrastructure only."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def blocks_of(width):
    return -(-width // BLOCK)


def quantize(x):
    """(codes uint8 [R, 16 nb], scales uint8 [R, nb]) of float64 x [R, W]."""
    rows, width = x.shape
    nb = blocks_of(width)
    v = np.zeros((rows, nb * BLOCK))
    v[:, :width] = x
    v = v.reshape(rows, nb, BLOCK)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    largest = np.abs(v).max(-1)
    _, above = np.frexp(largest)                       # largest = m 2^above, 1/2 <= m < 1
    e = np.where(largest > 0, np.maximum(above - 1 - 2, -127), -127)
    scaled = np.ldexp(np.abs(v), -e[..., None])
    code = np.zeros(v.shape, dtype=np.uint8)
    for i in range(7):                                 # up at the middle where the lower code is odd
        middle = (GRID[i] + GRID[i + 1]) / 2
        code += ((scaled > middle) | ((scaled == middle) & (i % 2 == 1))).astype(np.uint8)
    code |= np.where(np.signbit(v), 8, 0).astype(np.uint8)
    code[bad] = 0
    codes = (code[..., 0::2] | (code[..., 1::2] << 4)).reshape(rows, nb * 16)
    return codes, np.where(bad, 255, e + 127).astype(np.uint8)


def dequantize(codes, scales, width):
    """float64 [.., W]"""
    value = np.concatenate((GRID, -GRID))
    both = np.stack((value[codes & 15], value[codes >> 4]), axis=-1)
    v = both.reshape(scales.shape + (BLOCK,))
    e = scales.astype(np.int64) - 127
    with np.errstate(invalid='ignore'):
        v = np.where((scales == 255)[..., None], np.nan, np.ldexp(v, e[..., None]))
    return v.reshape(scales.shape[:-1] + (-1,))[..., :width]


def product_bound(x, w, values_off=0.0):
    """How far a bf16 result of x w^T may be from the value in 64 bits: half a step of bf16, and the
    fp32 sum, whose every step is off by half a step of fp32 (twice that, as the matrix cores' order and
    rounding are their own) of what has been added up so far."""
    exact = x @ w.T
    sums = np.abs(x) @ np.abs(w).T
    off = values_off + (x.shape[1] + 2) * 2.0 ** -23 * sums
    return exact, off + 2.0 ** -8 * (np.abs(exact) + off) + 2.0 ** -133


def route(logits, top_k):
    """int64 [T, k]: the largest first, of equal ones the lower index, what is no number last."""
    key = np.where(np.isnan(logits), -np.inf, logits)
    order = np.lexsort((np.arange(logits.shape[1])[None, :] + np.zeros_like(key), np.isnan(logits), -key), axis=-1)
    return order[:, :top_k]


def sparse_mlp(x, router, wi, wo, top_k, normalize, capacity, length):
    """(y, how far y may be off, logits as fp32, index): x [T, D], router [E, D], wi [E, F, D], wo [E, D, F]
    in float64."""
    tokens = x.shape[0]
    logits = (x @ router.T).astype(np.float32)
    index = route(logits, top_k)
    with np.errstate(invalid='ignore', over='ignore'):
        most = logits.astype(np.float64).max(-1, keepdims=True)
        p = np.exp(logits.astype(np.float64) - most)
        p = np.take_along_axis(p / p.sum(-1, keepdims=True), index, -1)
    if normalize:
        p = p / p.sum(-1, keepdims=True)
    # exp, the sum over the experts and two quotients in fp32
    p_off = (router.shape[0] + 16) * 2.0 ** -23
    y, off = np.zeros_like(x), np.zeros_like(x)
    for t in range(tokens):
        for j in range(top_k):
            e = index[t, j]
            before = sum(index[u, 0] == e for u in range(t - t % length, t)) if capacity else 0
            if capacity and before >= capacity:
                out, out_off = x[t], 0.0
            else:
                with np.errstate(invalid='ignore'):
                    h, h_off = product_bound(x[t][None], wi[e])
                    h, h_off = np.maximum(h, 0), np.where(h < -h_off, 0, h_off)
                    out = wo[e] @ h[0]
                    out_off = np.abs(wo[e]) @ h_off[0]
                    out_off = out_off + (wo.shape[2] + 2) * 2.0 ** -23 * (np.abs(wo[e]) @ (h + h_off)[0])
            with np.errstate(invalid='ignore'):
                y[t] += p[t, j] * out
                off[t] += p[t, j] * (out_off + p_off * (np.abs(out) + out_off))
    with np.errstate(invalid='ignore'):
        off = off + top_k * 2.0 ** -23 * (np.abs(y) + off)
        return y, off + 2.0 ** -8 * (np.abs(y) + off) + 2.0 ** -133, logits, index
