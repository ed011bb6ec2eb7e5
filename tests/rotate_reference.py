"""Heads normed and turned by position from the definition in 64 bits on the CPU, with bounds on what rounding may take: the oracle of
test_gpu_rotate.py.

Bounds.  w = 2^-23 is one step of 32 bits, u half a step of the results' type.  A head's mean square is a sum of D terms in no fixed order, D w of it, its root and
the products with it and the weight 6 w more: (D + 6) w of a normed element.  An angle is rounded to 32 bits as a fraction of a half-turn (pi w / 2), its sine and
cosine are off by 2 w more: 4 w of each of the two elements that are added, and 2 w for that: e = (D + 12) w of |a| + |b|.  The gradient of a normed element
is a difference of two terms, g and xh mean(g xh), the latter with another sum of D products: 2 e + (D + 6) w of their absolute sum."""
import numpy as np
import torch

from block_reference import U, W


def angles(shape, rotary_len, positions=None, lengths=None, q_lengths=None, base=10000.0, frequencies=None, sections=None):
    """(cos, sin) of (batch, tokens, 1, pairs) and which rows are there."""
    batch, tokens = shape[:2]
    pairs = rotary_len // 2
    count = [tokens] * batch if q_lengths is None else [min(max(int(x), 0), tokens) for x in q_lengths]
    there = np.arange(tokens)[None] < np.array(count).reshape(-1, 1)
    if positions is not None:
        where = np.asarray(positions, dtype=np.float64).reshape(batch, tokens, -1)
    else:
        start = np.zeros(batch) if lengths is None else np.asarray(lengths, dtype=np.float64) - count
        where = (start.reshape(-1, 1) + np.arange(tokens)[None])[:, :, None]
    axis = np.repeat(np.arange(where.shape[2]), (pairs,) if sections is None else sections)
    if frequencies is None:
        frequencies = [base ** (-i / max(pairs, 1)) for i in range(pairs)]
    t = where[:, :, axis] * np.asarray(frequencies, dtype=np.float64).reshape(-1)
    return np.cos(t)[:, :, None], np.sin(t)[:, :, None], there[:, :, None, None]


def split(x, rotary_len, interleaved):
    half = rotary_len // 2
    return (x[..., 0:rotary_len:2], x[..., 1:rotary_len:2]) if interleaved else (x[..., :half], x[..., half:rotary_len])


def turned(x, cos, sin, rotary_len, interleaved):
    out = np.array(x, dtype=np.float64)
    a, b = (t.copy() for t in split(out, rotary_len, interleaved))
    x, y = split(out, rotary_len, interleaved)
    x[...], y[...] = a * cos - b * sin, a * sin + b * cos
    return out


def both(x, rotary_len, interleaved):
    """|a| + |b| for the elements of a pair, |x| for the others."""
    out = np.abs(x)
    a, b = (t.copy() for t in split(out, rotary_len, interleaved))
    p, q = split(out, rotary_len, interleaved)
    p[...] = q[...] = a + b
    return out


def rotate(x, weight, cos, sin, there, rotary_len, interleaved=False, eps=1e-6, dout=None, dtype=None):
    """{"y", "dx", "dw": (value, bound)} of one side; x and dout (batch, tokens, heads, head_len)."""
    dtype = x.dtype if dtype is None else dtype
    u = U[dtype]
    f = lambda t: None if t is None else t.detach().cpu().double().numpy()
    x, weight, dout = f(x), f(weight), f(dout)
    x = np.where(there, x, 0.0)
    D = x.shape[-1]
    e = (D + 12) * W
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    xh, inverse = x, 1.0
    if weight is not None:
        inverse = np.where(there, 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps), 0.0)
        xh = x * inverse
    y = xh if weight is None else xh * weight
    out = turned(y, cos, sin, rotary_len, interleaved)
    got = {"y": (out, u * np.abs(out) + e * both(y, rotary_len, interleaved) + tiny)}
    if dout is None:
        return got
    dout = np.where(there, dout, 0.0)
    dy = turned(dout, cos, -sin, rotary_len, interleaved)
    size = both(dout, rotary_len, interleaved)
    if weight is None:
        got["dx"] = dy, u * np.abs(dy) + e * size + tiny
        return got
    rows = x.size // D
    dw = (dy * xh).sum((0, 1, 2))
    got["dw"] = dw, u * np.abs(dw) + (2 * e + rows * W) * (size * np.abs(xh)).sum((0, 1, 2)) + tiny
    g = dy * weight
    dot = (g * xh).mean(-1, keepdims=True)
    dx = (g - xh * dot) * inverse
    most = size * np.abs(weight)
    got["dx"] = dx, u * np.abs(dx) + (2 * e + (D + 6) * W) * (most + np.abs(xh) * (most * np.abs(xh)).mean(-1, keepdims=True)) * inverse + tiny
    return got


def check(got, want, what=""):
    """A tensor against (value, bound)."""
    value, bound = want
    x = got.detach().cpu().double().numpy()
    assert x.shape == value.shape, (what, x.shape, value.shape)
    assert np.isfinite(x).all(), (what, "not finite")
    over = np.abs(x - value) - bound
    if (over > 1e-30).any():
        i = np.unravel_index(np.argmax(over), over.shape)
        raise AssertionError("%s: %d of %d off; at %s got %r, expected %r, bound %g" % (what, (over > 1e-30).sum(), over.size, i, x[i], value[i], bound[i]))
