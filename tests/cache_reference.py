"""A cache of keys and values in 4 or 8 bits from its definition, in 64 bits on the CPU, and attention over it with bounds on what rounding may take: the
oracle of test_gpu_cache*.py.

Bounds of attention.  w = 2^-23 is one step of 32 bits, u half a step of the results' type.  Every held value is exact as an operand.  Scores are sums
of D products in 32 bits in no fixed order (queries in two or three exact parts, so 3 D terms at most): |dz| <= (3 D + 4) w sum |q k| |scale|, plus 2 w |z| for the
scaling, plus 4 w of the power of two.  Powers enter the second product in two bfloat16 parts, each the nearest (2^-9 2^-9 = 2^-18 of a power is
lost), or three for 32-bit results (2^-27); their sum in 32 bits takes n w, the product's sum of up to 3 n terms 3 n w, joining shares 16 w."""
import numpy as np
import torch

from block_reference import U, W, visible

MAGNITUDES = {4: np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]),
              8: np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119])}
TOP = {4: 125, 8: 119}
LARGEST = {torch.float32: float(np.finfo(np.float32).max), torch.float16: 65504.0, torch.bfloat16: float(torch.finfo(torch.bfloat16).max)}


def quantise(x, bits):
    """(codes, scales) of (..., head_len) values as the cache holds them: uint8 arrays."""
    x = np.asarray(x, dtype=np.float64)
    groups = x.reshape(x.shape[:-1] + (-1, 32))
    finite = np.isfinite(groups).all(-1, keepdims=True)
    groups = np.where(finite, groups, 0.0)
    most = np.abs(groups).max(-1, keepdims=True)
    table = MAGNITUDES[bits]
    # what rounds to the step above the largest element: in 4 bits the border itself (the largest element's code is odd), in 8 only beyond it
    border = 7.0 if bits == 4 else 464.0
    e = np.full(most.shape, -127)
    for power in range(-126, TOP[bits] + 1):
        over = most >= np.ldexp(border, e) if bits == 4 else most > np.ldexp(border, e)
        e = np.where(over, power, e)
    y = np.ldexp(np.abs(groups), -e)
    above = np.clip(np.searchsorted(table, y), 1, len(table) - 1)
    low, high = table[above - 1], table[above]
    up = (y - low > high - y) | ((y - low == high - y) & (above % 2 == 0))
    code = np.where(up, above, above - 1)
    code = np.where(np.signbit(groups), code + (1 << (bits - 1)), code)
    code = np.where(finite, code, 0).reshape(x.shape).astype(np.uint8)
    if bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    scales = np.where(finite, e + 127, 255)[..., 0].astype(np.uint8)
    return code, scales


def values(codes, scales, bits):
    """(..., head_len) 64-bit values of codes and scales."""
    codes = np.asarray(codes)
    if bits == 4:
        codes = np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[:-1] + (-1,))
    table = np.append(MAGNITUDES[bits], np.nan) if bits == 8 else MAGNITUDES[bits]
    table = np.concatenate((table, -table))
    scale = np.where(np.asarray(scales) == 255, np.nan, np.ldexp(1.0, np.asarray(scales).astype(np.int64) - 127))
    return table[codes] * np.repeat(scale, 32, -1)


def held(cache):
    """(k, v) of a KeyValueCache, (batch, kv_heads, keys, head_len) in 64 bits."""
    return tuple(values(c.cpu().numpy(), s.cpu().numpy(), cache.bits) for c, s in ((cache.k, cache.k_scales), (cache.v, cache.v_scales)))


def as_type(x, dtype):
    """64-bit values as read_cache gives them."""
    x = torch.from_numpy(np.clip(x, -LARGEST[dtype], LARGEST[dtype]))
    return x.to(dtype)


def attention(q, k, v, blocks=None, block=None, scale=None, causal=True, lengths=None, q_lengths=None):
    """(out, bound): k and v (batch, kv_heads, keys, head_len) in 64 bits."""
    dtype = q.dtype
    u, lost = U[dtype], 2.0 ** -27 if dtype == torch.float32 else 2.0 ** -18
    qn = q.detach().cpu().double().numpy()
    B, N, H, D = qn.shape
    G, M = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    kl = [M] * B if lengths is None else [min(max(x, 0), M) for x in lengths.tolist()]
    ql = [N] * B if q_lengths is None else [min(max(x, 0), N) for x in q_lengths.tolist()]
    out, bound = np.zeros(qn.shape), np.zeros(qn.shape)
    if blocks is not None:
        blocks = blocks.cpu().numpy()
    for b in range(B):
        for g in range(G):
            if blocks is not None:
                seen = visible(blocks, b, g, N, M, block, causal, kl[b], ql[b])
            else:
                j, i = np.arange(M)[None], np.arange(N)[:, None]
                seen = (j < kl[b]) & (i < ql[b]) & ((j <= kl[b] - ql[b] + i) | (not causal))
            rows, cols = seen.any(1), seen.any(0)
            if not rows.any():
                continue
            s = seen[np.ix_(rows, cols)]
            K, V = k[b, g, cols], v[b, g, cols]
            for h in range(g * (H // G), (g + 1) * (H // G)):
                Q = qn[b, rows, h]
                z = np.where(s, Q @ K.T * scale, -np.inf)
                dz = (3 * D + 4) * W * abs(scale) * (np.abs(Q) @ np.abs(K).T)
                z = z - z.max(1, keepdims=True)
                dz = np.where(s, dz + 2 * W * np.where(s, np.abs(z), 0) + 4 * W, 0).max(1, keepdims=True)
                p = np.exp(z)
                p /= p.sum(1, keepdims=True)
                n = s.sum(1, keepdims=True)
                o = p @ V
                out[b, rows, h] = o
                bound[b, rows, h] = u * np.abs(o) + (lost + 2 * dz + (4 * n + 16) * W) * (p @ np.abs(V))
                if dtype == torch.float16:
                    bound[b, rows, h] += 2.0 ** -24
    return out, bound


def check(got, want, bound, what=""):
    x = got.detach().cpu().double().numpy()
    assert x.shape == want.shape, (what, x.shape, want.shape)
    assert np.isfinite(x).all(), (what, "not finite")
    over = np.abs(x - want) - bound
    if (over > 1e-30).any():
        i = np.unravel_index(np.argmax(over), over.shape)
        raise AssertionError("%s: %d of %d off; at %s got %r, expected %r, bound %g" % (what, (over > 1e-30).sum(), over.size, i, x[i], want[i], bound[i]))
