"""Attention over selected blocks from its definition in 64 bits on the CPU, with bounds on what rounding may take: the oracle of
test_gpu_block_*.py.

Bounds.  u is the largest relative error of one rounding to the type (half a step), w = 2^-23 one step of 32 bits.  Scores are sums of D products
in 32 bits, whose order is not fixed: |dz| <= (D + 4) w sum |q k| |scale|, plus w |z| for the scaling and the power of two, whose own error is
below 4 w.  Probabilities are off by a factor e^dz and, where they are an operand of the second product in 16 bits, by u; a sum of n
terms adds n w of their absolute sum.  Results are rounded once more, u of their value."""
import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -24}
W = 2.0 ** -23


def visible(blocks, b, g, queries, keys, block, causal, k_len, q_len):
    """(queries, keys) booleans of one sequence and key head."""
    nb = -(-keys // block)
    chosen = np.zeros((queries, nb), dtype=bool)
    for i in range(q_len):
        for x in blocks[b, i, g]:
            if 0 <= x < nb:
                chosen[i, x] = True
    seen = np.repeat(chosen, block, axis=1)[:, :keys]
    j = np.arange(keys)
    seen &= j < k_len
    if causal:
        seen &= j[None] <= (k_len - q_len + np.arange(queries))[:, None]
    return seen


def attention(q, k, v, blocks, block, scale=None, causal=True, lengths=None, q_lengths=None, bias=None, bounds=None, dout=None):
    """{name: (value, bound on the kernel's error)} for out, and with dout for dq, dk, dv and dbias.  Tensors as ops.block_attention takes them."""
    dtype = q.dtype
    u, half = U[dtype], (0.0 if dtype == torch.float32 else U[dtype])         # half: operands of second products that are rounded
    f = lambda t: None if t is None else t.detach().cpu().double().numpy()
    qn, kn, vn, dn, bn = f(q), f(k), f(v), f(dout), f(bias)
    blocks = blocks.cpu().numpy()
    B, N, H, D = qn.shape
    M, G = kn.shape[1], kn.shape[2]
    scale = D ** -0.5 if scale is None else scale
    kl = [M] * B if lengths is None else [min(max(x, 0), M) for x in lengths.tolist()]
    ql = [N] * B if q_lengths is None else [min(max(x, 0), N) for x in q_lengths.tolist()]
    names = ["out"] + (["dq", "dk", "dv"] if dout is not None else []) + (["dbias"] if dout is not None and bias is not None else [])
    shapes = {"out": qn.shape, "dq": qn.shape, "dk": kn.shape, "dv": kn.shape, "dbias": None if bn is None else bn.shape}
    val = {n: np.zeros(shapes[n]) for n in names}
    tol = {n: np.zeros(shapes[n]) for n in names}
    for b in range(B):
        distance = (kl[b] - ql[b] + np.arange(N))[:, None] - np.arange(M)[None]
        bucket = None if bn is None else np.searchsorted(np.asarray(bounds, dtype=np.int64), distance, side="right")
        for h in range(H):
            g = h // (H // G)
            seen = visible(blocks, b, g, N, M, block, causal, kl[b], ql[b])
            rows, cols = seen.any(1), seen.any(0)
            if not rows.any():
                continue
            s = seen[np.ix_(rows, cols)]
            Q, K, V = qn[b, rows, h], kn[b, cols, g], vn[b, cols, g]
            z = Q @ K.T * scale
            add = 0.0 if bn is None else bn[bucket[np.ix_(rows, cols)], h]
            z = np.where(s, z + add, -np.inf)
            z = z - z.max(1, keepdims=True)
            p = np.exp(z)
            p /= p.sum(1, keepdims=True)
            n = s.sum(1, keepdims=True)
            dz = (D + 4) * W * abs(scale) * (np.abs(Q) @ np.abs(K).T) + 2 * W * (np.where(s, np.abs(z), 0) + np.abs(add)) + 4 * W
            dz = np.where(s, dz, 0).max(1, keepdims=True)                   # of the row: its sum and maximum carry them too
            o = p @ V
            mass = p @ np.abs(V)
            ep = half + 2 * dz + (n + 8) * W                                # relative error of a probability as an operand
            eo = ep * mass
            val["out"][b, rows, h] = o
            tol["out"][b, rows, h] = u * np.abs(o) + eo
            if dn is None:
                continue
            d = dn[b, rows, h]
            val["dv"][b, cols, g] += p.T @ d
            tol["dv"][b, cols, g] += (p * (ep + len(d) * W)).T @ np.abs(d)
            dp = d @ V.T
            delta = (p * dp).sum(1, keepdims=True)
            ds = p * (dp - delta)
            # delta comes from the rounded output and (in 16 bits) its rounded remainder
            edelta = ((np.abs(d) * (eo + max(u * u, W) * np.abs(o))).sum(1, keepdims=True) + D * W * (np.abs(d) * np.abs(o)).sum(1, keepdims=True))
            edp = D * W * (np.abs(d) @ np.abs(V).T)
            eds = p * (edp + edelta) + np.abs(ds) * (half + 2 * dz + 8 * W)
            val["dq"][b, rows, h] = ds @ K * scale
            tol["dq"][b, rows, h] = ((eds + n * W * np.abs(ds)) @ np.abs(K)) * abs(scale)
            val["dk"][b, cols, g] += ds.T @ Q * scale
            tol["dk"][b, cols, g] += ((eds + len(d) * W * np.abs(ds)).T @ np.abs(Q)) * abs(scale)
            if bn is not None:
                where = bucket[np.ix_(rows, cols)][s]
                val["dbias"][:, h] += np.bincount(where, ds[s], len(bn))
                tol["dbias"][:, h] += np.bincount(where, (p * (edp + edelta) + np.abs(ds) * (2 * dz + 8 * W + s.sum() * W))[s], len(bn))
    for x in names:
        if x != "out":
            tol[x] += u * np.abs(val[x])
        if dtype == torch.float16:
            tol[x] += 2.0 ** -24                                            # what falls below the type's normal numbers
    return {x: (val[x], tol[x]) for x in names}


def check(got, want, what=""):
    """got {name: tensor} against attention()'s answer."""
    for name, t in got.items():
        value, bound = want[name]
        x = t.detach().cpu().double().numpy()
        assert x.shape == value.shape, (what, name, x.shape, value.shape)
        assert np.isfinite(x).all(), (what, name, "not finite")
        over = np.abs(x - value) - bound
        if (over > 1e-30).any():
            i = np.unravel_index(np.argmax(over), over.shape)
            raise AssertionError("%s %s: %d of %d off; at %s got %r, expected %r, bound %g" % (what, name, (over > 1e-30).sum(), over.size, i, x[i], value[i], bound[i]))


def selection(q, pooled, num_keys, block, topk, causal, lengths, q_lengths, keep_first, keep_last):
    """ops.select_blocks by sorting exact scores."""
    B, N, H, D = q.shape
    G, nb = pooled.shape[1], pooled.shape[2]
    out = np.full((B, N, G, topk), -1, dtype=np.int32)
    means = pooled.cpu().double().numpy()
    summed = q.cpu().double().view(B, N, G, -1, D).sum(3).float().to(q.dtype).double().numpy()
    for b in range(B):
        k_len = num_keys if lengths is None else min(max(int(lengths[b]), 0), num_keys)
        q_len = N if q_lengths is None else min(max(int(q_lengths[b]), 0), N)
        for i in range(q_len):
            last = min(k_len - q_len + i, k_len - 1) if causal else k_len - 1
            n = last // block + 1 if last >= 0 else 0
            for g in range(G):
                score = means[b, g, :n] @ summed[b, i, g]
                score = np.where(np.isnan(score), -np.inf, score)
                kept = (np.arange(n) < keep_first) | (np.arange(n) >= n - keep_last)
                order = sorted(range(n), key=lambda x: (not kept[x], -score[x], x))[:topk]
                out[b, i, g, :len(order)] = sorted(order)
    return out
