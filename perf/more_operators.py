"""What stands around attention in a serving program and in training: queries and keys normed and rotated, and a cache of keys and values in 4 or
8 bits with the attention that reads it.  The work a user has these operators do, as cases that can be timed and compared.

  rotate   the RMS norm of every head of q and k and the rotation by position, of one or several axes, in one pass; forward, and with its
           gradients (ops.rotate_heads)
  store    new tokens' keys and values quantised into a cache, and a window of it read back (ops.write_cache, ops.read_cache)
  attend   softmax attention of a few queries over such a cache, whole or the blocks that a list names (ops.cache_attention)

q is (batch, tokens, heads, head_len), k and v (batch, tokens, kv_heads, head_len), slices of one fused projection.  A cache holds
(batch, kv_heads, keys, head_len) elements of 4 bits (sign, two bits of exponent, one of mantissa; the lower half of a byte first) or 8 (e4m3),
and for every 32 of them a power of two, as its exponent plus 127: the least with which the largest of them rounds to no more than
the largest element.  A sequence's last new token stands at its last key.

In their plain form the operators are elementary torch operations in 32 bits, angles and long sums in 64; `exact` computes them from their
definition in 64 bits.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6
# magnitudes of the elements, in the order of their codes
_MAGNITUDES = {4: [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
               8: [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119]}
_TOP_EXPONENT = {4: 125, 8: 119}            # with a larger power the largest element would leave the range of 32 bits


def listed():
    layer = dict(heads=32, kv_heads=8, head_len=128)
    turn = dict(op="rotate", train=False, norm=True, rotary_len=128, axes=1, interleaved=False, ragged=False, base=500000.0)
    store = dict(op="store", kv_heads=8, head_len=128, bits=4, ragged=False)
    attend = dict(op="attend", bits=4, block=0, topk=0, ragged=False, **layer)
    return [
        # all tokens of a long prompt
        dict(name="rotate_16k", dtype="bf16", batch=1, tokens=16384, past=0, **dict(turn, **layer)),
        # one new token for each of many requests, at far and unequal positions: latency
        dict(name="rotate_token_32", dtype="bf16", batch=32, tokens=1, past=32768, **dict(turn, **layer, ragged=True)),
        # a training step, both directions
        dict(name="rotate_train_2x4k", dtype="bf16", batch=2, tokens=4096, past=0, **dict(turn, heads=16, kv_heads=4, head_len=128, train=True)),
        # video in 32 bits: time, height and width, neighbouring elements turned, a part of each head as it is, both directions
        dict(name="rotate_train_video_f32", dtype="f32", batch=3, tokens=1237, past=0, heads=6, kv_heads=2, head_len=64,
             **dict(turn, train=True, rotary_len=48, axes=3, interleaved=True, base=10000.0)),
        # a prompt's keys and values go into a cache of 4 bits, and come back as later tokens will see them
        dict(name="store_16k", dtype="bf16", batch=1, tokens=16384, keys=16384, window=16384, **store),
        # one new token for each of many requests; its block of 64 keys comes back for the block's mean
        dict(name="store_token_32x32k", dtype="bf16", batch=32, tokens=1, keys=32768, window=64, **dict(store, ragged=True)),
        # a padded batch of odd lengths behind what is there, in 32 and 8 bits
        dict(name="store_odd_f32", dtype="f32", batch=3, tokens=1237, keys=5000, window=1500, **dict(store, kv_heads=2, head_len=64, bits=8, ragged=True)),
        # one new token for each of many requests over long caches
        dict(name="attend_token_32x32k", dtype="bf16", batch=32, queries=1, keys=32768, **attend),
        # one new token of one request: latency
        dict(name="attend_token_1x2k", dtype="f16", batch=1, queries=1, keys=2048, **dict(attend, heads=8, kv_heads=8, head_len=64, bits=8)),
        # three drafted tokens for each of eight requests of unequal lengths, over the blocks that they selected
        dict(name="attend_blocks_8x5000", dtype="bf16", batch=8, queries=3, keys=5000, **dict(attend, heads=16, kv_heads=2, block=64, topk=16, ragged=True)),
        # the last piece of a prompt behind what the cache holds of it
        dict(name="attend_piece_64_of_16k", dtype="bf16", batch=1, queries=64, keys=16384, **dict(attend, bits=8)),
        # an odd batch in 32 bits, every head with keys of its own
        dict(name="attend_odd_f32", dtype="f32", batch=3, queries=5, keys=1237, **dict(attend, heads=6, kv_heads=6, head_len=32, ragged=True)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "store", "attend", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 4, 8, 16])
    head_len = rng.choice([32, 64, 64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "rotate":
        train = rng.random() < 0.5
        most = 16384 * 40 * 128 * 2 // (_TYPES[dtype].itemsize * (heads + kv_heads) * head_len * (4 if train else 1))
        tokens = _log_int(rng, 1, min(16384, most))
        batch = _log_int(rng, 1, max(1, min(32, most // tokens)))
        axes = rng.choice([1, 1, 1, 2, 3])
        rotary_len = rng.choice([head_len, head_len, head_len // 2])
        return dict(op=op, train=train, dtype=dtype, batch=batch, tokens=tokens, past=0 if train or axes > 1 else rng.choice([0, _log_int(rng, 1, 131072)]),
                    heads=heads, kv_heads=kv_heads, head_len=head_len, norm=rng.random() < 0.8, rotary_len=rotary_len, axes=axes,
                    interleaved=rng.random() < 0.3, ragged=axes == 1 and batch > 1 and rng.random() < 0.5, base=rng.choice([10000.0, 500000.0, 1e6]))
    bits = rng.choice([4, 4, 8])
    if op == "store":
        most = 16384 * 8 * 128 * 2 // (_TYPES[dtype].itemsize * kv_heads * head_len)
        tokens = rng.choice([1, 1, 2, _log_int(rng, 3, min(16384, most))])
        batch = _log_int(rng, 1, max(1, min(32, most // tokens)))
        keys = min(32768, tokens + _log_int(rng, 1, 16384))
        window = min(keys, tokens if tokens > 2 else rng.choice([32, 64, 128, 256]))
        return dict(op=op, dtype=dtype, batch=batch, tokens=tokens, keys=keys, window=window, kv_heads=kv_heads, head_len=head_len, bits=bits,
                    ragged=batch > 1 and rng.random() < 0.6)
    queries = rng.choice([1, 1, 1, 2, 3, 5, _log_int(rng, 6, 64)])
    keys = max(queries, _log_int(rng, 1, 65536))
    # the plain form holds heads x queries x keys values: as many as the largest listed case at most
    batch = _log_int(rng, 1, max(1, min(32, 32 * 32768 * 8 * 128 * 4 // (keys * kv_heads * head_len * bits), 32 * 64 * 16384 // (keys * heads * queries))))
    block, topk = (rng.choice([32, 64, 64, 128, 256]), _log_int(rng, 1, 24)) if rng.random() < 0.4 else (0, 0)
    return dict(op=op, dtype=dtype, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, head_len=head_len, bits=bits, block=block,
                topk=topk, ragged=batch > 1 and rng.random() < 0.5)


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and "held" in s:
        from featgraph_amd import ops
        s["cache"] = ops.KeyValueCache(*s["held"]["k"], *s["held"]["v"], bits=s["case"]["bits"])
    return s


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    c, dtype = dict(case), _TYPES[case["dtype"]]
    b, n, hk, d = c["batch"], c.get("tokens", c.get("queries")), c["kv_heads"], c["head_len"]

    def normal(*shape, like=dtype):
        return torch.randn(shape, generator=gen, device="cuda", dtype=like)

    def counts(low, high):
        return torch.randint(low, high + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)

    s = dict(case=c, lengths=None, q_lengths=None)
    if c["op"] == "rotate":
        h = c["heads"]
        fused = normal(b, n, (h + 2 * hk), d)
        s["q"], s["k"] = fused[:, :, :h], fused[:, :, h:h + hk]
        if c["norm"]:
            s["q_weight"], s["k_weight"] = normal(d).mul_(0.2).add_(1.0), normal(d).mul_(0.2).add_(1.0)
        pairs = c["rotary_len"] // 2
        s["sections"] = {1: (pairs,), 2: (pairs // 2, pairs - pairs // 2),
                         3: (pairs // 4, (pairs - pairs // 4) // 2, pairs - pairs // 4 - (pairs - pairs // 4) // 2)}[c["axes"]]
        if c["axes"] > 1:
            # frames of 16 x 22 patches behind some text
            i, start = torch.arange(n, device="cuda", dtype=torch.int32), counts(0, 400)[:, None]
            grid = [start + i // 352, start + i % 352 // 22, start + i % 22]
            s["positions"] = torch.stack(grid if c["axes"] == 3 else grid[1:], 2).contiguous()
        elif c["ragged"]:
            # new tokens behind what each sequence has, fewer than the tensor has room for in some
            s["q_lengths"] = counts(max(1, n // 2), n)
            s["lengths"] = (s["q_lengths"] + counts(0, c["past"])).int()
        elif c["past"]:
            s["lengths"] = torch.full((b,), c["past"] + n, device="cuda", dtype=torch.int32)
        if c["train"]:
            s["dq"], s["dk"] = normal(b, n, h, d), normal(b, n, hk, d)
        return s
    m = c["keys"]
    full = torch.full((b,), m, device="cuda", dtype=torch.int32)
    if c["op"] == "store":
        fused = normal(b, n, 2 * hk, d)
        s["k"], s["v"] = fused[:, :, :hk], fused[:, :, hk:]
        lengths, q_lengths = full, torch.full_like(full, n)
        if c["ragged"]:
            s["q_lengths"] = q_lengths = counts(max(1, n // 2), n)
            s["lengths"] = lengths = torch.maximum(q_lengths, counts(max(1, m // 2), m))
        s["first"] = (lengths - c["window"]).clamp(min=0).int()
        there = torch.arange(n, device="cuda") < q_lengths[:, None]
        at, row = there.nonzero(as_tuple=True)
        s["rows"] = at, row, (lengths - q_lengths)[at].long() + row         # which row goes where, for the plain form
    else:
        s["q"] = normal(b, n, c["heads"], d)
        if c["ragged"]:
            s["lengths"] = torch.maximum(counts(max(1, m // 2), m), full * 0 + n)
        if c["topk"]:
            # the first block, the last ones, and others between, as a selection gives them
            nb = -(-m // c["block"])
            lengths = full if s["lengths"] is None else s["lengths"]
            position = lengths[:, None] - n + torch.arange(n, device="cuda", dtype=torch.int32)
            last = (position // c["block"]).view(b, n, 1, 1)
            few = min(c["topk"], nb)
            score = torch.rand((b, n, hk, nb), generator=gen, device="cuda")
            ids = torch.arange(nb, device="cuda")
            score = torch.where((ids == last) | ((ids == 0) & (few > 1)), 2.0, score).masked_fill_(ids > last, -1.0)
            best, where = score.topk(few, 3)
            where = torch.where(best < 0, nb, where).sort(3).values
            where = torch.where(where == nb, -1, where)
            s["blocks"] = torch.nn.functional.pad(where, (0, c["topk"] - few), value=-1).to(torch.int32).contiguous()
    held = {"k": [], "v": []}
    for i in range(b):                      # what earlier tokens left in the cache
        for x in "kv":
            held[x].append(_pack(normal(hk, m, d), c["bits"]))
    s["held"] = {x: tuple(torch.stack(t) for t in zip(*held[x])) for x in "kv"}
    return s


# ---- the operators in their plain form ------------------------------------------------------------------


def _angles(s):
    """cos and sin of every token's pairs, (batch, tokens, 1, pairs), and whether a row is there."""
    c, q = s["case"], s["q"]
    pairs = c["rotary_len"] // 2
    i = torch.arange(c["tokens"], device=q.device)
    there = None if s["q_lengths"] is None else (i < s["q_lengths"].long()[:, None])[:, :, None, None]
    if c["axes"] > 1:
        axis = torch.repeat_interleave(torch.arange(c["axes"], device=q.device), torch.tensor(s["sections"], device=q.device), output_size=pairs)
        position = s["positions"][:, :, axis].double()
    else:
        behind = c["tokens"] if s["q_lengths"] is None else s["q_lengths"].long()[:, None]
        position = (i if s["lengths"] is None else s["lengths"].long()[:, None] - behind + i).double().expand(c["batch"], -1)[:, :, None]
    turn = position * c["base"] ** (-torch.arange(pairs, device=q.device, dtype=torch.float64) / pairs)
    return torch.cos(turn).float()[:, :, None], torch.sin(turn).float()[:, :, None], there


def _turned(c, x, cos, sin):
    part, rest = x[..., :c["rotary_len"]], x[..., c["rotary_len"]:]
    if c["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        part = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = part.chunk(2, -1)
        part = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((part, rest), -1)


def _rotate(s):
    c = s["case"]
    cos, sin, there = _angles(s)
    got = {}

    def kept(x):
        return x if there is None else torch.where(there, x, torch.zeros((), device=x.device))

    for x in "qk":
        data = kept(s[x].float())
        if c["norm"]:
            weight = s[x + "_weight"].float()
            inverse = torch.rsqrt(data.square().mean(-1, keepdim=True) + _EPS)
            data = data * inverse
        got[x] = _turned(c, data * weight if c["norm"] else data, cos, sin).to(s[x].dtype)
        if not c["train"]:
            continue
        g = _turned(c, kept(s["d" + x].float()), cos, -sin)
        if c["norm"]:
            got["d%s_weight" % x] = (g * data).sum((0, 1, 2), dtype=torch.float64).float().to(s[x].dtype)
            g = g * weight
            g = (g - data * (g * data).mean(-1, keepdim=True)) * inverse
        got["d" + x] = g.to(s[x].dtype)
    return got


def _pack(x, bits):
    """(codes, scales) of (..., head_len) values."""
    x = x.float().unflatten(-1, (-1, 32))
    # the largest value's exponent, one more where it would round to beyond the largest element
    fraction, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    over = fraction >= 0.875 if bits == 4 else fraction > 0.90625
    exponent = torch.where(fraction == 0, -127, (exponent - (3 if bits == 4 else 9) + over)).clamp_(-127, _TOP_EXPONENT[bits])
    x = torch.ldexp(x, -exponent)
    size = x.abs()
    step = torch.exp2(torch.floor(torch.log2(size.clamp(min=1.0 if bits == 4 else 2.0 ** -6))) - (1 if bits == 4 else 3))
    size = (size / step).round_().mul_(step).clamp_(max=_MAGNITUDES[bits][-1])
    code = torch.bucketize(size, torch.tensor(_MAGNITUDES[bits], device=x.device), out_int32=True)
    code = torch.where(x < 0, code + (1 << (bits - 1)), code).to(torch.uint8).flatten(-2)
    if bits == 4:
        code = code[..., 0::2] + code[..., 1::2] * 16
    return code, (exponent.squeeze(-1) + 127).to(torch.uint8)


def _unpack(codes, scales, bits):
    table = torch.tensor(_MAGNITUDES[bits], device=codes.device)
    if bits == 8:
        table = torch.cat((table, table.new_zeros(1)))                  # the code of no number
    table = torch.cat((table, -table))
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return torch.ldexp(table[codes.int()].unflatten(-1, (-1, 32)), scales.int()[..., None] - 127).flatten(-2)


def _store(s):
    c = s["case"]
    at, row, position = s["rows"]
    got = {}
    window = s["first"].long()[:, None] + torch.arange(c["window"], device=s["k"].device)
    there = window < (c["keys"] if s["lengths"] is None else s["lengths"].long()[:, None])
    window = window.clamp(max=c["keys"] - 1)
    batch = torch.arange(c["batch"], device=window.device)[:, None]
    for x in "kv":
        codes, scales = s["held"][x]
        new = _pack(s[x][at, row], c["bits"])                           # (rows, kv_heads, ...)
        codes[at, :, position], scales[at, :, position] = new
        back = _unpack(codes[batch, :, window], scales[batch, :, window], c["bits"])
        got[x] = torch.where(there[:, :, None, None], back, torch.zeros((), device=back.device)).to(s[x].dtype)
    return got


def _attend(s):
    c, q = s["case"], s["q"]
    b, n, m, hk, d = c["batch"], c["queries"], c["keys"], c["kv_heads"], c["head_len"]
    key = torch.arange(m, device=q.device)
    out = torch.empty((b, n, c["heads"], d), dtype=q.dtype, device=q.device)
    for i in range(b):                      # one sequence at a time: the cache's values take eight times its room
        k, v = (_unpack(*(t[i] for t in s["held"][x]), c["bits"]) for x in "kv")
        length = m if s["lengths"] is None else s["lengths"][i].long()
        seen = (key <= length - n + torch.arange(n, device=q.device)[:, None])[None]
        if c["topk"]:
            nb = -(-m // c["block"])
            ids = s["blocks"][i].long().transpose(0, 1)                 # (kv_heads, queries, topk)
            chosen = torch.zeros((hk, n, nb + 1), dtype=torch.bool, device=q.device)
            chosen = chosen.scatter_(2, torch.where(ids < 0, nb, ids), True)
            seen = seen & chosen[..., :nb].repeat_interleave(c["block"], 2)[..., :m]
        rows = q[i].float().view(n, hk, -1, d).transpose(0, 1).reshape(hk, -1, d)       # (kv_heads, queries x group, d)
        score = torch.matmul(rows, k.transpose(1, 2).contiguous()).mul_(d ** -0.5).view(hk, n, -1, m)
        score = score.masked_fill_(~seen[:, :, None], -math.inf)
        power = score.sub_(score.amax(-1, keepdim=True)).exp_()
        power = power.div_(power.sum(-1, keepdim=True)).view(hk, -1, m)
        out[i] = torch.matmul(power, v).view(hk, n, -1, d).transpose(0, 1).reshape(n, -1, d).to(q.dtype)
    return {"out": out}


# ---- one pass -------------------------------------------------------------------------------------------


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rotate": _rotate, "store": _store, "attend": _attend}[c["op"]](s)
    from featgraph_amd import ops
    lengths = dict(lengths=s["lengths"], q_lengths=s["q_lengths"])
    if c["op"] == "store":
        ops.write_cache(s["cache"], s["k"], s["v"], **lengths)
        k, v = ops.read_cache(s["cache"], s["k"].dtype, first=s["first"], count=c["window"], lengths=s["lengths"])
        return {"k": k, "v": v}
    if c["op"] == "attend":
        if c["topk"]:
            lengths.update(blocks=s["blocks"], block_size=c["block"])
        return {"out": ops.cache_attention(s["q"], s["cache"], **lengths)}
    more = dict(lengths, base=c["base"], rotary_len=c["rotary_len"], interleaved=c["interleaved"])
    if c["axes"] > 1:
        more.update(positions=s["positions"], sections=s["sections"])
    names = ("q", "k") + (("q_weight", "k_weight") if c["norm"] else ())
    if not c["train"]:
        q, k = ops.rotate_heads(*(s[x] for x in names), eps=_EPS, **more)
        return {"q": q, "k": k}
    leaves = [s[x].detach().requires_grad_() for x in names]
    q, k = ops.rotate_heads(*leaves, eps=_EPS, **more)
    grads = torch.autograd.grad((q, k), leaves, (s["dq"], s["dk"]))
    return dict({"q": q.detach(), "k": k.detach()}, **{"d" + x: g for x, g in zip(names, grads)})


def work(case):
    c = case
    size, b, hk, d = _TYPES[c["dtype"]].itemsize, c["batch"], c["kv_heads"], c["head_len"]
    if c["op"] == "rotate":
        tokens = c["tokens"] * 3 / 4 if c["ragged"] and c["tokens"] > 1 else c["tokens"]
        values = int(b * tokens * (c["heads"] + hk) * d)
        once = 2 + ((3 if c["norm"] else 2) if c["train"] else 0)       # q and k in and out; they, dL/dout and the gradients
        return {"bytes": values * once * size, "flops": values * (7 + (14 if c["train"] else 0))}
    element = c["bits"] / 8 + 1 / 32
    if c["op"] == "store":
        tokens = c["tokens"] * 3 / 4 if c["ragged"] and c["tokens"] > 1 else c["tokens"]
        rows, back = b * tokens * hk * d * 2, b * c["window"] * hk * d * 2
        # of the window, what was not just written is read
        return {"bytes": int(rows * (size + element) + back * size + max(0, back - rows) * element), "flops": int(2 * (rows + back))}
    n, m = c["queries"], c["keys"] * 3 // 4 if c["ragged"] else c["keys"]
    seen = min(m, c["topk"] * c["block"]) if c["topk"] else m
    read = min(m, n * seen) if c["topk"] else m
    lists = 4 * b * n * hk * c["topk"]
    return {"bytes": int(2 * b * n * c["heads"] * d * size + 2 * b * hk * read * d * element + lists), "flops": 4 * b * n * c["heads"] * seen * d}


# ---- the definition in 64 bits --------------------------------------------------------------------------


def _exact_rotate(s):
    c = s["case"]
    b, n, length, half = c["batch"], c["tokens"], c["rotary_len"], c["rotary_len"] // 2
    device = s["q"].device
    place = torch.zeros((b, n, half), dtype=torch.float64, device=device)
    alive = torch.ones((b, n, 1, 1), dtype=torch.bool, device=device)
    axis_of = [a for a, many in enumerate(s["sections"]) for _ in range(many)]
    for i in range(b):
        rows = n if s["q_lengths"] is None else int(s["q_lengths"][i])
        alive[i, rows:] = False
        start = 0 if s["lengths"] is None else int(s["lengths"][i]) - rows
        for pair, axis in enumerate(axis_of):
            place[i, :, pair] = s["positions"][i, :, axis] if c["axes"] > 1 else start + torch.arange(n, device=device)
    speed = torch.tensor([c["base"] ** (-2.0 * pair / length) for pair in range(half)], dtype=torch.float64, device=device)
    circle = torch.polar(torch.ones_like(place), place * speed)[:, :, None]
    got = {}
    for x in "qk":
        data = torch.where(alive, s[x].double(), 0.0).requires_grad_(c["train"])
        y = data
        if c["norm"]:
            weight = s[x + "_weight"].double().requires_grad_(c["train"])
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / c["head_len"] + _EPS) * weight
        first = list(range(0, length, 2)) if c["interleaved"] else list(range(half))
        second = [i + 1 for i in first] if c["interleaved"] else [i + half for i in first]
        turned = torch.complex(y[..., first], y[..., second]) * circle
        order = torch.tensor(first + second + list(range(length, c["head_len"])), device=device)
        y = torch.cat((turned.real, turned.imag, y[..., length:]), -1)[..., torch.argsort(order)]
        got[x] = y.detach()
        if c["train"]:
            dy = torch.where(alive, s["d" + x].double(), 0.0)
            grads = torch.autograd.grad(y, [data] + ([weight] if c["norm"] else []), dy)
            got["d" + x] = grads[0]
            if c["norm"]:
                got["d%s_weight" % x] = grads[1]
    return got


def _nearest(x, bits):
    """Rows of head_len 64-bit values as the cache holds them, by comparing with every element."""
    table = torch.tensor(_MAGNITUDES[bits], dtype=torch.float64, device=x.device)
    border = (table[1:] + table[:-1]) / 2
    beyond = table[-1] + (table[-1] - table[-2]) / 2
    groups = x.reshape(-1, 32)
    most = groups.abs().amax(1, keepdim=True)
    power = torch.full_like(most, 2.0 ** -127)
    for e in range(-126, _TOP_EXPONENT[bits] + 1):
        # a tie above the largest element goes to the even code: 4-bit elements end with an odd one, 8-bit elements with an even one
        small = most < power * beyond if bits == 4 else most <= power * beyond
        power = torch.where(small, power, torch.full_like(power, 2.0 ** e))
    y = groups / power
    low, high = torch.bucketize(y.abs(), border), torch.bucketize(y.abs(), border, right=True)
    code = torch.where(low % 2 == 0, low, high)                         # they differ on a border only
    return (table[code] * torch.sign(y) * power).reshape(x.shape)


def _value_of(codes, scales, bits):
    """64-bit values of rows of codes."""
    if bits == 4:
        codes = codes.repeat_interleave(2, -1)
        codes = torch.where(torch.arange(codes.shape[-1], device=codes.device) % 2 == 0, codes % 16, torch.div(codes, 16, rounding_mode="floor"))
        exponent, mantissa, sign, least, width = codes // 2 % 4, codes % 2, codes // 8, 1, 2
    else:
        exponent, mantissa, sign, least, width = codes // 8 % 16, codes % 8, codes // 128, 7, 8
    exponent, mantissa = exponent.double(), mantissa.double()
    size = torch.where(exponent == 0, 2.0 ** (1 - least) * mantissa / width, 2.0 ** (exponent - least) * (1 + mantissa / width))
    return torch.where(sign > 0, -size, size) * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def exact(case, seed):
    s = _inputs(case, seed)
    c = s["case"]
    if c["op"] == "rotate":
        return _exact_rotate(s)
    held = s["held"]
    b, m, hk, d = c["batch"], c["keys"], c["kv_heads"], c["head_len"]
    if c["op"] == "store":
        got = {x: torch.zeros((b, c["window"], hk, d), dtype=torch.float64, device=s["k"].device) for x in "kv"}
        for i in range(b):
            new = c["tokens"] if s["q_lengths"] is None else int(s["q_lengths"][i])
            length = m if s["lengths"] is None else int(s["lengths"][i])
            first = int(s["first"][i])
            upto = min(length, first + c["window"])
            for x in "kv":
                for g in range(hk):
                    row = _value_of(*(t[i, g, first:upto] for t in held[x]), c["bits"])
                    behind = max(first, length - new)
                    row[behind - first:] = _nearest(s[x][i, behind - length + new:new, g].double(), c["bits"])
                    got[x][i, :upto - first, g] = row
        return got
    n, group = c["queries"], c["heads"] // hk
    out = torch.zeros((b, n, c["heads"], d), dtype=torch.float64, device=s["q"].device)
    for i in range(b):
        length = m if s["lengths"] is None else int(s["lengths"][i])
        for g in range(hk):
            k, v = (_value_of(*(t[i, g, :length] for t in held[x]), c["bits"]) for x in "kv")
            where = torch.arange(length, device=k.device)
            for r in range(n):
                upto = length - n + r + 1
                near = where[:upto]
                if c["topk"]:
                    near = near[torch.isin(near // c["block"], s["blocks"][i, r, g].long())]
                z = s["q"][i, r, g * group:(g + 1) * group].double() @ k[near].t() / math.sqrt(d)
                out[i, r, g * group:(g + 1) * group] = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) @ v[near]
    return {"out": out}
