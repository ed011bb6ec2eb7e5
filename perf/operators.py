"""Attention over blocks of keys that every query selects for itself: the work a user has these operators do, as cases that can be
timed and compared.

  select   every query's best blocks of keys by a cheap score: the keys' mean over each block, against the sum of the queries
           of the heads that share a key head (ops.pool_blocks, ops.select_blocks)
  attend   softmax attention of every query over the keys of its blocks, forward, with its gradients, and for single tokens
           over a long cache (ops.block_attention)
  biased   the same with a learned bias for each bucket of relative positions, with the bias's gradient
           (ops.block_attention, ops.position_bounds)

q is (batch, queries, heads, head_len), k and v (batch, keys, kv_heads, head_len); heads / kv_heads query heads share a key
head and its selection.  A sequence's last query stands at its last key.  Blocks are (batch, queries, kv_heads, topk), -1 behind
the last one.

In their plain form the operators are elementary torch operations in 32 bits, the scores that choose blocks in 64; `exact` computes
them from their definition in 64 bits, head by head.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    layer = dict(heads=32, kv_heads=8, head_len=128, block=64, topk=16, causal=True, ragged=False, buckets=0)
    return [
        # choosing blocks for all tokens of a long prompt
        dict(name="select_16k", op="select", train=False, dtype="bf16", batch=1, queries=16384, keys=16384, **layer),
        # one new token for each of many requests, from the pooled keys that a serving program keeps
        dict(name="select_token_32x32k", op="select", train=False, dtype="bf16", batch=32, queries=1, keys=32768, **layer),
        # a padded batch of odd lengths in 32 bits, three query heads to a key head
        dict(name="select_odd_f32", op="select", train=False, dtype="f32", batch=3, queries=1237, keys=1237, heads=6, kv_heads=2,
             head_len=64, block=32, topk=7, causal=True, ragged=True, buckets=0),
        # the forward pass over a prompt
        dict(name="attend_8k", op="attend", train=False, dtype="bf16", batch=1, queries=8192, keys=8192, **layer),
        # a training step's attention
        dict(name="attend_train_2x4k", op="attend", train=True, dtype="bf16", batch=2, queries=4096, keys=4096,
             **dict(layer, heads=16, kv_heads=4)),
        # training an encoder whose heads share one key head: sixteen to one, long blocks, nothing causal
        dict(name="attend_train_shared_8k", op="attend", train=True, dtype="f16", batch=1, queries=8192, keys=8192, heads=16, kv_heads=1,
             head_len=64, block=128, topk=8, causal=False, ragged=False, buckets=0),
        # a padded batch of odd lengths in 32 bits, every head with keys of its own
        dict(name="attend_train_odd_f32", op="attend", train=True, dtype="f32", batch=3, queries=1237, keys=1237, heads=8, kv_heads=8,
             head_len=64, block=32, topk=8, causal=True, ragged=True, buckets=0),
        # one new token for each of many requests over long caches
        dict(name="attend_token_32x32k", op="attend", train=False, dtype="bf16", batch=32, queries=1, keys=32768, **layer),
        # one new token of one request: latency
        dict(name="attend_token_1x2k", op="attend", train=False, dtype="f16", batch=1, queries=1, keys=2048, heads=8, kv_heads=8,
             head_len=64, block=64, topk=8, causal=True, ragged=False, buckets=0),
        # a training step with a learned bias of 32 distance buckets
        dict(name="biased_train_2x2k", op="biased", train=True, dtype="bf16", batch=2, queries=2048, keys=2048,
             **dict(layer, heads=16, kv_heads=4, topk=8, buckets=32)),
        # a short sequence, both directions
        dict(name="biased_train_517", op="biased", train=True, dtype="f16", batch=1, queries=517, keys=517, heads=4, kv_heads=4,
             head_len=32, block=32, topk=4, causal=False, ragged=False, buckets=16),
        # three new tokens at once for each of eight requests of unequal lengths
        dict(name="biased_tokens_8x5000", op="biased", train=False, dtype="bf16", batch=8, queries=3, keys=5000,
             **dict(layer, heads=16, kv_heads=2, ragged=True, buckets=32)),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "attend", "attend", "attend", "biased", "biased"])
    group = rng.choice([1, 1, 2, 3, 4, 4, 8, 16])
    kv_heads = rng.choice([1, 2, 4, 8])
    head_len = rng.choice([32, 64, 64, 128, 128])
    block = rng.choice([32, 64, 64, 128, 256])
    topk = _log_int(rng, 1, 24)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    causal = rng.random() < 0.75
    tokens = op != "select" and rng.random() < 0.35 or op == "select" and rng.random() < 0.3
    train = op != "select" and not tokens and rng.random() < 0.7
    heads = group * kv_heads
    if tokens:
        queries, keys = rng.choice([1, 1, 1, 2, 3, 5]), _log_int(rng, 1, 32768)
        most = max(1, min(32, 32 * 32768 * 8 * 128 // (keys * kv_heads * head_len)))
        batch = _log_int(rng, 1, most)
        keys = max(keys, queries)
    else:
        # the plain form holds heads x queries x keys values: at most what the largest listed cases of the kind hold
        most = 2 * 4096 * 4096 * 16 if train or op == "biased" else 8192 * 8192 * 16
        if op == "select":
            keys = _log_int(rng, 40, 16384)
            batch = _log_int(rng, 1, max(1, min(8, 16384 * 8 // (keys * kv_heads))))
        else:
            keys = _log_int(rng, 40, min(8192, math.isqrt(most // heads)))
            batch = _log_int(rng, 1, max(1, min(8, most // (heads * keys * keys))))
        queries = keys
    return dict(op=op, train=train, dtype=dtype, batch=batch, queries=queries, keys=keys, heads=heads, kv_heads=kv_heads, head_len=head_len,
                block=block, topk=topk, causal=causal, ragged=batch > 1 and rng.random() < 0.5,
                buckets=rng.choice([8, 16, 32, 32, 64]) if op == "biased" else 0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)
    c, dtype = dict(case), _TYPES[case["dtype"]]
    b, n, m, h, hk, d = c["batch"], c["queries"], c["keys"], c["heads"], c["kv_heads"], c["head_len"]

    def normal(*shape, like=dtype):
        return torch.randn(shape, generator=gen, device="cuda", dtype=like)

    # text speaks of a topic for a while and comes back to it later: a stretch of 128 keys shares a direction, and a stretch of
    # queries looks for some of those
    span = 128
    topics = normal(b, -(-m // span), hk, d)
    k = normal(b, m, hk, d).add_(topics.repeat_interleave(span, 1)[:, :m], alpha=0.7)
    wanted = torch.randint(topics.shape[1], (b, -(-n // span), 4), generator=gen, device="cuda")
    wish = topics[torch.arange(b, device="cuda")[:, None, None], wanted].sum(2).repeat_interleave(span, 1)[:, :n]
    q = normal(b, n, h, d).add_(wish.repeat_interleave(h // hk, 2), alpha=0.4)
    s = dict(case=c, q=q, k=k)
    if c["ragged"]:
        lengths = torch.randint(max(1, m // 2), m + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        lengths[0] = m
        s["lengths"] = lengths
        s["q_lengths"] = lengths if n == m else None        # a padded batch, or new tokens behind caches of unequal lengths
    else:
        s["lengths"] = s["q_lengths"] = None
    if c["op"] == "select":
        s["pooled"] = _pool(s) if n < m else None           # a serving program keeps the pooled keys of its cache
        return s
    s["v"] = normal(b, m, hk, d)
    s["blocks"] = _select(s, _pool(s))
    if c["buckets"]:
        s["bias"] = normal(c["buckets"], h).mul_(0.5)
        s["bounds"] = _bounds(c["buckets"], 128, c["causal"])
    if c["train"]:
        s["dout"] = normal(b, n, h, d)
    return s


def _bounds(buckets, far, causal):
    """First distance (query's position less key's) of each bucket but the first: the nearer half one by one, the others growing in
    proportion up to `far`; without causality the same on both sides."""
    one = buckets if causal else buckets // 2
    near = one // 2
    side = list(range(1, near + 1)) + [int(math.ceil(near * (far / near) ** ((i - near) / (one - near)))) for i in range(near + 1, one)]
    side = [max(x, i + 1) for i, x in enumerate(side)]
    return side if causal else [1 - x for x in reversed(side)] + [1] + [x + 1 for x in side][:buckets - 2 - len(side)]


# ---- the operators in their plain form ------------------------------------------------------------------


def _sizes(s):
    """(keys, queries) of every sequence, (batch,) each."""
    c, q = s["case"], s["q"]
    full = torch.ones(c["batch"], dtype=torch.int64, device=q.device)
    kl = full * c["keys"] if s["lengths"] is None else s["lengths"].long()
    ql = full * c["queries"] if s["q_lengths"] is None else s["q_lengths"].long()
    return kl, ql


def _positions(s):
    """Position of every query, (batch, queries): the last one's is the last key's; -1 for rows behind the last query."""
    c = s["case"]
    kl, ql = _sizes(s)
    i = torch.arange(c["queries"], device=kl.device)
    pos = kl[:, None] - ql[:, None] + i
    return torch.where(i < ql[:, None], pos, torch.full_like(pos, -1)), i < ql[:, None]


def _pool(s):
    """Mean of the keys of every block, (batch, kv_heads, blocks, head_len), in the keys' type."""
    c, k = s["case"], s["k"]
    kl, _ = _sizes(s)
    nb = -(-c["keys"] // c["block"])
    valid = torch.arange(c["keys"], device=k.device) < kl[:, None]
    x = torch.where(valid[:, :, None, None], k, torch.zeros((), dtype=k.dtype, device=k.device))
    x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, nb * c["block"] - c["keys"]))
    total = x.view(c["batch"], nb, c["block"], c["kv_heads"], c["head_len"]).sum(2, dtype=torch.float64)
    count = (kl[:, None] - torch.arange(nb, device=k.device) * c["block"]).clamp(0, c["block"])
    mean = total / count.clamp(min=1)[:, :, None, None]
    return mean.float().to(k.dtype).transpose(1, 2).contiguous()


def _select(s, pooled):
    """The topk best blocks of every query: those that it may see, its first and its own for certain, ties to the lower block."""
    c, q = s["case"], s["q"]
    b, n, hk, d = c["batch"], c["queries"], c["kv_heads"], c["head_len"]
    nb = pooled.shape[2]
    summed = q.view(b, n, hk, -1, d).sum(3, dtype=torch.float64).float().to(q.dtype)
    scores = torch.matmul(summed.double().transpose(1, 2).contiguous(), pooled.double().transpose(2, 3).contiguous())
    kl, _ = _sizes(s)
    pos, there = _positions(s)
    first = torch.arange(nb, device=q.device) * c["block"]
    last = pos if c["causal"] else (kl[:, None] - 1).expand_as(pos)
    seen = (first <= last[:, :, None]) & (first < kl[:, None, None]) & there[:, :, None]
    own_block = torch.div(last, c["block"], rounding_mode="floor")
    kept = seen & ((torch.arange(nb, device=q.device) == own_block[:, :, None]) | ((first == 0) & (c["topk"] > 1)))
    scores = torch.where(scores.isnan(), torch.full_like(scores, -math.inf), scores).clamp(min=-1e300, max=1e300)
    scores = torch.where(kept[:, None], torch.full_like(scores, math.inf), scores).masked_fill(~seen[:, None], -math.inf)
    best, at = torch.sort(scores, dim=3, descending=True, stable=True)
    best, at = best[..., :c["topk"]], at[..., :c["topk"]]
    at = torch.where(best == -math.inf, torch.full_like(at, nb), at).sort(3).values
    at = torch.where(at == nb, torch.full_like(at, -1), at)
    if at.shape[3] < c["topk"]:
        at = torch.nn.functional.pad(at, (0, c["topk"] - at.shape[3]), value=-1)
    return at.transpose(1, 2).to(torch.int32).contiguous()


def _softmax(scores, seen):
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(total.masked_fill_(total == 0, 1.0))


def _buckets_of(s, distance):
    bounds = torch.tensor(s["bounds"], device=distance.device)
    return torch.bucketize(distance, bounds, right=True)


def _attend_gathered(s):
    """A few queries: the keys of their blocks taken out of the cache first."""
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, n, hk, d, size = c["batch"], c["queries"], c["kv_heads"], c["head_len"], c["block"]
    kl, _ = _sizes(s)
    pos, there = _positions(s)
    key = (s["blocks"].long()[..., None] * size + torch.arange(size, device=q.device)).view(b, n, hk, -1)
    seen = (key >= 0) & (key < kl[:, None, None, None]) & there[:, :, None, None]
    if c["causal"]:
        seen &= key <= pos[:, :, None, None]
    at = key.clamp(0, c["keys"] - 1)
    where = (torch.arange(b, device=q.device)[:, None, None, None], at, torch.arange(hk, device=q.device)[:, None])
    ks, vs = k[where].float(), v[where].float()                     # (b, n, hk, keys, d)
    scores = torch.matmul(q.float().view(b, n, hk, -1, d), ks.transpose(3, 4).contiguous()) * d ** -0.5
    if c["buckets"]:
        bias = s["bias"].float()[_buckets_of(s, pos[:, :, None, None] - key)].view(b, n, hk, -1, hk, c["heads"] // hk)
        scores += torch.diagonal(bias, dim1=2, dim2=4).permute(0, 1, 4, 3, 2)
    p = _softmax(scores, seen[:, :, :, None])
    return {"out": torch.matmul(p, vs).view(b, n, c["heads"], d).to(q.dtype)}


def _attend_dense(s):
    """Many queries: every score, those outside the blocks masked; with the gradients where the step trains."""
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, n, m, h, hk, d = c["batch"], c["queries"], c["keys"], c["heads"], c["kv_heads"], c["head_len"]
    kl, _ = _sizes(s)
    pos, there = _positions(s)
    key = torch.arange(m, device=q.device)
    nb = -(-m // c["block"])
    blocks = s["blocks"].long().transpose(1, 2)
    chosen = torch.zeros((b, hk, n, nb + 1), dtype=torch.bool, device=q.device)
    chosen = chosen.scatter_(3, torch.where(blocks < 0, torch.full_like(blocks, nb), blocks), True)
    seen = chosen[..., :nb].repeat_interleave(c["block"], 3)[..., :m]
    seen = seen & (key < kl[:, None, None])[:, None] & there[:, None, :, None]
    if c["causal"]:
        seen &= (key <= pos[:, :, None])[:, None]
    seen = seen.unsqueeze(2)                                        # (b, hk, 1, n, m)

    def heads_first(x):
        return x.float().view(b, n, hk, -1, d).permute(0, 2, 3, 1, 4).reshape(b * hk, -1, d)

    def keys_first(x):
        return x.float().transpose(1, 2).reshape(b * hk, m, d)

    def back(x, rows):
        x = x.view(b, hk, -1, rows, d).permute(0, 3, 1, 2, 4).reshape(b, rows, -1, d)
        return x.to(q.dtype).contiguous()

    qf, kf, vf = heads_first(q), keys_first(k), keys_first(v)
    scores = torch.bmm(qf, kf.transpose(1, 2).contiguous()).mul_(d ** -0.5).view(b, hk, h // hk, n, m)
    if c["buckets"]:
        bucket = _buckets_of(s, pos[:, :, None] - key)              # (b, n, m)
        scores += s["bias"].float().t().contiguous()[:, bucket].view(hk, h // hk, b, n, m).permute(2, 0, 1, 3, 4)
    p = _softmax(scores, seen).view(b * hk, -1, m)
    of = torch.bmm(p, vf)
    got = {"out": back(of, n)}
    if c["train"]:
        do = heads_first(s["dout"])
        got["dv"] = back(torch.bmm(p.transpose(1, 2).contiguous(), do), m)
        dp = torch.bmm(do, vf.transpose(1, 2).contiguous())
        ds = dp.sub_((do * of).sum(-1, keepdim=True)).mul_(p)
        del dp, p
        got["dq"] = back(torch.bmm(ds, kf).mul_(d ** -0.5), n)
        got["dk"] = back(torch.bmm(ds.transpose(1, 2).contiguous(), qf).mul_(d ** -0.5), m)
        if c["buckets"]:                # long sums: in 64 bits
            head = torch.arange(h, device=q.device).view(1, hk, h // hk, 1, 1)
            cell = head * c["buckets"] + bucket[:, None, None]
            total = torch.bincount(cell.reshape(-1), weights=ds.view(cell.shape).double().reshape(-1), minlength=h * c["buckets"])
            got["dbias"] = total.view(h, c["buckets"]).t().to(q.dtype).contiguous()
    return got


# ---- one pass -------------------------------------------------------------------------------------------


def run(state):
    s, c = state, state["case"]
    if not own:
        if c["op"] == "select":
            pooled = _pool(s) if s["pooled"] is None else s["pooled"]
            return {"pooled": pooled, "blocks": _select(s, pooled)}
        return _attend_gathered(s) if c["queries"] < 16 else _attend_dense(s)
    from featgraph_amd import ops
    lengths = dict(lengths=s["lengths"], q_lengths=s["q_lengths"])
    if c["op"] == "select":
        pooled = ops.pool_blocks(s["k"], c["block"], s["lengths"]) if s["pooled"] is None else s["pooled"]
        return {"pooled": pooled, "blocks": ops.select_blocks(s["q"], pooled, c["keys"], c["block"], c["topk"], causal=c["causal"], **lengths)}
    if c["buckets"]:
        lengths.update(bias=s["bias"], bounds=s["bounds"])
    if not c["train"]:
        return {"out": ops.block_attention(s["q"], s["k"], s["v"], s["blocks"], c["block"], causal=c["causal"], **lengths)}
    leaves = {x: s[x].detach().requires_grad_() for x in ("q", "k", "v") + (("bias",) if c["buckets"] else ())}
    if c["buckets"]:
        lengths["bias"] = leaves["bias"]
    out = ops.block_attention(leaves["q"], leaves["k"], leaves["v"], s["blocks"], c["block"], causal=c["causal"], **lengths)
    grads = torch.autograd.grad(out, list(leaves.values()), s["dout"])
    return dict({"out": out.detach()}, **{"d" + x: g for x, g in zip(leaves, grads)})


def work(case):
    c = case
    size = _TYPES[c["dtype"]].itemsize
    b, n, m, h, hk, d = c["batch"], c["queries"], c["keys"], c["heads"], c["kv_heads"], c["head_len"]
    if c["ragged"]:
        m = m * 3 // 4
        n = m if c["queries"] == c["keys"] else n
    nb = -(-m // c["block"])
    lists = 4 * b * n * hk * c["topk"]
    if c["op"] == "select":
        pools = n == m                      # else the pooled keys are kept by the program
        return {"bytes": size * (b * n * h * d + b * hk * nb * d + (b * m * hk * d if pools else 0)) + lists,
                "flops": b * n * h * d + 2 * b * n * hk * nb * d + (b * m * hk * d if pools else 0)}
    # keys that a query attends to, and keys that any query reads
    most = min(c["topk"] * c["block"], m)
    pairs = sum(min(most, i + 1) for i in range(n)) if c["causal"] and n == m else n * most
    keys = min(m, n * most)
    rows = size * b * d
    passes, products = (2, 7) if c["train"] else (1, 2)
    once = rows * (2 * n * h + 2 * keys * hk) + lists
    if passes == 2:                         # q, k, v, dout, out in; dq, dk, dv out
        once += rows * (4 * n * h + 4 * keys * hk)
    return {"bytes": once, "flops": 2 * products * d * h * b * pairs}


# ---- the definition in 64 bits --------------------------------------------------------------------------


def _exact_select(s):
    c, q, k = s["case"], s["q"].double(), s["k"].double()
    b, n, m, hk, d, size = c["batch"], c["queries"], c["keys"], c["kv_heads"], c["head_len"], c["block"]
    group, nb = c["heads"] // hk, -(-m // size)
    dtype = s["q"].dtype
    kl, ql = [x.tolist() for x in _sizes(s)]
    pooled = torch.zeros((b, hk, nb, d), dtype=torch.float64, device=q.device)
    blocks = torch.full((b, n, hk, c["topk"]), -1, dtype=torch.int32, device=q.device)
    ids = torch.arange(nb, device=q.device)
    for i in range(b):
        for x in range(nb):
            if x * size < kl[i]:
                pooled[i, :, x] = k[i, x * size:min(kl[i], (x + 1) * size)].mean(0)
        means = pooled[i].float().to(dtype).double() if s["pooled"] is None else s["pooled"][i].double()
        for g in range(hk):
            rows = q[i, :ql[i], g * group:(g + 1) * group].sum(1).float().to(dtype).double()
            for r in range(0, ql[i], 512):
                part = rows[r:r + 512]
                score = torch.stack([(part * means[g, x]).sum(1) for x in range(nb)], 1)
                at = torch.arange(r, r + part.shape[0], device=q.device) + kl[i] - ql[i]
                last = at if c["causal"] else torch.full_like(at, kl[i] - 1)
                may = (ids * size <= last[:, None]) & (ids * size < kl[i])
                score[ids == last[:, None] // size] = math.inf
                if c["topk"] > 1:
                    score[:, 0] = math.inf
                # a block's rank: how many that may be chosen stand before it
                ahead = (score[:, None, :] > score[:, :, None]) | ((score[:, None, :] == score[:, :, None]) & (ids < ids[:, None]))
                rank = (ahead & may[:, None, :]).sum(2)
                taken = may & (rank < c["topk"])
                place = taken.cumsum(1) - 1
                row, block = taken.nonzero(as_tuple=True)
                blocks[i, r + row, g, place[row, block]] = block.to(torch.int32)
    return {"pooled": pooled if s["pooled"] is None else s["pooled"].double(), "blocks": blocks}


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "select":
        return _exact_select(s)
    b, n, m, h, hk, d, size = (c[x] for x in ("batch", "queries", "keys", "heads", "kv_heads", "head_len", "block"))
    group = h // hk
    kl, ql = [x.tolist() for x in _sizes(s)]
    q, k, v = s["q"], s["k"], s["v"]
    double = dict(dtype=torch.float64, device=q.device)
    got = {"out": torch.zeros((b, n, h, d), **double)}
    if c["train"]:
        got.update(dq=torch.zeros((b, n, h, d), **double), dk=torch.zeros((b, m, hk, d), **double), dv=torch.zeros((b, m, hk, d), **double))
        if c["buckets"]:
            got["dbias"] = torch.zeros((c["buckets"], h), **double)
    for i in range(b):
        rows, keys = ql[i], kl[i]
        at = torch.arange(rows, device=q.device) + keys - rows
        for g in range(hk):
            few = n < 16
            # the keys any of these rows may see: for a few rows those of their blocks alone, so that a long cache is not widened
            near = torch.arange(keys, device=q.device)
            if few:
                used = torch.unique(s["blocks"][i, :rows, g].clamp(min=-1))
                near = near[torch.isin(near // size, used)]
            kd, vd = k[i, near, g].double(), v[i, near, g].double()
            of_block = (near // size)
            open_ = torch.stack([(of_block[None] == s["blocks"][i, :rows, g, x, None]) for x in range(c["topk"])]).any(0)
            distance = at[:, None] - near
            if c["causal"]:
                open_ &= distance >= 0
            if c["buckets"]:
                bucket = sum((distance >= x).long() for x in s["bounds"])
            for e in range(g * group, (g + 1) * group):
                qd = q[i, :rows, e].double()
                z = qd @ kd.t() / math.sqrt(d)
                if c["buckets"]:
                    z = z + s["bias"][:, e].double()[bucket]
                z = torch.where(open_, z, -math.inf)
                a = torch.where(open_, torch.exp(z - torch.logsumexp(z, 1, keepdim=True)), 0.0)
                got["out"][i, :rows, e] = a @ vd
                if c["train"]:
                    do = s["dout"][i, :rows, e].double()
                    t = do @ vd.t()
                    z = a * (t - (a * t).sum(1, keepdim=True))
                    got["dv"][i, near, g] += a.t() @ do
                    got["dq"][i, :rows, e] = z @ kd / math.sqrt(d)
                    got["dk"][i, near, g] += z.t() @ qd / math.sqrt(d)
                    if c["buckets"]:
                        for x in range(c["buckets"]):
                            got["dbias"][x, e] += z[bucket == x].sum()
    return got
