"""Attention over a cache of 4 or 8 bits (ops.cache_attention) against the definition in 64 bits."""
import numpy as np
import pytest

import cache_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(dtype=BF16, batch=2, queries=1, keys=70, heads=4, kv_heads=2, head_len=64, bits=4, topk=0, block=32, seed=0):
    """(q, cache, options); every query names its own block and topk - 1 drawn ones, behind the keys and -1 among them."""
    from featgraph_amd import ops
    gen = torch.Generator().manual_seed(seed)
    new = lambda *shape: torch.randn(shape, generator=gen)
    cache = ops.new_cache(batch, keys, kv_heads, head_len, bits)
    if keys:
        ops.write_cache(cache, new(batch, keys, kv_heads, head_len).to(dtype).cuda(), new(batch, keys, kv_heads, head_len).to(dtype).cuda())
    options = {}
    if topk:
        nb = -(-keys // block)
        blocks = torch.randint(-1, nb + 1, (batch, queries, kv_heads, topk), generator=gen, dtype=torch.int32)
        blocks[..., 0] = ((torch.arange(queries) + keys - queries).clamp(min=0) // block)[None, :, None]
        options = dict(blocks=blocks.cuda(), block_size=block)
    return new(batch, queries, heads, head_len).to(dtype).cuda(), cache, options


def want(q, cache, blocks=None, block_size=None, **options):
    return ref.attention(q, *ref.held(cache), blocks, block_size, **options)


def check(q, cache, **options):
    from featgraph_amd import ops
    got = ops.cache_attention(q, cache, **options)
    ref.check(got, *want(q, cache, **options), what=str(sorted(options)))
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("head_len", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 2), (3, 1), (8, 1), (16, 1), (14, 2)])
def test_types_and_groups(bits, dtype, head_len, heads, kv_heads):
    for topk in (0, 2):
        q, cache, options = make(dtype, 2, 3, 70, heads, kv_heads, head_len, bits, topk)
        check(q, cache, **options)


@pytest.mark.parametrize("bits,dtype,head_len", [(4, BF16, 128), (8, F32, 64), (4, F16, 32), (8, BF16, 128)])
@pytest.mark.parametrize("queries,keys", [(1, 1), (1, 2), (1, 31), (1, 32), (1, 33), (2, 2), (1, 700), (5, 1000), (17, 17), (3, 4097), (40, 129), (64, 64), (100, 515)])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(bits, dtype, head_len, queries, keys, causal):
    q, cache, _ = make(dtype, 2, queries, keys, 4, 2, head_len, bits, seed=1)
    check(q, cache, causal=causal)


@pytest.mark.parametrize("bits,dtype,head_len", [(4, BF16, 128), (8, F16, 64), (4, F32, 32)])
@pytest.mark.parametrize("queries,keys,block,topk,causal", [(1, 700, 64, 5, True), (5, 1000, 128, 8, True), (3, 257, 32, 9, False), (33, 257, 32, 4, True),
                                                            (2, 6000, 64, 94, True), (1, 513, 256, 1, True), (20, 640, 128, 5, False)])
def test_blocks(bits, dtype, head_len, queries, keys, block, topk, causal):
    q, cache, options = make(dtype, 2, queries, keys, 6, 2, head_len, bits, topk, block, seed=2)
    check(q, cache, causal=causal, **options)
    if topk == 94:                          # all of them: as without a list
        options["blocks"][:] = torch.arange(94, dtype=torch.int32, device="cuda")
        check(q, cache, causal=causal, **options)


def test_more_blocks_than_one_window():
    q, cache, options = make(F32, 1, 2, 70001, 2, 1, 32, 4, 40, 32, seed=3)
    check(q, cache, **options)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("batch,heads,kv_heads,head_len", [(1, 8, 8, 64), (2, 32, 8, 128), (32, 4, 1, 128), (3, 5, 5, 32)])
def test_long_caches(bits, batch, heads, kv_heads, head_len):
    q, cache, _ = make(BF16, batch, 1, 9001, heads, kv_heads, head_len, bits, seed=4)
    lengths = torch.linspace(1, 9001, batch).int().cuda()
    check(q, cache, lengths=lengths)


@pytest.mark.parametrize("topk", [0, 3])
@pytest.mark.parametrize("causal", [True, False])
def test_ragged_batch_with_rubbish_behind_the_lengths(topk, causal):
    from featgraph_amd import ops
    q, cache, options = make(BF16, 5, 6, 130, 4, 2, 64, 4, topk, 32, seed=5)
    options.update(lengths=ints(130, 77, 1, 0, 40), q_lengths=ints(6, 5, 1, 3, 0), causal=causal)
    right = want(q, cache, **options)
    for b in range(5):
        n, m = int(options["q_lengths"][b]), int(options["lengths"][b])
        q[b, n:] = float("nan")
        cache.k_scales[b, :, m:] = 255      # no numbers
        cache.v_scales[b, :, m:] = 255
    got = ops.cache_attention(q, cache, **options)
    ref.check(got, *right)
    for b in range(5):
        assert not got[b, int(options["q_lengths"][b]):].any()
    assert not got[3].any()


def test_counts_outside_the_tensors_are_clamped():
    from featgraph_amd import ops
    q, cache, _ = make()
    full = ops.cache_attention(q, cache)
    assert torch.equal(full, ops.cache_attention(q, cache, lengths=ints(1000, 70), q_lengths=ints(1, 2 ** 31 - 1)))
    assert not ops.cache_attention(q, cache, lengths=ints(-5, 0)).any()
    assert not ops.cache_attention(q, cache, q_lengths=ints(-5, 0)).any()


def test_rows_that_see_nothing():
    # more queries than keys: the first stand before key 0; lists that name nothing
    q, cache, _ = make(F32, 2, 9, 70, seed=6)
    got = check(q, cache, lengths=ints(4, 70), q_lengths=ints(9, 9))
    assert not got[0, :5].any() and got[0, 5:].any()
    q, cache, options = make(F32, 2, 9, 70, topk=3, seed=6)
    options["blocks"][0], options["blocks"][1, 2] = -1, 7
    got = check(q, cache, **options)
    assert not got[0].any() and not got[1, 2].any()


def test_lists_in_any_order_twice_the_same_and_beyond():
    from featgraph_amd import ops
    q, cache, options = make(BF16, 2, 4, 500, topk=6, seed=7)
    one = ops.cache_attention(q, cache, **options)
    blocks = options["blocks"]
    other = torch.cat((blocks.flip(3), blocks[..., :2], torch.full_like(blocks[..., :1], 2 ** 31 - 1), torch.full_like(blocks[..., :1], -2 ** 31)), 3)
    assert torch.equal(one, ops.cache_attention(q, cache, blocks=other, block_size=32))


def test_empty():
    from featgraph_amd import ops
    for change in (dict(batch=0), dict(queries=0)):
        assert ops.cache_attention(*make(**change)[:2]).numel() == 0
    got = ops.cache_attention(*make(keys=0)[:2])
    assert got.shape == (2, 1, 4, 64) and not got.any()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("topk", [0, 8])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(bits, dtype, topk):
    from featgraph_amd import ops
    q, cache, options = make(dtype, 1, 5, 200, 4, 2, 64, bits, topk, 32, seed=8)
    if topk:
        options["blocks"][:] = torch.arange(8, dtype=torch.int32, device="cuda")
    clean = ops.cache_attention(q, cache, **options)
    # key 197 of head 0: seen by tokens 2, 3 and 4 of five whose last one stands at 199
    cache.v_scales[0, 0, 197, 1] = 255
    got = ops.cache_attention(q, cache, **options)
    bad = torch.zeros_like(got, dtype=torch.bool)
    bad[0, 2:, :2, 32:] = True
    assert torch.equal(torch.isnan(got), bad)
    assert torch.equal(got[~bad], clean[~bad])
    cache.k_scales[0, 1, 198, 0] = 255
    got = ops.cache_attention(q, cache, **options)
    bad[0, 3:, 2:] = True
    assert torch.equal(torch.isnan(got), bad)
    q[0, 0, 0, 0], q[0, 1, 3, 5] = float("inf"), float("nan")
    got = ops.cache_attention(q, cache, **options)
    assert torch.isnan(got[0, 1, 3]).all() and not torch.isnan(got[0, 1, 2]).any() and not torch.isnan(got[0, 0, 1:]).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_large_scores_and_scales(dtype):
    # one key takes all: its value to the last bit; and a softmax of one reference far from 0
    q, cache, _ = make(dtype, 2, 2, 300, seed=9)
    check(q * 30, cache)
    for scale in (0.0, -0.7, 3.0):
        check(q, cache, scale=scale)
    k, v = ref.held(cache)
    big = torch.from_numpy(k[:, :, 250]).float().cuda().repeat_interleave(2, 1)[:, None].expand(2, 2, 4, 64)
    from featgraph_amd import ops
    got = ops.cache_attention((big * 8).to(dtype), cache)[0, 0].cpu()
    want_v = torch.from_numpy(v[0, :, 250]).repeat_interleave(2, 0).to(dtype)
    # the others weigh e^-40 and less: far below half a step of a number, but what stands beside a value of 0
    assert torch.equal(torch.where(want_v == 0, 0, got), want_v) and (got[want_v == 0].float().abs() < 2.0 ** -30).all()


def test_float32_queries_keep_their_bits():
    # numbers of 24 bits near the largest and the smallest: parts of them are cut, never rounded up beyond the range
    from featgraph_amd import ops
    cache = ops.new_cache(1, 3, 1, 32)
    x = torch.zeros((1, 3, 1, 32), device="cuda")
    x[0, 0, 0, 0], x[0, 1, 0, 1], x[0, 2, 0, 2] = 1.0, 1.0, 1.0
    ops.write_cache(cache, x, x)
    q = torch.zeros((1, 1, 1, 32), device="cuda")
    q[..., 0], q[..., 1], q[..., 2] = 1 + 2.0 ** -23, 1.0, 1 + 2.0 ** -12
    for size in (2.0 ** 15, 2.0 ** 100):
        got = ops.cache_attention(q * size, cache, scale=1 / size * 1024, causal=False)
        z = np.array([1 + 2.0 ** -23, 1.0, 1 + 2.0 ** -12]) * 1024
        p = np.exp(z - z.max())
        p /= p.sum()
        assert np.abs(got[0, 0, 0, :3].cpu().double().numpy() - p).max() <= 1024 * 8 * 2.0 ** -23
    q[..., 3] = torch.finfo(F32).max
    assert torch.isfinite(ops.cache_attention(q, cache, scale=1.0, causal=False)).all()


def test_strides():
    from featgraph_amd import ops
    q, cache, options = make(F16, 3, 2, 100, topk=3, seed=10)
    right = ops.cache_attention(q, cache, **options)
    fused = torch.zeros((3, 2, 8, 64), dtype=F16, device="cuda")
    fused[:, :, 2:6] = q
    shifted = torch.empty(q.numel() + 1, dtype=F16, device="cuda")[1:].view(q.shape).copy_(q)
    for x in (fused[:, :, 2:6], q.transpose(0, 1).contiguous().transpose(0, 1), shifted, q.flip(3).contiguous().flip(3)):
        assert torch.equal(right, ops.cache_attention(x, cache, **options))
    blocks = options["blocks"].transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(right, ops.cache_attention(q, cache, blocks=blocks, block_size=32))
    one = q[:, :, :1].expand_as(q)
    assert torch.equal(ops.cache_attention(one, cache), ops.cache_attention(one.contiguous(), cache))


def test_refusals():
    from featgraph_amd import ops
    q, cache, options = make(topk=2)
    blocks = options["blocks"]
    for bad in (lambda: ops.cache_attention(q[:, :, :3], cache), lambda: ops.cache_attention(q[..., :32], cache), lambda: ops.cache_attention(q[:1], cache),
                lambda: ops.cache_attention(q[:, :, :0], cache), lambda: ops.cache_attention(q.cpu(), cache), lambda: ops.cache_attention(q.double(), cache),
                lambda: ops.cache_attention(q[0], cache), lambda: ops.cache_attention(q, cache, blocks=blocks), lambda: ops.cache_attention(q, cache, block_size=32),
                lambda: ops.cache_attention(q, cache, blocks=blocks, block_size=48), lambda: ops.cache_attention(q, cache, blocks=blocks.long(), block_size=32),
                lambda: ops.cache_attention(q, cache, blocks=blocks[..., :0], block_size=32), lambda: ops.cache_attention(q, cache, blocks=blocks[:, :, :1], block_size=32),
                lambda: ops.cache_attention(q, cache, lengths=ints(1)), lambda: ops.cache_attention(q, cache, q_lengths=ints(1, 1).long())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.cache_attention(q, cache, blocks=[0, 1], block_size=32)
    leaf = q.clone().requires_grad_()
    with pytest.raises(NotImplementedError, match="no gradient"):
        ops.cache_attention(leaf, cache)
    with torch.no_grad():
        assert torch.equal(ops.cache_attention(leaf, cache), ops.cache_attention(q, cache))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.cache_attention(dual, cache)


def test_offsets_beyond_32_bits():
    from featgraph_amd import ops
    keys = (1 << 26) + 77                   # 4.3 GB of codes in a head
    cache = ops.new_cache(1, keys, 2, 128, 4)
    gen = torch.Generator().manual_seed(11)
    k, v, q = (torch.randn((1, 40, n, 128), generator=gen).to(BF16).cuda() for n in (2, 2, 4))
    q = q[:, :1] * 8                        # so that the zeros before weigh little
    ops.write_cache(cache, k, v)
    got = ops.cache_attention(q, cache)
    # the rest of the cache: scores of 0 and values of 0
    near = [ref.values(*ref.quantise(x.cpu().double().numpy().transpose(0, 2, 1, 3), 4), 4) for x in (k, v)]
    z = np.einsum("hd,hkd->hk", q[0, 0].cpu().double().numpy(), np.repeat(near[0][0], 2, 0)) * 128 ** -0.5
    top = np.maximum(z.max(1, keepdims=True), 0)
    p = np.exp(z - top)
    total = p.sum(1, keepdims=True) + (keys - 40) * np.exp(-top)
    p /= total
    values = np.repeat(near[1][0], 2, 0)
    # sums of 2^26 equal terms in 32 bits, each wavefront's share one after the other: up to 2^26 / 32 / 4 steps of 2^-24 where one adds all
    out, bound = np.einsum("hk,hkd->hd", p, values), (2.0 ** -8 + 0.05) * np.einsum("hk,hkd->hd", p, np.abs(values)) + 1e-6
    assert (np.abs(got[0, 0].cpu().double().numpy() - out) <= bound).all()
    blocks = torch.tensor([keys // 64, keys // 64 - 1, 0], dtype=torch.int32, device="cuda").view(1, 1, 1, 3).expand(1, 1, 2, 3)
    got = ops.cache_attention(q, cache, blocks=blocks, block_size=64)
    seen = keys - (keys // 64 - 1) * 64 + 64
    p = np.exp(z - top)
    p /= p.sum(1, keepdims=True) + (seen - 40) * np.exp(-top)
    out = np.einsum("hk,hkd->hd", p, values)
    bound = 2.0 ** -8 * np.abs(out) + (2.0 ** -17 + 400 * 128 * 2.0 ** -23) * np.einsum("hk,hkd->hd", p, np.abs(values))
    assert (np.abs(got[0, 0].cpu().double().numpy() - out) <= bound).all()


def test_the_same_bits_on_every_call_and_two_streams_at_once():
    from featgraph_amd import ops
    q, cache, _ = make(BF16, 2, 1, 20000, 32, 8, 128, seed=12)
    other, second, _ = make(BF16, 2, 1, 20000, 32, 8, 128, seed=13)
    first, right = ops.cache_attention(q, cache), ops.cache_attention(other, second)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for s, x, c, to in zip(streams, (q, other), (cache, second), got):
            with torch.cuda.stream(s):
                to.append(ops.cache_attention(x, c))
    torch.cuda.synchronize()
    assert all(torch.equal(first, x) for x in got[0]) and all(torch.equal(right, x) for x in got[1])


def test_captured():
    from featgraph_amd import ops
    q, cache, _ = make(BF16, 2, 1, 5000, 8, 2, 128, seed=14)
    lengths = ints(5000, 4)
    graphs, outs = [], []
    for _ in range(2):                      # two graphs share no workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(ops.cache_attention(q, cache, lengths=lengths))
        graphs.append(graph)
    for i in range(4):
        q.copy_(make(BF16, 2, 1, 1, 8, 2, 128, seed=20 + i)[0])
        lengths.sub_(1)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        right = ops.cache_attention(q, cache, lengths=lengths)
        assert torch.equal(outs[0], right) and torch.equal(outs[1], right)


def test_a_decoding_layer():
    """Norms and positions, the new key into the cache, the block's mean renewed, blocks chosen, attention over them: a prompt, then tokens one by
    one and three at a time, equal to a layer that keeps its keys in float32 as the cache rounds them."""
    from featgraph_amd import ops
    gen = torch.Generator().manual_seed(15)
    batch, room, heads, kv_heads, head_len, block, topk = 3, 400, 8, 2, 64, 32, 4
    weights = tuple(1 + 0.2 * torch.randn(head_len, generator=gen).to(BF16).cuda() for _ in "qk")
    for bits in (4, 8):
        cache = ops.new_cache(batch, room, kv_heads, head_len, bits)
        pooled = torch.zeros((batch, kv_heads, -(-room // block), head_len), dtype=BF16, device="cuda")
        plain = [torch.zeros((batch, room, kv_heads, head_len), device="cuda") for _ in "kv"]
        lengths = ints(0, 0, 0)
        for tokens, new in ((250, ints(250, 31, 180)), (1, None), (1, None), (3, ints(3, 2, 1)), (1, ints(1, 0, 1)), (1, None)):
            fused = torch.randn((batch, tokens, heads + 2 * kv_heads, head_len), generator=gen).to(BF16).cuda()
            added = ints(*[tokens] * batch) if new is None else new
            lengths = lengths + added
            q, k = ops.rotate_heads(fused[:, :, :heads], fused[:, :, heads:heads + kv_heads], *weights, lengths=lengths, q_lengths=new)
            v = fused[:, :, heads + kv_heads:]
            ops.write_cache(cache, k, v, lengths, new)
            for b in range(batch):
                m, n = int(lengths[b]), int(added[b])
                for to, x in zip(plain, (k, v)):
                    if n:
                        to[b, m - n:m] = torch.from_numpy(ref.values(*ref.quantise(x[b, :n].cpu().double().numpy(), bits), bits)).float().cuda()
            if tokens > 3:                  # the prompt's means at once
                pooled = ops.pool_blocks(ops.read_cache(cache, lengths=lengths)[0], block, lengths)
            else:                           # the last two blocks of each, which hold the new keys
                first = ((lengths - 1).clamp(min=0) // block - 1).clamp(min=0)
                window = ops.read_cache(cache, first=first * block, count=2 * block, lengths=lengths)[0]
                means = ops.pool_blocks(window, block, (lengths - first * block).int())
                at = (first[:, None] + torch.arange(2, dtype=torch.int32, device="cuda")).long()
                pooled.scatter_(2, at[:, None, :, None].expand(-1, kv_heads, -1, head_len), means)
            assert torch.equal(pooled, ops.pool_blocks(plain[0].to(BF16), block, lengths))
            blocks = ops.select_blocks(q, pooled, room, block, topk, lengths=lengths, q_lengths=new)
            held = ref.held(cache)
            for x, y in zip(held, plain):
                for b in range(batch):
                    m = int(lengths[b])
                    assert np.array_equal(x[b, :, :m], y[b, :m].transpose(0, 1).cpu().double().numpy())
            for options in (dict(blocks=blocks, block_size=block), {}):
                got = ops.cache_attention(q, cache, lengths=lengths, q_lengths=new, **options)
                ref.check(got, *want(q, cache, lengths=lengths, q_lengths=new, **options))
            near = ops.block_attention(q, plain[0].to(BF16), plain[1].to(BF16), blocks, block, lengths=lengths, q_lengths=new)
            listed = ops.cache_attention(q, cache, blocks, block, lengths=lengths, q_lengths=new)
            # both round the same sum; two roundings to bfloat16 and the powers' own in the other operator
            assert (near.float() - listed.float()).abs().max() <= 2.0 ** -6 * listed.float().abs().max()
