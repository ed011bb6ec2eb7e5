"""Attention over a cache of 4 or 8 bits (ops.cache_attention): what rows that are padding cost, and values at the ends of their ranges."""
import numpy as np
import pytest

import cache_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def arbitrary(batch, keys, kv_heads, head_len, bits, seed=0):
    """A cache of arbitrary numbers of ordinary size."""
    from featgraph_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda low, high, row: torch.randint(low, high, (batch, kv_heads, keys, row), generator=gen, device="cuda", dtype=torch.uint8)
    codes = [new(0, 256 if bits == 4 else 127, head_len * bits // 8) for _ in "kv"]
    scales = [new(125, 128, head_len // 32) for _ in "kv"]
    return ops.KeyValueCache(codes[0], scales[0], codes[1], scales[1], bits)


def least_time(call, calls=5, tries=6):
    """Milliseconds of a call among others."""
    call()
    best = float("inf")
    for _ in range(tries):
        ends = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        ends[0].record()
        for _ in range(calls):
            call()
        ends[1].record()
        ends[1].synchronize()
        best = min(best, ends[0].elapsed_time(ends[1]) / calls)
    return best


@pytest.mark.parametrize("causal", [True, False])
def test_rows_behind_the_queries_walk_no_keys(causal):
    # 4,096 workgroups of 8 tokens each, many times what the card holds at once; with no token there none has anything to see
    from featgraph_amd import ops
    cache = arbitrary(64, 4096, 8, 128, 4)
    q = torch.randn((64, 64, 32, 128), device="cuda").to(BF16)
    few, none = torch.ones(64, dtype=torch.int32, device="cuda"), torch.zeros(64, dtype=torch.int32, device="cuda")
    took = [least_time(lambda: ops.cache_attention(q, cache, causal=causal, q_lengths=lengths)) for lengths in (None, few, none)]
    print("64 tokens %.3f ms, 1 of 64 %.3f ms, none %.3f ms" % tuple(took))
    assert took[2] < 0.25 * took[0] and took[1] < 0.75 * took[0]
    got = ops.cache_attention(q, cache, causal=causal, q_lengths=few)
    alone = ops.cache_attention(q[:, :1].contiguous(), cache, causal=causal)
    assert not got[:, 1:].any()
    # shares of the keys differ between the two calls, and so does the order of their sums
    torch.testing.assert_close(got[:, :1].float(), alone.float(), rtol=2.0 ** -7, atol=2.0 ** -7)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("head_len", [32, 64, 128])
@pytest.mark.parametrize("keys,queries", [(1, 1), (5, 3), (9001, 1), (700, 40)])
def test_float16_results_end_where_read_values_do(bits, head_len, keys, queries):
    # 65504 is held as 65536, every result is that value, and float16 ends between the two; 57344 is 65536 in 4 bits
    from featgraph_amd import ops
    cache = ops.new_cache(1, keys, 2, head_len, bits)
    x = torch.full((1, keys, 2, head_len), 65504.0, dtype=F16, device="cuda")
    x[..., 1::3] *= -1
    x[..., 2::3] = 57344.0
    ops.write_cache(cache, torch.randn(x.shape, device="cuda").to(F16), x)
    q = torch.randn((1, queries, 4, head_len), device="cuda").to(F16)
    held = ops.read_cache(cache, F16, count=1)[1][:, :, [0, 0, 1, 1]].expand_as(q)
    assert held.abs().max() == 65504
    lists = torch.arange(-(-keys // 32), dtype=torch.int32, device="cuda").expand(1, queries, 2, -1)
    for options in ({}, dict(causal=False), dict(blocks=lists, block_size=32)):
        got = ops.cache_attention(q, cache, **options)
        # an average of equal numbers is that number, within float16's step once sums are rounded
        assert torch.isfinite(got).all() and ((got - held).float().abs() <= 32).all() and torch.equal(got.abs() == 65504, held.abs() == 65504)
    cache.v_scales[0, 1, 0] = 255           # no numbers stay none
    got = ops.cache_attention(q, cache, causal=False)
    assert torch.isnan(got[:, :, 2:]).all() and torch.isfinite(got[:, :, :2]).all()


def check_large(q, cache, blocks=None, block_size=None, **options):
    """Powers of steps with large scales are 2^40 below their reference: the difference of score and reference is off by half a step of 32 bits at 2^6, 2^-18 at most
    (2^-19, and as much for what is added to a reference), powers below 2^-86 of the largest are lost, and what is lost of either reaches the sum of powers too."""
    from featgraph_amd import ops
    got = ops.cache_attention(q, cache, blocks, block_size, **options)
    k, v = ref.held(cache)
    out, bound = ref.attention(q, k, v, blocks, block_size, **options)
    assert np.isfinite(v).all()
    mean = ref.attention(q, k, np.abs(v), blocks, block_size, **options)[0]        # sum of p |v|
    ref.check(got, out, bound + 2 * np.log(2) * 2.0 ** -18 * mean + 2.0 ** -84 * cache.keys * np.abs(v).max())
    return got


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("keys,queries", [(1, 1), (2, 1), (300, 3), (9001, 1), (700, 40)])
def test_the_largest_values_of_a_cache_have_a_mean(bits, dtype, keys, queries):
    # sums of powers times values are beyond 32 bits, the result is not: 6 2^125 and 448 2^119, each with its sign
    from featgraph_amd import ops
    cache = ops.new_cache(2, keys, 2, 64, bits)
    largest = 6 * 2.0 ** 125 if bits == 4 else 448 * 2.0 ** 119
    x = torch.full((2, keys, 2, 64), largest, device="cuda")
    x[..., 1::2] *= -1
    ops.write_cache(cache, torch.randn(x.shape, device="cuda"), x)
    q = 3 * torch.randn((2, queries, 4, 64), device="cuda").to(dtype)
    lists = torch.arange(-(-keys // 32), dtype=torch.int32, device="cuda").expand(2, queries, 2, -1)
    for options in ({}, dict(causal=False), dict(blocks=lists, block_size=32)):
        got = check_large(q, cache, **options)
        assert (got[..., 0::2] > 0).all() and (got[..., 1::2] < 0).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,head_len", [(F32, 32), (BF16, 128), (F32, 128), (BF16, 64)])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
def test_values_of_very_different_sizes(bits, dtype, head_len, order):
    # sizes from 2^-20 to the largest, among them steps of 32 keys without a large one; scores that rise, fall or do neither along the keys
    from featgraph_amd import ops
    gen = torch.Generator().manual_seed(3)
    keys = 2000
    power = torch.where(torch.arange(keys) // 32 % 3 > 0, torch.randint(-20, 20, (keys,), generator=gen), torch.randint(70, 125, (keys,), generator=gen)).double()
    v = torch.randn((2, keys, 2, head_len), generator=gen).clamp(-3, 3).double() * torch.exp2(power)[:, None, None]
    k = torch.randn((2, keys, 2, head_len), generator=gen)
    if order != "mixed":
        k[..., :32] = torch.linspace(-1, 1, keys)[:, None, None] * (1 if order == "up" else -1)
    cache = ops.new_cache(2, keys, 2, head_len, bits)
    ops.write_cache(cache, k.cuda(), v.float().cuda())
    q = torch.randn((2, 3, 4, head_len), generator=gen)
    if order != "mixed":
        q = q.abs()
        q[..., :32] = 20 * head_len ** 0.5 / 32
    check_large((q * 2).to(dtype).cuda(), cache)
    few = torch.randint(0, 63, (2, 3, 2, 12), generator=gen, dtype=torch.int32).cuda()
    check_large((q * 2).to(dtype).cuda(), cache, few, 32)


def test_large_values_behind_what_a_row_sees_change_nothing():
    from featgraph_amd import ops
    cache = arbitrary(1, 500, 2, 64, 4)
    q = torch.randn((1, 3, 4, 64), device="cuda").to(BF16)
    clean = ops.cache_attention(q, cache, lengths=ints(400))
    cache.v_scales[:, :, 400:] = 250
    assert torch.equal(ops.cache_attention(q, cache, lengths=ints(400)), clean)
    cache.v_scales[:, :, 384:] = 250        # token 0 of three that end at 385 sees keys up to 383, and the step of 32 from 384 on only in passing
    got = ops.cache_attention(q, cache, lengths=ints(384 + 2), q_lengths=ints(3))
    clean = ops.cache_attention(q, cache, lengths=ints(384), q_lengths=ints(1))
    assert torch.equal(got[:, :1], clean[:, :1]) and torch.isfinite(got).all()


def test_many_equal_keys_far_apart():
    """Offsets beyond 32 bits again, bounded by the steps that are added up: 2^26 keys are cut into 256 shares of four wavefronts, so that one adds 2,048 steps of 32
    keys, in two parts each.  Every score is 0 and every power 1: their sums, of whole numbers up to 2^16, are exact, and values' sums are off by half a step of 32 bits for each addition."""
    from featgraph_amd import ops
    keys = 1 << 26
    cache = ops.new_cache(1, keys, 1, 32, 4)
    gen = torch.Generator(device="cuda").manual_seed(4)
    cache.v.copy_(torch.randint(0, 256, (16,), generator=gen, device="cuda", dtype=torch.uint8))        # the same key everywhere
    cache.v_scales.fill_(127)
    q = torch.randn((1, 1, 4, 32), device="cuda")
    got = ops.cache_attention(q, cache)
    want = ops.read_cache(cache, F32, count=1)[1].expand_as(q)
    assert ((got - want).abs() <= (2048 * 32 + 256 * 4) * 2.0 ** -24 * want.abs()).all()
    del cache


def test_sizes_are_whole_numbers_whatever_holds_them():
    from featgraph_amd import ops
    cache = arbitrary(2, 70, 2, 64, 4)
    other = ops.KeyValueCache(cache.k, cache.k_scales, cache.v, cache.v_scales, 4.0)
    q = torch.randn((2, 1, 4, 64), device="cuda")
    blocks = torch.zeros((2, 1, 2, 1), dtype=torch.int32, device="cuda")
    right = ops.cache_attention(q, cache, blocks, 32)
    assert torch.equal(ops.cache_attention(q, other, blocks, 32.0), right) and torch.equal(ops.cache_attention(q, cache, blocks, np.int64(32)), right)
    assert torch.equal(ops.read_cache(other, F32, count=np.int64(3))[0], ops.read_cache(cache, F32, count=3)[0])
    with pytest.raises(TypeError):
        ops.read_cache(cache, count=3.0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype,queries", [(F32, 1), (F16, 3), (BF16, 40)])
def test_large_values_beside_ones_that_are_no_numbers(bits, dtype, queries):
    # both in one step of 32 keys; float16 results end at 65504
    from featgraph_amd import ops
    cache = arbitrary(1, 200, 2, 64, bits)
    cache.v_scales[:, :, 128:160, 0] = 200 if bits == 8 else 240
    cache.v_scales[:, :, 140, 1] = 255
    q = torch.randn((1, queries, 4, 64), device="cuda").to(dtype)
    got = ops.cache_attention(q, cache)
    assert torch.isnan(got[..., 32:]).all() and torch.isfinite(got[..., :32]).all()
    if dtype == F16:
        assert got[..., :32].abs().max() == 65504
    else:
        cache.v_scales[:, :, 140, 1] = 127  # numbers again: the others keep their bits
        assert torch.equal(ops.cache_attention(q, cache)[..., :32], got[..., :32])
        if bits == 4:
            check_large(q, cache)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_values_captured(dtype):
    from featgraph_amd import ops
    cache = arbitrary(2, 3000, 2, 64, 4)
    q = torch.randn((2, 1, 4, 64), device="cuda").to(dtype)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.cache_attention(q, cache)
    for scale in (127, 250, 130, 251):
        cache.v_scales[:, :, 1000:1100] = scale
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.cache_attention(q, cache)) and torch.isfinite(out).all()
