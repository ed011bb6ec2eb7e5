"""Attention over a cache of 4 or 8 bits (ops.cache_attention): what rows that are padding cost, and values at the ends of their ranges."""
import pytest

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
