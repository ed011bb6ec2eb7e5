"""Writing keys and values into a cache of 4 or 8 bits and reading them back (ops.write_cache, ops.read_cache): equal to the definition bit by bit."""
import numpy as np
import pytest

import cache_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def rubbish(batch, keys, kv_heads, head_len, bits, seed=0):
    """A cache full of arbitrary codes and ordinary scales."""
    from featgraph_amd import ops
    gen = torch.Generator().manual_seed(seed)
    row = head_len * bits // 8
    codes = lambda: torch.randint(0, 256, (batch, kv_heads, keys, row), generator=gen, dtype=torch.uint8).cuda()
    scales = lambda: torch.randint(100, 140, (batch, kv_heads, keys, head_len // 32), generator=gen, dtype=torch.uint8).cuda()
    return ops.KeyValueCache(codes(), scales(), codes(), scales(), bits)


def parts(cache):
    return [t.cpu().numpy().copy() for t in (cache.k, cache.k_scales, cache.v, cache.v_scales)]


def expected(cache, k, v, lengths, q_lengths):
    """What parts(cache) has to be after a write."""
    held = parts(cache)
    tokens = k.shape[1]
    for b in range(cache.batch):
        n = tokens if q_lengths is None else min(max(int(q_lengths[b]), 0), tokens)
        m = cache.keys if lengths is None else min(max(int(lengths[b]), 0), cache.keys)
        for i in range(n):
            at = m - n + i
            if at < 0:
                continue
            for x, codes, scales in ((k, held[0], held[1]), (v, held[2], held[3])):
                codes[b, :, at], scales[b, :, at] = ref.quantise(x[b, i].cpu().double().numpy(), cache.bits)
    return held


def check_write(cache, k, v, lengths=None, q_lengths=None):
    from featgraph_amd import ops
    want = expected(cache, k, v, lengths, q_lengths)
    ops.write_cache(cache, k, v, lengths, q_lengths)
    for name, a, b in zip(("k", "k_scales", "v", "v_scales"), parts(cache), want):
        assert np.array_equal(a, b), (name, np.argwhere(a != b)[:3])


def values_of(kind, shape, dtype, gen):
    x = torch.randn(shape, generator=gen)
    if kind == "sizes":                     # rows of very different sizes
        x = x * torch.exp2(torch.randint(-20, 12, shape[:-1] + (1,), generator=gen).float())
    elif kind == "ties":                    # halfway between elements, and next to it
        x = torch.randint(-64, 65, shape, generator=gen).float() / 8
        x = x * torch.exp2(torch.randint(-8, 9, shape[:-1] + (1,), generator=gen).float())
    elif kind == "zeros":
        x = torch.where(torch.rand(shape, generator=gen) < 0.9, torch.zeros(()), x)
    return x.to(dtype).cuda()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("head_len", [32, 64, 128])
@pytest.mark.parametrize("kind", ["normal", "sizes", "ties", "zeros"])
def test_values(bits, dtype, head_len, kind):
    gen = torch.Generator().manual_seed(1)
    k, v = (values_of(kind, (2, 21, 3, head_len), dtype, gen) for _ in "kv")
    check_write(rubbish(2, 40, 3, head_len, bits), k, v)


@pytest.mark.parametrize("bits", [4, 8])
def test_borders_of_the_scale(bits):
    # the largest value a step below, on and above the border at which the scale doubles, for many powers; -0, subnormal numbers, the largest ones
    border = np.float32(7.0 if bits == 4 else 464.0)
    rows = []
    for power in list(range(-140, -120)) + [-30, -1, 0, 1, 30] + list(range(110, 126)):
        for x in (np.nextafter(border, np.float32(0)), border, np.nextafter(border, np.float32(1000))):
            with np.errstate(over="ignore"):
                top = np.float32(np.ldexp(np.float64(x), power))
            row = np.linspace(0, 1, 32, dtype=np.float32) * (top if np.isfinite(top) else np.float32(3e38))
            row[3], row[7] = -0.0, np.float32(1e-45)
            rows.append(row)
    rows.append(np.full(32, np.finfo(np.float32).max, np.float32))
    rows.append(np.zeros(32, np.float32))
    rows = np.stack(rows)
    x = torch.from_numpy(rows).cuda().view(1, -1, 1, 32)
    cache = rubbish(1, x.shape[1], 1, 32, bits)
    check_write(cache, x, -x)
    from featgraph_amd import ops
    k, v = ref.held(cache)
    got = ops.read_cache(cache, F32)
    assert np.array_equal(got[0].cpu().double().numpy(), k.transpose(0, 2, 1, 3)) and np.array_equal(got[1].cpu().double().numpy(), v.transpose(0, 2, 1, 3))
    assert torch.isfinite(got[0]).all()


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_what_is_not_finite_marks_its_32(bits, dtype):
    from featgraph_amd import ops
    gen = torch.Generator().manual_seed(2)
    k, v = (torch.randn((1, 5, 2, 128), generator=gen).to(dtype).cuda() for _ in "kv")
    k[0, 1, 0, 40], k[0, 2, 1, 127], v[0, 4, 1, 0] = float("nan"), float("inf"), float("-inf")
    cache = rubbish(1, 8, 2, 128, bits)
    check_write(cache, k, v)
    back = ops.read_cache(cache, dtype, first=ints(3), count=5)
    for x, places in ((back[0], [(1, 0, 1), (2, 1, 3)]), (back[1], [(4, 1, 0)])):
        bad = torch.zeros((5, 2, 4), dtype=torch.bool)
        for i, g, group in places:
            bad[i, g, group] = True
        assert torch.equal(torch.isnan(x[0]).cpu().view(5, 2, 4, 32), bad[..., None].expand(5, 2, 4, 32))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("batch,tokens,keys,kv_heads,head_len", [(1, 1, 1, 1, 32), (3, 1, 70, 2, 64), (2, 5, 5, 1, 128), (1, 257, 300, 3, 32), (4, 2, 1000, 8, 128)])
def test_lengths(bits, batch, tokens, keys, kv_heads, head_len):
    gen = torch.Generator().manual_seed(3)
    k, v = (torch.randn((batch, tokens, kv_heads, head_len), generator=gen).to(BF16).cuda() for _ in "kv")
    check_write(rubbish(batch, keys, kv_heads, head_len, bits), k, v)
    lengths = torch.randint(0, keys + 1, (batch,), generator=gen, dtype=torch.int32).cuda()
    q_lengths = torch.randint(0, tokens + 1, (batch,), generator=gen, dtype=torch.int32).cuda()
    check_write(rubbish(batch, keys, kv_heads, head_len, bits), k, v, lengths, q_lengths)


def test_counts_outside_the_tensors_are_clamped():
    gen = torch.Generator().manual_seed(4)
    k, v = (torch.randn((5, 6, 2, 32), generator=gen).cuda() for _ in "kv")
    for b, n in ((2, 0), (3, 0)):
        k[b, n:] = float("nan")
    check_write(rubbish(5, 9, 2, 32, 4), k, v, ints(2 ** 31 - 1, 3, 9, -8, -2 ** 31), ints(6, 100, 0, -5, 2 ** 31 - 1))


def test_more_tokens_than_room_keep_the_last_ones():
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn((2, 12, 1, 32), generator=gen).cuda() for _ in "kv")
    check_write(rubbish(2, 8, 1, 32, 8), k, v, ints(8, 4), ints(12, 7))
    check_write(rubbish(2, 8, 1, 32, 4), k, v, ints(8, 4))
    check_write(rubbish(2, 8, 1, 32, 4), k, v, None, ints(3, 0))


def test_a_cache_stays_as_it_was_made():
    import copy
    from featgraph_amd import ops
    cache = rubbish(1, 8, 1, 32, 4)
    with pytest.raises(AttributeError, match="as it was made"):
        cache.k = torch.zeros(1)
    other = copy.deepcopy(cache)
    x = torch.randn((1, 1, 1, 32), device="cuda")
    before = parts(cache)
    ops.write_cache(other, x, x)
    assert all(np.array_equal(a, b) for a, b in zip(before, parts(cache))) and not np.array_equal(before[0], parts(other)[0])
    for bad in (lambda: ops.KeyValueCache(cache.k[:, :, ::2], cache.k_scales, cache.v, cache.v_scales, 4), lambda: ops.KeyValueCache(cache.k, cache.k_scales, cache.v, cache.v_scales, 8),
                lambda: ops.KeyValueCache(cache.k, cache.v, cache.v, cache.v_scales, 4), lambda: ops.KeyValueCache(cache.k.int(), cache.k_scales, cache.v, cache.v_scales, 4),
                lambda: ops.write_cache(cache, x.expand(1, 9, 1, 32), x.expand(1, 9, 1, 32)), lambda: ops.write_cache(cache, x[..., :16], x[..., :16]),
                lambda: ops.write_cache(cache, x, x.half()), lambda: ops.write_cache(cache, x, x, lengths=torch.ones(1, device="cuda")),
                lambda: ops.write_cache(cache, x.expand(2, 1, 1, 32), x.expand(2, 1, 1, 32)), lambda: ops.read_cache(cache, torch.float64),
                lambda: ops.read_cache(cache, count=-1), lambda: ops.read_cache(cache, first=ints(1, 2)), lambda: ops.write_cache(cache, x.cpu(), x.cpu())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(NotImplementedError):
        ops.write_cache(cache, x.clone().requires_grad_(), x)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("head_len", [32, 64, 128])
def test_reading(bits, dtype, head_len):
    from featgraph_amd import ops
    cache = rubbish(3, 50, 2, head_len, bits, seed=6)
    if bits == 8:                           # no NaN among the arbitrary codes
        for t in (cache.k, cache.v):
            t[(t & 127) == 127] = 3
    k, v = ref.held(cache)
    for first, count, lengths in ((None, None, None), (ints(0, 7, 45), 9, None), (ints(0, 7, 45), 9, ints(50, 10, 49)), (ints(-3, -100, 60), 20, None),
                                  (ints(2 ** 31 - 1, -2 ** 31, 49), 1, ints(50, 50, 1000)), (None, 0, None), (None, 60, ints(-1, 0, 55))):
        got = ops.read_cache(cache, dtype, first=first, count=count, lengths=lengths)
        for x, y in zip(got, (k, v)):
            want = torch.zeros((3, 50 if count is None else count, 2, head_len), dtype=dtype)
            for b in range(3):
                for i in range(want.shape[1]):
                    at = i + (0 if first is None else int(first[b]))
                    if 0 <= at < min(50, 50 if lengths is None else int(lengths[b])):
                        want[b, i] = ref.as_type(y[b, :, at], dtype)
            assert torch.equal(x.cpu(), want)


def test_float16_takes_no_infinity():
    from featgraph_amd import ops
    x = torch.full((1, 1, 1, 32), 65504.0, dtype=F16, device="cuda")
    for bits in (4, 8):
        cache = ops.new_cache(1, 1, 1, 32, bits)
        ops.write_cache(cache, x, -x)
        k, v = ops.read_cache(cache, F16)
        assert (k == 65504).all() and (v == -65504).all()
        assert (ops.read_cache(cache, BF16)[0] == 65536).all()


def test_a_new_cache_holds_zeros_and_what_is_written_again_stays():
    from featgraph_amd import ops
    gen = torch.Generator().manual_seed(7)
    for bits in (4, 8):
        cache = ops.new_cache(2, 33, 2, 64, bits)
        assert not any(x.any() for x in ops.read_cache(cache, F32))
        x = torch.randn((2, 33, 2, 64), generator=gen).cuda()
        ops.write_cache(cache, x, 2 * x)
        k, v = ops.read_cache(cache, F32)
        assert torch.equal(v, 2 * k)        # a power of two only moves the scale
        ops.write_cache(cache, k, v)
        assert torch.equal(ops.read_cache(cache, F32)[0], k)


def test_strides():
    gen = torch.Generator().manual_seed(8)
    fused = torch.randn((2, 7, 10, 64), generator=gen).to(F16).cuda()
    k, v = fused[:, :, 3:5], fused[:, :, 8:10]
    check_write(rubbish(2, 7, 2, 64, 4), k, v)
    check_write(rubbish(2, 7, 2, 64, 4), k.transpose(1, 2).contiguous().transpose(1, 2), v.flip(3).contiguous().flip(3))
    check_write(rubbish(2, 7, 2, 64, 4), k[:, :, :1].expand(2, 7, 2, 64), v[:, :1].expand(2, 7, 2, 64))
    shifted = torch.empty(k.numel() + 1, dtype=F16, device="cuda")[1:].view(k.shape).copy_(k)
    check_write(rubbish(2, 7, 2, 64, 8), shifted, v)


def test_offsets_beyond_32_bits():
    from featgraph_amd import ops
    keys = (1 << 26) + 100                  # 4.3 GB of codes in a head, 8.6 in all
    cache = ops.new_cache(1, keys, 2, 128, 4)
    gen = torch.Generator().manual_seed(9)
    k, v = (torch.randn((1, 3, 2, 128), generator=gen).to(BF16).cuda() for _ in "kv")
    for m in (keys, 70, (1 << 25) + 1):
        ops.write_cache(cache, k, v, ints(m))
        got = ops.read_cache(cache, F32, first=ints(m - 4), count=4)
        for x, y in zip(got, (k, v)):
            want = ref.values(*ref.quantise(y.cpu().double().numpy(), 4), 4)
            assert not x[:, 0].any() and np.array_equal(x[:, 1:].cpu().double().numpy(), want)


def test_sources_and_results_beyond_32_bits():
    from featgraph_amd import ops
    tokens = (1 << 21) + 3                  # 2^31 elements of keys and more, 4.3 GB
    gen = torch.Generator(device="cuda").manual_seed(11)
    x = torch.empty((1, tokens, 8, 128), dtype=F16, device="cuda")
    for i in range(0, tokens, 1 << 17):
        x[:, i:i + (1 << 17)].normal_(generator=gen)
    cache, few = ops.new_cache(1, tokens, 8, 128, 4), ops.new_cache(1, 5, 8, 128, 4)
    ops.write_cache(cache, x, x)
    ops.write_cache(few, x[:, -5:], x[:, -5:])
    assert torch.equal(cache.k[:, :, -5:], few.k) and torch.equal(cache.v_scales[:, :, -5:], few.v_scales)
    back = ops.read_cache(cache, F16)
    assert all(torch.equal(a[:, -5:], b) for a, b in zip(back, ops.read_cache(few, F16)))


def test_captured_and_another_stream():
    from featgraph_amd import ops
    gen = torch.Generator().manual_seed(10)
    new = lambda: torch.randn((3, 1, 2, 64), generator=gen).to(BF16).cuda()
    k, v, lengths = new(), new(), ints(1, 5, 9)
    cache, eager = ops.new_cache(3, 20, 2, 64), ops.new_cache(3, 20, 2, 64)
    first = lengths - 2
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.write_cache(cache, k, v, lengths)
        got = ops.read_cache(cache, first=first, count=3, lengths=lengths)
    for _ in range(4):
        k.copy_(new()), v.copy_(new())
        graph.replay()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.write_cache(eager, k, v, lengths)
            want = ops.read_cache(eager, first=first, count=3, lengths=lengths)
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(np.array_equal(a, b) for a, b in zip(parts(cache), parts(eager)))
        lengths.add_(1)
        first.add_(1)
