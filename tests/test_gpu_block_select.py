"""Pooled keys and the choice of blocks (ops.pool_blocks, ops.select_blocks) against sorting exact scores, and selection, attention and gradients
as they are used together."""
import numpy as np
import pytest

import block_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(dtype, batch, queries, keys, heads, kv_heads, head_len, seed=0):
    gen = torch.Generator().manual_seed(seed)
    new = lambda *shape: torch.randn(shape, generator=gen).to(dtype).cuda()
    return new(batch, queries, heads, head_len), new(batch, keys, kv_heads, head_len)


def chosen(q, k, block, topk, causal=True, lengths=None, q_lengths=None, first=None, last=1, pooled=None):
    from featgraph_amd import ops
    pooled = ops.pool_blocks(k, block, lengths) if pooled is None else pooled
    got = ops.select_blocks(q, pooled, k.shape[1], block, topk, causal, lengths, q_lengths, first, last)
    first = (1 if topk > last else 0) if first is None else first
    want = ref.selection(q, pooled, k.shape[1], block, topk, causal, lengths, q_lengths, first, last)
    assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), want)
    return got


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("head_len", [32, 64, 128])
@pytest.mark.parametrize("keys,block", [(1, 32), (95, 32), (200, 64), (513, 128), (700, 256)])
def test_pooled_keys(dtype, head_len, keys, block):
    from featgraph_amd import ops
    _, k = make(dtype, 3, 1, keys, 2, 2, head_len)
    lengths = torch.tensor([keys, keys // 2, 0], dtype=torch.int32, device="cuda")
    for n in (None, lengths):
        x = k.clone()
        if n is not None:
            x[1, keys // 2:], x[2] = float("nan"), float("inf")             # not read
        got = ops.pool_blocks(x, block, n)
        want = torch.zeros(got.shape, dtype=torch.float64)
        for b in range(3):
            m = keys if n is None else int(n[b])
            for i in range(-(-m // block)):
                want[b, :, i] = k[b, i * block:min(m, (i + 1) * block)].cpu().double().mean(0)
        assert torch.equal(got.cpu(), want.float().to(dtype))               # exact sums, rounded as a conversion rounds
        assert torch.equal(ops.pool_blocks(torch.cat([x, x], 2)[:, :, 2:], block, n), got)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("queries,keys,heads,kv_heads,head_len,block,topk,causal", [
    (1, 1, 1, 1, 32, 32, 1, True), (17, 17, 2, 1, 64, 32, 3, True), (100, 900, 6, 2, 32, 32, 5, True), (40, 4500, 4, 4, 128, 32, 16, False),
    (3, 9000, 16, 1, 64, 64, 20, True), (2, 40000, 2, 2, 32, 32, 100, True), (130, 130, 8, 8, 128, 64, 1, True), (5, 60000, 4, 1, 128, 32, 7, False)])
def test_choice(dtype, queries, keys, heads, kv_heads, head_len, block, topk, causal):
    q, k = make(dtype, 2, queries, keys, heads, kv_heads, head_len, seed=1)
    chosen(q, k, block, topk, causal)


def test_ragged_batch():
    q, k = make(BF16, 5, 60, 300, 4, 2, 64, seed=2)
    lengths, q_lengths = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([300, 77, 1, 0, 10 ** 9], [60, 60, 60, 5, -1]))
    for causal in (True, False):
        got = chosen(q, k, 32, 3, causal, lengths, q_lengths)
        assert (got[3] == -1).all() and (got[4] == -1).all()
        assert (got[:, :, :, 0] >= got[:, :, :, 1]).logical_or(got[:, :, :, 1] > got[:, :, :, 0]).all()


@pytest.mark.parametrize("topk", [2, 3, 9, 40])
@pytest.mark.parametrize("causal", [True, False])
def test_lists_ascend_and_end_in_minus_one(topk, causal):
    from featgraph_amd import ops
    q, k = make(BF16, 4, 60, 1000, 4, 2, 64, seed=14)
    lengths, q_lengths = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([1000, 77, 0, 500], [60, 60, 60, 5]))
    got = ops.select_blocks(q, ops.pool_blocks(k, 32, lengths), 1000, 32, topk, causal, lengths, q_lengths)
    before, after = got[..., :-1], got[..., 1:]
    assert ((after == -1) | ((before >= 0) & (after > before))).all()
    assert (got >= -1).all() and (got < 32).all()


def test_first_and_last_blocks_are_kept():
    q, k = make(F16, 1, 80, 640, 2, 1, 32, seed=3)
    for first, last, topk in ((0, 0, 4), (2, 0, 4), (0, 3, 4), (2, 2, 4), (4, 0, 4), (0, 0, 1)):
        for causal in (True, False):
            chosen(q, k, 32, topk, causal, first=first, last=last)


def test_equal_scores_go_to_the_lower_block():
    q, k = make(BF16, 1, 33, 4000, 2, 1, 64, seed=4)
    chosen(torch.zeros_like(q), k, 32, 6)                                   # every score 0
    chosen(-torch.zeros_like(q), k, 32, 6)
    same = k[:, :32].repeat(1, 125, 1, 1)                                   # every block the same
    chosen(q, same, 32, 6)
    # whole numbers: many ties, every sum exact
    gen = torch.Generator().manual_seed(5)
    q, k = (torch.randint(-1, 2, t.shape, generator=gen).to(BF16).cuda() for t in (q, k))
    for dtype in (F32, BF16):
        pooled = torch.randint(-1, 2, (1, 1, 125, 64), generator=gen).to(dtype).cuda()
        chosen(q.to(dtype), k.to(dtype), 32, 6, pooled=pooled)


def test_scores_next_to_each_other():
    """Blocks that differ by the last bit of one element, around a common large score: 32-bit sums cannot order them."""
    for dtype, step in ((F32, 2.0 ** -23), (F16, 2.0 ** -10), (BF16, 2.0 ** -7)):
        gen = torch.Generator().manual_seed(6)
        q = torch.randn(1, 40, 1, 128, generator=gen).to(dtype).cuda()
        base = torch.randn(128, generator=gen).to(dtype)
        pooled = base.repeat(1, 1, 300, 1)
        # one element of each moves by one step, the query's weight on it is tiny: scores differ by 1e-6 of their size and less
        q[..., 7] = 1e-3
        pooled[0, 0, :, 7] = (1 + step * torch.randint(0, 40, (300,), generator=gen)).to(dtype)
        chosen(q, torch.zeros(1, 300 * 32, 1, 128, dtype=dtype, device="cuda"), 32, 9, pooled=pooled.cuda())


def test_few_scores_next_to_each_other():
    """A dozen blocks that 32-bit sums cannot order at the cut, among others that they can."""
    for dtype, step in ((F32, 2.0 ** -23), (F16, 2.0 ** -10), (BF16, 2.0 ** -7)):
        gen = torch.Generator().manual_seed(13)
        q = torch.randn(1, 40, 1, 64, generator=gen).abs().to(dtype).cuda()
        base = torch.randn(64, generator=gen).abs().to(dtype)
        pooled = base.repeat(1, 1, 100, 1)
        q[..., 7] = 1e-3
        pooled[0, 0, :, 7] = (1 + step * torch.randint(0, 40, (100,), generator=gen)).to(dtype)
        pooled[0, 0, 30:34] *= 2                         # four above the rest
        pooled[0, 0, 46:] /= 2                           # most below it
        pooled[0, 0, :30] /= 4
        for topk in (3, 9, 16):
            chosen(q, torch.zeros(1, 100 * 32, 1, 64, dtype=dtype, device="cuda"), 32, topk, causal=False, first=0, last=0, pooled=pooled.cuda())


def test_infinite_and_nan_scores():
    q, k = make(BF16, 1, 20, 3200, 2, 1, 64, seed=7)
    from featgraph_amd import ops
    pooled = ops.pool_blocks(k, 32)
    pooled[0, 0, 10, 3], pooled[0, 0, 20, 4], pooled[0, 0, 30, 5], pooled[0, 0, 40:90, 6] = float("nan"), float("inf"), float("-inf"), 3e38
    for topk in (3, 99):
        chosen(q, k, 32, topk, pooled=pooled)
    chosen(q * float("nan"), k, 32, 5)


def test_strides_and_streams():
    q, k = make(F16, 2, 50, 500, 4, 2, 64, seed=8)
    one = chosen(q, k, 32, 4)
    packed = torch.cat([q, q], 2)[:, :, 4:]
    turned = k.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(one, chosen(packed, turned, 32, 4))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = chosen(q, k, 32, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(one, other)


def test_refusals():
    from featgraph_amd import ops
    q, k = make(BF16, 2, 10, 100, 4, 2, 64)
    pooled = ops.pool_blocks(k, 32)
    assert not pooled.requires_grad
    for change in (dict(pooled=pooled[:, :, :3]), dict(num_keys=200), dict(num_keys=-1), dict(topk=0), dict(keep_last=5), dict(keep_first=-1), dict(block_size=31),
                   dict(pooled=pooled.half()), dict(q=q[:, :, :3]), dict(q=q.double()), dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))):
        args = dict(q=q, pooled=pooled, num_keys=100, block_size=32, topk=4)
        args.update(change)
        with pytest.raises(ValueError):
            ops.select_blocks(**args)
    for args in ((k[0], 32), (k, 33), (k.double(), 32), (k[..., :40], 32)):
        with pytest.raises(ValueError):
            ops.pool_blocks(*args)
    assert ops.pool_blocks(k[:, :0], 32).shape == (2, 2, 0, 64)
    none = ops.select_blocks(q, ops.pool_blocks(k[:, :0], 32), 0, 32, 3)
    assert (none == -1).all() and none.shape == (2, 10, 2, 3)
    with pytest.raises(ValueError, match="2048"):
        ops.select_blocks(q, q.new_zeros(2, 2, 2049, 64), 2049 * 32, 32, 3)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_layer_and_its_tokens(dtype):
    """A prompt's selection, attention and gradients, then new tokens one by one from the cache with pooled keys brought up to date: the same
    rows as the prompt's."""
    from featgraph_amd import ops
    q, k = make(dtype, 2, 150, 150, 4, 2, 64, seed=9)
    v = torch.randn(k.shape, generator=torch.Generator().manual_seed(10)).to(dtype).cuda()
    bias, bounds = torch.randn(16, 4, generator=torch.Generator().manual_seed(11)).to(dtype).cuda(), ops.position_bounds(16, 60)
    blocks = chosen(q, k, 32, 3)
    leaves = [t.detach().requires_grad_() for t in (q, k, v, bias)]
    out = ops.block_attention(leaves[0], leaves[1], leaves[2], blocks, 32, bias=leaves[3], bounds=bounds)
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(12)).to(dtype).cuda()
    grads = torch.autograd.grad(out, leaves, dout)
    want = ref.attention(q, k, v, blocks, 32, bias=bias, bounds=bounds, dout=dout)
    ref.check(dict(zip(("out", "dq", "dk", "dv", "dbias"), (out,) + grads)), want)
    for t in (0, 31, 32, 100, 149):
        lengths = torch.tensor([t + 1, t + 1], dtype=torch.int32, device="cuda")
        one = q[:, t:t + 1]
        got = ops.select_blocks(one, ops.pool_blocks(k, 32, lengths), 150, 32, 3, lengths=lengths)
        mine = ref.attention(one, k, v, got, 32, bias=bias, bounds=bounds, lengths=lengths)
        ref.check({"out": ops.block_attention(one, k, v, got, 32, lengths=lengths, bias=bias, bounds=bounds)}, mine)
        if (t + 1) % 32 == 0:                            # whole blocks only behind: the prompt's choice (its own block was pooled whole there too)
            assert torch.equal(got[:, 0], blocks[:, t])
