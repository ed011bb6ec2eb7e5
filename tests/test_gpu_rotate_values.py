"""Heads normed and turned by position (ops.rotate_heads) at the ends of float32's range and against its last bits."""
import numpy as np
import pytest

import rotate_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("head_len", [32, 64, 128])
@pytest.mark.parametrize("eps", [0.0, 2.0 ** -140])
def test_the_smallest_numbers_are_normed(dtype, head_len, eps):
    # whole multiples of the smallest number, 2^-149 (2^-133 in bfloat16), and of larger ones: squares are far below 32 bits.  Beside eps = 2^-140 the smaller ones are
    # x w 2^70, the larger ones normed
    from featgraph_amd import ops
    gen = torch.Generator().manual_seed(1)
    least = -149 if dtype == F32 else -133
    tokens = 2 + 133 + least + 149
    power = least + torch.arange(tokens)[:, None, None]                        # a token for each power
    x = torch.ldexp(torch.randint(-15, 16, (1, tokens, 3, head_len), generator=gen).double(), power)
    x[:, :, 0, 0] = torch.ldexp(torch.ones(tokens).double(), power[:, 0, 0])   # not all of a head 0
    x[:, :, 1:, 0] = x[:, :, :1, 0] * 3
    x = x.to(dtype)
    assert (x[0, 0].double() != 0).any()
    w = (1 + 0.3 * torch.randn(head_len, generator=gen)).to(dtype)
    cos, sin, there = ref.angles(x.shape, head_len)
    out = ops.rotate_heads(x.cuda(), x.cuda(), w.cuda(), w.cuda(), eps=eps)
    for y in out:
        ref.check(y, ref.rotate(x, w, cos, sin, there, head_len, eps=eps)["y"])
    # gradients of the largest ones, which are in 32 bits
    big = x[:, -20:].cuda().requires_grad_()
    dout = torch.randn(big.shape, generator=gen).to(dtype)
    y = ops.rotate_heads(big, big.detach(), w.cuda(), w.cuda(), eps=eps)[0]
    (grad,) = torch.autograd.grad(y, big, dout.cuda())
    cos, sin, there = ref.angles(big.shape, head_len)
    ref.check(grad, ref.rotate(x[:, -20:], w, cos, sin, there, head_len, eps=eps, dout=dout)["dx"])


@pytest.mark.parametrize("head_len", [32, 128])
def test_angles_are_those_of_64_bits(head_len):
    """What float32 takes from an angle is made up for: of (1, 0) turned by t the error in the angle's direction is no multiple of that remainder.  The sine's own rounding, up to 2^-24 and
    independent of it, leaves a slope of 2^-24 / (pi 2^-26 sqrt(n)), 0.02 for n = 10^4; without the remainder it is -1."""
    from featgraph_amd import ops
    tokens, pairs = 4000, head_len // 2
    q = torch.zeros((1, tokens, 1, head_len), device="cuda")
    q[..., :pairs] = 1
    got = ops.rotate_heads(q, q, lengths=ints(131072 + 17))[0].cpu().double().numpy()[0, :, 0]
    position = np.arange(tokens) + 131072 + 17 - tokens
    turns = np.array([10000.0 ** (-i / pairs) / (2 * np.pi) for i in range(pairs)])
    t = position[:, None] * turns
    t = 2 * (t - np.rint(t))
    rest = np.pi * (t - t.astype(np.float32).astype(np.float64))
    cos, sin = np.cos(np.pi * t), np.sin(np.pi * t)
    off = got[:, pairs:] * cos - got[:, :pairs] * sin                          # of the angle
    assert np.abs(off).max() <= 3 * 2.0 ** -24
    assert abs((off * rest).sum() / (rest * rest).sum()) < 0.1


def test_weights_gradients_of_many_rows():
    """Rows of ones and minus ones are their own norm, so that the weights' gradient is a plain sum of the outputs' gradients with signs: 2^20 rows in 4,096 wavefronts.  A lane adds 16 in
    32 bits (additions 2 to 16 of numbers whose sum grows like sqrt(i), each off by 2^-24 / sqrt(3) of it at most: 2.8 of 2^-48 together), then sums are 64 bits up to a workgroup's, rounded, and the result, rounded.
    All of 256 rows in 32 bits would give 43 in place of 2.8."""
    from featgraph_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = [torch.randint(0, 2, (1, 1 << 20, 1, 32), generator=gen, device="cuda").float() * 2 - 1 for _ in "qk"]
    w = [torch.ones(32, device="cuda").requires_grad_() for _ in "qk"]
    dout = [torch.randn(t.shape, generator=gen, device="cuda") for t in x]
    grads = torch.autograd.grad(ops.rotate_heads(*x, *w, rotary_len=0, eps=0.0), w, dout)
    want = [(t.double() * d.double()).sum((0, 1, 2)) for t, d in zip(x, dout)]
    off = torch.cat([g.double() - v for g, v in zip(grads, want)])
    assert float(off.norm() / torch.cat(want).norm()) <= (2.8 + 1 / 3 + 1 / 3) ** 0.5 * 2.0 ** -24


@pytest.mark.parametrize("tokens,heads,kv_heads,head_len", [(700, 40, 1, 64), (3000, 5, 17, 32), (9000, 9, 4, 128)])
def test_weights_gradients_across_sums_of_rows(tokens, heads, kv_heads, head_len):
    # rows that do not come in sixteens, wavefronts of one group of heads and of all of a token's, captured and replayed
    from featgraph_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *shape: torch.randn(shape, generator=gen, device="cuda")
    q, k, w = new(1, tokens, heads, head_len), new(1, tokens, kv_heads, head_len), [1 + 0.3 * new(head_len) for _ in "qk"]
    douts = new(*q.shape), new(*k.shape)
    leaves = [t.requires_grad_() for t in [q, k] + w]
    there_are = ints(tokens - 3)
    step = lambda: torch.autograd.grad(ops.rotate_heads(*leaves, q_lengths=there_are), leaves, douts)
    got = step()
    cos, sin, there = ref.angles(q.shape, head_len, q_lengths=[tokens - 3])
    for i, (x, weight, dout) in enumerate(zip((q, k), w, douts)):
        want = ref.rotate(x, weight, cos, sin, there, head_len, dout=dout)
        ref.check(got[i], want["dx"])
        # the terms' own rounding, and sixteen rows, a workgroup's sum and the result in 32 bits, in place of all rows
        e = (head_len + 12) * ref.W
        value, bound = want["dw"]
        rows = x.numel() // head_len
        ref.check(got[2 + i], (value, bound * (2 * e + 20 * ref.W) / (2 * e + rows * ref.W) + ref.U[F32] * np.abs(value)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, got))
        step()
