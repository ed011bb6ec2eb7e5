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
