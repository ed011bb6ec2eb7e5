"""Heads normed and turned by position (ops.rotate_heads) and the gradients, against the definition in 64 bits."""
import pytest

import rotate_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(dtype=F32, batch=2, tokens=9, heads=4, kv_heads=2, head_len=64, norm=True, seed=0):
    gen = torch.Generator().manual_seed(seed)
    new = lambda *shape: torch.randn(shape, generator=gen).to(dtype).cuda()
    fused = new(batch, tokens, heads + 2 * kv_heads, head_len)
    s = dict(q=fused[:, :, :heads], k=fused[:, :, heads:heads + kv_heads])
    s["weights"] = (1 + 0.3 * new(head_len), 1 + 0.3 * new(head_len)) if norm else (None, None)
    s["douts"] = new(batch, tokens, heads, head_len), new(batch, tokens, kv_heads, head_len)
    return s


def step(s, **options):
    """Outputs and gradients by name."""
    from featgraph_amd import ops
    leaves = [t.detach().requires_grad_() for t in (s["q"], s["k"]) + tuple(w for w in s["weights"] if w is not None)]
    out = ops.rotate_heads(*leaves, **options)
    grads = torch.autograd.grad(out, leaves, s["douts"])
    got = dict(zip(("q.y", "k.y", "q.dx", "k.dx", "q.dw", "k.dw"), tuple(out) + grads))
    return got


def want(s, rotary_len=None, positions=None, lengths=None, q_lengths=None, base=10000.0, frequencies=None, sections=None, interleaved=False, eps=1e-6):
    length = s["q"].shape[3] if rotary_len is None else rotary_len
    cpu = lambda t: None if t is None else t.cpu().numpy()
    cos, sin, there = ref.angles(s["q"].shape, length, cpu(positions), cpu(lengths), cpu(q_lengths), base, frequencies, sections)
    found = {}
    for x, weight, dout in zip("qk", s["weights"], s["douts"]):
        for name, pair in ref.rotate(s[x], weight, cos, sin, there, length, interleaved, eps, dout).items():
            found["%s.%s" % (x, name)] = pair
    return found


def check(s, **options):
    from featgraph_amd import ops
    got, right = step(s, **options), want(s, **options)
    assert set(got) == set(right)
    for name in got:
        ref.check(got[name], right[name], name)
    with torch.no_grad():
        q, k = ops.rotate_heads(s["q"], s["k"], *(w for w in s["weights"] if w is not None), **options)
    assert torch.equal(q, got["q.y"]) and torch.equal(k, got["k.y"])
    return got


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("head_len", [32, 64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [True, False])
def test_types_and_lengths(dtype, head_len, interleaved, norm):
    check(make(dtype, head_len=head_len, norm=norm), interleaved=interleaved)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch,tokens,heads,kv_heads", [(1, 1, 1, 1), (3, 1, 32, 8), (1, 2, 5, 3), (2, 37, 33, 1), (1, 300, 1, 17), (5, 850, 3, 1), (2, 2100, 2, 2)])
def test_sizes(dtype, batch, tokens, heads, kv_heads):
    check(make(dtype, batch, tokens, heads, kv_heads, 64, seed=1))


@pytest.mark.parametrize("dtype,head_len", [(F32, 32), (F16, 128), (BF16, 64), (F32, 128)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_a_part_of_each_head(dtype, head_len, interleaved):
    for rotary_len in range(0, head_len + 1, 16):
        got = check(make(dtype, head_len=head_len, norm=rotary_len % 32 == 0, seed=2), rotary_len=rotary_len, interleaved=interleaved)
        if rotary_len % 32:                                     # what is not turned and not normed passes as it is
            s = make(dtype, head_len=head_len, norm=False, seed=2)
            assert torch.equal(got["q.y"][..., rotary_len:], s["q"][..., rotary_len:])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("sections,axes", [((32,), 1), ((8, 24), 2), ((8, 12, 12), 3), ((0, 32), 2), ((5, 1, 9, 17), 4), ((4,) * 8, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_axes(dtype, sections, axes, interleaved):
    gen = torch.Generator().manual_seed(3)
    positions = torch.randint(-50, 4000, (2, 9, axes), generator=gen, dtype=torch.int32).cuda()
    check(make(dtype, seed=3), positions=positions, sections=sections, interleaved=interleaved, q_lengths=ints(9, 4))
    if axes == 1:
        one = step(make(dtype, seed=3), positions=positions[:, :, 0].t().contiguous().t())
        many = step(make(dtype, seed=3), positions=positions, sections=sections)
        assert all(torch.equal(one[x], many[x]) for x in one)


def test_frequencies():
    fast = [3.0, -0.25] + [10.0 ** -i for i in range(14)]
    check(make(seed=4), rotary_len=32, frequencies=fast)
    check(make(seed=4), base=1e6)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_far_positions_keep_their_angles(dtype):
    # rounded to 32 bits before it is reduced the first pair's angle would be off by 0.06 at 2^20, and by all there is at 2^31
    check(make(dtype, batch=4, seed=5), lengths=ints(2 ** 20, 131072 + 5, 9, 2 ** 31 - 1))
    check(make(dtype, batch=4, seed=5), lengths=ints(3, 0, -7, -2 ** 31), q_lengths=ints(9, 9, 9, 9))


def test_ragged_batch_with_rubbish_behind_the_lengths():
    s = make(BF16, 4, 13, seed=6)
    options = dict(lengths=ints(100, 13, 5, 0), q_lengths=ints(13, 7, 1, 0))
    right = want(s, **options)
    for b, n in enumerate((13, 7, 1, 0)):
        s["q"][b, n:], s["k"][b, n:] = float("nan"), float("inf")
        for d in s["douts"]:
            d[b, n:] = float("nan")
    got = step(s, **options)
    for name in got:
        ref.check(got[name], right[name], name)
    for b, n in enumerate((13, 7, 1, 0)):
        assert not any(got[x][b, n:].any() for x in ("q.y", "k.y", "q.dx", "k.dx"))


def test_counts_outside_the_tensors_are_clamped():
    s = make(seed=7)
    full, over = step(s), step(s, q_lengths=ints(1000, 9))
    assert all(torch.equal(full[x], over[x]) for x in full)
    none = step(s, q_lengths=ints(-1, 0))
    assert not any(none[x].any() for x in none)


def test_empty():
    for change in (dict(batch=0), dict(tokens=0)):
        got = step(make(**change))
        assert got["q.y"].numel() == 0 and got["q.dx"].numel() == 0 and not got["q.dw"].any() and not got["k.dw"].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_squares_beyond_32_bits(dtype):
    # x^2 overflows, the mean square of the scaled values does not; with eps = 0 a head's size does not matter
    s = make(dtype, seed=8)
    plain = step(s, eps=0.0)
    for power in (2.0 ** 90, 2.0 ** -40, 2.0 ** -80, 2.0 ** -110):
        got = step(dict(s, q=s["q"] * power, k=s["k"] * power), eps=0.0)
        ref.check(got["q.y"], want(s, eps=0.0)["q.y"])
        ref.check(got["q.dw"], want(s, eps=0.0)["q.dw"])
        ref.check(got["k.dx"].double() * power, want(s, eps=0.0)["k.dx"])
    mixed = dict(s, q=s["q"] * torch.exp2(torch.tensor([-110.0, 0.0, 90.0, 3.0], device="cuda")).to(dtype)[:, None])      # side by side in a wavefront
    ref.check(step(mixed, eps=0.0)["q.y"], want(s, eps=0.0)["q.y"])
    tiny = step(dict(s, q=s["q"] * 2.0 ** -80))["q.y"]             # beside an eps of ordinary size: x w / sqrt(eps)
    ref.check(tiny.double() * 2.0 ** 80, (want(dict(s, q=s["q"] * 2.0 ** -80))["q.y"][0] * 2.0 ** 80, want(dict(s, q=s["q"] * 2.0 ** -80))["q.y"][1] * 2.0 ** 80))
    assert not torch.isnan(plain["q.y"]).any()


def test_rows_that_are_not_finite_stay_alone():
    s = make(seed=9)
    clean = step(s)
    s["q"][0, 3, 1, 5], s["k"][1, 2, 0, 0] = float("nan"), float("inf")
    got = step(s)
    assert torch.isnan(got["q.y"][0, 3, 1]).all() and torch.isnan(got["k.y"][1, 2, 0]).any()
    for name, b, i, h in (("q.y", 0, 3, 1), ("k.y", 1, 2, 0), ("q.dx", 0, 3, 1), ("k.dx", 1, 2, 0)):
        got[name][b, i, h] = clean[name][b, i, h]
        assert torch.equal(got[name], clean[name]), name


def test_a_zero_head_has_a_gradient():
    s = make(seed=10)
    s["q"][0, 0, 0] = 0
    check(s)


def test_strides():
    s = make(BF16, seed=11)
    right = step(s)
    head_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    shifted = torch.empty(s["q"].numel() + 1, dtype=BF16, device="cuda")[1:].view(s["q"].shape).copy_(s["q"])     # not at 16 bytes
    for change in (dict(q=head_first(s["q"]), douts=tuple(head_first(d) for d in s["douts"])), dict(q=shifted),
                   dict(k=s["k"].flip(3).contiguous().flip(3)), dict(weights=tuple(w.repeat_interleave(2)[::2] for w in s["weights"]))):
        got = step(dict(s, **change))
        assert all(torch.equal(right[x], got[x]) for x in right)
    # one head for all: gradients of what is broadcast add up
    one = s["k"][:, :, :1].detach().requires_grad_()
    from featgraph_amd import ops
    out = ops.rotate_heads(s["q"], one.expand_as(s["k"]), *s["weights"])[1]
    (grad,) = torch.autograd.grad(out, one, s["douts"][1])
    each = step(dict(s, k=one.detach().expand_as(s["k"]).contiguous()))["k.dx"]
    torch.testing.assert_close(grad, each.sum(2, keepdim=True), rtol=2 ** -7, atol=2 ** -7)


def test_gradients_by_differences():
    """What is linear by one difference, whatever its size: the weights, and without norms the inputs.  Along a direction for the rest: the error of a
    central difference is h^2 of a third derivative, and the outputs' rounding over h."""
    from featgraph_amd import ops
    s = make(seed=12)
    got = step(s)
    loss = lambda q, k, *w: sum((y.double() * d.double()).sum() for y, d in zip(ops.rotate_heads(q, k, *w), s["douts"]))
    gen = torch.Generator().manual_seed(13)
    draw = lambda t: torch.randn(t.shape, generator=gen).to(t.dtype).cuda()
    w, dw = s["weights"], tuple(draw(t) for t in s["weights"])
    mass = sum(float((y.detach().abs().double() * d.abs().double()).sum()) for y, d in zip((got["q.y"], got["k.y"]), s["douts"]))
    slope = loss(s["q"], s["k"], *(a + b for a, b in zip(w, dw))) - loss(s["q"], s["k"], *w)
    exact = sum((got[x].double() * d.double()).sum() for x, d in zip(("q.dw", "k.dw"), dw))
    assert abs(float(slope - exact)) <= 8 * (64 + 12) * 2.0 ** -23 * mass
    dx = draw(s["q"]), draw(s["k"])
    h = 2.0 ** -8
    ends = [loss(s["q"] + e * dx[0], s["k"] + e * dx[1], *w) for e in (h, -h)]
    exact = sum((got[x].double() * d.double()).sum() for x, d in zip(("q.dx", "k.dx"), dx))
    # third derivatives of a normed row along a direction of its own size are below 50 of its size
    assert abs(float((ends[0] - ends[1]) / (2 * h) - exact)) <= (50 * h * h + (64 + 12) * 2.0 ** -23 / h) * 2 * mass


def test_one_sided_gradients_and_second_ones():
    from featgraph_amd import ops
    s = make(seed=14)
    q = s["q"].detach().requires_grad_()
    out, _ = ops.rotate_heads(q, s["k"], *s["weights"])
    (grad,) = torch.autograd.grad(out, q, s["douts"][0])
    assert torch.equal(grad, step(s)["q.dx"])
    (grad,) = torch.autograd.grad(ops.rotate_heads(q, s["k"], *s["weights"])[0].square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        grad.sum().backward()
    with pytest.raises(TypeError):
        ops.rotate_heads(s["q"], s["k"], sections=[16.5, 15.5], positions=torch.zeros((2, 9, 2), dtype=torch.int32, device="cuda"))
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(s["q"].contiguous(), torch.ones_like(s["q"].contiguous()))
        with pytest.raises(Exception):
            ops.rotate_heads(dual, s["k"], *s["weights"])


def test_the_same_bits_on_every_call_and_another_stream():
    s = make(BF16, 3, 700, 16, 4, 128, seed=15)
    first = step(s)
    for _ in range(3):
        again = step(s)
        assert all(torch.equal(first[x], again[x]) for x in first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(s)
    side.synchronize()
    assert all(torch.equal(first[x], other[x]) for x in first)


def test_a_row_is_the_same_whoever_stands_beside_it():
    from featgraph_amd import ops
    s = make(BF16, 2, 1300, 20, 3, 64, seed=24)     # 2,600 tokens: a wavefront each; alone a wavefront for every group of heads
    s["q"][0, 7, 3] *= 2.0 ** 100                   # squares out of range, in the same wavefront as others
    positions = torch.arange(1300, dtype=torch.int32, device="cuda").expand(2, 1300)
    q, k = ops.rotate_heads(s["q"], s["k"], *s["weights"], positions=positions)
    for i in (0, 7, 1299):
        one = ops.rotate_heads(s["q"][:, i:i + 1], s["k"][:, i:i + 1], *s["weights"], positions=positions[:, i:i + 1])
        assert torch.equal(one[0], q[:, i:i + 1]) and torch.equal(one[1], k[:, i:i + 1])


def test_offsets_beyond_32_bits():
    from featgraph_amd import ops
    tokens = (1 << 18) + 5                          # 2^31 elements of queries and more, 4.3 GB
    gen = torch.Generator(device="cuda").manual_seed(25)
    q = torch.empty((1, tokens, 64, 128), dtype=BF16, device="cuda")
    for i in range(0, tokens, 1 << 14):
        q[:, i:i + (1 << 14)].normal_(generator=gen)
    k, w = q[:, :, :1], torch.ones(128, dtype=BF16, device="cuda")
    out, _ = ops.rotate_heads(q, k, w, w)
    few = ops.rotate_heads(q[:, -3:], k[:, -3:], w, w, lengths=ints(tokens))[0]
    assert torch.equal(out[:, -3:], few)
    from featgraph_amd.module import rotate
    plan = rotate.check(q, k, w, w, None, None, None, 10000.0, None, None, None, False, 1e-6)
    dq = rotate.backward(q, k, w, w, plan, None, None, None, q, k)[0]
    plan = rotate.check(q[:, -3:], k[:, -3:], w, w, None, ints(tokens), None, 10000.0, None, None, None, False, 1e-6)
    assert torch.equal(dq[:, -3:], rotate.backward(q[:, -3:], k[:, -3:], w, w, plan, None, ints(tokens), None, q[:, -3:], k[:, -3:])[0])


def test_captured():
    from featgraph_amd import ops
    s = make(BF16, 2, 50, 8, 2, 128, seed=16)
    lengths = ints(300, 77)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.rotate_heads(s["q"], s["k"], *s["weights"], lengths=lengths)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, k = ops.rotate_heads(s["q"], s["k"], *s["weights"], lengths=lengths)
    for seed in (17, 18, 19):
        s["q"].copy_(make(BF16, 2, 50, 8, 2, 128, seed=seed)["q"])
        lengths.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        right = ops.rotate_heads(s["q"], s["k"], *s["weights"], lengths=lengths)
        assert torch.equal(q, right[0]) and torch.equal(k, right[1])


def test_captured_training_step():
    from featgraph_amd import ops
    s = make(F16, 2, 600, 8, 2, 64, seed=20)
    leaves = [t.detach().clone().requires_grad_() for t in (s["q"], s["k"]) + s["weights"]]

    def run():
        out = ops.rotate_heads(*leaves)
        return torch.autograd.grad(out, leaves, s["douts"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grads = run()
    for seed in (21, 22, 23):
        with torch.no_grad():
            leaves[0].copy_(make(F16, 2, 600, 8, 2, 64, seed=seed)["q"])
        graph.replay()
        torch.cuda.synchronize()
        got = step(dict(s, q=leaves[0].detach()))
        assert all(torch.equal(a, got[x]) for a, x in zip(grads, ("q.dx", "k.dx", "q.dw", "k.dw")))
