"""Attention over selected blocks of keys (ops.block_attention) and its gradients against the definition in 64 bits."""
import numpy as np
import pytest

import block_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def make(dtype=F32, batch=2, queries=70, keys=70, heads=4, kv_heads=2, head_len=32, block=32, topk=2, buckets=0, causal=True, seed=0):
    """Inputs on the GPU; every query names its own block and topk - 1 drawn ones, behind the keys and -1 among them."""
    gen = torch.Generator().manual_seed(seed)
    new = lambda *shape: torch.randn(shape, generator=gen).to(dtype).cuda()
    nb = -(-keys // block)
    blocks = torch.randint(-1, nb + 1, (batch, queries, kv_heads, topk), generator=gen, dtype=torch.int32)
    blocks[..., 0] = ((torch.arange(queries) + keys - queries).clamp(min=0) // block)[None, :, None]
    s = dict(q=new(batch, queries, heads, head_len), k=new(batch, keys, kv_heads, head_len), v=new(batch, keys, kv_heads, head_len),
             blocks=blocks.cuda(), block_size=block, causal=causal, lengths=None, q_lengths=None, bias=None, bounds=None)
    if buckets:
        from featgraph_amd import ops
        s["bias"], s["bounds"] = new(buckets, heads), ops.position_bounds(buckets, max(buckets, 40), causal)
    return s, new(batch, queries, heads, head_len)


def call(s, **change):
    from featgraph_amd import ops
    s = dict(s, **change)
    return ops.block_attention(s["q"], s["k"], s["v"], s["blocks"], s["block_size"], causal=s["causal"], lengths=s["lengths"],
                               q_lengths=s["q_lengths"], bias=s["bias"], bounds=s["bounds"])


def step(s, dout, **change):
    """Output and gradients of one training step."""
    names = [x for x in ("q", "k", "v", "bias") if s[x] is not None]
    leaves = {x: s[x].detach().requires_grad_() for x in names}
    out = call(s, **leaves, **change)
    grads = torch.autograd.grad(out, list(leaves.values()), dout)
    return dict({"out": out}, **{"d" + x: g for x, g in zip(names, grads)})


def want(s, dout=None):
    return ref.attention(s["q"], s["k"], s["v"], s["blocks"], s["block_size"], causal=s["causal"], lengths=s["lengths"], q_lengths=s["q_lengths"],
                         bias=s["bias"], bounds=s["bounds"], dout=dout)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("head_len", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (4, 2), (3, 1), (8, 1), (16, 1), (14, 2)])
def test_types_and_groups(dtype, head_len, heads, kv_heads):
    s, dout = make(dtype, heads=heads, kv_heads=kv_heads, head_len=head_len)
    ref.check(step(s, dout), want(s, dout))
    ref.check({"out": call(s)}, want(s))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("queries,keys,block,topk,causal", [
    (1, 1, 32, 1, True), (1, 1, 256, 3, False), (2, 33, 32, 2, True), (1, 700, 64, 5, True), (5, 1000, 128, 8, True), (31, 31, 64, 1, True),
    (33, 257, 32, 9, False), (130, 130, 64, 2, False), (200, 513, 256, 2, True), (300, 300, 32, 10, True), (64, 640, 128, 5, False)])
def test_lengths_and_blocks(dtype, queries, keys, block, topk, causal):
    s, dout = make(dtype, 2, queries, keys, 4, 2, 64, block, topk, causal=causal, seed=3)
    ref.check(step(s, dout), want(s, dout))


@pytest.mark.parametrize("dtype,head_len,block,buckets", [(F32, 32, 32, 8), (F16, 64, 128, 0), (BF16, 128, 64, 32), (BF16, 32, 32, 16), (F32, 128, 64, 0)])
@pytest.mark.parametrize("batch,queries,heads,kv_heads,causal", [(4, 1030, 8, 8, True), (2, 1030, 16, 4, False), (1, 2060, 16, 1, True), (2, 2610, 6, 2, True)])
def test_many_queries(dtype, head_len, block, buckets, batch, queries, heads, kv_heads, causal):
    """Enough of them for the kernels that take several tiles at a time (256 workgroups)."""
    s, dout = make(dtype, batch, queries, queries, heads, kv_heads, head_len, block, 3, buckets, causal, seed=4)
    s["blocks"][:, 700:705] = -1
    ref.check(step(s, dout), want(s, dout))
    ref.check({"out": call(s)}, want(s))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("buckets,heads,kv_heads,queries,keys", [(32, 4, 2, 200, 200), (16, 3, 1, 90, 90), (64, 2, 2, 33, 150), (4, 16, 1, 70, 70), (7, 4, 4, 1, 300)])
def test_bias(dtype, causal, buckets, heads, kv_heads, queries, keys):
    s, dout = make(dtype, 2, queries, keys, heads, kv_heads, 64, 32, 5, buckets, causal, seed=5)
    ref.check(step(s, dout), want(s, dout))


def test_bias_of_one_bucket_changes_nothing_and_far_bounds_hold():
    s, dout = make(BF16, queries=100, keys=100, topk=3)
    plain = step(s, dout)
    one = step(dict(s, bias=torch.full((1, 4), 0.5, dtype=BF16, device="cuda"), bounds=()), dout)
    for x in plain:
        torch.testing.assert_close(plain[x].float(), one[x].float(), rtol=2 ** -7, atol=1e-2)
    # softmax does not see a shift: the exact gradient is 0, and sums of dS leave their rounding
    s["bias"], s["bounds"] = torch.randn(3, 4, device="cuda").to(BF16), (-3000, 1000)
    ref.check(step(s, dout), want(s, dout))


def test_long_rows_are_joined_and_many_queries_of_one_block_cut():
    # every query names block 0: its list is cut into pieces; with few queries a row's blocks go to several workgroups
    s, dout = make(F32, 1, 2500, 2500, 2, 2, 32, 64, 3, seed=8)
    s["blocks"][..., 1] = 0
    ref.check(step(s, dout), want(s, dout))
    s, dout = make(BF16, 1, 2, 6000, 4, 2, 64, 64, 94, seed=9)
    s["blocks"][:] = torch.arange(94, dtype=torch.int32, device="cuda")
    ref.check(step(s, dout), want(s, dout))


def test_more_blocks_than_one_window():
    # 2,048 blocks are listed at a time
    s, dout = make(F32, 1, 20, 70001, 2, 1, 32, 32, 40, seed=10)
    ref.check(step(s, dout), want(s, dout))


def test_ragged_batch_with_rubbish_behind_the_lengths():
    for causal in (True, False):
        s, dout = make(BF16, 5, 96, 130, 4, 2, 64, 32, 4, 8, causal, seed=11)
        s["lengths"], s["q_lengths"] = ints(130, 77, 1, 0, 40), ints(96, 50, 1, 3, 0)
        value = want(s, dout)                            # from clean inputs
        for b in range(5):
            n, m = int(s["q_lengths"][b]), int(s["lengths"][b])
            s["q"][b, n:], dout[b, n:], s["k"][b, m:], s["v"][b, m:] = float("nan"), float("inf"), float("nan"), float("-inf")
        got = step(s, dout)
        ref.check(got, value)
        for b in range(5):
            n, m = int(s["q_lengths"][b]), int(s["lengths"][b])
            assert not got["out"][b, n:].any() and not got["dq"][b, n:].any() and not got["dk"][b, m:].any() and not got["dv"][b, m:].any()


def test_counts_outside_the_tensors_are_clamped():
    s, dout = make(F32)
    full = step(s, dout)
    got = step(dict(s, lengths=ints(1000, 70), q_lengths=ints(70, 2 ** 31 - 1)), dout)
    assert all(torch.equal(full[x], got[x]) for x in full)
    got = step(dict(s, lengths=ints(-5, 0), q_lengths=ints(70, 70)), dout)
    assert not any(got[x].any() for x in got)


def test_rows_without_a_visible_key():
    s, dout = make(BF16, queries=90, keys=90, topk=2)
    s["blocks"][:, ::3] = -1
    s["blocks"][:, 1::7] = 5                             # behind the keys
    s["blocks"][:, 2, :, :] = 2                          # behind the query
    got = step(s, dout)
    ref.check(got, want(s, dout))
    assert not got["out"][:, ::3].any() and not got["dq"][:, 2].any()


def test_ids_twice_in_any_order_and_out_of_range():
    s, dout = make(F32, queries=128, keys=128, topk=3)
    some = step(s, dout)
    b = s["blocks"]
    rubbish = torch.tensor([2 ** 31 - 1, -2 ** 31, 4, 67108864], dtype=torch.int32, device="cuda").expand(2, 128, 2, 4)
    again = step(dict(s, blocks=torch.cat([b.flip(3), rubbish, b], 3)), dout)
    assert all(torch.equal(some[x], again[x]) for x in some)


@pytest.mark.parametrize("batch", [1, 120])
def test_masked_infinities_and_nan_reach_nobody(batch):
    """Keys and values that are not finite in blocks that a neighbouring query selects and this one does not, and behind a causal query; in the
    first sequence of a batch that is small, or large enough for the kernels that take many queries (looked at in that sequence)."""
    def step(s, dout):
        got = globals()["step"](s, dout)
        if batch > 1:
            assert all(torch.isfinite(t[1:]).all() for t in got.values())
            assert all(torch.equal(got[x][1], clean_step[x][1]) for x in got) if clean_step else True
        return {x: t[:1] for x, t in got.items()}

    def want(s, dout):
        return globals()["want"](dict(s, **{x: s[x][:1] for x in ("q", "k", "v", "blocks")}), dout[:1])

    for dtype in (F32, BF16):
        s, dout = make(dtype, batch, 96, 96, 2, 1, 64, 32, 1, seed=12)
        clean_step = None
        s["blocks"][:] = 0
        s["blocks"][:, 70:80] = 1                        # these rows alone see block 1
        clean = dict(s, k=s["k"].clone(), v=s["v"].clone())
        value = want(clean, dout)
        clean_step = globals()["step"](clean, dout)
        for rubbish in (float("nan"), float("inf"), float("-inf")):
            for name in ("k", "v"):
                t = clean[name].clone()
                t[0, 40, 0, 3] = rubbish
                t[0, 20, 0, 5] = rubbish                 # rows 0 .. 19 are before it
                got = step(dict(s, **{name: t}), dout)
                hit = np.zeros(96, dtype=bool)
                hit[20:] = True
                for x in ("out", "dq"):
                    keep = got[x][:, ~hit]
                    ref.check({x: keep}, {x: tuple(a[:, ~hit] for a in value[x])}, (dtype, rubbish, name))
                if name == "v":
                    assert not torch.isfinite(got["out"][0, 20:70, :, 5]).any() and torch.isfinite(got["out"][0, 20:70, :, 6]).all()
                    assert not torch.isfinite(got["out"][0, 70:80, :, 3]).any() and torch.isfinite(got["out"][0, 70:80, :, 5]).all()
                    expect = torch.isposinf if rubbish == float("inf") else torch.isneginf if rubbish < 0 else torch.isnan
                    assert expect(got["out"][0, 20:70, :, 5]).all() and expect(got["out"][0, 70:80, :, 3]).all()
        # a row of Q or of the gradient that is not finite: keys that do not see it keep their gradients
        for name in ("q", "dout"):
            t = (dout if name == "dout" else clean["q"]).clone()
            t[0, 75, 0, 2] = float("nan")
            got = step(dict(s, q=t) if name == "q" else s, t if name == "dout" else dout)
            for x in ("dk", "dv"):
                far = list(range(32)) + list(range(76, 96))      # keys 32 .. 75 of block 1 are seen by row 75
                ref.check({x: got[x][:, far]}, {x: tuple(a[:, far] for a in value[x])}, (dtype, name))


def test_scores_of_infinite_size():
    s, dout = make(F32, 1, 40, 40, 1, 1, 32, 32, 2, seed=13)
    s["blocks"][..., 0], s["blocks"][..., 1] = 0, 1
    s["bias"], s["bounds"] = torch.zeros(2, 1, device="cuda"), (5,)
    low = torch.finfo(F32).min
    s["bias"][0] = low                                   # distances below 5 at the type's lowest value: as good as masked where others are seen
    got, value = call(s), want(s)
    ref.check({"out": got}, value)                       # rows 0 .. 4 see nothing else: their softmax is over equal scores
    s["bias"][0] = float("-inf")
    got = call(s)
    assert not got[:, :5].any()                          # every score -inf: 0
    ref.check({"out": got[:, 5:]}, {"out": tuple(a[:, 5:] for a in value["out"])})
    s["bias"][0] = float("inf")
    assert call(s).isnan().all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("batch,heads,kv_heads", [(2, 2, 1), (64, 8, 8)])
def test_bias_of_the_lowest_value(dtype, batch, heads, kv_heads):
    """Distances below 5 have the type's lowest value, as a mask: the first five rows of a block see nothing else."""
    s, dout = make(dtype, batch, 150, 150, heads, kv_heads, 64, 32, 1, seed=20)
    masked = torch.arange(150, device="cuda") % 32 < 5
    # their queries are 0, so that their softmax is the one over equal scores; 2^-140 and 2^-1000000 are both nothing beside the other rows' scores
    s["q"][:, masked] = 0
    s["bias"], s["bounds"] = torch.randn(3, heads, generator=torch.Generator().manual_seed(1)).to(dtype).cuda(), (5, 20)
    low = s["bias"].clone()
    s["bias"][0], low[0] = -97, torch.finfo(dtype).min
    value = want(dict(s, **{x: s[x][:1] for x in ("q", "k", "v", "blocks")}), dout[:1]) if batch > 2 else want(s, dout)
    got = step(dict(s, bias=low), dout)
    assert all(torch.isfinite(t).all() for t in got.values())
    if batch > 2:                                        # the first of them alone: the bias's gradient is all sequences'
        got = {x: t[:1] for x, t in got.items() if x != "dbias"}
    ref.check(got, value)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch", [1, 64])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_scales(dtype, batch, scale):
    from featgraph_amd import ops
    s, dout = make(dtype, batch, 70, 70, 8, 8, 32, 32, 2, seed=21)
    leaves = [s[x].detach().requires_grad_() for x in ("q", "k", "v")]
    out = ops.block_attention(*leaves, s["blocks"], 32, scale)
    got = [out] + list(torch.autograd.grad(out, leaves, dout))
    value = ref.attention(*(s[x][:1] for x in ("q", "k", "v", "blocks")), 32, scale, dout=dout[:1])
    ref.check({x: t[:1] for x, t in zip(("out", "dq", "dk", "dv"), got)}, value)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("size", [-6000, 6000])
@pytest.mark.parametrize("batch,queries,heads,kv_heads,head_len", [(2, 70, 4, 2, 64), (1, 5, 16, 1, 32), (4, 1030, 8, 8, 32), (2, 1030, 16, 4, 128)])
def test_rows_of_large_scores_leave_their_neighbours_alone(dtype, size, batch, queries, heads, kv_heads, head_len):
    """One head of a few tokens has scores of thousands, near enough to one another for a softmax over many keys; the rest are ordinary."""
    s, dout = make(dtype, batch, queries, queries, heads, kv_heads, head_len, 32, 3, seed=25)
    s["k"][..., 0] = 64                                  # all of a row's scores move together
    odd = s["k"][:, 1::2]
    odd.copy_(s["k"][:, :2 * odd.shape[1]:2])            # keys in pairs of equal ones: no row is one key's alone
    s["q"][:, 4::37, 0, 0] = size / 64 * head_len ** 0.5
    ref.check(step(s, dout), want(s, dout))


@pytest.mark.parametrize("batch", [2, 64])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 26, -2.0 ** 28])
def test_queries_gradients_of_scores_that_hold_no_fraction(batch, size):
    """Keys that are equal where the query is not 0 have equal scores, whatever rounding makes of them: a row's softmax is the one of a query
    of zeros.  From 2^24 on a score and the logarithm of a row's sum do not fit one 32-bit number."""
    s, dout = make(F32, batch, 90, 90, 8, 4, 64, 32, 2, seed=26)
    s["k"][..., 0] = 2.0 ** 10
    s["q"].zero_()
    value = ref.attention(*(s[x][:2] for x in ("q", "k", "v", "blocks")), 32, dout=dout[:2])
    s["q"][:, 3::5, 1, 0] = size / 2 ** 10 * 8
    got = step(s, dout)
    ref.check({x: got[x][:2] for x in ("out", "dq")}, value)


@pytest.mark.parametrize("batch,queries,block", [(2, 90, 32), (64, 90, 128), (1, 1030, 64)])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 26, -2.0 ** 28])
def test_keys_gradients_of_scores_that_hold_no_fraction(batch, queries, block, size):
    """As the queries' gradients.  The upper half of a query meets zeros in every key: the keys' gradients there are large and know nothing of the
    scores but the softmax."""
    s, dout = make(F32, batch, queries, queries, 8, 4, 64, block, 2, seed=27)
    s["q"].zero_()
    s["k"][..., 32:] = 0
    s["k"][..., 0] = 2.0 ** 10
    s["q"][..., 32:] = torch.randn(s["q"].shape[:3] + (32,), generator=torch.Generator().manual_seed(1)).cuda()      # meets zeros alone
    value = ref.attention(*(s[x][:2] for x in ("q", "k", "v", "blocks")), block, dout=dout[:2])
    s["q"][:, 3::5, 1, 0] = size / 2 ** 10 * 8
    got = step(s, dout)
    ref.check({"dv": got["dv"][:2]}, value)
    ref.check({"dk": got["dk"][:2, :, :, 32:]}, {"dk": tuple(a[..., 32:] for a in value["dk"])})


# Shapes of the two kernels for queries, and of blocks whose keys one wavefront has and several share
HALF_SHAPES = [(2, 70, 4, 2, 64, 32, 0), (1, 40, 16, 1, 128, 128, 8), (4, 1030, 8, 8, 32, 64, 0), (2, 1030, 16, 4, 128, 64, 16)]


@pytest.mark.parametrize("batch,queries,heads,kv_heads,head_len,block,buckets", HALF_SHAPES)
@pytest.mark.parametrize("long", ["q", "k"])
@pytest.mark.parametrize("size", [2.0 ** -16, 2.0 ** -12])
def test_small_gradients_of_16_bits(batch, queries, heads, kv_heads, head_len, block, buckets, long, size):
    """Scores' gradients of 1e-6 are below float16's normal numbers, the results that long keys (queries) make of them are not."""
    s, dout = make(F16, batch, queries, queries, heads, kv_heads, head_len, block, 3, buckets, seed=28)
    s[long] *= 64
    s["k" if long == "q" else "q"] /= 64
    dout = (dout.float() * size).half()
    ref.check(step(s, dout), want(s, dout))


@pytest.mark.parametrize("batch,queries,heads,kv_heads,head_len,block,buckets", HALF_SHAPES)
@pytest.mark.parametrize("values,gradients", [(64, 512), (4096, 1 / 16), (2 ** -6, 1024), (4096, 64)])
def test_large_score_gradients_of_16_bits(batch, queries, heads, kv_heads, head_len, block, buckets, values, gradients):
    """<dout, v> beyond float16's largest number; what comes of it, with short queries and keys, is within."""
    s, dout = make(F16, batch, queries, queries, heads, kv_heads, head_len, block, 3, 0, seed=29)
    s["q"] /= 1024
    s["k"] /= 1024
    s["v"] *= values
    dout = (dout.float() * gradients).half()
    ref.check(step(s, dout), want(s, dout))


@pytest.mark.parametrize("batch,queries,heads,kv_heads,head_len,block,buckets", HALF_SHAPES)
def test_gradients_of_small_values_of_16_bits(batch, queries, heads, kv_heads, head_len, block, buckets):
    """Outputs of a few times float16's smallest number: <dout, out> has to hold what their rounding took, for keys have much in common."""
    s, dout = make(F16, batch, queries, queries, heads, kv_heads, head_len, block, 3, buckets, seed=35)
    s["k"] += 64
    s["q"] /= 64
    s["v"] *= 2.0 ** -20
    dout *= 1024
    ref.check(step(s, dout), want(s, dout))


@pytest.mark.parametrize("batch,queries,heads,kv_heads,head_len,block,buckets", HALF_SHAPES)
def test_gradients_of_16_bits_of_values_that_cancel(batch, queries, heads, kv_heads, head_len, block, buckets):
    """Equal keys with opposite values, but for the last bit of one element: outputs far below the values, whose differences are not."""
    s, dout = make(F16, batch, queries, queries, heads, kv_heads, head_len, block, 3, buckets, causal=False, seed=36)
    s["k"][:, 1::2], s["v"][:, 1::2] = s["k"][:, ::2], -s["v"][:, ::2]
    s["v"][:, 1::2, :, 0] *= 1 + 2.0 ** -10
    if buckets:
        s["bias"][:] = s["bias"][:1]                     # equal keys in two buckets keep equal scores
    ref.check(step(s, dout), want(s, dout))


def test_gradients_of_16_bits_of_unequal_rows():
    """Rows whose gradients are 2^20 times their neighbours'; keys that only the small ones see, and rows that come before and after them."""
    s, dout = make(F16, 2, 200, 200, 4, 2, 64, 32, 2, seed=30)
    s["k"] *= 64
    s["q"] /= 64
    s["blocks"][..., 1] = -1                             # each its own block
    dout = (dout.float() * 2.0 ** -12).half()
    dout[:, 40::32] *= 2.0 ** 14
    dout[:, 60::64, 1] *= 2.0 ** 14
    ref.check(step(s, dout), want(s, dout))


@pytest.mark.parametrize("keys,block", [(1000, 64), (600, 32)])
def test_shares_below_the_normal_numbers_of_16_bits(keys, block):
    """One key has most of a row and the others 6e-6 each, between two multiples of float16's smallest number."""
    nb = -(-keys // block)
    s, dout = make(F16, 1, 1, keys, 1, 1, 32, block, nb, causal=False, seed=31)
    s["blocks"][:] = torch.arange(nb, dtype=torch.int32, device="cuda")
    s["q"].zero_(), s["k"].zero_()
    s["q"][..., 0] = 32 ** 0.5                           # in float16 5.65625
    top = [x for x in np.arange(11.5, 12.5, 2.0 ** -7) if 0.4 < 2.0 ** 24 / (np.exp(x * 5.65625 / 32 ** 0.5) + keys - 1) % 1 < 0.6][0]
    s["k"][0, 5, 0, 0] = top
    dout.fill_(2048)
    ref.check(step(s, dout), want(s, dout))


@pytest.mark.parametrize("batch,queries", [(1, 1), (2, 40), (64, 32)])
def test_outputs_of_shares_below_the_normal_numbers_of_16_bits(batch, queries):
    """One key has most of a row and a value of 0; the others have 6e-7 each, and all of the output."""
    s, _ = make(F16, batch, queries, 1000, 16, 1, 32, 64, 16, causal=False, seed=33)
    s["blocks"][:] = torch.arange(16, dtype=torch.int32, device="cuda")
    s["q"].zero_(), s["k"].zero_()
    s["q"][..., 0] = 32 ** 0.5                           # in float16 5.65625
    s["k"][:, 5, 0, 0] = [x for x in np.arange(14, 15, 2.0 ** -7) if 0.4 < 2.0 ** 24 * np.exp(-x * 5.65625 / 32 ** 0.5) % 1 < 0.6][0]
    s["v"][:] = 1
    s["v"][:, 5] = 0
    value = ref.attention(*(s[x][:1] for x in ("q", "k", "v", "blocks")), 64, causal=False)
    ref.check({"out": call(s)[:1]}, value)
    ref.check({"out": call(s, q=s["q"].detach().requires_grad_())[:1]}, value)


@pytest.mark.parametrize("batch", [2, 64])
@pytest.mark.parametrize("name", ["k", "v"])
def test_small_gradients_of_16_bits_beside_infinities(batch, name):
    s, dout = make(F16, batch, 96, 96, 4, 4, 64, 32, 1, seed=32)
    s["q"] /= 64
    s["k"] *= 64
    s["blocks"][:] = 0
    s["blocks"][:, 70:80] = 1                            # these rows alone see block 1
    dout = (dout.float() * 2.0 ** -14).half()
    value = ref.attention(*(s[x][:2] for x in ("q", "k", "v", "blocks")), 32, dout=dout[:2])
    s[name][:, 40, :, 3] = float("inf")
    got = step(s, dout)
    keep = [i for i in range(96) if not 70 <= i < 80]
    ref.check({x: got[x][:2, keep] for x in ("out", "dq")}, {x: tuple(a[:, keep] for a in value[x]) for x in ("out", "dq")})
    ref.check({x: got[x][:2, :32] for x in ("dk", "dv")}, {x: tuple(a[:, :32] for a in value[x]) for x in ("dk", "dv")})


def test_more_blocks_than_one_list_of_many_queries():
    """256 blocks are listed at a time where there are queries to fill the card; a row's blocks lie in several lists."""
    for dtype in (F32, BF16):
        s, dout = make(dtype, 256, 8, 17000, 16, 1, 32, 32, 3, seed=22)
        got = step(s, dout)
        for b in (0, 255):
            value = want(dict(s, **{x: s[x][b:b + 1] for x in ("q", "k", "v", "blocks")}), dout[b:b + 1])
            ref.check({x: t[b:b + 1] for x, t in got.items()}, value)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("batch,queries,heads,keys,ends", [(1, 20, 2, 70001, (1023, 1024, 2047, 2048)), (256, 8, 16, 17000, (255, 256, 511, 512))])
def test_blocks_at_the_ends_of_windows(dtype, batch, queries, heads, keys, ends):
    """Few queries list 1,024 blocks at a time, many 256: the last of a list and the first of the next."""
    s, dout = make(dtype, batch, queries, keys, heads, 1, 32, 32, 6, seed=37)
    s["blocks"][..., 1:5] = ints(*ends)
    got = step(s, dout)
    value = want(dict(s, **{x: s[x][:1] for x in ("q", "k", "v", "blocks")}), dout[:1])
    ref.check({x: t[:1] for x, t in got.items()}, value)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("queries", [40, 2100])
def test_the_most_buckets(dtype, queries):
    s, dout = make(dtype, 1, queries, queries, 16, 1, 128, 32, 2, seed=23)
    s["bias"], s["bounds"] = torch.randn(64, 16, generator=torch.Generator().manual_seed(1)).to(dtype).cuda(), tuple(range(-31, 31)) + (4063,)
    ref.check(step(s, dout), want(s, dout))


@pytest.mark.parametrize("batch,queries,keys", [(0, 30, 30), (2, 0, 30), (2, 30, 0), (2, 30, 30)])
def test_gradients_of_nothing_are_zero(batch, queries, keys):
    s, dout = make(BF16, 2, 30, 30, buckets=8, seed=24)
    s.update(q=s["q"][:batch, :queries], k=s["k"][:batch, :keys], v=s["v"][:batch, :keys], blocks=torch.full_like(s["blocks"], -1)[:batch, :queries])
    torch.full((2 ** 20,), float("nan"), device="cuda")          # memory that the gradients may come to lie in
    got = step(s, dout[:batch, :queries])
    assert all(not t.any() for t in got.values()) and got["dbias"].shape == (8, 4) and got["dk"].shape == s["k"].shape


def test_strides_and_alignment():
    for dtype in (F32, BF16):
        s, dout = make(dtype, 2, 70, 70, 4, 4, 64, 32, 3, seed=14)
        base = step(s, dout)
        packed = torch.cat([s["q"], s["k"], s["v"]], 2)                     # (b, n, 12, d), taken apart as views
        q, k, v = packed.split(4, 2)
        others = [dict(q=q, k=k, v=v), dict(q=s["q"].transpose(1, 2).contiguous().transpose(1, 2), k=s["k"].transpose(0, 1).contiguous().transpose(0, 1)),
                  dict(q=torch.cat([s["q"], s["q"]], 3)[..., 1:65].copy_(s["q"]), v=s["v"].flip(3).flip(3)),
                  dict(blocks=s["blocks"].transpose(0, 1).contiguous().transpose(0, 1))]
        for change in others:
            got = step(dict(s, **change), dout)
            assert all(torch.equal(base[x], got[x]) for x in base)
        odd = torch.empty(dout.numel() + 1, dtype=dtype, device="cuda")[1:].view(dout.shape).copy_(dout)      # not at a 16-byte address
        for d in (odd, torch.cat([dout, dout], 3)[..., :64]):
            got = step(s, d)
            assert all(torch.equal(base[x], got[x]) for x in base)
        # one key head's tensor for both sequences: an expanded axis
        shared = step(dict(s, k=s["k"][:1].expand(2, -1, -1, -1)), dout)
        ref.check(shared, want(dict(s, k=s["k"][:1].expand(2, -1, -1, -1).contiguous()), dout))
        ones = dout.new_ones(()).expand(dout.shape)
        ref.check(step(s, ones), want(s, ones.contiguous()))


def test_gradients_of_some_inputs_only():
    s, dout = make(BF16, queries=100, keys=100, topk=3, buckets=8)
    full = step(s, dout)
    for name in ("q", "k", "v", "bias"):
        leaf = s[name].detach().requires_grad_()
        (g,) = torch.autograd.grad(call(s, **{name: leaf}), leaf, dout)
        assert torch.equal(g, full["d" + name])
    # the same tensor as keys and values: both gradients add up
    kv = s["k"].detach().requires_grad_()
    (g,) = torch.autograd.grad(call(s, k=kv, v=kv), kv, dout)
    part = step(dict(s, v=s["k"]), dout)
    torch.testing.assert_close(g, part["dk"] + part["dv"])


@pytest.mark.parametrize("dtype,batch,queries,keys,topk", [(F16, 2, 70, 70, 2), (BF16, 2, 70, 70, 2), (BF16, 3, 1, 5000, 60), (F16, 1, 5, 3000, 40), (F32, 64, 70, 70, 2)])
def test_outputs_with_and_without_gradients_are_the_same(dtype, batch, queries, keys, topk):
    """Of a few queries in every type, and of any number of them in 32 bits."""
    s, _ = make(dtype, batch, queries, keys, 8, 4, 64, 32, topk, 8, seed=34)
    with torch.no_grad():
        plain = call(s, q=s["q"].detach().requires_grad_())
    assert torch.equal(plain, call(s)) and torch.equal(plain, call(s, q=s["q"].detach().requires_grad_()))


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("batch,queries,heads,kv_heads,head_len,block,buckets", HALF_SHAPES)
def test_gradients_of_16_bits_are_off_by_their_own_rounding(dtype, batch, queries, heads, kv_heads, head_len, block, buckets):
    """The root mean square error is that of rounding the exact results, r.  Operands in two parts are off by 2^-16 (float16: 2^-22) and less,
    independent of one another from term to term; even with sums 30 times as large as what is left of them that is below r / 4,
    and the two together below 1.05 r.  One part alone, off by as much as the result, would make 1.4 r."""
    s, dout = make(dtype, batch, queries, queries, heads, kv_heads, head_len, block, 3, buckets, seed=38)
    got, value = step(s, dout), want(s, dout)
    for x in ("out", "dq", "dk", "dv"):
        exact = value[x][0]
        own = torch.from_numpy(exact).to(dtype).double().numpy() - exact
        error = got[x].detach().cpu().double().numpy() - exact
        assert np.sqrt((error ** 2).mean()) <= 1.05 * np.sqrt((own ** 2).mean()), x


def test_gradients_against_differences():
    s, dout = make(F32, 1, 40, 40, 2, 1, 32, 32, 2, 6, seed=15)
    got = step(s, dout)
    gen = torch.Generator().manual_seed(2)
    for name in ("q", "k", "v", "bias"):
        along = torch.randn(s[name].shape, generator=gen).cuda()
        # central differences in 64 bits of the definition: their own error is of the order h^2, 1e-6 of the value here
        h = 1e-3
        f = lambda t: float((ref.attention(**{**{x: s[x] for x in ("q", "k", "v", "blocks", "bias", "bounds", "causal")}, "block": 32, name: t})["out"][0]
                             * dout.cpu().double().numpy()).sum())
        difference = (f(s[name].double() + h * along.double()) - f(s[name].double() - h * along.double())) / (2 * h)
        slope = float((got["d" + name].double() * along.double()).sum())
        mass = float((got["d" + name].double() * along.double()).abs().sum())
        assert abs(slope - difference) <= 1e-5 * mass + 1e-5 * abs(difference), name


def test_the_same_bits_every_time_and_on_another_stream():
    s, dout = make(BF16, 2, 700, 700, 8, 2, 64, 64, 5, 16, seed=16)
    first = step(s, dout)
    side = torch.cuda.Stream()
    for _ in range(3):
        again = step(s, dout)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step(s, dout)
        third = step(s, dout)                            # beside it
        torch.cuda.current_stream().wait_stream(side)
        for x in first:
            assert torch.equal(first[x], again[x]) and torch.equal(first[x], other[x]) and torch.equal(first[x], third[x])


def test_captured_steps_and_eager_ones_share_nothing():
    from featgraph_amd.module import block_attention as low
    s, dout = make(BF16, 1, 500, 500, 4, 2, 64, 32, 6, 16, seed=17)
    few, _ = make(BF16, 2, 1, 3000, 4, 2, 64, 64, 40, seed=18)

    def train(q, k, v):
        args = (q, k, v, s["blocks"], 32, 0.125, True, None, None, s["bias"], s["bounds"])
        out, lse, rest = low.block_attention_forward(*args, True)
        return (out,) + low.block_attention_backward(*args, out, lse, rest, dout)

    train(s["q"], s["k"], s["v"]), call(few)             # the kernels are loaded
    torch.cuda.synchronize()
    q, k, v = (s[x].clone() for x in ("q", "k", "v"))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(train(q, k, v) + (call(few),))
        graphs.append(graph)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for _ in range(3):
        for t in (q, k, v, few["q"]):
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        value = train(q, k, v) + (call(few),)
        for o in outs:
            for t in o:
                t.fill_(float("nan"))
        graphs[0].replay(), graphs[1].replay()
        eager = train(q, k, v)
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, value))
        assert all(torch.equal(a, b) for a, b in zip(eager, value))


def test_rows_beyond_32_bit_offsets():
    """A sequence that begins more than 2^32 elements behind the first."""
    far = 2 ** 32 + 2 ** 20
    cache = torch.empty(far + 2 ** 20, dtype=BF16, device="cuda")
    s, dout = make(BF16, 2, 40, 100, 4, 2, 64, 32, 3, seed=19)
    views = {}
    for i, x in enumerate(("k", "v")):
        t = cache.as_strided(s[x].shape, (far, 2 * 2 * 64, 2 * 64, 1), i * 64)    # key heads of K and V in turn
        views[x] = t.copy_(s[x])
    got, value = step(dict(s, **views), dout), step(s, dout)
    assert all(torch.equal(got[x], value[x]) for x in got)


def test_tangents_are_refused():
    import torch.autograd.forward_ad as forward
    s, _ = make(BF16, buckets=8)
    plain = call(s)
    with forward.dual_level():
        torch.testing.assert_close(call(s), plain, rtol=2 ** -7, atol=1e-2)
        for name in ("q", "k", "v", "bias"):
            dual = forward.make_dual(s[name], torch.ones_like(s[name]))
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="jvp"):
                    call(s, **{name: dual})
    assert torch.equal(call(s), plain)


def test_refusals():
    from featgraph_amd import ops
    s, _ = make(BF16)
    bad = [dict(q=s["q"].double()), dict(k=s["k"].half()), dict(v=s["v"][:, 1:]), dict(q=s["q"][..., :16]), dict(q=s["q"][0]), dict(block_size=48),
           dict(q=s["q"][:, :, :3]), dict(blocks=s["blocks"].long()), dict(blocks=s["blocks"][:, 1:]), dict(blocks=s["blocks"][..., :0]), dict(blocks=s["blocks"].cpu()),
           dict(lengths=ints(1)), dict(q_lengths=ints(1, 2).long()), dict(lengths=ints(1, 2).cpu()), dict(bias=torch.zeros(4, 4, device="cuda").to(BF16)),
           dict(bias=torch.zeros(4, 4, device="cuda").to(BF16), bounds=(1, 2)), dict(bias=torch.zeros(4, 4, device="cuda").to(BF16), bounds=(3, 2, 4)),
           dict(bias=torch.zeros(3, 4, device="cuda").to(BF16), bounds=(0, 5000)), dict(bias=torch.zeros(65, 4, device="cuda").to(BF16), bounds=range(64)),
           dict(bias=torch.zeros(3, 2, device="cuda").to(BF16), bounds=(1, 2)), dict(bias=torch.zeros(3, 4, device="cuda"), bounds=(1, 2))]
    for change in bad:
        with pytest.raises(ValueError):
            call(s, **change)
    with pytest.raises(TypeError):
        call(s, lengths=[70, 70])
    q = s["q"].detach().requires_grad_()
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        (g,) = torch.autograd.grad(call(s, q=q).float().square().sum(), q, create_graph=True)
        g.float().sum().backward()
    assert ops.block_attention(s["q"][:0], s["k"][:0], s["v"][:0], s["blocks"][:0], 32).shape == (0, 70, 4, 32)
    empty = s["k"][:, :0]
    assert not ops.block_attention(s["q"], empty, empty, s["blocks"], 32).any()
    none = {x: t.detach().requires_grad_() for x, t in (("q", s["q"][:, :0]), ("k", s["k"]), ("v", s["v"]))}
    out = ops.block_attention(none["q"], none["k"], none["v"], s["blocks"][:, :0], 32)
    grads = torch.autograd.grad(out, list(none.values()), torch.zeros_like(out))
    assert out.shape == (2, 0, 4, 32) and not any(g.any() for g in grads)
