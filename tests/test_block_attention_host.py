"""Attention over selected blocks without a GPU: bounds of buckets, and what the C interface and the functions refuse before they look
at device memory."""
import ctypes

import numpy as np
import pytest
import torch

from featgraph_amd import _lib, ops


def _args(**change):
    a = _lib.FgBlockAttentionArgs()
    a.type, a.batch, a.queries, a.keys, a.heads, a.kv_heads, a.head_len, a.block, a.topk = 2, 1, 100, 200, 8, 2, 64, 64, 4
    a.scale, a.causal = 0.125, 1
    for x in (a.q_strides, a.k_strides, a.v_strides):
        x[0], x[1], x[2] = 64 * 200 * 8, 64 * 8, 64
    for name, value in change.items():
        if name == "bounds":
            for i, x in enumerate(value):
                a.bounds[i] = x
        elif name.endswith("strides"):
            for i, x in enumerate(value):
                getattr(a, name)[i] = x
        else:
            setattr(a, name, value)
    return a


@pytest.mark.parametrize("change,status,words", [
    (dict(type=3), -1, "type"), (dict(batch=-1), -1, "negative"), (dict(topk=0), -1, "no heads or blocks"), (dict(kv_heads=0), -1, "no heads"),
    (dict(head_len=48), -2, "48"), (dict(block=16), -2, "16"), (dict(block=96), -2, "96"), (dict(kv_heads=3), -2, "1 to 16"),
    (dict(heads=34), -2, "1 to 16"), (dict(topk=1 << 24), -2, "too long a list"), (dict(keys=(1 << 30) + 1), -2, "2\\^30"), (dict(n_buckets=65), -2, "65"), (dict(n_buckets=-1), -2, "buckets"),
    (dict(n_buckets=3, bounds=(5, 5)), -1, "ascend"), (dict(n_buckets=3, bounds=(0, 4095)), -2, "apart"),
    (dict(n_buckets=2, bounds=((1 << 30) + 1,)), -2, "apart"), (dict(q_strides=(1, 512, 64)), -1, "16 bytes"), (dict(k=8), -1, "16 bytes")])
def test_c_interface_refuses(change, status, words):
    L = _lib.lib()
    a = _args(**change)
    for call in (lambda: L.fg_block_attention_workspace(ctypes.byref(a)), lambda: L.fg_block_attention_backward_workspace(ctypes.byref(a)),
                 lambda: L.fg_block_attention(ctypes.byref(a), None, 0, None),
                 lambda: L.fg_block_attention_backward(ctypes.byref(a), ctypes.byref(_lib.FgBlockAttentionGrads()), None, 0, None)):
        assert call() == status
        with pytest.raises(ValueError, match=words):
            _lib.check(status)


def test_c_interface_refuses_null_pointers_and_small_workspaces():
    L = _lib.lib()
    a = _args()
    assert L.fg_block_attention(None, None, 0, None) == -1
    assert L.fg_block_attention(ctypes.byref(a), None, 0, None) == -1
    assert L.fg_block_attention_backward(ctypes.byref(a), None, None, 0, None) == -1
    # few queries: their lists are dealt out, and the sums need a place
    a = _args(queries=1, keys=8192, topk=64, q=64, k=64, v=64, blocks=64, out=64, lse=64)
    need = L.fg_block_attention_workspace(ctypes.byref(a))
    assert need > 0
    assert L.fg_block_attention(ctypes.byref(a), None, 0, None) == -1
    assert L.fg_block_attention(ctypes.byref(a), ctypes.c_void_p(256), need - 1, None) == -1
    grads = _lib.FgBlockAttentionGrads(dout=64, dout_strides=a.q_strides, dq=64, dk=64, dv=64)
    need = L.fg_block_attention_backward_workspace(ctypes.byref(a))
    assert need > 0
    assert L.fg_block_attention_backward(ctypes.byref(a), ctypes.byref(grads), ctypes.c_void_p(256), need - 1, None) == -1
    grads.dv = None                                                 # dk alone
    assert L.fg_block_attention_backward(ctypes.byref(a), ctypes.byref(grads), ctypes.c_void_p(256), need, None) == -1
    # nothing to do is no error
    for empty in (dict(batch=0), dict(queries=0)):
        a = _args(**empty)
        assert L.fg_block_attention(ctypes.byref(a), None, 0, None) == 0


def test_c_interface_refuses_what_vector_accesses_cannot_reach():
    L = _lib.lib()
    good = dict(queries=1, keys=8192, topk=64, q=64, k=64, v=64, blocks=64, out=64, lse=64, rest=64)
    work = ctypes.c_void_p(256)
    for name, value in (("out", 72), ("rest", 80 + 2), ("lse", 68), ("q", 72), ("k", 66), ("v", 68), ("blocks", 66), ("lengths", 66), ("q_lengths", 65), ("bias", 65)):
        a = _args(**dict(good, **{name: value}))
        if name == "bias":
            a.n_buckets = 1
        assert L.fg_block_attention(ctypes.byref(a), work, 1 << 40, None) == -1, name
        with pytest.raises(ValueError, match="bytes"):
            _lib.check(-1)
    a = _args(**good)
    assert L.fg_block_attention(ctypes.byref(a), ctypes.c_void_p(264), 1 << 40, None) == -1
    with pytest.raises(ValueError, match="bytes"):
        _lib.check(-1)
    for name, value in (("dout", 72), ("dq", 72), ("dk", 66), ("dv", 68), ("dbias", 65)):
        grads = _lib.FgBlockAttentionGrads(**dict(dict(dout=64, dout_strides=a.q_strides, dq=64, dk=64, dv=64), **{name: value}))
        assert L.fg_block_attention_backward(ctypes.byref(a), ctypes.byref(grads), work, 1 << 40, None) == -1, name
        with pytest.raises(ValueError, match="bytes"):
            _lib.check(-1)
    grads = _lib.FgBlockAttentionGrads(dout=64, dout_strides=a.q_strides, dq=64, dk=64, dv=64)
    assert L.fg_block_attention_backward(ctypes.byref(a), ctypes.byref(grads), ctypes.c_void_p(264), 1 << 40, None) == -1


def test_c_interface_refuses_lists_beyond_32_bits():
    L = _lib.lib()
    size = 1 << 20
    a = _args(batch=64, queries=size, keys=size, topk=16, q_strides=(size * 512, 512, 64), k_strides=(size * 128, 128, 64), v_strides=(size * 128, 128, 64))
    assert L.fg_block_attention_workspace(ctypes.byref(a)) >= 0
    assert L.fg_block_attention_backward_workspace(ctypes.byref(a)) == -2
    with pytest.raises(ValueError, match="32-bit lists"):
        _lib.check(-2)
    a.batch = 1
    # the lists' sums stay within some times the gradients' memory (K's: 256 MiB in 16 bits)
    assert 0 < L.fg_block_attention_backward_workspace(ctypes.byref(a)) < 2 ** 33


@pytest.mark.parametrize("queries,heads,kv_heads,head_len,block,topk", [(8192, 16, 1, 64, 128, 8), (16384, 32, 8, 128, 256, 16), (4096, 16, 4, 128, 64, 16)])
def test_gradients_reserve_no_more_pieces_than_there_can_be(queries, heads, kv_heads, head_len, block, topk):
    L = _lib.lib()
    a = _args(type=1, queries=queries, keys=queries, heads=heads, kv_heads=kv_heads, head_len=head_len, block=block, topk=topk)
    for x, h in ((a.q_strides, heads), (a.k_strides, kv_heads), (a.v_strides, kv_heads)):
        x[0], x[1], x[2] = queries * h * head_len, h * head_len, head_len
    # a list of n tokens has floor(n / piece) + 1 pieces at most, and a piece some 768 rows at least; beside their sums there are rows of delta, marks
    # (a bit for each token and block) and the lists
    entries, blocks = queries * kv_heads * topk, kv_heads * queries // block
    sums = (entries * (heads // kv_heads) // 768 + blocks) * 2 * block * head_len * 4
    rest = 4 * queries * heads + blocks * queries // 8 + 4 * entries + 2 ** 20
    need = L.fg_block_attention_backward_workspace(ctypes.byref(a))
    assert 0 < need <= sums + rest
    rows = entries * (heads // kv_heads)
    piece = min(max(2048, rows // 8192), max(768, rows // 1024))
    assert need <= (entries * (heads // kv_heads) // piece + blocks) * 2 * block * head_len * 4 + rest


def test_pool_and_select_refuse():
    L = _lib.lib()
    strides = (ctypes.c_int64 * 3)(64 * 200 * 2, 64 * 2, 64)

    def pool(type=1, batch=1, keys=200, kv_heads=2, head_len=64, block=32, k=64):
        return L.fg_block_pool(type, k, strides, None, 64, batch, keys, kv_heads, head_len, block, None)

    def select(type=1, batch=1, queries=10, keys=200, heads=4, kv_heads=2, head_len=64, block=32, topk=4, first=1, last=1, q=64, out=64):
        return L.fg_block_select(type, q, strides, 64, None, None, out, batch, queries, keys, heads, kv_heads, head_len, block, topk, 1, first, last, None)

    assert pool(type=5) == -1 and pool(batch=-1) == -1 and pool(k=None) == -1 and pool(k=72) == -1
    assert pool(head_len=20) == -2 and pool(block=48) == -2 and pool(keys=(1 << 30) + 1) == -2
    assert pool(batch=0) == 0 and pool(keys=0) == 0
    assert select(topk=0) == -1 and select(first=3, last=2) == -1 and select(first=-1) == -1 and select(q=None) == -1 and select(out=None) == -1
    assert select(heads=5) == -2 and select(keys=2048 * 32 + 1) == -2 and select(head_len=256) == -2
    assert select(batch=0) == 0 and select(queries=0) == 0


def test_functions_refuse_what_is_not_on_a_gpu():
    q = torch.zeros(1, 4, 2, 32)
    for call in (lambda: ops.pool_blocks(q, 32), lambda: ops.select_blocks(q, torch.zeros(1, 2, 1, 32), 4, 32, 1),
                 lambda: ops.block_attention(q, q, q, torch.zeros(1, 4, 2, 1, dtype=torch.int32), 32)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(TypeError, match="torch tensor"):
        ops.pool_blocks(np.zeros((1, 4, 2, 32)), 32)


@pytest.mark.parametrize("buckets,far,causal", [(2, 128, True), (3, 10, True), (8, 128, True), (32, 128, True), (32, 2000, True), (64, 64, True),
                                                (4, 128, False), (5, 64, False), (16, 128, False), (32, 128, False), (64, 500, False)])
def test_position_bounds(buckets, far, causal):
    bounds = ops.position_bounds(buckets, far, causal)
    assert len(bounds) == buckets - 1 and all(x < y for x, y in zip(bounds, bounds[1:]))
    if causal:
        near = buckets // 2                                         # distances 0 .. near - 1 have buckets of their own
        assert bounds[:near] == tuple(range(1, near + 1))
        assert bounds[-1] <= max(far, buckets)
    else:
        assert 0 in bounds and 1 in bounds                          # distance 0 is apart from both sides
        assert bounds[0] <= 0 and 1 < bounds[-1]                    # negative distances, 0, and positive ones


def test_position_bounds_refuses():
    for buckets, far, causal in ((1, 128, True), (65, 128, True), (3, 128, False), (32, 20, True), (32, 3000, True)):
        with pytest.raises(ValueError):
            ops.position_bounds(buckets, far, causal)
