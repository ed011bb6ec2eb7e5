"""Calls on caches and rotations that a launch cannot take, fewer than 2^32 threads, are refused for what they are, without a GPU."""
import ctypes

import pytest

from featgraph_amd import _lib

STRIDES = (ctypes.c_int64 * 3)(64 << 30, 64, 64)


def refused(status):
    assert status == -2
    with pytest.raises(ValueError, match="workgroups do not fit a launch"):
        _lib.check(status)


@pytest.mark.parametrize("tokens", [(1 << 26) - 3, 1 << 26, 1 << 30])
def test_rotations(tokens):
    a = _lib.FgRotateArgs(type=2, batch=1, tokens=tokens, heads=1, kv_heads=1, head_len=64, rotary_len=64, interleaved=0, axes=1, eps=1e-6, q=64, k=64,
                          q_strides=STRIDES, k_strides=STRIDES, q_out=64, k_out=64)
    L = _lib.lib()
    refused(L.fg_rotate_heads(ctypes.byref(a), None))
    refused(L.fg_rotate_heads_backward_workspace(ctypes.byref(a)))
    a.tokens = (1 << 26) - 4                # a wavefront each
    assert L.fg_rotate_heads_backward_workspace(ctypes.byref(a)) == 0


@pytest.mark.parametrize("batch,keys,tokens", [(1 << 23, 128, 128), (1 << 30, 1, 1)])
def test_writing_and_reading(batch, keys, tokens):
    L = _lib.lib()
    c = _lib.FgKvCache(bits=4, batch=batch, keys=keys, kv_heads=1, head_len=128, k=64, k_scales=64, v=64, v_scales=64)
    refused(L.fg_cache_write(ctypes.byref(c), 2, 64, STRIDES, 64, STRIDES, tokens, None, None, None))
    refused(L.fg_cache_read(ctypes.byref(c), 2, 64, 64, tokens, None, None, None))


@pytest.mark.parametrize("batch,queries", [(1 << 24, 1), (1 << 20, 256)])
def test_attention(batch, queries):
    L = _lib.lib()
    a = _lib.FgCacheAttentionArgs(type=2, queries=queries, heads=1, causal=1, block=0, topk=0, scale=0.125, q=64, q_strides=STRIDES, blocks=None, out=64)
    a.cache = _lib.FgKvCache(bits=4, batch=batch, keys=1, kv_heads=1, head_len=64, k=64, k_scales=64, v=64, v_scales=64)
    if queries == 1:
        refused(L.fg_cache_attention_workspace(ctypes.byref(a)))
        refused(L.fg_cache_attention(ctypes.byref(a), None, 0, None))
    else:                                   # 32 tokens of one head a workgroup
        assert L.fg_cache_attention_workspace(ctypes.byref(a)) == 0
        a.queries = 512
        refused(L.fg_cache_attention(ctypes.byref(a), None, 0, None))
