"""A cache in 4 or 8 bits and heads normed and rotated without a GPU: what the C interface and the functions refuse before they look at device
memory, and the oracles against one another."""
import ctypes

import numpy as np
import pytest
import torch

import cache_reference
import rotate_reference
from featgraph_amd import _lib, ops

STRIDES = (ctypes.c_int64 * 3)(64 * 200 * 2, 64 * 2, 64)


def _cache(**change):
    c = _lib.FgKvCache(bits=4, batch=2, keys=200, kv_heads=2, head_len=64, k=64, k_scales=64, v=64, v_scales=64)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def _attention(cache=None, **change):
    a = _lib.FgCacheAttentionArgs(type=2, queries=1, heads=8, causal=1, block=0, topk=0, scale=0.125, q=64, q_strides=STRIDES, blocks=None, out=64)
    a.cache = _cache(**(cache or {}))
    for name, value in change.items():
        setattr(a, name, (ctypes.c_int64 * 3)(*value) if name == "q_strides" else value)
    return a


def _rotate(**change):
    a = _lib.FgRotateArgs(type=2, batch=2, tokens=10, heads=8, kv_heads=2, head_len=64, rotary_len=64, interleaved=0, axes=1, eps=1e-6, q=64, k=64,
                          q_strides=STRIDES, k_strides=STRIDES, q_weight=64, k_weight=64, q_out=64, k_out=64)
    for name, value in change.items():
        if name == "axis":
            a.axis[3] = value
        else:
            setattr(a, name, (ctypes.c_int64 * 3)(*value) if name.endswith("strides") else value)
    return a


def _refused(status, got, words):
    assert got == status
    with pytest.raises(ValueError, match=words):
        _lib.check(got)


@pytest.mark.parametrize("change,status,words", [
    (dict(bits=2), -1, "4 or 8 bits"), (dict(bits=16), -1, "4 or 8 bits"), (dict(batch=-1), -1, "negative"), (dict(keys=-1), -1, "negative"),
    (dict(kv_heads=0), -1, "no heads"), (dict(head_len=48), -2, "48"), (dict(head_len=256), -2, "256"), (dict(keys=(1 << 30) + 1), -2, "2\\^30"),
    (dict(k=72), -1, "16 bytes"), (dict(v=8), -1, "16 bytes"), (dict(k_scales=66), -1, "4 bytes"), (dict(v_scales=65), -1, "4 bytes"),
    (dict(k=None), -1, "null"), (dict(v_scales=None), -1, "null")])
def test_what_is_no_cache(change, status, words):
    L = _lib.lib()
    c = _cache(**change)
    _refused(status, L.fg_cache_write(ctypes.byref(c), 2, 64, STRIDES, 64, STRIDES, 1, None, None, None), words)
    _refused(status, L.fg_cache_read(ctypes.byref(c), 2, 64, 64, 1, None, None, None), words)
    a = _attention(cache=change)
    if words in ("16 bytes", "4 bytes", "null"):
        assert L.fg_cache_attention_workspace(ctypes.byref(a)) >= 0         # looks at sizes alone
    else:
        _refused(status, L.fg_cache_attention_workspace(ctypes.byref(a)), words)
    _refused(status, L.fg_cache_attention(ctypes.byref(a), None, 0, None), words)


def test_writing_and_reading_refuse():
    L = _lib.lib()
    c = _cache()
    odd = (ctypes.c_int64 * 3)(64 * 200 * 2, 64 * 2 + 1, 64)

    def write(cache=c, type=2, k=64, ks=STRIDES, v=64, vs=STRIDES, tokens=1, lengths=None, q_lengths=None):
        return L.fg_cache_write(cache if cache is None else ctypes.byref(cache), type, k, ks, v, vs, tokens, lengths, q_lengths, None)

    def read(cache=c, type=2, k=64, v=64, count=1, first=None, lengths=None):
        return L.fg_cache_read(cache if cache is None else ctypes.byref(cache), type, k, v, count, first, lengths, None)

    for call, words in ((lambda: write(cache=None), "null"), (lambda: write(type=3), "type"), (lambda: write(tokens=-1), "new tokens"), (lambda: write(k=None), "null"), (lambda: write(v=None), "null"),
                       (lambda: write(ks=None), "null"), (lambda: write(k=72), "16 bytes"), (lambda: write(vs=odd), "16 bytes"), (lambda: write(lengths=66), "4 bytes"),
                       (lambda: write(q_lengths=65), "4 bytes"), (lambda: read(cache=None), "null"), (lambda: read(type=-1), "type"), (lambda: read(count=-1), "to read"),
                       (lambda: read(k=None), "null"), (lambda: read(v=72), "16 bytes"), (lambda: read(first=66), "4 bytes"), (lambda: read(lengths=66), "4 bytes")):
        _refused(-1, call(), words)
    # more workgroups than a launch takes
    big = _cache(batch=1 << 12, keys=1 << 20, kv_heads=64, head_len=128)
    _refused(-2, write(cache=big, tokens=1 << 20), "workgroups")
    _refused(-2, read(cache=big, count=1 << 20), "workgroups")
    assert write(tokens=0) == 0 and read(count=0) == 0 and write(cache=_cache(batch=0)) == 0 and write(cache=_cache(keys=0)) == 0


@pytest.mark.parametrize("change,status,words", [
    (dict(type=7), -1, "type"), (dict(queries=-1), -1, "negative"), (dict(heads=0), -1, "no heads"), (dict(heads=7), -2, "1 to 16"), (dict(heads=34), -2, "1 to 16"),
    (dict(queries=(1 << 30) + 1), -2, "2\\^30"), (dict(topk=-1), -1, "blocks a query"), (dict(topk=2, block=48), -2, "48"), (dict(topk=1 << 24, block=64), -2, "too long"),
    (dict(q=72), -1, "16 bytes"), (dict(q_strides=(1, 64, 64)), -1, "16 bytes"), (dict(out=72), -1, "16 bytes"), (dict(topk=1, block=64, blocks=66), -1, "4 bytes"),
    (dict(lengths=66), -1, "4 bytes"), (dict(q_lengths=66), -1, "4 bytes")])
def test_attention_refuses(change, status, words):
    L = _lib.lib()
    a = _attention(**change)
    _refused(status, L.fg_cache_attention_workspace(ctypes.byref(a)), words)
    _refused(status, L.fg_cache_attention(ctypes.byref(a), None, 0, None), words)


def test_attention_refuses_null_pointers_and_small_workspaces():
    L = _lib.lib()
    assert L.fg_cache_attention(None, None, 0, None) == -1 and L.fg_cache_attention_workspace(None) == -1
    for change in (dict(q=None), dict(out=None), dict(topk=1, block=64)):
        _refused(-1, L.fg_cache_attention(ctypes.byref(_attention(**change)), None, 0, None), "null")
    a = _attention(cache=dict(keys=100000))
    need = L.fg_cache_attention_workspace(ctypes.byref(a))
    assert need > 0
    _refused(-1, L.fg_cache_attention(ctypes.byref(a), None, 0, None), "workspace")
    _refused(-1, L.fg_cache_attention(ctypes.byref(a), ctypes.c_void_p(256), need - 1, None), "needed")
    _refused(-1, L.fg_cache_attention(ctypes.byref(a), ctypes.c_void_p(264), need, None), "16 bytes")
    for a in (_attention(queries=0), _attention(cache=dict(batch=0))):
        assert L.fg_cache_attention(ctypes.byref(a), None, 0, None) == 0


@pytest.mark.parametrize("change,status,words", [
    (dict(type=3), -1, "type"), (dict(batch=-1), -1, "negative"), (dict(heads=0), -1, "no heads"), (dict(kv_heads=0), -1, "no heads"), (dict(head_len=96), -2, "96"),
    (dict(rotary_len=8), -2, "multiple of 16"), (dict(rotary_len=80), -2, "multiple of 16"), (dict(rotary_len=-16), -2, "multiple of 16"),
    (dict(axes=0), -1, "axes"), (dict(axes=9), -1, "axes"), (dict(axes=2), -1, "positions"), (dict(eps=-1.0), -1, "eps"), (dict(eps=float("nan")), -1, "eps"), (dict(axis=1), -1, "axis 1 of 1"),
    (dict(q_weight=None), -1, "come together"), (dict(q=72), -1, "16 bytes"), (dict(k_strides=(64, 1, 64)), -1, "16 bytes"), (dict(k_weight=72), -1, "16 bytes"),
    (dict(positions=66), -1, "4 bytes"), (dict(lengths=66), -1, "4 bytes"), (dict(q_out=72), -1, "16 bytes"), (dict(tokens=(1 << 30) + 1), -2, "2\\^30"),
    (dict(tokens=1 << 30, batch=1 << 10, heads=1 << 10), -2, "workgroups")])
def test_rotation_refuses(change, status, words):
    L = _lib.lib()
    a = _rotate(**change)
    grads = _lib.FgRotateGrads()
    _refused(status, L.fg_rotate_heads(ctypes.byref(a), None), words)
    _refused(status, L.fg_rotate_heads_backward_workspace(ctypes.byref(a)), words)
    _refused(status, L.fg_rotate_heads_backward(ctypes.byref(a), ctypes.byref(grads), None, 0, None), words)


def test_rotation_refuses_null_pointers_and_small_workspaces():
    L = _lib.lib()
    assert L.fg_rotate_heads(None, None) == -1 and L.fg_rotate_heads_backward_workspace(None) == -1
    for change in (dict(q=None), dict(k=None), dict(q_out=None), dict(k_out=None)):
        _refused(-1, L.fg_rotate_heads(ctypes.byref(_rotate(**change)), None), "null")
    a = _rotate()
    need = L.fg_rotate_heads_backward_workspace(ctypes.byref(a))
    assert need > 0 and L.fg_rotate_heads_backward_workspace(ctypes.byref(_rotate(q_weight=None, k_weight=None))) == 0
    good = dict(dq_out=64, dk_out=64, dq_out_strides=STRIDES, dk_out_strides=STRIDES, dq=64, dk=64, dq_weight=64, dk_weight=64)
    call = lambda work, size, **change: L.fg_rotate_heads_backward(ctypes.byref(a), ctypes.byref(_lib.FgRotateGrads(**dict(good, **change))), work, size, None)
    _refused(-1, L.fg_rotate_heads_backward(ctypes.byref(a), None, None, 0, None), "null")
    work = ctypes.c_void_p(256)
    _refused(-1, call(None, 0), "workspace")
    _refused(-1, call(work, need - 1), "needed")
    _refused(-1, call(ctypes.c_void_p(264), need), "16 bytes")
    for name in ("dq_out", "dk_out", "dq", "dk", "dq_weight", "dk_weight"):
        _refused(-1, call(work, need, **{name: None}), "null")
    for name, value in (("dq_out", 72), ("dk", 72), ("dq_weight", 65)):
        _refused(-1, call(work, need, **{name: value}), "bytes")
    for empty in (dict(batch=0), dict(tokens=0)):
        assert L.fg_rotate_heads(ctypes.byref(_rotate(**empty)), None) == 0


def test_functions_refuse_what_is_not_on_a_gpu():
    q = torch.zeros(1, 4, 2, 32)
    codes = torch.zeros(1, 2, 4, 16, dtype=torch.uint8)
    for call in (lambda: ops.rotate_heads(q, q), lambda: ops.KeyValueCache(codes, codes, codes, codes, 4), lambda: ops.new_cache(1, 4, 2, 32, device="cpu")):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    for call in (lambda: ops.rotate_heads(np.zeros((1, 4, 2, 32)), q), lambda: ops.KeyValueCache(np.zeros(4), codes, codes, codes, 4),
                 lambda: ops.write_cache(codes, q, q), lambda: ops.read_cache(None), lambda: ops.cache_attention(q, (codes, codes))):
        with pytest.raises(TypeError):
            call()
    for bad in (dict(bits=5), dict(head_len=48), dict(kv_heads=0), dict(batch=-1), dict(keys=-1)):
        with pytest.raises(ValueError):
            ops.new_cache(**dict(dict(batch=1, keys=4, kv_heads=2, head_len=32), **bad))


@pytest.mark.parametrize("bits", [4, 8])
def test_the_oracle_of_a_cache(bits):
    table = cache_reference.MAGNITUDES[bits]
    assert (np.diff(table) > 0).all() and len(table) == (8 if bits == 4 else 127)
    if bits == 8:                           # torch's own e4m3
        assert np.array_equal(table, torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy())
        gen = torch.Generator().manual_seed(0)
        x = torch.randn((50, 32), generator=gen)
        x[:, 0] = 448                       # the scale is 1: rounding is torch's
        codes, scales = cache_reference.quantise(x.numpy(), 8)
        assert (scales == 127).all() and np.array_equal(codes, x.to(torch.float8_e4m3fn).view(torch.uint8).numpy())
    # no element of the same scale is nearer, and half the scale would not hold the largest value
    rng = np.random.default_rng(1)
    x = rng.standard_normal((200, 32)) * 2.0 ** rng.integers(-60, 60, (200, 1))
    codes, scales = cache_reference.quantise(x, bits)
    got, scale = cache_reference.values(codes, scales, bits), 2.0 ** (scales.astype(int) - 127.0)
    every = np.concatenate((table, -table)) * scale[..., None]
    assert np.array_equal(np.abs(got - x), np.abs(every[:, None, :].reshape(200, 1, -1) - x[..., None]).min(-1))
    assert (np.abs(x).max(1) > table[-1] * scale[:, 0] / 2).all() and (np.abs(x).max(1) <= (table[-1] + (table[-1] - table[-2]) / 2) * scale[:, 0]).all()


def test_the_oracle_of_a_rotation_by_differences():
    gen = torch.Generator().manual_seed(2)
    x, dout, step = (torch.randn((2, 3, 2, 32), generator=gen, dtype=torch.float64) for _ in range(3))
    w, dw = (torch.randn(32, generator=gen, dtype=torch.float64) for _ in range(2))
    for interleaved in (False, True):
        cos, sin, there = rotate_reference.angles(x.shape, 16, lengths=[9, 2], q_lengths=[3, 2])
        loss = lambda x, w: (rotate_reference.rotate(x, w, cos, sin, there, 16, interleaved)["y"][0] * dout.numpy() * there).sum()
        got = rotate_reference.rotate(x, w, cos, sin, there, 16, interleaved, dout=dout)
        h = 1e-5
        slope = (loss(x + h * step, w) - loss(x - h * step, w)) / (2 * h)
        assert abs(slope - (got["dx"][0] * step.numpy()).sum()) < 1e-7
        slope = (loss(x, w + h * dw) - loss(x, w - h * dw)) / (2 * h)
        assert abs(slope - (got["dw"][0] * dw.numpy()).sum()) < 1e-7
