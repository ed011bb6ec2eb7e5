"""Attention over blocks of keys that every query selects, on the matrix cores: the calls of the C interface on torch tensors.

The graph of this attention -- which blocks of keys a query attends to -- is made on the GPU by every call's data, so there is nothing
to lay out ahead of a call and no module to build: the operators are functions of their tensors (`featgraph_amd.ops`).  Outputs and
workspaces come from torch's allocator on the current stream, so calls on several streams, and captured ones, share nothing.
The reference has no such operator.
"""
import ctypes
import functools
import struct

import torch

from .. import _lib
from . import common

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
HEAD_LENGTHS, BLOCK_SIZES, MAX_GROUP, MAX_BUCKETS, MAX_SPAN = (32, 64, 128), (32, 64, 128, 256), 16, 64, 4094


def _check(name, t, dims, like=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor on the GPU, got %s" % (name, type(t)))
    if not t.is_cuda:
        raise ValueError("%s is on %s: there is no CPU path" % (name, t.device))
    if t.dtype not in _TYPES:
        raise ValueError("%s must be float32, float16 or bfloat16, got %s" % (name, t.dtype))
    if t.dim() != dims:
        raise ValueError("%s must have %d axes, got shape %s" % (name, dims, tuple(t.shape)))
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError("%s is %s on %s, the queries are %s on %s" % (name, t.dtype, t.device, like.dtype, like.device))


def _check_counts(name, t, batch, device):
    if t is None:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError("%s must be a torch tensor, got %s" % (name, type(t)))
    if t.dtype != torch.int32 or t.device != device or tuple(t.shape) != (batch,) or not t.is_contiguous():
        raise ValueError("%s must be %d int32 values on %s, got %s of %s on %s" % (name, batch, device, tuple(t.shape), t.dtype, t.device))


def _check_sizes(head_len, block_size, heads=None, kv_heads=None):
    if head_len not in HEAD_LENGTHS:
        raise ValueError("heads of 32, 64 or 128 elements, got %d" % head_len)
    if block_size not in BLOCK_SIZES:
        raise ValueError("blocks of 32, 64, 128 or 256 keys, got %s" % (block_size,))
    if heads is not None and (kv_heads < 1 or heads % kv_heads or not 1 <= heads // kv_heads <= MAX_GROUP):
        raise ValueError("%d query heads over %d key heads: 1 to %d of the former to each of the latter" % (heads, kv_heads, MAX_GROUP))


def _rows(t):
    """The tensor itself where the kernels can address it -- dense heads at 16-byte addresses -- or else a dense copy."""
    a, b, c, d = t.stride()
    if d == 1 and not (a | b | c) * t.element_size() % 16 and not t.data_ptr() % 16:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _call(device, f):
    """f(library, current stream) with `device` current; the common case, where it is already, without the guard's 2 us."""
    if torch.cuda.current_device() == device.index:
        return f(_lib.lib(), common.stream_ptr())
    with torch.cuda.device(device):
        return f(_lib.lib(), common.stream_ptr())


def _launch(device, function, *args):
    """function(*args, current stream) of the library with `device` current, its status checked."""
    if torch.cuda.current_device() == device.index:
        status = function(*args, common.stream_ptr())
    else:
        with torch.cuda.device(device):
            status = function(*args, common.stream_ptr())
    if status < 0:
        _lib.check(status)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _strides(t):
    return _Strides(*t.stride()[:3])


_Strides = ctypes.c_int64 * 3


def block_pool(k, block_size, lengths):
    _check("k", k, 4)
    batch, keys, kv_heads, head_len = k.shape
    _check_sizes(head_len, block_size)
    _check_counts("lengths", lengths, batch, k.device)
    if kv_heads < 1:
        raise ValueError("k has no heads: shape %s" % (tuple(k.shape),))
    k = _rows(k)
    pooled = torch.empty((batch, kv_heads, -(-keys // block_size), head_len), dtype=k.dtype, device=k.device)
    _lib.check(_call(k.device, lambda L, stream: L.fg_block_pool(
        _TYPES[k.dtype], k.data_ptr(), _strides(k), _ptr(lengths), pooled.data_ptr(), batch, keys, kv_heads, head_len, block_size, stream)))
    return pooled


def block_select(q, pooled, num_keys, block_size, topk, causal, lengths, q_lengths, keep_first, keep_last):
    _check("q", q, 4)
    _check("pooled", pooled, 4, q)
    batch, queries, heads, head_len = q.shape
    kv_heads = pooled.shape[1]
    _check_sizes(head_len, block_size, heads, kv_heads)
    if num_keys < 0 or tuple(pooled.shape) != (batch, kv_heads, -(-num_keys // block_size), head_len):
        raise ValueError("pooled keys of %s keys in blocks of %d must be (%d, kv_heads, blocks, %d), got %s"
                         % (num_keys, block_size, batch, head_len, tuple(pooled.shape)))
    if topk < 1 or keep_first < 0 or keep_last < 0 or keep_first + keep_last > topk:
        raise ValueError("topk must be at least 1 and hold the first %s and the last %s blocks, got %s" % (keep_first, keep_last, topk))
    _check_counts("lengths", lengths, batch, q.device)
    _check_counts("q_lengths", q_lengths, batch, q.device)
    q, pooled = _rows(q), pooled.contiguous()
    if pooled.data_ptr() % 16:
        pooled = pooled.clone()
    blocks = torch.empty((batch, queries, kv_heads, topk), dtype=torch.int32, device=q.device)
    _lib.check(_call(q.device, lambda L, stream: L.fg_block_select(
        _TYPES[q.dtype], q.data_ptr(), _strides(q), pooled.data_ptr(), _ptr(lengths), _ptr(q_lengths), blocks.data_ptr(), batch, queries, num_keys,
        heads, kv_heads, head_len, block_size, topk, int(causal), keep_first, keep_last, stream)))
    return blocks


def _plain(q, k, v, blocks, block_size):
    """Whether the arguments are fine as they are, at a glance (1 us); what is not is looked at one by one for the message."""
    try:
        batch, queries, heads, head_len = q.shape
        _, keys, kv_heads, _ = k.shape
        device, dtype = q.device, q.dtype
        return (k.shape == (batch, keys, kv_heads, head_len) and v.shape == k.shape and blocks.shape[:3] == (batch, queries, kv_heads)
                and blocks.dim() == 4 and blocks.shape[3] > 0 and blocks.dtype == torch.int32 and dtype in _TYPES and k.dtype == dtype and v.dtype == dtype
                and device.type == "cuda" and k.device == device and v.device == device and blocks.device == device and head_len in HEAD_LENGTHS
                and block_size in BLOCK_SIZES and kv_heads > 0 and heads % kv_heads == 0 and 1 <= heads // kv_heads <= MAX_GROUP)
    except (AttributeError, ValueError, TypeError, IndexError):
        return False


def check_attention(q, k, v, blocks, block_size, lengths, q_lengths, bias, bounds):
    """The bounds as a tuple, after everything that can be seen of the arguments without looking at their values on the GPU."""
    if bias is None and bounds is None and lengths is None and q_lengths is None and _plain(q, k, v, blocks, block_size):
        return ()
    _check("q", q, 4)
    _check("k", k, 4, q)
    _check("v", v, 4, q)
    batch, queries, heads, head_len = q.shape
    keys, kv_heads = k.shape[1], k.shape[2]
    if tuple(k.shape) != (batch, keys, kv_heads, head_len) or k.shape != v.shape:
        raise ValueError("k and v must be (%d, keys, kv_heads, %d), got %s and %s" % (batch, head_len, tuple(k.shape), tuple(v.shape)))
    _check_sizes(head_len, block_size, heads, kv_heads)
    if not isinstance(blocks, torch.Tensor):
        raise TypeError("blocks must be a torch tensor, got %s" % type(blocks))
    if blocks.dtype != torch.int32 or blocks.device != q.device or blocks.dim() != 4 or tuple(blocks.shape[:3]) != (batch, queries, kv_heads) \
            or blocks.shape[3] < 1:
        raise ValueError("blocks must be int32 (%d, %d, %d, topk) on %s, got %s of %s on %s"
                         % (batch, queries, kv_heads, q.device, tuple(blocks.shape), blocks.dtype, blocks.device))
    _check_counts("lengths", lengths, batch, q.device)
    _check_counts("q_lengths", q_lengths, batch, q.device)
    if (bias is None) != (bounds is None):
        raise ValueError("bias and bounds come together")
    if bias is None:
        return ()
    _check("bias", bias, 2, q)
    bounds = tuple(int(x) for x in bounds)
    if not 1 <= bias.shape[0] <= MAX_BUCKETS or bias.shape[1] != heads or len(bounds) != bias.shape[0] - 1:
        raise ValueError("bias must be (buckets, %d) with 1 to %d buckets and one bound less, got %s and %d bounds"
                         % (heads, MAX_BUCKETS, tuple(bias.shape), len(bounds)))
    if any(x >= y for x, y in zip(bounds, bounds[1:])):
        raise ValueError("the bounds must ascend, got %s" % (bounds,))
    if bounds and (bounds[-1] - bounds[0] > MAX_SPAN or max(-bounds[0], bounds[-1]) > 2 ** 30):
        raise ValueError("the last bound must be within %d of the first, got %s" % (MAX_SPAN, bounds))
    return bounds


# fg_block_attention_args as bytes: whole numbers, scale, buckets and bounds; pointers and strides
_SIZES = struct.Struct("=10ifi63i4x")
_REST = struct.Struct("=3Q9q7Q")
assert ctypes.sizeof(_lib.FgBlockAttentionArgs) == _SIZES.size + _REST.size and _lib.FgBlockAttentionArgs.q.offset == _SIZES.size


class _Sizes(object):
    """The part of a call's arguments that goes by its tensors' sizes, and the device memory that it needs."""

    def __init__(self, sizes, bounds, buckets):
        self.bytes = _SIZES.pack(*sizes, buckets, *bounds, *(0,) * (63 - len(bounds)))
        self._need = [None, None]

    def workspace(self, backward):
        if self._need[backward] is None:
            L, raw = _lib.lib(), self.bytes + bytes(_REST.size)
            self._need[backward] = _lib.check((L.fg_block_attention_backward_workspace if backward else L.fg_block_attention_workspace)(raw))
        return self._need[backward]


@functools.lru_cache(maxsize=1024)
def _sizes(*key):
    return _Sizes(*key)


def _arguments(q, k, v, blocks, block_size, scale, causal, lengths, q_lengths, bias, bounds, out, lse, rest):
    """(the part of fg_block_attention_args that goes by sizes, all of it as bytes)."""
    batch, queries, heads, head_len = q.shape
    _, keys, kv_heads, _ = k.shape
    sizes = _sizes((_TYPES[q.dtype], batch, queries, keys, heads, kv_heads, head_len, block_size, blocks.shape[3], causal, scale), bounds,
                   0 if bias is None else len(bounds) + 1)
    return sizes, sizes.bytes + _REST.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                                           blocks.data_ptr(), _ptr(lengths), _ptr(q_lengths), _ptr(bias), out.data_ptr(), _ptr(lse), _ptr(rest))


def block_attention_forward(q, k, v, blocks, block_size, scale, causal, lengths, q_lengths, bias, bounds, train):
    """(out, lse, rest) of checked arguments; with `train` the latter are what the gradients start from: every row's reference and
    the logarithm of its sum and, in 16 bits, what rounding took from `out`."""
    q, k, v, blocks = _rows(q), _rows(k), _rows(v), blocks.contiguous()
    bias = None if bias is None else bias.contiguous()
    device = q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    lse = torch.empty(q.shape[:3] + (2,), dtype=torch.float32, device=device) if train else None
    rest = torch.empty_like(out) if train and q.dtype != torch.float32 else None
    sizes, raw = _arguments(q, k, v, blocks, block_size, scale, causal, lengths, q_lengths, bias, bounds, out, lse, rest)
    need = sizes.workspace(False)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _lib.check(_call(device, lambda L, stream: L.fg_block_attention(raw, _ptr(work), need, stream)))
    return out, lse, rest


def block_attention_backward(q, k, v, blocks, block_size, scale, causal, lengths, q_lengths, bias, bounds, out, lse, rest, dout, keys_too=True):
    """(dq, dk, dv, dbias) for dL/d(out) = dout; dk and dv None unless `keys_too`, dbias None without a bias."""
    q, k, v, blocks, dout = _rows(q), _rows(k), _rows(v), blocks.contiguous(), _rows(dout)
    bias = None if bias is None else bias.contiguous()
    new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)
    dq = new(q)
    dk, dv = (new(k), new(v)) if keys_too else (None, None)
    dbias = None if bias is None else new(bias)
    sizes, raw = _arguments(q, k, v, blocks, block_size, scale, causal, lengths, q_lengths, bias, bounds, out, lse, rest)
    grads = _lib.FgBlockAttentionGrads(dout.data_ptr(), _strides(dout), dq.data_ptr(), _ptr(dk), _ptr(dv), _ptr(dbias))
    need = sizes.workspace(True)
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _lib.check(_call(q.device, lambda L, stream: L.fg_block_attention_backward(raw, ctypes.byref(grads), _ptr(work), need, stream)))
    return dq, dk, dv, dbias
