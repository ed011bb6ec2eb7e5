"""A cache of keys and values in 4 or 8 bits: writing new tokens into it, reading it back, and the attention that takes it as it is held.  The calls
of the C interface on torch tensors.

Like the attention over float caches these are functions of their tensors (`featgraph_amd.ops`); what they share is the cache itself, four
byte arrays that the caller owns.  Outputs and workspaces come from torch's allocator on the current stream.
The reference has no such operator.
"""
import ctypes
import functools
import operator
import struct

import torch

from .. import _lib
from .block_attention import _TYPES, HEAD_LENGTHS, MAX_GROUP, _check, _check_counts, _check_sizes, _launch, _ptr, _rows

GROUP = 32                                 # elements of one scale

# fg_kv_cache as bytes
_CACHE = struct.Struct("=5i4x4Q")
assert ctypes.sizeof(_lib.FgKvCache) == _CACHE.size


class KeyValueCache(object):
    """Keys and values of `batch` sequences, `keys` of them each, in `bits` (4 or 8) an element.

    k and v: uint8 (batch, kv_heads, keys, head_len * bits / 8), a head's elements in order, 4-bit ones the lower half of a byte first; k_scales and
    v_scales: uint8 (batch, kv_heads, keys, head_len / 32), the exponent plus 127 of the power of two that 32 neighbouring elements
    share (255: none of the 32 is a number).  Elements have a sign and two bits of exponent and one of mantissa (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6) or four and
    three (e4m3, up to 448; not its codes 127 and 255, which are no numbers).  Scales reach 2^125 and 2^119.  The tensors are the caller's: dense, on one GPU, at
    multiples of 16 bytes (scales of 4); zeros hold zeros.  A cache's tensors are not replaced once it is made."""
    __slots__ = ("k", "k_scales", "v", "v_scales", "bits", "batch", "keys", "kv_heads", "head_len", "device")

    def __init__(self, k, k_scales, v, v_scales, bits):
        if bits not in (4, 8):
            raise ValueError("elements of 4 or 8 bits, got %s" % (bits,))
        for name, t in (("k", k), ("k_scales", k_scales), ("v", v), ("v_scales", v_scales)):
            if not isinstance(t, torch.Tensor):
                raise TypeError("%s must be a torch tensor on the GPU, got %s" % (name, type(t)))
            if not t.is_cuda:
                raise ValueError("%s is on %s: there is no CPU path" % (name, t.device))
            if t.dtype != torch.uint8 or t.dim() != 4 or t.device != k.device:
                raise ValueError("%s must be uint8 with 4 axes on %s, got %s of %s on %s" % (name, k.device, tuple(t.shape), t.dtype, t.device))
            if not t.is_contiguous() or t.data_ptr() % (4 if "scales" in name else 16):
                raise ValueError("%s must be dense and stand at a multiple of %d bytes" % (name, 4 if "scales" in name else 16))
        bits = int(bits)
        batch, kv_heads, keys, row = k.shape
        head_len = row * 8 // bits
        if head_len not in HEAD_LENGTHS or row * 8 != head_len * bits:
            raise ValueError("heads of 32, 64 or 128 elements, got rows of %d bytes with %d bits an element" % (row, bits))
        scales = (batch, kv_heads, keys, head_len // GROUP)
        if v.shape != k.shape or tuple(k_scales.shape) != scales or tuple(v_scales.shape) != scales:
            raise ValueError("k is %s: v must be alike and scales %s, got %s, %s and %s"
                             % (tuple(k.shape), scales, tuple(v.shape), tuple(k_scales.shape), tuple(v_scales.shape)))
        if kv_heads < 1:
            raise ValueError("the cache has no heads: shape %s" % (tuple(k.shape),))
        for name, value in zip(self.__slots__, (k, k_scales, v, v_scales, bits, batch, keys, kv_heads, head_len, k.device)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        raise AttributeError("a cache's %s is as it was made: make another KeyValueCache" % name)      # checked once, addressed by every call

    def __reduce__(self):
        return KeyValueCache, (self.k, self.k_scales, self.v, self.v_scales, self.bits)

    def raw(self):
        """fg_kv_cache as bytes."""
        return _CACHE.pack(self.bits, self.batch, self.keys, self.kv_heads, self.head_len, self.k.data_ptr(), self.k_scales.data_ptr(),
                           self.v.data_ptr(), self.v_scales.data_ptr())


def new(batch, keys, kv_heads, head_len, bits, device):
    if min(batch, keys) < 0 or kv_heads < 1 or head_len not in HEAD_LENGTHS or bits not in (4, 8):
        raise ValueError("a cache of %s sequences with room for %s keys, %s heads of %s elements (32, 64 or 128) of %s bits (4 or 8)"
                         % (batch, keys, kv_heads, head_len, bits))
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError("the cache is on %s: there is no CPU path" % device)
    zeros = lambda row: torch.zeros((batch, kv_heads, keys, row), dtype=torch.uint8, device=device)
    row = head_len * bits // 8
    return KeyValueCache(zeros(row), zeros(head_len // GROUP), zeros(row), zeros(head_len // GROUP), bits)


def _check_cache(cache):
    if not isinstance(cache, KeyValueCache):
        raise TypeError("cache must be a KeyValueCache, got %s" % type(cache))


def _check_write(cache, k, v):
    _check_cache(cache)
    _check("k", k, 4)
    _check("v", v, 4, k)
    if k.shape != v.shape or (k.shape[0], k.shape[2], k.shape[3]) != (cache.batch, cache.kv_heads, cache.head_len):
        raise ValueError("k and v must be (%d, tokens, %d, %d) as the cache is, got %s and %s"
                         % (cache.batch, cache.kv_heads, cache.head_len, tuple(k.shape), tuple(v.shape)))
    if k.device != cache.device:
        raise ValueError("k is on %s, the cache on %s" % (k.device, cache.device))


_STRIDES = struct.Struct("=3q")


def write(cache, k, v, lengths, q_lengths):
    try:                                    # whether the arguments are fine as they are, at a glance; what is not is looked at one by one for the message
        batch, tokens, kv_heads, head_len = k.shape
        plain = (v.shape == k.shape and k.dtype in _TYPES and v.dtype == k.dtype and k.device == cache.device and v.device == cache.device
                 and batch == cache.batch and kv_heads == cache.kv_heads and head_len == cache.head_len)
    except (AttributeError, ValueError, TypeError):
        plain = False
    if not plain:
        _check_write(cache, k, v)
    device = cache.device
    if lengths is not None:
        _check_counts("lengths", lengths, batch, device)
    if q_lengths is not None:
        _check_counts("q_lengths", q_lengths, batch, device)
    if tokens > cache.keys and lengths is None and q_lengths is None:
        raise ValueError("%d new tokens for a cache of %d keys" % (tokens, cache.keys))
    k, v = _rows(k), _rows(v)
    _launch(device, _lib.lib().fg_cache_write, cache.raw(), _TYPES[k.dtype], k.data_ptr(), _STRIDES.pack(*k.stride()[:3]), v.data_ptr(),
            _STRIDES.pack(*v.stride()[:3]), tokens, _ptr(lengths), _ptr(q_lengths))


def read(cache, dtype, first, count, lengths):
    _check_cache(cache)
    if dtype not in _TYPES:
        raise ValueError("values are read as float32, float16 or bfloat16, got %s" % (dtype,))
    device = cache.device
    _check_counts("first", first, cache.batch, device)
    _check_counts("lengths", lengths, cache.batch, device)
    count = cache.keys if count is None else operator.index(count)
    if count < 0:
        raise ValueError("%d keys to read" % count)
    shape = (cache.batch, count, cache.kv_heads, cache.head_len)
    k, v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
    _launch(device, _lib.lib().fg_cache_read, cache.raw(), _TYPES[dtype], k.data_ptr(), v.data_ptr(), count, _ptr(first), _ptr(lengths))
    return k, v


# fg_cache_attention_args as bytes, but for the cache between its parts
_HEAD, _REST = struct.Struct("=6if4x"), struct.Struct("=Q3q4Q")
assert ctypes.sizeof(_lib.FgCacheAttentionArgs) == _HEAD.size + _CACHE.size + _REST.size


@functools.lru_cache(maxsize=1024)
def _plan(dtype, queries, heads, causal, block, topk, scale, *cache_sizes):
    """(the part of a call's arguments that goes by its sizes, the device memory that it needs)."""
    head = _HEAD.pack(_TYPES[dtype], queries, heads, causal, block, topk, scale)
    return head, _lib.check(_lib.lib().fg_cache_attention_workspace(head + _CACHE.pack(*cache_sizes, 0, 0, 0, 0) + bytes(_REST.size)))


def _check_blocks(blocks, block_size, batch, queries, cache):
    if blocks is None or block_size is None:
        raise ValueError("blocks and block_size come together")
    _check_sizes(cache.head_len, block_size)
    if not isinstance(blocks, torch.Tensor):
        raise TypeError("blocks must be a torch tensor, got %s" % type(blocks))
    if blocks.dtype != torch.int32 or blocks.device != cache.device or blocks.dim() != 4 or tuple(blocks.shape[:3]) != (batch, queries, cache.kv_heads) \
            or blocks.shape[3] < 1:
        raise ValueError("blocks must be int32 (%d, %d, %d, topk) on %s, got %s of %s on %s"
                         % (batch, queries, cache.kv_heads, cache.device, tuple(blocks.shape), blocks.dtype, blocks.device))


def _check_attention(q, cache):
    _check_cache(cache)
    _check("q", q, 4)
    batch, queries, heads, head_len = q.shape
    if batch != cache.batch or head_len != cache.head_len or q.device != cache.device:
        raise ValueError("q must be (%d, queries, heads, %d) on %s as the cache is, got %s on %s"
                         % (cache.batch, cache.head_len, cache.device, tuple(q.shape), q.device))
    if heads % cache.kv_heads or not 1 <= heads // cache.kv_heads <= MAX_GROUP:
        raise ValueError("%d query heads over %d key heads: 1 to %d of the former to each of the latter" % (heads, cache.kv_heads, MAX_GROUP))


def attention(q, cache, blocks, block_size, scale, causal, lengths, q_lengths):
    try:
        batch, queries, heads, head_len = q.shape
        dtype, device = q.dtype, q.device
        plain = (batch == cache.batch and head_len == cache.head_len and device == cache.device and dtype in _TYPES and not heads % cache.kv_heads
                 and 1 <= heads // cache.kv_heads <= MAX_GROUP)
    except (AttributeError, ValueError, TypeError):
        plain = False
    if not plain:
        _check_attention(q, cache)
    topk = 0
    if blocks is not None or block_size is not None:
        _check_blocks(blocks, block_size, batch, queries, cache)
        blocks, block_size, topk = blocks.contiguous(), int(block_size), blocks.shape[3]
    if lengths is not None:
        _check_counts("lengths", lengths, batch, device)
    if q_lengths is not None:
        _check_counts("q_lengths", q_lengths, batch, device)
    q = _rows(q)
    head, need = _plan(dtype, queries, heads, causal, block_size or 0, topk, head_len ** -0.5 if scale is None else float(scale), cache.bits, batch,
                       cache.keys, cache.kv_heads, head_len)
    out = q.new_empty(q.shape)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    raw = head + cache.raw() + _REST.pack(q.data_ptr(), *q.stride()[:3], _ptr(blocks), _ptr(lengths), _ptr(q_lengths), out.data_ptr())
    _launch(device, _lib.lib().fg_cache_attention, raw, _ptr(work), need)
    return out
