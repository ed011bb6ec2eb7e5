"""RMS norm of every head of queries and keys and their rotation by position, in one pass, with its gradients: the calls of the C interface on
torch tensors (`featgraph_amd.ops.rotate_heads`).  Outputs and workspaces come from torch's allocator on the current stream.
The reference has no such operator.
"""
import ctypes
import functools
import math
import struct

import torch

from .. import _lib
from .block_attention import _TYPES, HEAD_LENGTHS, _call, _check, _check_counts, _ptr, _rows, _strides

MAX_AXES = 8

# fg_rotate_args as bytes: what goes by sizes, the angles, pointers and strides
_SIZES, _ANGLES, _REST = struct.Struct("=9if"), struct.Struct("=64d64B"), struct.Struct("=2Q6q7Q")
assert ctypes.sizeof(_lib.FgRotateArgs) == _SIZES.size + _ANGLES.size + _REST.size and _lib.FgRotateArgs.q.offset == _SIZES.size + _ANGLES.size


@functools.lru_cache(maxsize=256)
def _angles(rotary_len, sections, base, frequencies):
    """turns and axis of every pair, as bytes."""
    pairs = rotary_len // 2
    if frequencies is None:
        frequencies = [base ** (-i / pairs) for i in range(pairs)]
    axis = [a for a, many in enumerate(sections) for _ in range(many)]
    none = 64 - pairs
    return _ANGLES.pack(*[f / (2 * math.pi) for f in frequencies], *[0.0] * none, *axis, *[0] * none)


def check(q, k, q_weight, k_weight, positions, lengths, q_lengths, base, frequencies, sections, rotary_len, interleaved, eps):
    """What a call's arguments come to beside its tensors: (rotary_len, interleaved, axes, eps, angles)."""
    _check("q", q, 4)
    _check("k", k, 4, q)
    batch, tokens, heads, head_len = q.shape
    if tuple(k.shape[:2]) != (batch, tokens) or k.shape[3] != head_len or heads < 1 or k.shape[2] < 1:
        raise ValueError("q and k must be (batch, tokens, heads, head_len) of as many tokens, got %s and %s" % (tuple(q.shape), tuple(k.shape)))
    if head_len not in HEAD_LENGTHS:
        raise ValueError("heads of 32, 64 or 128 elements, got %d" % head_len)
    if (q_weight is None) != (k_weight is None):
        raise ValueError("weights for queries and keys come together")
    if q_weight is not None:
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            _check(name, w, 1, q)
            if w.shape[0] != head_len:
                raise ValueError("%s must be (%d,), got %s" % (name, head_len, tuple(w.shape)))
    rotary_len = head_len if rotary_len is None else rotary_len
    if rotary_len < 0 or rotary_len > head_len or rotary_len % 16:
        raise ValueError("a multiple of 16 elements of a head of %d can be turned, got %s" % (head_len, rotary_len))
    pairs = rotary_len // 2
    sections = (pairs,) if sections is None else tuple(int(x) for x in sections)
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError("sections must share the %d pairs out to 1 to %d axes, got %s" % (pairs, MAX_AXES, sections))
    if frequencies is not None:
        frequencies = tuple(float(x) for x in frequencies)
        if len(frequencies) != pairs or not all(math.isfinite(x) for x in frequencies):
            raise ValueError("frequencies must be %d finite numbers, got %s" % (pairs, frequencies))
    elif not (base > 0 and math.isfinite(base)):
        raise ValueError("base must be a number above 0, got %s" % (base,))
    if not eps >= 0:
        raise ValueError("eps must be 0 or more, got %s" % (eps,))
    if positions is None:
        if len(sections) > 1:
            raise ValueError("positions must be given for %d axes" % len(sections))
    else:
        if not isinstance(positions, torch.Tensor):
            raise TypeError("positions must be a torch tensor, got %s" % type(positions))
        shapes = [(batch, tokens, len(sections))] + ([(batch, tokens)] if len(sections) == 1 else [])
        if positions.dtype != torch.int32 or positions.device != q.device or tuple(positions.shape) not in shapes:
            raise ValueError("positions must be int32 %s on %s, got %s of %s on %s"
                             % (shapes[-1], q.device, tuple(positions.shape), positions.dtype, positions.device))
        if lengths is not None:
            raise ValueError("either positions or lengths say where tokens stand")
    _check_counts("lengths", lengths, batch, q.device)
    _check_counts("q_lengths", q_lengths, batch, q.device)
    return rotary_len, bool(interleaved), len(sections), float(eps), _angles(rotary_len, sections, float(base), frequencies)


def _vector(w):
    if w is None:
        return None
    w = w.contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _arguments(dtype, q_shape, kv_heads, q, k, q_weight, k_weight, spec, positions, lengths, q_lengths, q_out, k_out):
    batch, tokens, heads, head_len = q_shape
    rotary_len, interleaved, axes, eps, angles = spec
    none = (0, 0, 0)
    return (_SIZES.pack(_TYPES[dtype], batch, tokens, heads, kv_heads, head_len, rotary_len, interleaved, axes, eps) + angles
            + _REST.pack(_ptr(q), _ptr(k), *(none if q is None else q.stride()[:3]), *(none if k is None else k.stride()[:3]), _ptr(q_weight), _ptr(k_weight),
                         _ptr(positions), _ptr(lengths), _ptr(q_lengths), _ptr(q_out), _ptr(k_out)))


def forward(q, k, q_weight, k_weight, spec, positions, lengths, q_lengths):
    """(q, k) normed and turned, of checked arguments."""
    q, k, q_weight, k_weight = _rows(q), _rows(k), _vector(q_weight), _vector(k_weight)
    positions = None if positions is None else positions.contiguous()
    new = lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device)
    q_out, k_out = new(q), new(k)
    raw = _arguments(q.dtype, q.shape, k.shape[2], q, k, q_weight, k_weight, spec, positions, lengths, q_lengths, q_out, k_out)
    _lib.check(_call(q.device, lambda L, stream: L.fg_rotate_heads(raw, stream)))
    return q_out, k_out


def backward(q, k, q_weight, k_weight, spec, positions, lengths, q_lengths, dq_out, dk_out):
    """(dq, dk, dq_weight, dk_weight); q and k None without weights."""
    dq_out, dk_out, q_weight, k_weight = _rows(dq_out), _rows(dk_out), _vector(q_weight), _vector(k_weight)
    if q is not None:
        q, k = _rows(q), _rows(k)
    positions = None if positions is None else positions.contiguous()
    new = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)
    dq, dk, dq_weight, dk_weight = new(dq_out), new(dk_out), new(q_weight), new(k_weight)
    raw = _arguments(dq.dtype, dq.shape, dk.shape[2], q, k, q_weight, k_weight, spec, positions, lengths, q_lengths, None, None)
    grads = _lib.FgRotateGrads(dq_out.data_ptr(), dk_out.data_ptr(), _strides(dq_out), _strides(dk_out), dq.data_ptr(), dk.data_ptr(),
                               _ptr(dq_weight), _ptr(dk_weight))
    need = _lib.check(_lib.lib().fg_rotate_heads_backward_workspace(raw))
    work = torch.empty(need, dtype=torch.uint8, device=dq.device) if need else None
    _lib.check(_call(dq.device, lambda L, stream: L.fg_rotate_heads_backward(raw, ctypes.byref(grads), _ptr(work), need, stream)))
    return dq, dk, dq_weight, dk_weight
