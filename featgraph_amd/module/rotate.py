"""RMS norm of every head of queries and keys and their rotation by position, in one pass, with its gradients: the calls of the C interface on
torch tensors (`featgraph_amd.ops.rotate_heads`).  Outputs and workspaces come from torch's allocator on the current stream.
The reference has no such operator.
"""
import ctypes
import functools
import math
import operator
import struct

import torch

from .. import _lib
from .block_attention import _TYPES, HEAD_LENGTHS, _check, _check_counts, _launch, _ptr, _rows

MAX_AXES = 8

# fg_rotate_args as bytes: what goes by sizes, the angles, pointers and strides
_SIZES, _ANGLES, _REST = struct.Struct("=9if"), struct.Struct("=64d64B"), struct.Struct("=2Q6q7Q")
assert ctypes.sizeof(_lib.FgRotateArgs) == _SIZES.size + _ANGLES.size + _REST.size and _lib.FgRotateArgs.q.offset == _SIZES.size + _ANGLES.size


_GRADS = struct.Struct("=2Q6q4Q")
assert ctypes.sizeof(_lib.FgRotateGrads) == _GRADS.size


def _host(name, x):
    """What a tensor holds as Python numbers (one on the GPU is waited for), everything else as it is."""
    if not isinstance(x, torch.Tensor):
        return x
    if x.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("%s have no gradient; detach them or run under torch.no_grad()" % name)
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise ValueError("%s are numbers on the host: a tensor on the GPU cannot be read during capture" % name)
    return x.tolist()


def _options(base, frequencies, sections, rotary_len, interleaved, eps):
    """A call's options as numbers and tuples of numbers, by whose values its plan is kept."""
    if type(base) is not float:
        base = float(_host("base", base))
    if type(eps) is not float:
        eps = float(_host("eps", eps))
    if frequencies is not None and (type(frequencies) is not tuple or any(type(x) is not float for x in frequencies)):
        frequencies = tuple([float(_host("frequencies", x)) for x in _host("frequencies", frequencies)])
    if sections is not None and (type(sections) is not tuple or any(type(x) is not int for x in sections)):
        sections = tuple([operator.index(_host("sections", x)) for x in _host("sections", sections)])
    if rotary_len is not None and type(rotary_len) is not int:
        rotary_len = operator.index(_host("rotary_len", rotary_len))
    return base, frequencies, sections, rotary_len, bool(interleaved), eps


class _Plan(object):
    """What a call's sizes and options come to: the part of its arguments that goes by them, and the gradients' device memory."""

    def __init__(self, axes, sizes):
        self.axes, self.sizes = axes, sizes
        self._need = None

    def workspace(self, raw):
        if self._need is None:
            self._need = _lib.check(_lib.lib().fg_rotate_heads_backward_workspace(raw))
        return self._need


@functools.lru_cache(maxsize=1024)
def _plan(dtype, q_shape, k_shape, normed, base, frequencies, sections, rotary_len, interleaved, eps):
    if len(q_shape) != 4 or len(k_shape) != 4 or q_shape[:2] != k_shape[:2] or q_shape[3] != k_shape[3] or q_shape[2] < 1 or k_shape[2] < 1:
        raise ValueError("q and k must be (batch, tokens, heads, head_len) of as many tokens, got %s and %s" % (tuple(q_shape), tuple(k_shape)))
    batch, tokens, heads, head_len = q_shape
    if head_len not in HEAD_LENGTHS:
        raise ValueError("heads of 32, 64 or 128 elements, got %d" % head_len)
    rotary_len = head_len if rotary_len is None else rotary_len
    if rotary_len < 0 or rotary_len > head_len or rotary_len % 16:
        raise ValueError("a multiple of 16 elements of a head of %d can be turned, got %s" % (head_len, rotary_len))
    pairs = rotary_len // 2
    sections = (pairs,) if sections is None else sections
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0 or sum(sections) != pairs:
        raise ValueError("sections must share the %d pairs out to 1 to %d axes, got %s" % (pairs, MAX_AXES, sections))
    if frequencies is not None:
        if len(frequencies) != pairs or not all(math.isfinite(x) for x in frequencies):
            raise ValueError("frequencies must be %d finite numbers, got %s" % (pairs, frequencies))
    elif not (base > 0 and math.isfinite(base)):
        raise ValueError("base must be a number above 0, got %s" % (base,))
    else:
        frequencies = [base ** (-i / pairs) for i in range(pairs)]
    if not eps >= 0:
        raise ValueError("eps must be 0 or more, got %s" % (eps,))
    axis = [a for a, many in enumerate(sections) for _ in range(many)]
    none = [0] * (64 - pairs)
    sizes = _SIZES.pack(_TYPES[dtype], batch, tokens, heads, k_shape[2], head_len, rotary_len, interleaved, len(sections), eps)
    return _Plan(len(sections), sizes + _ANGLES.pack(*[f / (2 * math.pi) for f in frequencies], *none, *axis, *none))


def _plain(q, k, q_weight, k_weight):
    """Whether types and devices are fine as they are, at a glance; what is not is looked at one by one for the message."""
    try:
        dtype, device = q.dtype, q.device
        if dtype not in _TYPES or k.dtype != dtype or device.type != "cuda" or k.device != device:
            return False
        if q_weight is None or k_weight is None:
            return q_weight is k_weight
        shape = q.shape[3:]
        return (q_weight.shape == shape and k_weight.shape == shape and q_weight.dtype == dtype and k_weight.dtype == dtype
                and q_weight.device == device and k_weight.device == device)
    except AttributeError:
        return False


def _check_tensors(q, k, q_weight, k_weight):
    _check("q", q, 4)
    _check("k", k, 4, q)
    if (q_weight is None) != (k_weight is None):
        raise ValueError("weights for queries and keys come together")
    if q_weight is not None:
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            _check(name, w, 1, q)
            if w.shape[0] != q.shape[3]:
                raise ValueError("%s must be (%d,), got %s" % (name, q.shape[3], tuple(w.shape)))


def check(q, k, q_weight, k_weight, positions, lengths, q_lengths, base, frequencies, sections, rotary_len, interleaved, eps):
    """The call's plan, after everything that can be seen of its arguments without looking at their values on the GPU."""
    if not _plain(q, k, q_weight, k_weight):
        _check_tensors(q, k, q_weight, k_weight)
    plan = _plan(q.dtype, q.shape, k.shape, q_weight is not None, *_options(base, frequencies, sections, rotary_len, interleaved, eps))
    if positions is None and lengths is None and q_lengths is None and plan.axes == 1:
        return plan
    batch, tokens = q.shape[:2]
    if positions is None:
        if plan.axes > 1:
            raise ValueError("positions must be given for %d axes" % plan.axes)
    else:
        if not isinstance(positions, torch.Tensor):
            raise TypeError("positions must be a torch tensor, got %s" % type(positions))
        shapes = [(batch, tokens, plan.axes)] + ([(batch, tokens)] if plan.axes == 1 else [])
        if positions.dtype != torch.int32 or positions.device != q.device or tuple(positions.shape) not in shapes:
            raise ValueError("positions must be int32 %s on %s, got %s of %s on %s"
                             % (shapes[-1], q.device, tuple(positions.shape), positions.dtype, positions.device))
        if lengths is not None:
            raise ValueError("either positions or lengths say where tokens stand")
    _check_counts("lengths", lengths, batch, q.device)
    _check_counts("q_lengths", q_lengths, batch, q.device)
    return plan


def _vector(w):
    if w is None or w.is_contiguous() and not w.data_ptr() % 16:
        return w
    return w.contiguous().clone()


def _new(t):
    return t.new_empty(t.shape)


_NOTHING = (0, 0, 0)


def _arguments(plan, q, k, q_weight, k_weight, positions, lengths, q_lengths, q_out, k_out):
    """fg_rotate_args as bytes."""
    return plan.sizes + _REST.pack(_ptr(q), _ptr(k), *(_NOTHING if q is None else q.stride()[:3]), *(_NOTHING if k is None else k.stride()[:3]),
                                   _ptr(q_weight), _ptr(k_weight), _ptr(positions), _ptr(lengths), _ptr(q_lengths), _ptr(q_out), _ptr(k_out))


def forward(q, k, q_weight, k_weight, plan, positions, lengths, q_lengths):
    """(q, k) normed and turned, of checked arguments."""
    q, k, q_weight, k_weight = _rows(q), _rows(k), _vector(q_weight), _vector(k_weight)
    positions = None if positions is None else positions.contiguous()
    q_out, k_out = _new(q), _new(k)
    raw = _arguments(plan, q, k, q_weight, k_weight, positions, lengths, q_lengths, q_out, k_out)
    _launch(q.device, _lib.lib().fg_rotate_heads, raw)
    return q_out, k_out


def backward(q, k, q_weight, k_weight, plan, positions, lengths, q_lengths, dq_out, dk_out):
    """(dq, dk, dq_weight, dk_weight); q and k None without weights."""
    dq_out, dk_out, q_weight, k_weight = _rows(dq_out), _rows(dk_out), _vector(q_weight), _vector(k_weight)
    if q is not None:
        q, k = _rows(q), _rows(k)
    positions = None if positions is None else positions.contiguous()
    dq, dk = _new(dq_out), _new(dk_out)
    dq_weight, dk_weight = (None, None) if q_weight is None else (_new(q_weight), _new(k_weight))
    raw = _arguments(plan, q, k, q_weight, k_weight, positions, lengths, q_lengths, None, None)
    grads = _GRADS.pack(dq_out.data_ptr(), dk_out.data_ptr(), *dq_out.stride()[:3], *dk_out.stride()[:3], dq.data_ptr(), dk.data_ptr(),
                        _ptr(dq_weight), _ptr(dk_weight))
    need = plan.workspace(raw)
    work = torch.empty(need, dtype=torch.uint8, device=dq.device) if need else None
    _launch(dq.device, _lib.lib().fg_rotate_heads_backward, raw, grads, _ptr(work), need)
    return dq, dk, dq_weight, dk_weight
