"""gspmm / gsddmm with the call signatures of DGL's `dgl.ops`, over a `featgraph_amd.autograd.Graph`.

The reference's README (README.md:9-14) points to generalised SpMM / SDDMM kernels and to their integration
into DGL, whose message-passing layer calls exactly these two functions; the reference snapshot itself holds
neither.  Operand conventions are DGL's: node features of the source nodes are `(num_src, ...)`, of the
destination nodes `(num_dst, ...)`, edge features `(nnz, ...)` in the graph's CSR edge order, and the feature
shapes of two operands broadcast against each other the numpy way.

Gradients: every call routes to a differentiable operator (weighted sums; sum / mean / max / min of add / sub /
mul / div messages and copies; per-edge add / sub / mul / div and dot products of node features); what is left --
operators between two operands on the same target, dot products that involve edge features or broadcasting --
runs forward only and refuses inputs that require grad.

pool_blocks / select_blocks / block_attention are attention over a graph that the data itself makes on the GPU: every query selects
blocks of keys by a cheap score and attends to the keys in them.
"""
import math

import torch

from . import autograd
from .module import block_attention as _block

_BINARY = ("add", "sub", "mul", "div")


def _no_grad_inputs(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError("%s has no gradient here; detach the inputs or run under torch.no_grad()" % what)


def gspmm(g, op, reduce_op, lhs_data, rhs_data):
    """out[v] = reduce_op over the edges e = (u -> v) of  lhs_data[u] op rhs_data[e].

    op: 'add' | 'sub' | 'mul' | 'div' | 'copy_lhs' | 'copy_rhs'; reduce_op: 'sum' | 'mean' | 'max' | 'min'
    (rows without edges give 0).  lhs_data lives on the source nodes, rhs_data on the edges; the operand a
    copy does not use may be None."""
    if reduce_op not in ("sum", "mean", "max", "min"):
        raise ValueError("reduce_op must be 'sum', 'mean', 'max' or 'min'")
    if op == "copy_lhs":
        x = lhs_data
        if x.dim() == 1:
            return g.aggregate(x[:, None], reduce_op)[:, 0]
        return g.aggregate(x.reshape(x.shape[0], -1), reduce_op).reshape((g.shape[0],) + tuple(x.shape[1:]))
    if op == "copy_rhs":
        return g.gspmm("copy_e", rhs_data, reduce=reduce_op)
    if op not in _BINARY:
        raise ValueError("op must be one of %s, 'copy_lhs', 'copy_rhs'" % (_BINARY,))
    if op == "mul" and reduce_op == "sum" and lhs_data.dim() in (2, 3):
        # one weight per edge (or per edge and head): the weighted-sum kernels with their source partitions
        heads = lhs_data.shape[1] if lhs_data.dim() == 3 else 1
        if rhs_data.dim() == 1 and lhs_data.dim() == 2:
            return g.spmm(lhs_data, rhs_data)
        if lhs_data.dim() == 3 and tuple(rhs_data.shape[1:]) == (heads, 1):
            return g.spmm(lhs_data, rhs_data[:, :, 0])
        if lhs_data.dim() == 2 and tuple(rhs_data.shape[1:]) == (1,):
            return g.spmm(lhs_data, rhs_data[:, 0])
    return g.gspmm("u_%s_e" % op, lhs_data, rhs_data, reduce_op)


def gsddmm(g, op, lhs_data, rhs_data, lhs_target="u", rhs_target="v"):
    """out[e] = lhs_data[lhs_target of e] op rhs_data[rhs_target of e] for every edge e.

    op: 'add' | 'sub' | 'mul' | 'div' | 'dot' | 'copy_lhs' | 'copy_rhs'; targets: 'u' (source node), 'v'
    (destination node), 'e' (the edge).  'dot' contracts the last feature axis and keeps it with length 1,
    as DGL does.  out is (nnz, ...) in the graph's CSR edge order."""
    if op == "copy_lhs":
        return _copy_to_edges(g, lhs_data, lhs_target)
    if op == "copy_rhs":
        return _copy_to_edges(g, rhs_data, rhs_target)
    if op == "dot":
        same = (lhs_target, rhs_target) == ("u", "v") and lhs_data.shape[1:] == rhs_data.shape[1:]
        if same and lhs_data.dim() in (2, 3):
            return g.sddmm(lhs_data, rhs_data).unsqueeze(-1)
        if (lhs_target, rhs_target) == ("v", "u") and lhs_data.shape[1:] == rhs_data.shape[1:] and lhs_data.dim() in (2, 3):
            return g.sddmm(rhs_data, lhs_data).unsqueeze(-1)
        _no_grad_inputs("a dot product between these targets / shapes", lhs_data, rhs_data)
        return g._bcast_sddmm_raw("dot", lhs_target, rhs_target, [lhs_data, rhs_data]).unsqueeze(-1)
    if op not in _BINARY:
        raise ValueError("op must be one of %s, 'dot', 'copy_lhs', 'copy_rhs'" % (_BINARY,))
    if lhs_target != rhs_target:
        return g.gsddmm(op, lhs_data, rhs_data, lhs_target, rhs_target)
    _no_grad_inputs("gsddmm(%s) between '%s' and '%s'" % (op, lhs_target, rhs_target), lhs_data, rhs_data)
    return g._bcast_sddmm_raw(op, lhs_target, rhs_target, [lhs_data, rhs_data])


def _copy_to_edges(g, x, target):
    if target == "e":
        return x
    # a copy is the per-edge sum of x with zeros on the edges: differentiable through gsddmm
    zeros = torch.zeros((g.nnz,) + (1,) * (x.dim() - 1), dtype=x.dtype, device=x.device)
    return g.gsddmm("add", x, zeros, target, "e")


def edge_softmax(g, scores):
    """Softmax of the edge scores over the edges of each destination node, per head (dgl.ops.edge_softmax with
    norm_by='dst')."""
    squeeze = scores.dim() == 3 and scores.shape[-1] == 1
    a = g.edge_softmax(scores[..., 0] if squeeze else scores)
    return a.unsqueeze(-1) if squeeze else a


def pool_blocks(k, block_size, lengths=None):
    """Mean of the keys of every block, (batch, kv_heads, ceil(keys / block_size), head_len), in the keys' type (summed in 64 bits, rounded to
    32 and then to the type); 0 for a block without keys.  k (batch, keys, kv_heads, head_len); lengths: int32 (batch,), the keys of each
    sequence, the rest is not read.  head_len 32, 64 or 128, block_size 32, 64, 128 or 256.  Not differentiable."""
    return _block.block_pool(k.detach() if isinstance(k, torch.Tensor) else k, block_size, lengths)


def select_blocks(q, pooled, num_keys, block_size, topk, causal=True, lengths=None, q_lengths=None, keep_first=None, keep_last=1):
    """The topk blocks of keys that every query scores highest, int32 (batch, queries, kv_heads, topk), ascending, -1 behind the last.

    q (batch, queries, heads, head_len) against pooled = pool_blocks(k, ...) of `num_keys` keys; a block's score is its pooled key times the
    sum of the queries of the heads that share the key head (rounded to 32 bits and then to their type), compared as exact numbers, equal ones
    by the lower id.  A sequence's last query stands at its last key; with `causal` a query may choose its own block and those before.
    The first `keep_first` blocks (default 1, or 0 with topk = 1) and the last `keep_last` a query may choose are always among
    them.  Rows behind q_lengths are -1.  At most 2048 blocks.  Not differentiable."""
    if keep_first is None:
        keep_first = 1 if topk > keep_last else 0
    q, pooled = (t.detach() if isinstance(t, torch.Tensor) else t for t in (q, pooled))
    return _block.block_select(q, pooled, num_keys, block_size, topk, causal, lengths, q_lengths, keep_first, keep_last)


def block_attention(q, k, v, blocks, block_size, scale=None, causal=True, lengths=None, q_lengths=None, bias=None, bounds=None):
    """out[b, i, h] = sum over the keys j that query i sees of softmax(scale <q[b, i, h], k[b, j, g]> + bias[bucket, h]) v[b, j, g]

    q (batch, queries, heads, head_len), k and v (batch, keys, kv_heads, head_len), float32, float16 or bfloat16; heads / kv_heads (1 to
    16) query heads share key head g.  blocks: int32 (batch, queries, kv_heads, topk) as select_blocks returns them, in any order;
    ids outside the keys name nothing, one that stands twice counts once.  lengths / q_lengths: int32 (batch,), each
    sequence's keys and queries (default: all); what lies behind them is not read, and their rows of the output are 0.  Query i stands
    at position lengths - q_lengths + i, so that one new token attends to a whole cache and a prompt to itself; with `causal`
    it sees no key behind that.  A query that sees no key gives 0.  scale: 1 / sqrt(head_len) unless given.

    bias (buckets, heads), at most 64 buckets, with `bounds`, buckets - 1 ascending distances (position_bounds): query position less key
    position is in bucket (number of bounds that are not above it).

    Differentiable in q, k, v and bias.  The same bits on every call, whatever else runs; but in float16 and bfloat16 a call over enough
    queries to fill the card rounds the softmax's powers to the type, half a step each, where no gradient is wanted, and keeps what that takes
    where one is: with and without gradients its outputs differ by about their own rounding (also under checkpointing that runs the
    first forward pass without).  head_len 32, 64 or 128, block_size 32, 64, 128 or 256."""
    bounds = _block.check_attention(q, k, v, blocks, block_size, lengths, q_lengths, bias, bounds)
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else float(scale)
    return autograd.block_attention(q, k, v, bias, blocks, (block_size, scale, bool(causal)), lengths, q_lengths, bounds)


def position_bounds(num_buckets, max_distance=128, causal=True):
    """Bounds of `num_buckets` buckets of relative positions: the nearer half of them one distance each, the others growing in proportion
    up to max_distance, the last one for all beyond; without `causal` half of the buckets on either side.  At least 2 buckets (4
    without `causal`)."""
    sides = [num_buckets] if causal else [num_buckets // 2, num_buckets - num_buckets // 2]
    if sides[0] < 2 or num_buckets > _block.MAX_BUCKETS or max_distance < sides[-1] or max_distance > _block.MAX_SPAN // 2:
        raise ValueError("%d buckets up to distance %d" % (num_buckets, max_distance))

    def ends(side):                     # first distance of each of a side's buckets but the nearest
        near = side // 2
        x = list(range(1, near + 1)) + [math.ceil(near * (max_distance / near) ** ((i - near) / (side - near))) for i in range(near + 1, side)]
        return [max(d, i + 1) for i, d in enumerate(x)]

    if causal:
        return tuple(ends(sides[0]))
    return tuple([1 - x for x in reversed(ends(sides[0]))] + [1] + [x + 1 for x in ends(sides[1])])
