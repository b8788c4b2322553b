"""Differentiable attention cores beside the encoder's masked attention: `relpos_attention` (a learned relative position bias by buckets) and
`diff_attention` (the difference of two softmax maps with a learned weight per head), forward and backward on the kernels of
`ops.relpos_attention_fwd / _bwd` and `ops.diff_attention_fwd / _bwd`, where shapes, types and masks are documented.

    buckets = ops.relpos_buckets(32, 128)                                  # once
    o = relpos_attention(q, k, v, table, buckets, kvalid=kvalid)           # table: [32, H] parameter
    o = diff_attention(q, k, v, lam, kvalid=kvalid)                        # lam: [H], e.g. exp(a1 . b1) - exp(a2 . b2) + lam0 of four parameters

Under `torch.no_grad()`, or when nothing requires a gradient, they are the forward calls alone: a few new tokens against a cache of keys and
values (`q_offset` = how many came before) run the kernel that splits the keys.

Derivatives are first ones, in reverse mode; others are refused.

A step that is captured into a graph is captured whole, forward and backward, on one stream, with no autograd graph of another stream alive that
holds the same leaves.  Where such a graph was made by these functions, the call is refused; those of other operations on the same leaves (a weight whose
loss of an eager step is still referenced) are not seen here and have to be released before the capture."""
from __future__ import annotations

import itertools
import random
import weakref

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops

# autograd nodes of this module that are alive, by a number; their leaves carry (number, stream) pairs, which are copied and saved with a leaf without
# harm: numbers start at random, so that another process's mean nothing here
_nodes = {}
_numbers = itertools.count(random.getrandbits(62))


def _once(backward):
    """torch's once_differentiable, whose wrapping costs 5 us: only where a second derivative could be asked for (create_graph)."""
    guarded = once_differentiable(backward)

    def once(ctx, do):
        _check_tangents(do)
        return guarded(ctx, do) if torch.is_grad_enabled() else backward(ctx, do)
    return once


def _check_tangents(*tensors):
    """Forward-mode differentiation: the kernels would drop the tangents without a word."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("attention: forward-mode differentiation is not implemented")


class _RelposAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, buckets, kvalid, opts):
        o, lse, (ctx.dims, *operands) = ops._relpos_fwd(q, k, v, table, buckets, kvalid, *opts)
        ctx.save_for_backward(*operands, o, lse)
        return o

    @staticmethod
    @_once
    def backward(ctx, do):
        return *ops._relpos_bwd(do, ctx.dims, *ctx.saved_tensors, ctx.needs_input_grad[3]), None, None, None


class _DiffAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lam, kvalid, opts):
        o, lse, o2, (ctx.dims, *operands) = ops._diff_fwd(q, k, v, lam, kvalid, *opts, True)
        ctx.save_for_backward(*operands, o, o2, lse)
        return o

    @staticmethod
    @_once
    def backward(ctx, do):
        return *ops._diff_bwd(do, ctx.dims, *ctx.saved_tensors, ctx.needs_input_grad[3]), None, None


def _apply(function, leaves, *args):
    """function.apply(*args), which differentiates `leaves`.  A gradient accumulator lives as long as some autograd graph of its leaf does, and autograd's
    engine makes the stream it was made on wait for a backward pass: during a capture that joins a stream outside it, which ends the process in
    capture_end, not in an error.  So every graph made here is noted on its leaves, and a capture is refused while one of another stream is alive.
    (Whether a graph of another operation holds a leaf cannot be asked of torch.)"""
    on_gpu = leaves[0].is_cuda
    stream = ops._stream_of(leaves[0]) if on_gpu else 0
    leaves = [t for t in leaves if t.requires_grad and t.is_leaf]
    if on_gpu and leaves and torch.cuda.is_current_stream_capturing():
        _check_capture(leaves, stream)
    o = function.apply(*args)
    if leaves:
        n = next(_numbers)
        _nodes[n] = weakref.ref(o.grad_fn, lambda _, nodes=_nodes: nodes.pop(n, None))
        for t in leaves:                                     # (a graph beside others shares their accumulator, made on the first one's stream)
            alive = [p for p in getattr(t, "_attention_graphs", ()) if p[0] in _nodes]
            t._attention_graphs = alive + [(n, alive[0][1] if alive else stream)]
    return o


def _check_capture(leaves, stream):
    if any(n in _nodes and s != stream for t in leaves for n, s in getattr(t, "_attention_graphs", ())):
        raise RuntimeError("attention: an autograd graph made outside this capture still holds a leaf of the captured call; release its outputs "
                           "before the capture, or pass the captured call leaves of its own")


def _needs_grad(*tensors):
    _check_tangents(*tensors)
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def relpos_attention(q, k, v, table, buckets, kvalid=None, q_offset=0, causal=False, scale=None):
    """o [B, Sq, H, D] of ops.relpos_attention_fwd, differentiable in q, k, v and table (a table of another type is used, and gets its gradient, through
    a cast to fp32)."""
    opts = (q_offset, causal, scale)
    if not _needs_grad(q, k, v, table):
        return ops.relpos_attention_fwd(q, k, v, table, buckets, kvalid, *opts)[0]
    if ops._elsewhere(q):
        with torch.cuda.device(q.device):
            return relpos_attention(q, k, v, table, buckets, kvalid, *opts)
    return _apply(_RelposAttention, (q, k, v, table), q, k, v, table.float(), buckets, kvalid, opts)


def diff_attention(q, k, v, lam, kvalid=None, q_offset=0, causal=False, scale=None):
    """o [B, Sq, H, 2 D] of ops.diff_attention_fwd, differentiable in q, k, v and lam (a lam of another type through a cast to fp32)."""
    opts = (q_offset, causal, scale)
    if not _needs_grad(q, k, v, lam):
        return ops.diff_attention_fwd(q, k, v, lam, kvalid, *opts)[0]
    if ops._elsewhere(q):
        with torch.cuda.device(q.device):
            return diff_attention(q, k, v, lam, kvalid, *opts)
    return _apply(_DiffAttention, (q, k, v, lam), q, k, v, lam.float(), kvalid, opts)
