"""Attention of queries and keys of different lengths on the B200 kernels:

    cross_attention(q, k, v, mask)                      keys of another sequence
    relative_bias_attention(q, k, v, table, mask, ...)  a learned bias by bucketed relative position
    shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths)
                                                        a batch behind one shared prefix of keys

q is [B, H, Nq, D]; k and v are [B, Hkv, Nk, D] with Hkv dividing H: query
head h reads key head h // (H // Hkv).  Types, head dims (64 and 128), the
scale 1/sqrt(D), FP32 inputs (computed in bf16 and cast back), the refusal of
CPU tensors and the meaning of a mask (bool, True = attend, a row that keeps
nothing gives 0) are those of ``sparse_attention``.  Masks broadcast:
[B or 1, H or 1, Nq or 1, Nk]; a padding mask is [B, 1, 1, Nk].

Inputs need not be contiguous: views with a contiguous last axis and 16-byte
steps (such as a [B, N, H, D] projection transposed) are read in place, others
are copied.  Work is enqueued on the current stream of the tensors' device.

Keys that no query keeps may hold anything, NaN and infinities included;
under gradients that holds behind a padding mask, and every other key, query
and incoming gradient must be finite.  A gradient cannot be differentiated
again (refused).  With gradients at most 65536 keys, and 2048 steps of 64
queries over the heads that share a key head.  Without, past 65536 keys they
are read again for every 16 query rows of a key head instead of every 128:
B1 H8 D128 with 1024 queries takes 0.36 ms over 65536 keys and 1.64 over one
more, with 16 queries 0.06 either way.
"""

import ctypes
import functools

import torch

from . import _lib
from .sparse_attn_cuda import _require


def cross_attention(q, k, v, mask=None, scale=None):
    """Masked-softmax attention of q [B, H, Nq, D] over k, v [B, Hkv, Nk, D],
    the states of another sequence (an encoder's, a cache's); returns
    [B, H, Nq, D] in the input dtype.  ``mask``: bool, broadcastable to
    [B, H, Nq, Nk], True = attend; None keeps every key."""
    return _lib.ops().cross_attention(q, k, v, mask, scale)


@functools.lru_cache(maxsize=64)
def _bucket_starts(side, max_distance):
    """Smallest distance of each of one side's ``side`` buckets: distances
    below side // 2 have a bucket each, the rest of the buckets grow
    geometrically up to ``max_distance`` and the last one holds everything
    beyond.  Bucket e + j (e = side // 2, n = side - e) starts at the smallest
    d with (d / e) ** n >= (max_distance / e) ** j, decided in whole numbers."""
    e = side // 2
    n = side - e
    starts, d = list(range(e)), e
    for j in range(n):
        bound = max_distance**j * e**n
        while d**n * e**j < bound:
            d += 1
        starts.append(d)
    return (ctypes.c_int32 * side)(*starts)


@functools.lru_cache(maxsize=64)
def _side(buckets, bidirectional, max_distance):
    """Address and number of one side's bucket starts (and their owner)."""
    side = buckets // 2 if bidirectional else buckets
    _require(not bidirectional or buckets % 2 == 0, "a bidirectional bias needs an even number of buckets")
    _require(2 <= side <= _lib.SMA_MAX_BIAS_SIDE, f"2 to {_lib.SMA_MAX_BIAS_SIDE} buckets per side are supported")
    _require(
        side // 2 < max_distance <= _lib.SMA_MAX_BIAS_DISTANCE,
        f"max_distance must exceed the buckets of one distance each and be at most {_lib.SMA_MAX_BIAS_DISTANCE}",
    )
    starts = _bucket_starts(side, max_distance)
    return ctypes.addressof(starts), side, starts


def relative_bias_attention(q, k, v, table, mask=None, bidirectional=True, max_distance=128, query_offset=0, scale=None):
    """``cross_attention`` with a learned bias: table[bucket(j - i -
    query_offset), h] is added to the scaled score of query i and key j of
    head h.

    ``table``: [num_buckets, H], of q's dtype or FP32 (the kernels read it
    rounded to q's dtype; its gradient, a sum over all queries, stays FP32).
    ``bidirectional``: half of the buckets are for keys after the query; else
    those keys all count as distance 0.  Half of a side's buckets hold one
    distance each, the others grow geometrically up to ``max_distance``, and
    the last one takes every larger distance.  ``query_offset``: how many keys
    stand in front of query 0 (a cache's length while generating), an int or
    an int32 tensor [B] on the device."""
    _require(table.dim() == 2, "table must be [num_buckets, H]")
    bidirectional = bool(bidirectional)
    starts, side, _owner = _side(table.shape[0], bidirectional, int(max_distance))
    offset, offsets = 0, None
    if isinstance(query_offset, torch.Tensor):
        offsets = query_offset
    else:
        offset = int(query_offset)
        _require(abs(offset) < 1 << 30, "query_offset out of range")
    return _lib.ops().relative_bias_attention(q, k, v, table, mask, starts, side, bidirectional, offset, offsets, scale)


def shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths=None, scale=None):
    """Attention of new tokens q [B, H, T, D] behind a prefix that the whole
    batch shares: k_prefix, v_prefix [Hkv, P, D], then each sequence's own
    k, v [B, Hkv, S, D], of which the first lengths[b] are in use (int32 [B]
    on the device, clamped to [0, S]; None: all S).  The T queries are the
    last T of a sequence's own tokens: each keeps the prefix and its own keys
    up to itself.  Own keys that no query keeps may hold anything.  Returns
    [B, H, T, D]; forward only."""
    return _lib.ops().shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths, scale)
