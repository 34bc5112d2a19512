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
"""

import ctypes
import functools
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib, sparse_attn_cuda
from .sparse_attn_cuda import _empty, _require, _strided

_DTYPES = (torch.float16, torch.bfloat16)


def _check_qkv(q, k, v):
    _require(q.is_cuda and k.is_cuda and v.is_cuda, "attention requires CUDA tensors (no CPU fallback)")
    _require(q.device == k.device == v.device, "q/k/v must be on the same device")
    _require(q.dim() == 4 and k.dim() == 4, "q must be [B, H, Nq, D], k and v [B, Hkv, Nk, D]")
    _require(k.shape == v.shape, "k and v must have the same shape")
    _require(q.dtype == k.dtype == v.dtype, "q/k/v must have the same dtype")
    _require(q.dtype in _DTYPES or q.dtype == torch.float32, "Unsupported dtype, need BF16, FP16 or FP32")
    B, H, _, D = q.shape
    _require(k.shape[0] == B and k.shape[3] == D, "q/k/v must agree in batch and head dim")
    _require(D in (64, 128), "head dim must be 64 or 128")
    Hkv = k.shape[1]
    _require((Hkv > 0 and H % Hkv == 0) or H == 0, "the key heads must divide the query heads")


def _check_mask(mask, q, k):
    if mask is None:
        return
    B, H, Nq, _ = q.shape
    _require(mask.device == q.device, "mask must be on the same device as q")
    _require(mask.dtype == torch.bool, "mask must be a bool tensor")
    want = (B, H, Nq, k.shape[2])
    _require(
        mask.dim() == 4 and mask.shape[3] == want[3] and all(n in (1, w) for n, w in zip(mask.shape[:3], want)),
        f"mask must broadcast to {want} along its first three axes, got {tuple(mask.shape)}",
    )


def _scale_of(scale, D):
    if scale is None:
        return 1.0 / math.sqrt(D)
    scale = float(scale)
    _require(0.0 < scale < math.inf, "scale must be finite and > 0")
    return scale


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


def _few_rows(q, k, mask, bias):
    """Whether the streaming kernel is taken (16 rows of a key head at a time,
    the keys read again for every 16) instead of the 128-row tiles.

    With no mask, or one that all rows of a key head share, and R rows per key
    head in T tiles of 128, the first takes (measured on a B200) about 8 us +
    B Hkv Nk D ceil(R / 16) * 0.57e-6 us, the second (which also packs the
    mask) 18 us + B Hkv Nk D T * 0.9e-6 us (D = 64) or 0.77e-6 us (D = 128).
    For instance B8 Hkv8 Nk1000 D64: 12.8 against 22.3 us at 64 rows, 22.9
    against 25.0 at 128; B16 H12 Nk1500 D128: 31 against 50 us at 16 rows, 58
    against 49 at 24.  Masks of the rows' own and a bias cost the first more:
    B16 H12 Nk500 D64 with a mask 19.4 against 20.9 us at 16 rows, 35.5 against
    21.0 at 32, so there it is taken for one tile of 16 rows only."""
    B, H, Nq, D = q.shape
    Hkv, Nk = k.shape[1:3]
    if Nk > _lib.SMA_MAX_SEQ_LEN:
        return True
    rows = H // max(Hkv, 1) * Nq
    if rows <= 16 or rows > 128:
        return rows <= 16
    if bias is not None or (mask is not None and (mask.shape[1] != 1 or mask.shape[2] != 1)):
        return False
    return B * Hkv * Nk * D * ((0.6 if D == 64 else 0.75) * ((rows + 15) // 16) - 1.0) <= 15e6


class CrossAttentionFunction(Function):
    """Autograd node of cross_attention (table and bias None) and
    relative_bias_attention: ``table`` is the differentiable input, the rest
    of the bias comes with ``bias``."""

    @staticmethod
    def forward(ctx, q, k, v, table, mask, scale, bias):
        q, k, v = _strided(q), _strided(k), _strided(v)
        offsets = None
        if bias is not None:
            bias = bias._replace(table=table)
            offsets = bias.offsets
            ctx.bias = bias._replace(table=None, offsets=None)
        else:
            ctx.bias = None
        out = _empty(q)
        saved, ctx.mask_strides = sparse_attn_cuda.cross_forward(q, k, v, out, scale, mask, bias, training=True)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, out, saved, table, offsets)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, saved, table, offsets = ctx.saved_tensors
        if q.numel() == 0 or k.numel() == 0:
            dtable = None if table is None else torch.zeros_like(table)
            return torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), dtable, None, None, None
        dout = dout.contiguous()
        if dout.data_ptr() % 16 != 0:
            dout = dout.clone()
        bias = None if ctx.bias is None else ctx.bias._replace(table=table, offsets=offsets)
        dq, dk, dv, dtable = sparse_attn_cuda.cross_backward(dout, q, k, v, out, ctx.scale, saved, ctx.mask_strides, bias)
        return dq, dk, dv, dtable, None, None, None


# With gradients: 64-row steps of the queries of all heads that share a key head.
_MAX_STEPS = 2048


def _attention(q, k, v, mask, scale, bias):
    """out [B, H, Nq, D] of checked fp16 / bf16 inputs."""
    table = None if bias is None else bias.table
    if _needs_grad(q, k, v) or (table is not None and _needs_grad(table)):
        Nk, steps = k.shape[2], q.shape[1] // max(k.shape[1], 1) * ((q.shape[2] + 63) // 64)
        _require(Nk <= _lib.SMA_MAX_SEQ_LEN, f"with gradients at most {_lib.SMA_MAX_SEQ_LEN} keys are supported")
        _require(steps <= _MAX_STEPS, f"with gradients at most {_MAX_STEPS} steps of 64 queries may share a key head")
        return CrossAttentionFunction.apply(q, k, v, table, mask, scale, bias)
    q, k, v = _strided(q), _strided(k), _strided(v)
    out = _empty(q)
    if _few_rows(q, k, mask, bias):
        sparse_attn_cuda.rows_forward(q, k, v, out, scale, mask=mask, bias=bias)
    else:
        sparse_attn_cuda.cross_forward(q, k, v, out, scale, mask, bias)
    return out


def cross_attention(q, k, v, mask=None, scale=None):
    """Masked-softmax attention of q [B, H, Nq, D] over k, v [B, Hkv, Nk, D],
    the states of another sequence (an encoder's, a cache's); returns
    [B, H, Nq, D] in the input dtype.  ``mask``: bool, broadcastable to
    [B, H, Nq, Nk], True = attend; None keeps every key."""
    _check_qkv(q, k, v)
    _check_mask(mask, q, k)
    scale = _scale_of(scale, q.shape[-1])
    if q.dtype == torch.float32:
        return _attention(q.bfloat16(), k.bfloat16(), v.bfloat16(), mask, scale, None).float()
    return _attention(q, k, v, mask, scale, None)


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


def _make_bias(table, q, bidirectional, max_distance, query_offset):
    _require(table.device == q.device, "table must be on the same device as q")
    _require(table.dim() == 2 and table.shape[1] == q.shape[1], "table must be [num_buckets, H]")
    _require(table.dtype == q.dtype or table.dtype == torch.float32, "table must have the dtype of q or be FP32")
    buckets = table.shape[0]
    side = buckets // 2 if bidirectional else buckets
    _require(not bidirectional or buckets % 2 == 0, "a bidirectional bias needs an even number of buckets")
    _require(2 <= side <= _lib.SMA_MAX_BIAS_SIDE, f"2 to {_lib.SMA_MAX_BIAS_SIDE} buckets per side are supported")
    max_distance = int(max_distance)
    _require(
        side // 2 < max_distance <= _lib.SMA_MAX_BIAS_DISTANCE,
        f"max_distance must exceed the buckets of one distance each and be at most {_lib.SMA_MAX_BIAS_DISTANCE}",
    )
    offset, offsets = 0, None
    if isinstance(query_offset, torch.Tensor):
        offsets = query_offset
        _require(
            offsets.device == q.device and offsets.dtype == torch.int32 and tuple(offsets.shape) == (q.shape[0],),
            "query_offset must be an int or an int32 tensor [B] on the device of q",
        )
        offsets = offsets.contiguous()
    else:
        offset = int(query_offset)
        _require(abs(offset) < 1 << 30, "query_offset out of range")
    return _bucket_starts(side, max_distance), bool(bidirectional), offset, offsets


def relative_bias_attention(q, k, v, table, mask=None, bidirectional=True, max_distance=128, query_offset=0, scale=None):
    """``cross_attention`` with a learned bias: table[bucket(j - i -
    query_offset), h] is added to the scaled score of query i and key j of
    head h.

    ``table``: [num_buckets, H], of q's dtype or FP32 (rounded to q's dtype).
    ``bidirectional``: half of the buckets are for keys after the query; else
    those keys all count as distance 0.  Half of a side's buckets hold one
    distance each, the others grow geometrically up to ``max_distance``, and
    the last one takes every larger distance.  ``query_offset``: how many keys
    stand in front of query 0 (a cache's length while generating), an int or
    an int32 tensor [B] on the device."""
    _check_qkv(q, k, v)
    _check_mask(mask, q, k)
    starts, two_sided, offset, offsets = _make_bias(table, q, bidirectional, max_distance, query_offset)
    scale = _scale_of(scale, q.shape[-1])
    dtype = q.dtype
    if dtype == torch.float32:
        q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
    table = table.to(q.dtype).contiguous()
    out = _attention(q, k, v, mask, scale, sparse_attn_cuda.Bias(table, starts, two_sided, offset, offsets))
    return out.float() if dtype == torch.float32 else out


def shared_prefix_attention(q, k_prefix, v_prefix, k, v, lengths=None, scale=None):
    """Attention of new tokens q [B, H, T, D] behind a prefix that the whole
    batch shares: k_prefix, v_prefix [Hkv, P, D], then each sequence's own
    k, v [B, Hkv, S, D], of which the first lengths[b] are in use (int32 [B]
    on the device, clamped to [0, S]; None: all S).  The T queries are the
    last T of a sequence's own tokens: each keeps the prefix and its own keys
    up to itself.  Own keys that no query keeps may hold anything.  Returns
    [B, H, T, D]; forward only."""
    _check_qkv(q, k, v)
    _require(k_prefix.is_cuda and v_prefix.is_cuda, "attention requires CUDA tensors (no CPU fallback)")
    B, H, T, D = q.shape
    Hkv, S = k.shape[1:3]
    _require(k_prefix.device == q.device == v_prefix.device, "the prefix must be on the same device as q")
    _require(k_prefix.dtype == q.dtype == v_prefix.dtype, "the prefix must have the dtype of q")
    _require(
        k_prefix.dim() == 3 and k_prefix.shape == v_prefix.shape and k_prefix.shape[0] == Hkv and k_prefix.shape[2] == D,
        "k_prefix and v_prefix must be [Hkv, P, D]",
    )
    _require(not _needs_grad(q, k_prefix, v_prefix, k, v), "shared_prefix_attention is forward only (use torch.no_grad())")
    if lengths is not None:
        _require(
            lengths.device == q.device and lengths.dtype == torch.int32 and tuple(lengths.shape) == (B,),
            "lengths must be an int32 tensor [B] on the device of q",
        )
        lengths = lengths.contiguous()
    elif T > 1:
        lengths = torch.full((B,), S, dtype=torch.int32, device=q.device)
    scale = _scale_of(scale, D)
    dtype = q.dtype
    if dtype == torch.float32:
        q, k_prefix, v_prefix, k, v = (t.bfloat16() for t in (q, k_prefix, v_prefix, k, v))
    q, k_prefix, v_prefix, k, v = (_strided(t) for t in (q, k_prefix, v_prefix, k, v))
    out = _empty(q)
    prefix = (k_prefix, v_prefix)
    if k_prefix.shape[1] == 0 or S > _lib.SMA_MAX_SEQ_LEN:
        sparse_attn_cuda.rows_forward(q, k, v, out, scale, lengths=lengths, prefix=prefix)
    else:
        sparse_attn_cuda.prefix_forward(q, k, v, out, scale, prefix, lengths)
    return out.float() if dtype == torch.float32 else out
