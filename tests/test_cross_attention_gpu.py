"""cross_attention, relative_bias_attention and shared_prefix_attention
(forward) against their plain form in 64 bits; the bounds are derived in
cross_ref.py."""

import pytest
import torch

from cross_ref import Ref, buckets_of
from python import cross_attention, relative_bias_attention, shared_prefix_attention, sparse_attn_cuda

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def heads(gen, B, H, N, D, dtype, layout="bhnd"):
    if layout == "bnhd":
        return torch.randn(B, N, H, D, generator=gen, device=DEV).to(dtype).transpose(1, 2)
    if layout == "sliced":  # rows of a wider buffer
        return torch.randn(B, H, N + 3, D + 8, generator=gen, device=DEV).to(dtype)[:, :, 2 : N + 2, :D]
    return torch.randn(B, H, N, D, generator=gen, device=DEV).to(dtype)


def make_mask(gen, kind, B, H, Nq, Nk):
    if kind == "none":
        return None
    if kind == "padding":  # one sequence keeps nothing, one keeps all
        lengths = torch.randint(0, Nk + 1, (B,), generator=gen, device=DEV)
        lengths[0] = 0 if B > 1 else Nk
        lengths[-1] = Nk
        return (torch.arange(Nk, device=DEV)[None] < lengths[:, None]).view(B, 1, 1, Nk)
    if kind == "causal":
        return torch.ones(Nq, Nk, dtype=torch.bool, device=DEV).tril().view(1, 1, Nq, Nk)
    m = torch.rand(B if kind != "shared" else 1, H if kind == "heads" else 1, Nq, Nk, generator=gen, device=DEV) < 0.3
    m[:, :, Nq // 2] = False  # a row that keeps nothing
    if kind == "sliced":  # rows of a wider buffer, an odd first byte
        wide = torch.zeros(*m.shape[:3], Nk + 5, dtype=torch.bool, device=DEV)
        wide[..., 1 : Nk + 1] = m
        m = wide[..., 1 : Nk + 1]
    return m


SHAPES = [  # B, H, Hkv, Nq, Nk
    (1, 1, 1, 1, 1),
    (2, 3, 3, 1, 31),
    (3, 4, 2, 1, 32),
    (1, 8, 1, 1, 33),
    (2, 2, 1, 3, 64),
    (2, 4, 4, 16, 257),
    (2, 6, 2, 17, 129),
    (1, 2, 2, 65, 500),
    (2, 4, 2, 130, 333),
    (1, 2, 1, 257, 1025),
    (2, 32, 8, 1, 3001),
    (1, 2, 2, 1, 20011),
]


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (64, BF16), (128, F16)])
@pytest.mark.parametrize("mask", ["none", "padding", "heads", "batch", "shared", "sliced"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_cross_attention(shape, mask, D, dtype):
    B, H, Hkv, Nq, Nk = shape
    gen = torch.Generator(device=DEV).manual_seed(Nq * 1000 + Nk)
    q = heads(gen, B, H, Nq, D, dtype)
    k, v = (heads(gen, B, Hkv, Nk, D, dtype) for _ in range(2))
    m = make_mask(gen, mask, B, H, Nq, Nk)
    out = cross_attention(q, k, v, m)
    sparse_attn_cuda.device_status()
    assert out.shape == q.shape and out.dtype == dtype and out.is_contiguous()
    Ref(q, k, v, m).check_out(out)


@pytest.mark.parametrize("layout", ["bnhd", "sliced"])
@pytest.mark.parametrize("Nq,D", [(1, 64), (5, 128), (200, 64), (150, 128)])
def test_strided_inputs(layout, Nq, D):
    gen = torch.Generator(device=DEV).manual_seed(Nq)
    q = heads(gen, 2, 4, Nq, D, BF16, layout)
    k, v = (heads(gen, 2, 2, 300, D, BF16, layout) for _ in range(2))
    m = make_mask(gen, "padding", 2, 4, Nq, 300)
    out = cross_attention(q, k, v, m)
    assert torch.equal(out, cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), m))
    Ref(q, k, v, m).check_out(out)


def test_odd_strides_and_expanded_keys_are_copied():
    gen = torch.Generator(device=DEV).manual_seed(4)
    q = torch.randn(2, 2, 7, 131, generator=gen, device=DEV).half()[..., 3:67]  # 2-byte aligned rows
    k = torch.randn(1, 1, 90, 64, generator=gen, device=DEV).half().expand(2, 2, 90, 64)
    v = torch.randn(2, 2, 64, 90, generator=gen, device=DEV).half().transpose(2, 3)
    Ref(q, k, v).check_out(cross_attention(q, k, v))


def test_fp32_inputs_are_computed_in_bf16():
    gen = torch.Generator(device=DEV).manual_seed(5)
    q, k, v = (torch.randn(2, 2, n, 64, generator=gen, device=DEV) for n in (9, 70, 70))
    out = cross_attention(q, k, v)
    assert out.dtype == torch.float32
    assert torch.equal(out, cross_attention(q.bfloat16(), k.bfloat16(), v.bfloat16()).float())


@pytest.mark.parametrize("Nq", [1, 40, 200])
def test_padding_may_hold_anything(Nq):
    """Keys and values behind a padding mask may be infinite or NaN."""
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = heads(gen, 2, 4, Nq, 64, F16), heads(gen, 2, 4, 500, 64, F16), heads(gen, 2, 4, 500, 64, F16)
    m = torch.zeros(2, 1, 1, 500, dtype=torch.bool, device=DEV)
    m[0, ..., :333] = True
    m[1, ..., 7:490] = True
    want = cross_attention(q, k, v, m)
    gone = ~m.view(2, 1, 500, 1)
    k2, v2 = k.masked_fill(gone, float("nan")), v.masked_fill(gone, float("inf"))
    assert torch.equal(cross_attention(q, k2, v2, m), want)


def test_no_keys_and_no_queries():
    q = torch.randn(2, 2, 3, 64, device=DEV).half()
    none = torch.empty(2, 1, 0, 64, device=DEV).half()
    assert torch.equal(cross_attention(q, none, none), torch.zeros_like(q))
    assert cross_attention(q[:, :, :0], q, q).shape == (2, 2, 0, 64)
    assert cross_attention(q[:0], q[:0], q[:0]).shape == (0, 2, 3, 64)


def test_large_scores():
    """Scores in the hundreds: the running maximum keeps the sums finite."""
    gen = torch.Generator(device=DEV).manual_seed(8)
    for Nq in (2, 150):
        q, k = (20 * torch.randn(1, 2, n, 64, generator=gen, device=DEV).half() for n in (Nq, 400))
        v = torch.randn(1, 2, 400, 64, generator=gen, device=DEV).half()
        Ref(q, k, v).check_out(cross_attention(q, k, v))


BIAS = [  # buckets, max_distance, two_sided
    (32, 128, True),
    (32, 128, False),
    (16, 64, True),
    (64, 256, False),
    (4, 5, True),
    (2, 3, False),
]


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("buckets,distance,two_sided", BIAS)
@pytest.mark.parametrize(
    "shape,offset,mask",
    [
        ((1, 2, 2, 1, 1), 0, "none"),
        ((2, 4, 2, 1, 700), 699, "padding"),
        ((2, 4, 2, 1, 700), 12, "none"),
        ((2, 8, 2, 3, 90), 50, "batch"),
        ((1, 3, 3, 200, 200), 0, "causal"),
        ((2, 2, 2, 300, 300), 0, "heads"),
        ((1, 4, 2, 190, 777), -37, "padding"),
        ((1, 2, 1, 129, 1200), 1071, "none"),
    ],
)
def test_relative_bias(shape, offset, mask, buckets, distance, two_sided, D, dtype):
    B, H, Hkv, Nq, Nk = shape
    gen = torch.Generator(device=DEV).manual_seed(Nq + Nk)
    q = heads(gen, B, H, Nq, D, dtype)
    k, v = (heads(gen, B, Hkv, Nk, D, dtype) for _ in range(2))
    table = (2 * torch.randn(buckets, H, generator=gen, device=DEV)).to(dtype)
    m = make_mask(gen, mask, B, H, Nq, Nk)
    out = relative_bias_attention(q, k, v, table, m, bidirectional=two_sided, max_distance=distance, query_offset=offset)
    sparse_attn_cuda.device_status()
    add = table.double().cpu().t()[:, buckets_of(Nq, Nk, buckets, distance, two_sided, offset)]
    Ref(q, k, v, m, add).check_out(out)


@pytest.mark.parametrize("Nq", [1, 140])
def test_bias_offsets_per_sequence(Nq):
    gen = torch.Generator(device=DEV).manual_seed(9)
    q, k, v = heads(gen, 3, 4, Nq, 64, BF16), heads(gen, 3, 4, 400, 64, BF16), heads(gen, 3, 4, 400, 64, BF16)
    table = torch.randn(32, 4, generator=gen, device=DEV)  # FP32 parameters are rounded to the inputs' type
    offsets = torch.tensor([0, 260, 399], dtype=torch.int32, device=DEV)
    out = relative_bias_attention(q, k, v, table, bidirectional=False, query_offset=offsets)
    for b in range(3):
        one = relative_bias_attention(q[b : b + 1], k[b : b + 1], v[b : b + 1], table.bfloat16(), bidirectional=False,
                                      query_offset=int(offsets[b]))
        add = table.bfloat16().double().cpu().t()[:, buckets_of(Nq, 400, 32, 128, False, int(offsets[b]))]
        Ref(q[b : b + 1], k[b : b + 1], v[b : b + 1], None, add).check_out(out[b : b + 1])
        Ref(q[b : b + 1], k[b : b + 1], v[b : b + 1], None, add).check_out(one)


def prefix_ref(q, kp, vp, k, v, lengths):
    """The prefix in front of the sequence's own keys, causal among the last T."""
    B, H, T, D = q.shape
    P, S = kp.shape[1], k.shape[2]
    n = (lengths.cpu().long() if lengths is not None else torch.full((B,), S)).clamp(0, S)
    last = n[:, None] - T + 1 + torch.arange(T)
    keep = torch.cat([torch.ones(B, T, P, dtype=torch.bool), torch.arange(S) < last[..., None]], -1)
    keys, values = (torch.cat([a.expand(B, *a.shape), b], 2) for a, b in ((kp, k), (vp, v)))
    return Ref(q, keys, values, keep[:, None])


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize(
    "B,H,Hkv,T,P,S",
    [
        (1, 1, 1, 1, 1, 1),
        (3, 2, 2, 1, 64, 5),
        (4, 8, 2, 1, 500, 33),
        (5, 6, 2, 1, 1000, 70),
        (2, 4, 4, 7, 129, 20),
        (3, 8, 2, 9, 300, 40),
        (16, 4, 1, 2, 2049, 65),
        (2, 2, 2, 150, 260, 170),
        (3, 4, 2, 40, 0, 50),
        (2, 4, 2, 1, 90, 0),
    ],
)
def test_shared_prefix(B, H, Hkv, T, P, S, D, dtype):
    gen = torch.Generator(device=DEV).manual_seed(P + S)
    q = heads(gen, B, H, T, D, dtype)
    kp, vp = (heads(gen, 1, Hkv, P, D, dtype)[0] for _ in range(2))
    k, v = (heads(gen, B, Hkv, S, D, dtype) for _ in range(2))
    cases = [None]
    if S:
        some = torch.randint(0, S + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
        some[0] = 0
        cases += [some, torch.full((B,), S, dtype=torch.int32, device=DEV)]
    for lengths in cases:
        out = shared_prefix_attention(q, kp, vp, k, v, lengths)
        sparse_attn_cuda.device_status()
        prefix_ref(q, kp, vp, k, v, lengths).check_out(out)


@pytest.mark.parametrize("T", [1, 6, 90])
def test_prefix_lengths_are_clamped_and_the_rest_unread(T):
    gen = torch.Generator(device=DEV).manual_seed(11)
    B, S = 3, 100
    q, k, v = heads(gen, B, 4, T, 64, F16), heads(gen, B, 2, S, 64, F16), heads(gen, B, 2, S, 64, F16)
    kp, vp = (heads(gen, 1, 2, 200, 64, F16)[0] for _ in range(2))
    lengths = torch.tensor([-5, S + 77, 41], dtype=torch.int32, device=DEV)
    want = shared_prefix_attention(q, kp, vp, k, v, lengths.clamp(0, S))
    assert torch.equal(shared_prefix_attention(q, kp, vp, k, v, lengths), want)
    used = torch.arange(S, device=DEV)[None] < lengths[:, None]
    junk = ~used[:, None, :, None]
    got = shared_prefix_attention(q, kp, vp, k.masked_fill(junk, float("nan")), v.masked_fill(junk, float("nan")), lengths)
    assert torch.equal(got, want)


def test_results_do_not_change_from_run_to_run():
    gen = torch.Generator(device=DEV).manual_seed(12)
    q, k, v = heads(gen, 2, 8, 1, 64, F16), heads(gen, 2, 2, 9000, 64, F16), heads(gen, 2, 2, 9000, 64, F16)
    want = cross_attention(q, k, v)
    for _ in range(20):
        assert torch.equal(cross_attention(q, k, v), want)


@pytest.mark.parametrize("Nq,D", [(3, 64), (100, 64), (300, 128)])
def test_keys_that_no_row_keeps_may_hold_anything(Nq, D):
    """Masks with rows of their own (causal and padded, say): keys that no
    query keeps may be infinite or NaN."""
    gen = torch.Generator(device=DEV).manual_seed(13)
    q = heads(gen, 2, 2, Nq, D, BF16)
    k, v = (heads(gen, 2, 2, 400, D, BF16) for _ in range(2))
    m = torch.rand(2, 2, Nq, 400, generator=gen, device=DEV) < 0.5
    m[0, ..., 333:] = False
    m[1, ..., :130] = False
    m[1, 0, :, 200] = False
    want = cross_attention(q, k, v, m)
    gone = ~m.any(2)[..., None]
    got = cross_attention(q, k.masked_fill(gone, float("nan")), v.masked_fill(gone, float("-inf")), m)
    assert torch.equal(got, want)
