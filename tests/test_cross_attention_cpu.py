"""Refusals of the operators on queries and keys of different lengths, and
the bucket bounds of the relative position bias.  CPU only: no call here
launches work."""

import ctypes
import math

import pytest
import torch

import python as sma
import python._lib as L
from cross_ref import buckets_of, starts_of
from python.cross_attention import _bucket_starts


@pytest.fixture(scope="module")
def lib():
    return L.load()


STARTS = (ctypes.c_int32 * 4)(0, 1, 2, 8)
FIELDS = ("dtype scale B H Hkv Nq Nk D P q k v qb qh qn kb kh kn vb vh vn kp vp kph kpn vph vpn mask mb mh mn lengths table "
          "starts offsets offset side two_sided out lse words distance out_lo").split()


def raw(**kw):
    """sma_attn_args of a small valid call (never-read addresses) with some fields replaced."""
    d = dict.fromkeys(FIELDS, 0)
    d.update(dtype=0, scale=0.125, B=2, H=4, Hkv=2, Nq=1, Nk=64, D=64, q=16, k=16, v=16, qb=256, qh=64, qn=64, kb=8192,
             kh=4096, kn=64, vb=8192, vh=4096, vn=64, kph=4096, kpn=64, vph=4096, vpn=64, out=16)
    assert set(kw) <= set(d)
    d.update(kw)
    return L.ATTN_ARGS.pack(*(d[f] for f in FIELDS))


FAR = (ctypes.c_int32 * 2)(0, L.SMA_MAX_BIAS_DISTANCE + 1)
BIAS = dict(table=16, starts=ctypes.addressof(STARTS), side=4)


@pytest.mark.parametrize(
    "kw,code",
    [
        (dict(dtype=5), L.SMA_ERR_DTYPE),
        (dict(D=96), L.SMA_ERR_UNSUPPORTED_D),
        (dict(B=-1), L.SMA_ERR_ARG),
        (dict(Nk=(1 << 30) + 1), L.SMA_ERR_UNSUPPORTED_N),
        (dict(P=(1 << 30) + 1, kp=16, vp=16), L.SMA_ERR_UNSUPPORTED_N),
        (dict(scale=0.0), L.SMA_ERR_ARG),
        (dict(scale=math.nan), L.SMA_ERR_ARG),
        (dict(scale=math.inf), L.SMA_ERR_ARG),
        (dict(Hkv=3), L.SMA_ERR_ARG),
        (dict(Hkv=0), L.SMA_ERR_ARG),
        (dict(q=0), L.SMA_ERR_ARG),
        (dict(k=0), L.SMA_ERR_ARG),
        (dict(out=0), L.SMA_ERR_ARG),
        (dict(P=8), L.SMA_ERR_ARG),  # no prefix pointers
        (dict(v=24), L.SMA_ERR_ARG),
        (dict(lse=2), L.SMA_ERR_ARG),
        (dict(qb=260), L.SMA_ERR_ARG),
        (dict(kn=0), L.SMA_ERR_ARG),
        (dict(vh=-64), L.SMA_ERR_ARG),
        (dict(P=8, kp=16, vp=16, kpn=4), L.SMA_ERR_ARG),
        (dict(mask=1, lengths=16), L.SMA_ERR_ARG),
        (dict(lengths=2), L.SMA_ERR_ARG),
        (dict(mask=1, mn=-1), L.SMA_ERR_ARG),
        (dict(BIAS, side=0), L.SMA_ERR_ARG),
        (dict(BIAS, side=129), L.SMA_ERR_ARG),
        (dict(BIAS, starts=0), L.SMA_ERR_ARG),
        (dict(BIAS, starts=ctypes.addressof(STARTS) + 4, side=2), L.SMA_ERR_ARG),  # does not start at 0
        (dict(BIAS, side=1, two_sided=1), L.SMA_ERR_ARG),
        (dict(BIAS, offset=1 << 30), L.SMA_ERR_ARG),
        (dict(BIAS, P=8, kp=16, vp=16), L.SMA_ERR_ARG),
        (dict(BIAS, table=17), L.SMA_ERR_ARG),
    ],
)
def test_library_refuses(lib, kw, code):
    assert lib.sma_rows_attn_fwd(raw(**kw), None) == code
    assert lib.sma_last_error()


def test_library_refuses_no_arguments(lib):
    assert lib.sma_rows_attn_fwd(None, None) == L.SMA_ERR_ARG


MASK = dict(mask=1, mn=64, words=16)
TRAIN = dict(lse=16, out_lo=16)


@pytest.mark.parametrize(
    "kw,code",
    [
        (dict(D=96), L.SMA_ERR_UNSUPPORTED_D),
        (dict(Nk=L.SMA_MAX_SEQ_LEN + 1), L.SMA_ERR_UNSUPPORTED_N),
        (dict(P=8, kp=16, vp=16), L.SMA_ERR_ARG),
        (dict(MASK, words=0), L.SMA_ERR_ARG),
        (dict(MASK, words=8), L.SMA_ERR_ARG),
        (dict(MASK, mask=0), L.SMA_ERR_ARG),  # words that nothing fills
        (dict(MASK, lengths=16), L.SMA_ERR_ARG),
        (dict(out_lo=8), L.SMA_ERR_ARG),
        (dict(BIAS), L.SMA_ERR_ARG),  # no room for the bias by distance
        (dict(BIAS, distance=8), L.SMA_ERR_ARG),
        (dict(BIAS, starts=ctypes.addressof(FAR), side=2, distance=16), L.SMA_ERR_UNSUPPORTED_N),
    ],
)
def test_tile_entry_refuses(lib, kw, code):
    assert lib.sma_cross_attn_fwd(raw(**kw), None) == code
    assert lib.sma_last_error()


@pytest.mark.parametrize(
    "kw,code",
    [
        (dict(), L.SMA_ERR_ARG),  # no prefix
        (dict(P=8, kp=16, vp=16, mask=1, words=16), L.SMA_ERR_ARG),
        (dict(P=8, kp=16, vp=16, lse=16), L.SMA_ERR_ARG),
        (dict(P=8, kp=16, vp=16, out_lo=16), L.SMA_ERR_ARG),
        (dict(P=8, kp=16, vp=16, Nk=L.SMA_MAX_SEQ_LEN + 1), L.SMA_ERR_UNSUPPORTED_N),
        (dict(P=8, kp=16), L.SMA_ERR_ARG),
    ],
)
def test_prefix_entry_refuses(lib, kw, code):
    assert lib.sma_prefix_attn_fwd(raw(**kw), None) == code
    assert lib.sma_last_error()


@pytest.mark.parametrize(
    "kw,pointers,code",
    [
        (dict(), {}, L.SMA_ERR_ARG),  # no lse, no out_lo
        (dict(lse=16), {}, L.SMA_ERR_ARG),
        (dict(TRAIN, Nk=0), {}, L.SMA_ERR_ARG),
        (dict(TRAIN, Nq=0), {}, L.SMA_ERR_ARG),
        (dict(TRAIN, lengths=16), {}, L.SMA_ERR_ARG),
        (dict(TRAIN, P=8, kp=16, vp=16), {}, L.SMA_ERR_ARG),
        (dict(TRAIN, Nk=L.SMA_MAX_SEQ_LEN + 1), {}, L.SMA_ERR_UNSUPPORTED_N),
        (dict(TRAIN), dict(dout=None), L.SMA_ERR_ARG),
        (dict(TRAIN), dict(dq=8), L.SMA_ERR_ARG),
        (dict(TRAIN), dict(scratch=None), L.SMA_ERR_ARG),
        (dict(TRAIN, **BIAS, distance=16), dict(dtable=None), L.SMA_ERR_ARG),
        (dict(TRAIN, **BIAS, distance=16), dict(dtable=17), L.SMA_ERR_ARG),
    ],
)
def test_backward_entry_refuses(lib, kw, pointers, code):
    at = dict(dict(dout=16, dq=16, dk=16, dv=16, dtable=16, scratch=16), **pointers)
    assert lib.sma_cross_attn_bwd(raw(**kw), *at.values(), None) == code
    assert lib.sma_last_error()


def test_backward_scratch_of_refused_arguments(lib):
    for kw in (dict(D=96), dict(Nk=0), dict(B=0), dict(Nk=L.SMA_MAX_SEQ_LEN + 1), dict(BIAS)):
        assert lib.sma_cross_attn_bwd_scratch(raw(**kw)) == -1
    assert lib.sma_cross_attn_bwd_scratch(None) == -1


def test_nothing_to_write_is_ok(lib):
    for kw in (dict(B=0), dict(H=0), dict(Nq=0)):
        assert lib.sma_rows_attn_fwd(raw(**kw), None) == L.SMA_OK


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(1, 2, 3, 64).half(), torch.zeros(1, 2, 5, 64).half()
    with pytest.raises(RuntimeError, match="CUDA"):
        sma.cross_attention(q, k, k)
    with pytest.raises(RuntimeError, match="CUDA"):
        sma.relative_bias_attention(q, k, k, torch.zeros(32, 2).half())
    with pytest.raises(RuntimeError, match="CUDA"):
        sma.shared_prefix_attention(q, k[0], k[0], k, k)


@pytest.mark.parametrize("side,distance", [(16, 128), (32, 128), (8, 64), (64, 256), (2, 3), (3, 9), (128, 1000), (5, 1 << 16)])
def test_bucket_starts(side, distance):
    """Against the definition in exact fractions; a query's own distance is
    bucket 0, and `distance` and everything beyond it fall in the last one."""
    starts = list(_bucket_starts(side, distance))
    if distance < 5000:
        assert starts == starts_of(side, distance)
    assert starts == sorted(starts) and starts[: side // 2] == list(range(side // 2))
    assert starts[-1] <= distance


def test_buckets_of_both_sides():
    b = buckets_of(300, 300, 32, 128, True)
    assert b[5, 5] == 0 and b[5, 4] == 1 and b[4, 5] == 17 and b[299, 0] == 15 and b[0, 299] == 31
    one = buckets_of(300, 300, 32, 128, False)
    assert one[0, 299] == 0 and one[299, 0] == 31 and one[20, 4] == 16
