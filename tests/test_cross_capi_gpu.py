"""The C entries on sma_attn_args where the package's functions do not reach
them: the LSE of sma_rows_attn_fwd, and a prefix together with a mask.

Bound on the LSE of a row of n keys: every score is off by at most s_max 2^-20
(cross_ref.py); base-2 exponentials, the logarithm and the merges of warps and
pieces by a few 2^-22; and a thread adds at most n / 16 + 64 exponentials in a
row, each addition off by 2^-24 of the sum."""

import numpy as np
import pytest
import torch

import python._lib as L
from cross_ref import Ref, buckets_of
from python import sparse_attn_cuda
from test_cross_attention_cpu import raw
from test_cross_attention_gpu import heads, make_mask, prefix_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
FLT_MAX = float(np.finfo(np.float32).max)


def rows_entry(q, k, v, **kw):
    """out and lse of sma_rows_attn_fwd."""
    B, H, Nq, D = q.shape
    out, lse = torch.empty_like(q), torch.empty(B, H, Nq, device=DEV)
    at = dict(dtype=int(q.dtype == BF16), scale=D**-0.5, B=B, H=H, Hkv=k.shape[1], Nq=Nq, Nk=k.shape[2], D=D,
              q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr())
    for n, t in (("q", q), ("k", k), ("v", v)):
        at.update({n + "b": t.stride(0), n + "h": t.stride(1), n + "n": t.stride(2)})
    L.check(L.load().sma_rows_attn_fwd(raw(**at, **kw), torch.cuda.current_stream().cuda_stream))
    sparse_attn_cuda.device_status()
    return out, lse


def check(ref, out, lse):
    ref.check_out(out)
    lse, n = lse.double().cpu(), ref.keep.shape[-1]
    some = torch.isfinite(ref.lse)
    assert torch.all(lse[~some] == -FLT_MAX)
    bound = 1.05 * (ref.s_max[..., 0] * 2.0**-20 + ref.lse.abs() * 2.0**-22 + (n / 16 + 64) * 2.0**-24) + 2.0**-20
    assert torch.all((lse - ref.lse).abs()[some] <= bound[some])


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("mask", ["none", "padding", "heads"])
@pytest.mark.parametrize("B,H,Hkv,Nq,Nk", [(2, 3, 3, 1, 31), (2, 6, 2, 17, 129), (1, 8, 1, 1, 20011), (2, 4, 2, 3, 3001)])
def test_lse_under_a_mask(B, H, Hkv, Nq, Nk, mask, D, dtype):
    gen = torch.Generator(device=DEV).manual_seed(Nk)
    q = heads(gen, B, H, Nq, D, dtype)
    k, v = (heads(gen, B, Hkv, Nk, D, dtype) for _ in range(2))
    m = make_mask(gen, mask, B, H, Nq, Nk)
    kw = {}
    if m is not None:
        sb, sh, sq = (0 if m.shape[i] == 1 else m.stride(i) for i in range(3))
        kw = dict(mask=m.data_ptr(), mb=sb, mh=sh, mn=sq)
    check(Ref(q, k, v, m), *rows_entry(q, k, v, **kw))


@pytest.mark.parametrize("P,S", [(0, 40), (500, 33), (9000, 70)])
def test_lse_behind_a_prefix(P, S):
    """Lengths, one of them 0, and a prefix in front."""
    gen = torch.Generator(device=DEV).manual_seed(P)
    q = heads(gen, 3, 4, 2, 64, F16)
    kp, vp = (heads(gen, 1, 2, P, 64, F16)[0] for _ in range(2))
    k, v = (heads(gen, 3, 2, S, 64, F16) for _ in range(2))
    n = torch.tensor([0, S, S // 2], dtype=torch.int32, device=DEV)
    at = dict(kp=kp.data_ptr(), vp=vp.data_ptr(), P=P) if P else {}
    for x, t in (("kp", kp), ("vp", vp)):
        at.update({x + "h": t.stride(0), x + "n": t.stride(1)})
    check(prefix_ref(q, kp, vp, k, v, n), *rows_entry(q, k, v, lengths=n.data_ptr(), **at))


def test_lse_with_a_bias():
    from python.cross_attention import _side

    gen = torch.Generator(device=DEV).manual_seed(3)
    q = heads(gen, 2, 4, 5, 64, BF16)
    k, v = (heads(gen, 2, 4, 700, 64, BF16) for _ in range(2))
    table = torch.randn(32, 4, generator=gen, device=DEV).bfloat16()
    starts, side, _owner = _side(32, True, 128)
    got = rows_entry(q, k, v, table=table.data_ptr(), starts=starts, side=side, two_sided=1, offset=300)
    check(Ref(q, k, v, None, table.double().cpu().t()[:, buckets_of(5, 700, 32, 128, True, 300)]), *got)


@pytest.mark.parametrize("Nq,P", [(1, 77), (7, 2000)])
def test_prefix_and_mask_together(Nq, P):
    """The mask is over the own keys; every row keeps the prefix."""
    gen = torch.Generator(device=DEV).manual_seed(P)
    q = heads(gen, 2, 4, Nq, 128, BF16)
    kp, vp = (heads(gen, 1, 2, P, 128, BF16)[0] for _ in range(2))
    k, v = (heads(gen, 2, 2, 90, 128, BF16) for _ in range(2))
    m = torch.rand(2, 4, Nq, 90, generator=gen, device=DEV) < 0.4
    at = dict(kp=kp.data_ptr(), vp=vp.data_ptr(), P=P, mask=m.data_ptr(), mb=m.stride(0), mh=m.stride(1), mn=m.stride(2))
    for x, t in (("kp", kp), ("vp", vp)):
        at.update({x + "h": t.stride(0), x + "n": t.stride(1)})
    keys, values = (torch.cat([a.expand(2, -1, -1, -1), b], 2) for a, b in ((kp, k), (vp, v)))
    keep = torch.cat([torch.ones(2, 4, Nq, P, dtype=torch.bool, device=DEV), m], -1)
    check(Ref(q, keys, values, keep), *rows_entry(q, k, v, **at))
