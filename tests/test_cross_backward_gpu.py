"""Gradients of cross_attention and relative_bias_attention against the
formulas in 64 bits and against differences of the 64-bit forward.

Bounds, with u = eps / 2 of the type.  The kernel rebuilds P from the LSE
(FP32), rounds P and dS to the type for the products (u each) and uses
Delta = rowsum(dO * O) with O rounded (off by 2 u A + u |O| at most, see
cross_ref).  So, elementwise and to first order:
  dV: u (|P|^T |dO|), and u |dV| for the result
  dS: e = P (2 u A_d + FP32 terms), A_d = sum_d |dO_d| (2 A + |O|), and u |dS|
  dQ = scale (dS K): scale (|e| + u |dS|) |K|, and u |dQ|;  dK alike
  dtable: the sum of e over the bucket's pairs, and u |dtable|
FP32 sums: 2^-20 of the sum of magnitudes.  In fp16 values below 2^-14 are
rounded by at most 2^-25 instead of u times themselves; P and dS get that
much more.  A factor of 1.1 covers second-order terms."""

import pytest
import torch

from cross_ref import Ref, buckets_of
from python import cross_attention, relative_bias_attention, sparse_attn_cuda
from test_cross_attention_gpu import BIAS, heads, make_mask

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


class RefGrads(Ref):
    def __init__(self, q, k, v, dout, keep=None, add=None, scale=None, dtype=None):
        super().__init__(q, k, v, keep, add, scale)
        u = torch.finfo(dtype).eps / 2
        tiny = 2.0**-25 if dtype == F16 else 0.0
        f = 2.0**-20
        do = dout.double().cpu()
        p, k64, v64, q64 = self.p, self.k, self.v, self.q
        dp = do @ v64.transpose(2, 3)
        delta = (do * self.out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        dp_mag = do.abs() @ v64.abs().transpose(2, 3)
        e_delta = (do.abs() * (2 * u * self.A + u * self.out.abs() + 2 * tiny * self.V)).sum(-1, keepdim=True)
        # P itself is off by the FP32 error of its scores and of the LSE.
        e_p = p * f * (2 * self.s_max + 4)
        e_ds = e_p * (dp - delta).abs() + p * (e_delta + f * (dp_mag + (do.abs() * self.A).sum(-1, keepdim=True)))
        r_ds = e_ds + (u + f) * ds.abs() + tiny * self.keep
        r_p = e_p + (u + f) * p + tiny * self.keep
        B, H, Nq, Nk = p.shape
        Hkv = H // self.G
        share = lambda t: t.view(B, Hkv, self.G, Nk, -1).sum(2)  # noqa: E731
        self.grads = {
            "dq": self.scale * (ds @ k64),
            "dk": self.scale * share(ds.transpose(2, 3) @ q64),
            "dv": share(p.transpose(2, 3) @ do),
        }
        mags = {
            "dq": self.scale * (r_ds @ k64.abs()),
            "dk": self.scale * share(r_ds.transpose(2, 3) @ q64.abs()),
            "dv": share(r_p.transpose(2, 3) @ do.abs()),
        }
        self.bounds = {n: 1.1 * (m + u * self.grads[n].abs()) + 1e-6 for n, m in mags.items()}
        self.ds, self.e_ds, self.u, self.f = ds, e_ds, u, f

    def with_table(self, bucket, n):
        member = torch.nn.functional.one_hot(bucket, n).double()  # [Nq, Nk, n]
        self.grads["dtable"] = torch.einsum("bhqk,qkn->nh", self.ds, member)
        e = torch.einsum("bhqk,qkn->nh", self.e_ds + self.f * self.ds.abs(), member)
        self.bounds["dtable"] = 1.1 * (e + self.u * self.grads["dtable"].abs()) + 1e-6
        return self

    def check(self, **got):
        for n, g in got.items():
            assert torch.isfinite(g).all(), f"{n}: non-finite values"
            assert tuple(g.shape) == tuple(self.grads[n].shape)
            err = (g.double().cpu() - self.grads[n]).abs()
            worst = float((err / self.bounds[n]).max()) if err.numel() else 0.0
            assert worst <= 1.0, f"{n} is off by {worst:.2f} of its bound (largest error {float(err.max()):.3e})"


SHAPES = [  # B, H, Hkv, Nq, Nk
    (1, 1, 1, 1, 1),
    (2, 3, 3, 1, 40),
    (1, 4, 2, 16, 33),
    (2, 6, 2, 20, 129),
    (1, 8, 1, 30, 260),
    (2, 4, 2, 64, 64),
    (1, 2, 1, 130, 77),
    (2, 4, 2, 257, 300),
    (1, 2, 2, 300, 1025),
]


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (64, BF16), (128, F16)])
@pytest.mark.parametrize("mask", ["none", "padding", "heads", "batch", "shared", "sliced"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_cross_attention_gradients(shape, mask, D, dtype):
    B, H, Hkv, Nq, Nk = shape
    gen = torch.Generator(device=DEV).manual_seed(Nq * 1000 + Nk + 1)
    q = heads(gen, B, H, Nq, D, dtype).requires_grad_(True)
    k, v = (heads(gen, B, Hkv, Nk, D, dtype).requires_grad_(True) for _ in range(2))
    dout = heads(gen, B, H, Nq, D, dtype)
    m = make_mask(gen, mask, B, H, Nq, Nk)
    out = cross_attention(q, k, v, m)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    sparse_attn_cuda.device_status()
    ref = RefGrads(q, k, v, dout, m, dtype=dtype)
    ref.check_out(out.detach())
    ref.check(dq=dq, dk=dk, dv=dv)
    empty_rows = ~ref.keep.any(-1)
    assert torch.all(dq.cpu()[empty_rows] == 0), "rows that keep no key get dq = 0"


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("buckets,distance,two_sided", BIAS)
@pytest.mark.parametrize(
    "shape,offset,mask",
    [
        ((1, 2, 2, 1, 1), 0, "none"),
        ((2, 4, 2, 1, 300), 299, "padding"),
        ((1, 3, 3, 200, 200), 0, "causal"),
        ((2, 2, 2, 300, 300), 0, "heads"),
        ((1, 4, 2, 190, 777), -37, "padding"),
        ((2, 4, 1, 40, 500), 333, "batch"),
        ((1, 2, 1, 129, 1200), 1071, "none"),
    ],
)
def test_relative_bias_gradients(shape, offset, mask, buckets, distance, two_sided, D, dtype):
    B, H, Hkv, Nq, Nk = shape
    gen = torch.Generator(device=DEV).manual_seed(Nq + Nk + 2)
    q = heads(gen, B, H, Nq, D, dtype).requires_grad_(True)
    k, v = (heads(gen, B, Hkv, Nk, D, dtype).requires_grad_(True) for _ in range(2))
    table = (2 * torch.randn(buckets, H, generator=gen, device=DEV)).to(dtype).requires_grad_(True)
    dout = heads(gen, B, H, Nq, D, dtype)
    m = make_mask(gen, mask, B, H, Nq, Nk)
    out = relative_bias_attention(q, k, v, table, m, bidirectional=two_sided, max_distance=distance, query_offset=offset)
    dq, dk, dv, dtable = torch.autograd.grad(out, (q, k, v, table), dout)
    sparse_attn_cuda.device_status()
    bucket = buckets_of(Nq, Nk, buckets, distance, two_sided, offset)
    add = table.detach().double().cpu().t()[:, bucket]
    ref = RefGrads(q, k, v, dout, m, add, dtype=dtype).with_table(bucket, buckets)
    ref.check_out(out.detach())
    ref.check(dq=dq, dk=dk, dv=dv, dtable=dtable)


def test_bias_offsets_per_sequence_and_long_distances():
    """Offsets on the device, a last bucket farther out than any key, FP32
    parameters."""
    gen = torch.Generator(device=DEV).manual_seed(21)
    q, k, v, dout = (heads(gen, 3, 2, n, 64, BF16) for n in (70, 400, 400, 70))
    table = torch.randn(24, 2, generator=gen, device=DEV)
    offsets = torch.tensor([0, 260, 330], dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    out = relative_bias_attention(q, k, v, table, max_distance=5000, query_offset=offsets)
    dq, dk, dv, dtable = torch.autograd.grad(out, leaves, dout)
    assert dtable.dtype == torch.float32
    total = torch.zeros(24, 2).double()
    bound = torch.zeros(24, 2).double()
    for b in range(3):
        bucket = buckets_of(70, 400, 24, 5000, True, int(offsets[b]))
        add = table.detach().bfloat16().double().cpu().t()[:, bucket]
        one = [t[b : b + 1] for t in (q, k, v, dout)]
        ref = RefGrads(*one, None, add, dtype=BF16).with_table(bucket, 24)
        ref.check(dq=dq[b : b + 1], dk=dk[b : b + 1], dv=dv[b : b + 1])
        total += ref.grads["dtable"]
        bound += ref.bounds["dtable"]
    assert torch.all((dtable.cpu().double() - total).abs() <= bound + 2.0**-8 * total.abs())


def test_gradient_against_differences():
    """dq, dk, dv and dtable along random directions against central
    differences of the 64-bit forward (bf16 results: 2^-8 of the norms)."""
    gen = torch.Generator(device=DEV).manual_seed(22)
    q, k, v, dout = (heads(gen, 1, 2, n, 64, BF16) for n in (50, 90, 90, 50))
    table = torch.randn(32, 2, generator=gen, device=DEV).bfloat16()
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    out = relative_bias_attention(q, k, v, table)
    grads = torch.autograd.grad(out, leaves, dout)
    bucket = buckets_of(50, 90, 32, 128, True)

    def loss(x):
        add = x[3].t()[:, bucket]
        return float((Ref(x[0], x[1], x[2], None, add).out * dout.double().cpu()).sum())

    base = [t.detach().double().cpu() for t in leaves]
    for i, g in enumerate(grads):
        step = torch.randn(base[i].shape, generator=torch.Generator().manual_seed(i)).double()
        h = 1e-4
        up = [t + h * step if j == i else t for j, t in enumerate(base)]
        down = [t - h * step if j == i else t for j, t in enumerate(base)]
        want = (loss(up) - loss(down)) / (2 * h)
        got = float((g.double().cpu() * step).sum())
        # Each element of g is off by about 2^-8 of its magnitude (rounding of
        # P, dS and the result); the directions are independent of it.
        assert abs(got - want) <= 4 * 2.0**-8 * float(g.double().norm()), (i, got, want)


def test_expanded_and_strided_inputs():
    """Gradients of a key shared by expansion, of transposed projections and
    of an expanded upstream gradient."""
    gen = torch.Generator(device=DEV).manual_seed(23)
    x = torch.randn(2, 150, 4, 64, generator=gen, device=DEV).half().requires_grad_(True)
    k1 = torch.randn(1, 1, 90, 64, generator=gen, device=DEV).half().requires_grad_(True)
    out = cross_attention(x.transpose(1, 2), k1.expand(2, 2, 90, 64), k1.expand(2, 2, 90, 64))
    gx, gk = torch.autograd.grad(out.float().sum(), (x, k1))
    q = x.detach().transpose(1, 2)
    k = k1.detach().expand(2, 2, 90, 64)
    ref = RefGrads(q, k, k, torch.ones_like(q), dtype=F16)
    ref.check(dq=gx.transpose(1, 2))
    want = (ref.grads["dk"] + ref.grads["dv"]).sum((0, 1), keepdim=True)
    bound = (ref.bounds["dk"] + ref.bounds["dv"]).sum((0, 1), keepdim=True) + 2.0**-8 * want.abs() + 1e-3
    assert torch.all((gk.double().cpu() - want).abs() <= bound)


def test_dk_dv_dtable_do_not_change_from_run_to_run():
    gen = torch.Generator(device=DEV).manual_seed(24)
    q, k, v, dout = (heads(gen, 2, 4, 500, 64, BF16) for _ in range(4))
    table = torch.randn(32, 4, generator=gen, device=DEV).bfloat16()
    leaves = [t.requires_grad_(True) for t in (q, k, v, table)]
    first = None
    for _ in range(5):
        grads = torch.autograd.grad(relative_bias_attention(q, k, v, table), leaves, dout)
        if first is not None:
            assert all(torch.equal(a, b) for a, b in zip(grads[1:], first[1:]))
        first = grads


def test_second_derivative_is_refused():
    q = torch.randn(1, 1, 20, 64, device=DEV).half().requires_grad_(True)
    (g,) = torch.autograd.grad(cross_attention(q, q, q).float().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_empty_inputs_have_zero_gradients():
    q = torch.randn(2, 2, 3, 64, device=DEV).half().requires_grad_(True)
    k = torch.empty(2, 2, 0, 64, device=DEV).half().requires_grad_(True)
    gq, gk = torch.autograd.grad(cross_attention(q, k, k).sum(), (q, k))
    assert torch.all(gq == 0) and gk.shape == k.shape


def test_too_many_query_tiles_are_refused():
    q = torch.empty(1, 2049, 1, 64, device=DEV).half().requires_grad_(True)
    k = torch.empty(1, 1, 8, 64, device=DEV).half()
    with pytest.raises(RuntimeError, match="2048"):
        cross_attention(q, k, k)


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("Nq,D", [(5, 64), (200, 64), (130, 128)])
def test_padding_may_hold_anything(Nq, D, bias):
    """Keys and values behind a padding mask may be infinite or NaN: their
    gradients are 0 and nothing else changes."""
    gen = torch.Generator(device=DEV).manual_seed(25)
    q, dout = heads(gen, 2, 4, Nq, D, BF16), heads(gen, 2, 4, Nq, D, BF16)
    k, v = (heads(gen, 2, 2, 300, D, BF16) for _ in range(2))
    table = torch.randn(32, 4, generator=gen, device=DEV).bfloat16()
    m = torch.zeros(2, 1, 1, 300, dtype=torch.bool, device=DEV)
    m[0, ..., :133] = True
    m[1, ..., 7:290] = True
    gone = ~m.view(2, 1, 300, 1)

    def run(k, v):
        leaves = [t.clone().requires_grad_(True) for t in ((q, k, v, table) if bias else (q, k, v))]
        out = relative_bias_attention(*leaves, m) if bias else cross_attention(*leaves, m)
        return out.detach(), torch.autograd.grad(out, leaves, dout)

    out0, want = run(k, v)
    out1, got = run(k.masked_fill(gone, float("nan")), v.masked_fill(gone, float("inf")))
    assert torch.equal(out0, out1)
    for i, (a, b) in enumerate(zip(got, want)):
        if i == 0:  # dq: FP32 adds in another order
            assert torch.allclose(a.float(), b.float(), rtol=2.0**-7, atol=1e-4)
        else:
            assert torch.equal(a, b)
    assert torch.all(got[1].masked_select(gone.expand_as(k)) == 0) and torch.all(got[2].masked_select(gone.expand_as(v)) == 0)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("mask,bias", [("none", False), ("padding", False), ("heads", False), ("padding", True)])
def test_items_that_do_not_fill_the_last_round(mask, bias, D, dtype):
    """A few more (batch, head, query tile) items than run at once."""
    B, H, Nq, Nk = 10, 30, 20, 1100
    gen = torch.Generator(device=DEV).manual_seed(D)
    q, k, v = (heads(gen, B, H, n, D, dtype).requires_grad_(True) for n in (Nq, Nk, Nk))
    dout = heads(gen, B, H, Nq, D, dtype)
    m = make_mask(gen, mask, B, H, Nq, Nk)
    if bias:
        table = torch.randn(32, H, generator=gen, device=DEV).to(dtype)
        out = relative_bias_attention(q, k, v, table, m, query_offset=500)
        add = table.double().cpu().t()[:, buckets_of(Nq, Nk, 32, 128, True, 500)]
    else:
        out, add = cross_attention(q, k, v, m), None
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), dout)))
    sparse_attn_cuda.device_status()
    ref = RefGrads(q, k, v, dout, m, add, dtype=dtype)
    ref.check_out(out.detach())
    ref.check(**got)
    again = (relative_bias_attention(q, k, v, table, m, query_offset=500) if bias else cross_attention(q, k, v, m)).detach()
    assert torch.equal(out.detach(), again)
