"""Calls of cross_attention and relative_bias_attention at the edges of what
they take: bias tables with large, infinite or FP32 entries, losses on
gradients, no keys and more than the tiles take, expanded masks.  Bounds as in
test_cross_backward_gpu.py."""

import math

import pytest
import torch

from cross_ref import Ref, buckets_of
from python import cross_attention, relative_bias_attention, sparse_attn_cuda
from test_cross_attention_gpu import heads, make_mask
from test_cross_backward_gpu import RefGrads

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,entry", [(F16, 12.0), (F16, 20.0), (F16, 100.0), (BF16, 100.0)])
@pytest.mark.parametrize("mask", ["none", "padding", "heads"])
@pytest.mark.parametrize("Nq", [5, 70, 190])
def test_large_bias_entries(Nq, mask, dtype, entry, D):
    """exp(entry) passes what fp16 (11.09) or FP32 (88.7) holds: only the LSE
    of a row may ever stand next to it, and rows past the last query of a step
    of 64 have none."""
    B, H, Hkv, Nk = 2, 4, 2, 300
    gen = torch.Generator(device=DEV).manual_seed(Nq)
    q = heads(gen, B, H, Nq, D, dtype).requires_grad_(True)
    k, v = (heads(gen, B, Hkv, Nk, D, dtype).requires_grad_(True) for _ in range(2))
    table = torch.randn(32, H, generator=gen, device=DEV)
    table[[0, 3, 15, 31]] = entry
    table[20] = -entry
    table = table.to(dtype).requires_grad_(True)
    dout = heads(gen, B, H, Nq, D, dtype)
    m = make_mask(gen, mask, B, H, Nq, Nk)
    out = relative_bias_attention(q, k, v, table, m)
    dq, dk, dv, dtable = torch.autograd.grad(out, (q, k, v, table), dout)
    sparse_attn_cuda.device_status()
    bucket = buckets_of(Nq, Nk, 32, 128, True)
    add = table.detach().double().cpu().t()[:, bucket]
    ref = RefGrads(q, k, v, dout, m, add, dtype=dtype).with_table(bucket, 32)
    ref.check_out(out.detach())
    ref.check(dq=dq, dk=dk, dv=dv, dtable=dtable)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("Nq", [5, 70, 200])
def test_minus_infinity_in_the_table(Nq, D, dtype):
    """A bucket that a table closes: as if a mask closed it, also where it
    leaves a row nothing (O = 0 and no gradient, dtable's entry 0)."""
    B, H, Nk = 2, 2, Nq
    gen = torch.Generator(device=DEV).manual_seed(65)
    q, k, v, dout = (heads(gen, B, H, Nq, D, dtype) for _ in range(4))
    table = torch.randn(32, H, generator=gen, device=DEV).to(dtype)
    table[0] = -math.inf  # distance 0 and later keys: the first query keeps nothing
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, table)]
    out = relative_bias_attention(*leaves, bidirectional=False)
    got = dict(zip(("dq", "dk", "dv", "dtable"), torch.autograd.grad(out, leaves, dout)))
    bucket = buckets_of(Nq, Nk, 32, 128, False)
    add = table.masked_fill(table == -math.inf, 0.0).double().cpu().t()[:, bucket]
    ref = RefGrads(q, k, v, dout, (bucket != 0).view(1, 1, Nq, Nk), add, dtype=dtype).with_table(bucket, 32)
    ref.check_out(out.detach())
    ref.check(**got)
    with torch.no_grad():
        one = relative_bias_attention(q[:, :, :1], k, v, table, bidirectional=False)
        assert torch.all(one == 0)
        two = relative_bias_attention(q[:, :, 4:5], k, v, table, bidirectional=False, query_offset=4)
        Ref(q[:, :, 4:5], k, v, (bucket != 0)[4:5].view(1, 1, 1, Nk), add[:, 4:5]).check_out(two)


@pytest.mark.parametrize("Nk", [150, 9000])
@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_row_without_a_sum_is_not_one_that_keeps_nothing(bad, D, dtype, Nk):
    """NaN or infinity in a query: NaN in its output, its dq and the gradients
    of every key it keeps, not zeros; other rows are as without it."""
    gen = torch.Generator(device=DEV).manual_seed(66)
    q, dout = heads(gen, 1, 2, 70, D, dtype), heads(gen, 1, 2, 70, D, dtype)
    k, v = (heads(gen, 1, 2, Nk, D, dtype) for _ in range(2))
    m = make_mask(gen, "batch", 1, 2, 70, Nk)
    q[0, 1, 7, 3] = bad
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = cross_attention(*leaves, m)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    sparse_attn_cuda.device_status()
    assert out[0, 1, 7].isnan().all() and dq[0, 1, 7].isnan().all()
    kept = m[0, 0, 7]
    assert dk[0, 1][kept].isnan().all() and dv[0, 1][kept].isnan().all()
    others = torch.arange(70, device=DEV) != 7
    assert torch.isfinite(out[0, 1][others]).all() and torch.isfinite(out[0, 0]).all()
    assert all(torch.isfinite(t[0, 0]).all() for t in (dq, dk, dv))


@pytest.mark.parametrize("bias", [False, True])
def test_second_derivatives_of_a_mixed_loss_are_refused(bias):
    """A penalty on a gradient whose incoming gradient is a constant: it still
    depends on q, k, v and the table, and must not be dropped in silence."""
    gen = torch.Generator(device=DEV).manual_seed(63)
    leaves = [heads(gen, 1, 2, n, 64, F16).requires_grad_(True) for n in (20, 30, 30)]
    if bias:
        leaves.append(torch.randn(16, 2, generator=gen, device=DEV).half().requires_grad_(True))
    attend = relative_bias_attention if bias else cross_attention
    for leaf in leaves:
        out = attend(*leaves)
        g, = torch.autograd.grad(out.sum(), leaf, create_graph=True)
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="differentiated again"):
            (out.sum() + g.square().sum()).backward()
    # First derivatives under create_graph are as ever.
    out = attend(*leaves)
    plain = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
    kept = torch.autograd.grad(out.sum(), leaves, create_graph=True)
    for i, (a, b) in enumerate(zip(plain, kept)):
        if i:  # dq: FP32 adds in another order
            assert torch.equal(a, b.detach())


@pytest.mark.parametrize("Nq", [1, 40, 200])
@pytest.mark.parametrize("mask", ["padding", "heads", "shared"])
@pytest.mark.parametrize("bias", [False, True])
def test_no_keys_under_a_mask(bias, mask, Nq):
    """Zeros, as without a mask: with and without gradients."""
    gen = torch.Generator(device=DEV).manual_seed(64)
    q = heads(gen, 2, 4, Nq, 64, F16)
    k = torch.empty(2, 2, 0, 64, device=DEV, dtype=F16)
    table = torch.randn(16, 4, generator=gen, device=DEV).half()
    m = make_mask(gen, mask, 2, 4, Nq, 5)[..., :0]

    def run(*leaves):
        return relative_bias_attention(*leaves, m) if bias else cross_attention(*leaves, m)

    leaves = (q, k, k.clone(), table) if bias else (q, k, k.clone())
    assert torch.equal(run(*leaves), torch.zeros_like(q))
    leaves = [t.clone().requires_grad_(True) for t in leaves]
    out = run(*leaves)
    assert torch.equal(out.detach(), torch.zeros_like(q))
    for leaf, g in zip(leaves, torch.autograd.grad(out.sum(), leaves)):
        assert g.shape == leaf.shape and torch.all(g == 0)
    sparse_attn_cuda.device_status()


def coherent(dtype=F16):
    """A call whose dtable is large: all of a bucket's dS have one sign."""
    gen = torch.Generator(device=DEV).manual_seed(61)
    q, k = heads(gen, 4, 2, 300, 64, dtype), heads(gen, 4, 2, 300, 64, dtype)
    v = torch.where(torch.arange(300, device=DEV) < 150, 0.5, -0.5)[:, None].expand(4, 2, 300, 64).to(dtype).contiguous()
    dout = (500 + torch.randn(4, 2, 300, 64, generator=gen, device=DEV)).to(dtype)
    table = torch.randn(32, 2, generator=gen, device=DEV).to(dtype)
    return q, k, v, table, dout


def test_fp32_table_gets_an_fp32_gradient():
    """Not by way of the queries' type: beyond its range, and not rounded to it."""
    q, k, v, table, dout = coherent()
    leaf = table.float().requires_grad_(True)
    got, = torch.autograd.grad(relative_bias_attention(q, k, v, leaf), leaf, dout)
    assert got.dtype == torch.float32
    bucket = buckets_of(300, 300, 32, 128, True)
    ref = RefGrads(q, k, v, dout, None, table.double().cpu().t()[:, bucket], dtype=F16).with_table(bucket, 32)
    want = ref.grads["dtable"]
    assert float(want.abs().max()) > 2 * torch.finfo(F16).max
    ref.check(dtable=got)
    small = (dout.float() / 512).to(F16)
    got, = torch.autograd.grad(relative_bias_attention(q, k, v, leaf), leaf, small)
    half = table.clone().requires_grad_(True)
    rounded, = torch.autograd.grad(relative_bias_attention(q, k, v, half), half, small)
    assert rounded.dtype == F16 and torch.isfinite(rounded).all()
    assert torch.equal(got.half(), rounded) and not torch.equal(got, rounded.float())


@pytest.mark.parametrize("inputs", [F16, BF16, torch.float32])
@pytest.mark.parametrize("turned", [False, True])
def test_fp32_tables_of_every_input_type(inputs, turned):
    """Contiguous or a transposed view; the parameter's own gradient."""
    gen = torch.Generator(device=DEV).manual_seed(62)
    kernel = BF16 if inputs == torch.float32 else inputs
    q, k, v, dout = (heads(gen, 2, 4, n, 64, kernel) for n in (70, 133, 133, 70))
    table = torch.randn(16, 4, generator=gen, device=DEV)
    leaf = (table.t().contiguous() if turned else table.clone()).requires_grad_(True)
    x = [t.to(inputs) for t in (q, k, v)]
    out = relative_bias_attention(*x, leaf.t() if turned else leaf, query_offset=63)
    assert out.dtype == inputs
    out.backward(dout.to(inputs))
    assert leaf.grad.dtype == torch.float32 and leaf.grad.shape == leaf.shape
    bucket = buckets_of(70, 133, 16, 128, True, 63)
    add = table.to(kernel).double().cpu().t()[:, bucket]
    ref = RefGrads(q, k, v, dout, None, add, dtype=kernel).with_table(bucket, 16)
    ref.check(dtable=leaf.grad.t() if turned else leaf.grad)


@pytest.mark.parametrize("B,H,Hkv,Nq,Nk", [(2, 4, 2, 1, 300), (2, 4, 4, 64, 500), (2, 8, 2, 10, 700), (1, 4, 2, 200, 300)])
def test_expanded_masks_are_taken_as_broadcast(B, H, Hkv, Nq, Nk):
    """A padding mask expanded over heads and queries: the same kernel, so the
    same bits."""
    gen = torch.Generator(device=DEV).manual_seed(67)
    q = heads(gen, B, H, Nq, 64, F16)
    k, v = (heads(gen, B, Hkv, Nk, 64, F16) for _ in range(2))
    m = make_mask(gen, "padding", B, H, Nq, Nk)
    want = cross_attention(q, k, v, m)
    assert torch.equal(cross_attention(q, k, v, m.expand(B, H, Nq, Nk)), want)
    Ref(q, k, v, m).check_out(want)


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("kind", ["none", "padding", "heads", "bias"])
def test_more_keys_than_the_tiles_take(kind, D, dtype):
    """Past 65536 keys every forward streams them."""
    Nq, Nk = 33, 65536 + 77
    gen = torch.Generator(device=DEV).manual_seed(68)
    q = heads(gen, 1, 2, Nq, D, dtype)
    k, v = (heads(gen, 1, 1, Nk, D, dtype) for _ in range(2))
    m, add = make_mask(gen, "none" if kind == "bias" else kind, 1, 2, Nq, Nk), None
    if kind == "bias":
        table = torch.randn(32, 2, generator=gen, device=DEV).to(dtype)
        add = table.double().cpu().t()[:, buckets_of(Nq, Nk, 32, 128, True, 65500)]
        out = relative_bias_attention(q, k, v, table, query_offset=65500)
    else:
        out = cross_attention(q, k, v, m)
    sparse_attn_cuda.device_status()
    Ref(q, k, v, m, add).check_out(out)
    leaf = q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="65536"):
        cross_attention(leaf, k, v, m)


def test_fp32_table_in_a_captured_step():
    """Forward and backward in one graph, replayed on new values of the table."""
    q, k, v, table, dout = coherent(BF16)
    leaf = table.float().requires_grad_(True)

    def step():
        out = relative_bias_attention(q, k, v, leaf)
        return out.detach(), torch.autograd.grad(out, leaf, dout)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for shift in (0.5, -1.0):
        with torch.no_grad():
            leaf.add_(shift * torch.arange(32, device=DEV)[:, None] / 32)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
    assert got[1].dtype == torch.float32
    sparse_attn_cuda.device_status()
