"""The autograd node of cross_attention and relative_bias_attention: which
gradients it returns, how often it can be run, hooks on what it saves, and the
errors it raises."""

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from python import _lib, cross_attention, relative_bias_attention, shared_prefix_attention, sparse_attn_cuda

pytestmark = pytest.mark.gpu


def case(seed=0, Nq=70, Nk=133, D=64, dtype=torch.float16):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn(2, 4, Nq, D, generator=gen, device="cuda").to(dtype)
    k, v = (torch.randn(2, 2, Nk, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    table = torch.randn(16, 4, generator=gen, device="cuda").to(dtype)
    mask = torch.rand(2, 1, Nq, Nk, generator=gen, device="cuda") < 0.5
    dout = torch.randn(2, 4, Nq, D, generator=gen, device="cuda").to(dtype)
    return q, k, v, table, mask, dout


def grads(wanted, run=relative_bias_attention):
    q, k, v, table, mask, dout = case()
    leaves = dict(q=q, k=k, v=v, table=table)
    for n in wanted:
        leaves[n].requires_grad_(True)
    out = run(q, k, v, table, mask)
    return dict(zip(wanted, torch.autograd.grad(out, [leaves[n] for n in wanted], dout)))


def same(a, b, exact):
    """dq is summed in FP32 in any order (a sum of at most 133 keys' products,
    2 ** -24 of their size each, before its rounding by half a step)."""
    if exact:
        return torch.equal(a, b)
    return torch.allclose(a.double(), b.double(), rtol=2 * torch.finfo(a.dtype).eps, atol=133 * 2.0**-24 * 16)


@pytest.mark.parametrize("wanted", [("q",), ("k",), ("v",), ("table",), ("q", "table"), ("k", "v")])
def test_each_gradient_alone(wanted):
    every, some = grads(("q", "k", "v", "table")), grads(wanted)
    for n in wanted:
        assert same(some[n], every[n], n != "q"), n


def test_nothing_is_built_without_gradients():
    q, k, v, table, mask, _ = case()
    assert not cross_attention(q, k, v, mask).requires_grad
    q.requires_grad_(True)
    with torch.no_grad():
        assert not cross_attention(q, k, v, mask).requires_grad
    out = cross_attention(q, k, v, mask)
    assert out.requires_grad and not out.is_leaf
    with pytest.raises(RuntimeError, match="forward only"):
        shared_prefix_attention(q, k[0], v[0], k, v)


def test_backward_once_unless_retained():
    q, k, v, table, mask, dout = case()
    v.requires_grad_(True)
    out = cross_attention(q, k, v, mask)
    first, = torch.autograd.grad(out, v, dout, retain_graph=True)
    second, = torch.autograd.grad(out, v, dout)
    assert torch.equal(first, second)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out, v, dout)


def test_second_derivatives_are_refused():
    q, k, v, table, mask, dout = case()
    k.requires_grad_(True)
    dout.requires_grad_(True)
    dk, = torch.autograd.grad(cross_attention(q, k, v, mask), k, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated again"):
        dk.sum().backward()


def test_forward_mode_is_refused():
    """Not dropped in silence, with or without inputs that require gradients."""
    q, k, v, table, mask, _ = case()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        for run in (lambda: cross_attention(dual, k, v, mask), lambda: relative_bias_attention(q, k, v, dual[0, :, :16, 0].t()),
                    lambda: shared_prefix_attention(dual, k[0], v[0], k, v)):
            with pytest.raises(RuntimeError):
                run()


def test_changed_inputs_are_noticed():
    q, k, v, table, mask, dout = case()
    q.requires_grad_(True)
    out = cross_attention(q, k, v, mask)
    k.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, q, dout)


@pytest.mark.parametrize("how", ["checkpoint", "on_cpu", "fp32"])
def test_saved_tensors_that_come_back_elsewhere(how):
    """Recomputed, or moved to the host and back: the same gradients."""
    names = ("q", "k", "v", "table")
    want = grads(names)

    def run(q, k, v, table, mask):
        if how == "checkpoint":
            return checkpoint(relative_bias_attention, q, k, v, table, mask, use_reentrant=False)
        if how == "on_cpu":
            with torch.autograd.graph.save_on_cpu():
                return relative_bias_attention(q, k, v, table, mask)
        # An FP32 table: its gradient is rounded to the queries' type on the way.
        return relative_bias_attention(q, k, v, table.float(), mask)

    got = grads(names, run)
    for n in names:
        assert same(got[n], want[n], n != "q"), n
    sparse_attn_cuda.device_status()


def test_strided_and_misaligned_incoming_gradients():
    q, k, v, table, mask, dout = case()
    v.requires_grad_(True)
    want, = torch.autograd.grad(cross_attention(q, k, v, mask), v, dout)
    turned = dout.transpose(1, 2).contiguous().transpose(1, 2)
    shifted = torch.empty(dout.numel() + 1, dtype=dout.dtype, device="cuda")[1:].view_as(dout).copy_(dout)
    for d in (turned, shifted):
        got, = torch.autograd.grad(cross_attention(q, k, v, mask), v, d)
        assert torch.equal(got, want)
    got, = torch.autograd.grad(cross_attention(q, k, v, mask).sum(), v)
    ones, = torch.autograd.grad(cross_attention(q, k, v, mask), v, torch.ones_like(dout))
    assert torch.equal(got, ones)


def test_views_with_odd_strides_of_single_rows():
    """Axes of length 1 may have any stride."""
    q, k, v, table, mask, _ = case()
    one = torch.empty_strided((1, 1, 1, 64), (7, 3, 5, 1), dtype=q.dtype, device="cuda").copy_(q[:1, :1, :1])
    keys = torch.empty_strided((1, 1, 133, 64), (11, 9, 64, 1), dtype=q.dtype, device="cuda").copy_(k[:1, :1])
    want = cross_attention(q[:1, :1, :1].contiguous(), k[:1, :1].contiguous(), k[:1, :1].contiguous())
    assert torch.equal(cross_attention(one, keys, keys), want)
    one.requires_grad_(True)
    assert torch.autograd.grad(cross_attention(one, keys, keys).sum(), one)[0].shape == one.shape


def test_errors_keep_their_types():
    q, k, v, table, mask, _ = case()
    with pytest.raises(RuntimeError, match="scale must be finite") as e:
        cross_attention(q, k, v, mask, scale=0.0)
    assert "Exception raised" not in str(e.value)
    with pytest.raises(_lib.SmaError) as e:  # finite, but 0 in FP32: refused by the library
        cross_attention(q, k, v, mask, scale=1e-60)
    assert e.value.code == _lib.SMA_ERR_ARG
    with pytest.raises(TypeError):
        cross_attention(q, k, v, mask, scale="large")
    B = 1 << 20  # a copy of the expanded queries would take 4 TB
    wide_k = k[:1, :1].expand(B, 2, -1, -1)
    with pytest.raises(torch.OutOfMemoryError):
        cross_attention(q[:1, :1, :1].expand(B, 2, 1 << 14, -1), wide_k, wide_k)
    sparse_attn_cuda.device_status()
    assert torch.isfinite(cross_attention(q, k, v, mask)).all()
