"""Calls of cross_attention and relative_bias_attention at the edges of what
they take: bias tables with large entries.  Bounds as in
test_cross_backward_gpu.py."""

import pytest
import torch

from cross_ref import buckets_of
from python import relative_bias_attention, sparse_attn_cuda
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
