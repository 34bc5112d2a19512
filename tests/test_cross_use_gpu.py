"""The operators on queries and keys of different lengths as a program uses
them: an encoder-decoder training step and its generation, other streams,
threads, captured and replayed graphs, and caches whose offsets pass 32 bits."""

import threading

import pytest
import torch

from cross_ref import Ref, buckets_of
from python import (cross_attention, relative_bias_attention, shared_prefix_attention, sparse_attention,
                    sparse_attn_cuda)
from test_cross_attention_gpu import heads, make_mask, prefix_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def bias_add(table, Nq, Nk, two_sided, offset=0):
    return table.detach().double().cpu().t()[:, buckets_of(Nq, Nk, table.shape[0], 128, two_sided, offset)]


def test_training_step_then_generation():
    """An encoder (two-sided bias over a padded batch), a decoder (causal bias,
    then attention to the encoder's states with shared key heads), one
    backward through all of it, and generation: a token with its cache, and
    samples behind the shared prompt.  Every stage against its plain form on
    the same inputs, and the tokens against the full pass."""
    gen = torch.Generator(device=DEV).manual_seed(31)
    B, H, Hkv, Ns, Nt, D = 2, 4, 2, 150, 70, 64
    x = heads(gen, B, H, Ns, D, BF16).requires_grad_(True)
    y = heads(gen, B, H, Nt, D, BF16).requires_grad_(True)
    t_enc, t_dec = (torch.randn(32, H, generator=gen, device=DEV).bfloat16().requires_grad_(True) for _ in range(2))
    pad = (torch.arange(Ns, device=DEV)[None] < torch.tensor([Ns, 97], device=DEV)[:, None]).view(B, 1, 1, Ns)
    causal = torch.ones(Nt, Nt, dtype=torch.bool, device=DEV).tril().view(1, 1, Nt, Nt)
    enc = relative_bias_attention(x, x, x, t_enc, pad)
    Ref(x, x, x, pad, bias_add(t_enc, Ns, Ns, True)).check_out(enc.detach())
    dec = relative_bias_attention(y, y, y, t_dec, causal, bidirectional=False)
    Ref(y, y, y, causal, bias_add(t_dec, Nt, Nt, False)).check_out(dec.detach())
    keys, values = enc[:, :Hkv], enc[:, Hkv:]  # views of the encoder's states
    out = cross_attention(dec, keys, values, pad)
    Ref(dec, keys, values, pad).check_out(out.detach())
    loss = out.float().square().mean()
    loss.backward()
    for t in (x, y, t_enc, t_dec):
        assert t.grad is not None and torch.isfinite(t.grad).all() and float(t.grad.float().abs().max()) > 0
    # The same loss through the plain form in FP32 agrees along the gradients:
    # bf16 intermediates (enc, dec, out) are off by 2^-8 of their size each,
    # the gradient by as much per stage, three stages; 2^-5 covers them.
    xs = [t.detach().float().cpu().requires_grad_(True) for t in (x, y, t_enc, t_dec)]

    def plain(q, k, v, keep, add):
        s = q @ k.transpose(2, 3) / 8.0 + add
        return s.masked_fill(~keep, float("-inf")).softmax(-1) @ v

    def add(t, Nq, two):
        return t.t()[:, buckets_of(Nq, Nq, 32, 128, two)]

    e = plain(xs[0], xs[0], xs[0], pad.cpu(), add(xs[2], Ns, True))
    d = plain(xs[1], xs[1], xs[1], causal.cpu(), add(xs[3], Nt, False))
    G = H // Hkv
    o = plain(d, e[:, :Hkv].repeat_interleave(G, 1), e[:, Hkv:].repeat_interleave(G, 1), pad.cpu(), 0.0)
    o.square().mean().backward()
    for got, want in zip((x, y, t_enc, t_dec), xs):
        err = float((got.grad.float().cpu() - want.grad).norm() / want.grad.norm())
        assert err <= 2.0**-5, err
    with torch.no_grad():
        # The last decoder position again, as one token with its cache.
        one = relative_bias_attention(y[:, :, -1:], y, y, t_dec, bidirectional=False, query_offset=Nt - 1)
        assert (one - dec[:, :, -1:]).float().abs().max() <= 2.0**-7 * dec.float().abs().max()
        tok = cross_attention(dec[:, :, -1:], keys, values, pad)
        assert (tok - out[:, :, -1:]).float().abs().max() <= 2.0**-7 * out.float().abs().max()
        # Samples of one prompt: the first sequence's states as the prefix.
        kp, vp = keys[0].contiguous(), values[0].contiguous()
        k, v = heads(gen, B, Hkv, 40, D, BF16), heads(gen, B, Hkv, 40, D, BF16)
        lengths = torch.tensor([40, 13], dtype=torch.int32, device=DEV)
        got = shared_prefix_attention(dec[:, :, -3:], kp, vp, k, v, lengths)
        prefix_ref(dec[:, :, -3:], kp, vp, k, v, lengths).check_out(got)
    sparse_attn_cuda.device_status()


def test_square_masks_agree_with_sparse_attention():
    """On square inputs cross_attention is sparse_attention (both rounded once
    from FP32 sums taken in another order)."""
    gen = torch.Generator(device=DEV).manual_seed(32)
    for D, dtype in ((64, F16), (128, BF16)):
        q, k, v = (heads(gen, 2, 3, 200, D, dtype) for _ in range(3))
        m = make_mask(gen, "heads", 2, 3, 200, 200)
        a, b = sparse_attention(q, k, v, m), cross_attention(q, k, v, m)
        ref = Ref(q, k, v, m)
        ref.check_out(b)
        ref.check_out(a)


CALLS = {
    "rows": lambda t: cross_attention(t["q1"], t["k"], t["v"], t["pad"]),
    "rows_bias": lambda t: relative_bias_attention(t["q1"], t["k"], t["v"], t["table"], query_offset=1999),
    "tiles": lambda t: cross_attention(t["q"], t["k"], t["v"], t["mask"]),
    "tiles_split": lambda t: cross_attention(t["q"][:1, :2], t["k"][:1, :1], t["v"][:1, :1], t["mask"][:1, :2]),
    "tiles_bias": lambda t: relative_bias_attention(t["q"], t["k"], t["v"], t["table"], t["pad"], query_offset=500),
    "prefix_rows": lambda t: shared_prefix_attention(t["q1"], t["k"][0], t["v"][0], t["k"][:, :, :40], t["v"][:, :, :40],
                                                     t["lengths"]),
    "prefix_tiles": lambda t: shared_prefix_attention(t["q"], t["k"][0], t["v"][0], t["k"][:, :, :300],
                                                      t["v"][:, :, :300], t["lengths"]),
    "prefix_shared": lambda t: shared_prefix_attention(t["qs"], t["kl"], t["vl"], t["ks"], t["vs"], t["lengths_s"]),
}


def tensors(seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t = {"q": heads(gen, 2, 8, 300, 64, BF16), "q1": heads(gen, 2, 8, 1, 64, BF16),
         "k": heads(gen, 2, 4, 2000, 64, BF16), "v": heads(gen, 2, 4, 2000, 64, BF16)}
    t["table"] = torch.randn(32, 8, generator=gen, device=DEV).bfloat16()
    t["mask"] = torch.rand(2, 8, 300, 2000, generator=gen, device=DEV) < 0.4
    t["pad"] = (torch.arange(2000, device=DEV)[None] < torch.randint(1, 2001, (2, 1), generator=gen, device=DEV)).view(
        2, 1, 1, 2000)
    t["lengths"] = torch.randint(0, 300, (2,), generator=gen, device=DEV, dtype=torch.int32)
    t["qs"] = heads(gen, 64, 4, 1, 64, BF16)
    t["kl"], t["vl"] = (heads(gen, 1, 4, 9000, 64, BF16)[0] for _ in range(2))
    t["ks"], t["vs"] = (heads(gen, 64, 4, 50, 64, BF16) for _ in range(2))
    t["lengths_s"] = torch.randint(0, 51, (64,), generator=gen, device=DEV, dtype=torch.int32)
    return t


@pytest.mark.parametrize("name", CALLS)
def test_graph_capture_and_replay(name):
    """A captured call replayed on new inputs gives what an eager call gives."""
    t = tensors(41)
    CALLS[name](t)  # outside the capture: shared-memory limits, pools
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = CALLS[name](t)
    for seed in (42, 43):
        for x, y in zip(t.values(), tensors(seed).values()):
            x.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, CALLS[name](t))
    sparse_attn_cuda.device_status()


def test_two_graphs_and_an_eager_call_together():
    """Two captured graphs of one shape replayed at once on two streams, with an
    eager call on a third: their scratch is their own."""
    sets = [tensors(s) for s in (44, 45, 46)]
    for name in ("tiles_split", "rows", "prefix_shared"):
        call = CALLS[name]
        want = [call(t) for t in sets]
        torch.cuda.synchronize()
        graphs, outs = [], []
        for t in sets[:2]:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(call(t))
            graphs.append(g)
        streams = [torch.cuda.Stream() for _ in range(3)]
        for _ in range(10):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
            with torch.cuda.stream(streams[2]):
                eager = call(sets[2])
            torch.cuda.synchronize()
            assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


def test_captured_training_step():
    """Forward and backward in one graph (gradients by torch.autograd.grad)."""
    gen = torch.Generator(device=DEV).manual_seed(47)
    leaves = [heads(gen, 2, 4, n, 64, BF16).requires_grad_(True) for n in (200, 333, 333)]
    table = torch.randn(32, 4, generator=gen, device=DEV).bfloat16().requires_grad_(True)
    m = make_mask(gen, "batch", 2, 4, 200, 333)
    dout = heads(gen, 2, 4, 200, 64, BF16)

    def step():
        out = relative_bias_attention(*leaves, table, m, query_offset=133)
        return (out.detach(), *torch.autograd.grad(out, (*leaves, table), dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    with torch.no_grad():
        for x in (*leaves, table, dout):
            x.copy_(torch.randn(x.shape, generator=gen, device=DEV))
    g.replay()
    torch.cuda.synchronize()
    want = step()
    for i, (a, b) in enumerate(zip(got, want)):
        if i == 1:  # dq: FP32 adds in another order
            assert torch.allclose(a.float(), b.float(), rtol=2.0**-7, atol=1e-4)
        else:
            assert torch.equal(a, b)


def test_other_stream_and_threads():
    """Calls on a stream of their own and from threads whose first CUDA work
    they are."""
    t = tensors(48)
    want = {n: c(t) for n, c in CALLS.items()}
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = {n: c(t) for n, c in CALLS.items()}
    s.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in CALLS)
    results, errors = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                r = {n: c(t) for n, c in CALLS.items()}
                torch.cuda.current_stream().synchronize()
            results[i] = r
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    assert all(torch.equal(r[n], want[n]) for r in results.values() for n in CALLS)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes (2.2e9 elements each for K and V): the
    last sequence's result equals that of a call with it alone."""
    B, Hkv, Nk, D = 33, 8, 65536, 128
    gen = torch.Generator(device=DEV).manual_seed(49)
    k = torch.zeros(B, Hkv, Nk, D, dtype=BF16, device=DEV)
    v = torch.zeros(B, Hkv, Nk, D, dtype=BF16, device=DEV)
    assert k.numel() > 1 << 31
    k[-1].normal_(generator=gen)
    v[-1].normal_(generator=gen)
    for Nq in (1, 40):
        q = heads(gen, B, 8, Nq, D, BF16)
        out = cross_attention(q, k, v)
        one = cross_attention(q[-1:], k[-1:].clone(), v[-1:].clone())
        diff = (out[-1:] - one).float().abs().max()
        assert diff <= 2.0**-7 * one.float().abs().max(), (Nq, diff)
        assert torch.all(out[:-1] == 0)
    kp, vp = k.view(B * Hkv, Nk, D)[-8:], v.view(B * Hkv, Nk, D)[-8:]
    q = heads(gen, 3, 8, 2, D, BF16)
    out = shared_prefix_attention(q, kp, vp, k[:3, :, :5], v[:3, :, :5])
    one = shared_prefix_attention(q, kp.clone(), vp.clone(), k[:3, :, :5].clone(), v[:3, :, :5].clone())
    assert torch.equal(out, one)


def test_prefix_longer_than_one_launch():
    """A shared prefix past 65536 keys goes in stretches that are merged."""
    gen = torch.Generator(device=DEV).manual_seed(50)
    P = 65536 + 1000
    q = heads(gen, 40, 2, 1, 64, F16)
    kp, vp = (heads(gen, 1, 2, P, 64, F16)[0] for _ in range(2))
    k, v = (heads(gen, 40, 2, 7, 64, F16) for _ in range(2))
    prefix_ref(q, kp, vp, k, v, None).check_out(shared_prefix_attention(q, kp, vp, k, v))
    none = k[:, :, :0]
    prefix_ref(q, kp, vp, none, none, None).check_out(shared_prefix_attention(q, kp, vp, none, none))


def test_refused_calls_leave_the_device_usable():
    q, k = torch.randn(2, 2, 3, 64, device=DEV).half(), torch.randn(2, 2, 9, 64, device=DEV).half()
    t = torch.randn(32, 2, device=DEV).half()
    bad = [
        lambda: cross_attention(q, k[:1], k[:1]),
        lambda: cross_attention(q, k, k.bfloat16()),
        lambda: cross_attention(q, k[..., :32], k[..., :32]),
        lambda: cross_attention(q.double(), k.double(), k.double()),
        lambda: cross_attention(q[:, :1], k, k),
        lambda: cross_attention(q, k, k.cpu()),
        lambda: cross_attention(q, k, k, torch.ones(2, 2, 3, 8, dtype=torch.bool, device=DEV)),
        lambda: cross_attention(q, k, k, torch.ones(2, 2, 3, 9, device=DEV)),
        lambda: cross_attention(q, k, k, torch.ones(3, 9, dtype=torch.bool, device=DEV)),
        lambda: cross_attention(q, k, k, scale=0.0),
        lambda: cross_attention(q, k, k, scale=float("nan")),
        lambda: relative_bias_attention(q, k, k, t[:, :1]),
        lambda: relative_bias_attention(q, k, k, t.bfloat16()),
        lambda: relative_bias_attention(q, k, k, t[:31]),
        lambda: relative_bias_attention(q, k, k, t[:2]),
        lambda: relative_bias_attention(q, k, k, t, max_distance=8),
        lambda: relative_bias_attention(q, k, k, t, max_distance=1 << 20),
        lambda: relative_bias_attention(q, k, k, t, query_offset=1 << 30),
        lambda: relative_bias_attention(q, k, k, t, query_offset=torch.zeros(2, device=DEV)),
        lambda: relative_bias_attention(q, k, k, torch.zeros(600, 2, device=DEV).half()),
        lambda: shared_prefix_attention(q, k[0, :1], k[0, :1], k, k),
        lambda: shared_prefix_attention(q, k[0], k[0, :, :3], k, k),
        lambda: shared_prefix_attention(q, k[0], k[0], k, k, torch.ones(2, device=DEV)),
        lambda: shared_prefix_attention(q, k[0], k[0], k, k, torch.ones(3, dtype=torch.int32, device=DEV)),
        lambda: shared_prefix_attention(q.clone().requires_grad_(True), k[0], k[0], k, k),
    ]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
    Ref(q, k, k).check_out(cross_attention(q, k, k))
