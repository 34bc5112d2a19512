"""Plain 64-bit forms of the operators on queries and keys of different
lengths, and the bounds that their tests hold the kernels to.

Forward bound, per element of O = sum_j P_j v_j.  With u = eps / 2 of the
type, the kernels round every P_j to the type (off by at most u P_j; in fp16,
below 2^-14, by at most 2^-25 of the row's largest P instead) and divide by
the sum of the rounded values, so O moves by at most
u (sum_j P_j |v_j| + |O|) <= 2 u A with A = sum_j P_j |v_j|, plus
2^-25 sum_j |v_j| over the kept keys; the result is rounded once more,
u |O|.  Scores are FP32 sums of exact products: |s| 2^-20 covers their
rounding and that of the exponential (D <= 128 additions and the scaling),
which moves every P_j by that share.  A factor of 1.05 covers products of
these terms."""

import math

import torch


def starts_of(side, distance):
    """Bucket starts by the definition with exact fractions: the smallest d of
    bucket e + j has (d / e) ** n >= (distance / e) ** j."""
    from fractions import Fraction

    e = side // 2
    n = side - e
    out = list(range(e))
    for j in range(n):
        d = e
        while Fraction(d, e) ** n < Fraction(distance, e) ** j:
            d += 1
        out.append(d)
    return out


def buckets_of(Nq, Nk, num_buckets, distance, two_sided, offset=0):
    """Bucket of every (query, key) pair, [Nq, Nk]."""
    side = num_buckets // 2 if two_sided else num_buckets
    starts = torch.tensor(starts_of(side, distance))
    d = torch.arange(Nk)[None, :] - (torch.arange(Nq)[:, None] + offset)
    far = d.abs() if two_sided else (-d).clamp_min(0)
    bucket = (far[..., None] >= starts).sum(-1) - 1
    return bucket + side * (d > 0) if two_sided else bucket


class Ref:
    """Attention in 64 bits of q [B, H, Nq, D] over k, v [B, Hkv, Nk, D]:
    out, lse and A = P @ |v| (the scale of the rounding error)."""

    def __init__(self, q, k, v, keep=None, add=None, scale=None):
        B, H, Nq, D = q.shape
        G = H // k.shape[1]
        self.scale = 1.0 / math.sqrt(D) if scale is None else scale
        q, k, v = (t.detach().double().cpu() for t in (q, k, v))
        self.q, self.k, self.v = q, k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
        self.G = G
        Nk = k.shape[2]
        keep = torch.ones(B, H, Nq, Nk, dtype=torch.bool) if keep is None else keep.cpu().expand(B, H, Nq, Nk)
        # A key that no query keeps may hold anything.
        used = keep.any(2)[..., None]
        self.k, self.v = self.k.masked_fill(~used, 0.0), self.v.masked_fill(~used, 0.0)
        s = self.q @ self.k.transpose(2, 3) * self.scale
        if add is not None:
            s = s + add.double().cpu()
        self.s_max = s.masked_fill(~keep, 0.0).abs().amax(-1, keepdim=True) if Nk else torch.zeros(B, H, Nq, 1).double()
        s = s.masked_fill(~keep, -math.inf)
        self.lse = torch.logsumexp(s, -1) if Nk else torch.full((B, H, Nq), -math.inf).double()
        some = torch.isfinite(self.lse)[..., None]
        self.p = torch.where(some, torch.exp(s - torch.where(some, self.lse[..., None], 0.0)), 0.0)
        self.keep = keep
        self.out = self.p @ self.v
        self.A = self.p @ self.v.abs()
        self.V = keep.double() @ self.v.abs()

    def out_bound(self, dtype):
        u = torch.finfo(dtype).eps / 2
        tail = 2.0**-25 * self.V if dtype == torch.float16 else 0.0
        return 1.05 * (u * self.out.abs() + 2 * u * self.A + self.s_max * 2.0**-20 * 2 * self.A + tail) + 1e-7

    def check_out(self, out):
        err = (out.double().cpu() - self.out).abs()
        bound = self.out_bound(out.dtype)
        worst = float((err / bound).max()) if err.numel() else 0.0
        assert torch.isfinite(out).all(), "non-finite output"
        assert worst <= 1.0, f"out is off by {worst:.2f} of its bound (largest error {float(err.max()):.3e})"
        empty = ~self.keep.any(-1)
        assert torch.all(out.cpu()[empty] == 0), "rows that keep no key give 0"
