"""The library's operators on queries and keys of different lengths, as they are measured:

  cross     cross_attention          queries over the states of another sequence (encoder states, a cache)
  bias      relative_bias_attention  masked attention with a learned bias by bucketed relative position
  prefix    shared_prefix_attention  a batch whose sequences share one long prefix

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, rounded once), or, where
``own`` is set, through the library's public entry points.  ``exact`` restates each operator in 64 bits.
"""

import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # One answer token over a short source: latency alone.
        dict(name="cross_token_small", op="cross", B=1, H=12, Hkv=12, Nq=1, Nk=128, D=64, dtype="fp16", mask="none",
             train=False, layout="bhnd"),
        # One token for each of 16 requests over long padded sources, key heads shared by four query heads.
        dict(name="cross_token_long", op="cross", B=16, H=32, Hkv=8, Nq=1, Nk=8192, D=128, dtype="bf16",
             mask="padding", train=False, layout="bhnd"),
        # A decoder's pass over padded encoder states of odd length, projections left as [B, N, H, D].
        dict(name="cross_forward_odd", op="cross", B=16, H=12, Hkv=12, Nq=448, Nk=1500, D=64, dtype="fp16",
             mask="padding", train=False, layout="bnhd"),
        # Training with a random mask of its own for every head, the headline workload's mask on another key length.
        dict(name="cross_train_sparse", op="cross", B=8, H=12, Hkv=12, Nq=512, Nk=1024, D=64, dtype="fp16",
             mask="bernoulli", train=True, layout="bhnd"),
        # Training with shared key heads and a block mask that all heads share.
        dict(name="cross_train_shared", op="cross", B=4, H=32, Hkv=8, Nq=1024, Nk=2048, D=128, dtype="bf16",
             mask="block", train=True, layout="bhnd"),
        # The headline workload (random mask per head) with a two-sided bias.
        dict(name="bias_forward", op="bias", B=16, H=12, Hkv=12, Nq=512, Nk=512, D=64, dtype="fp16",
             mask="bernoulli", train=False, layout="bhnd", buckets=32, distance=128, two_sided=True, offset=0),
        # A causal decoder's training step.
        dict(name="bias_train_causal", op="bias", B=4, H=16, Hkv=16, Nq=1024, Nk=1024, D=64, dtype="bf16",
             mask="causal", train=True, layout="bhnd", buckets=32, distance=128, two_sided=False, offset=0),
        # An encoder's training step on a padded batch of odd length.
        dict(name="bias_train_odd", op="bias", B=8, H=16, Hkv=16, Nq=777, Nk=777, D=128, dtype="bf16",
             mask="padding", train=True, layout="bhnd", buckets=32, distance=128, two_sided=True, offset=0),
        # One generated token for each of 32 sequences, the query standing behind 2048 cached keys.
        dict(name="bias_token", op="bias", B=32, H=16, Hkv=16, Nq=1, Nk=2049, D=64, dtype="bf16", mask="none",
             train=False, layout="bhnd", buckets=32, distance=128, two_sided=False, offset=2048),
        # A few samples of one short prompt: latency alone.
        dict(name="prefix_small", op="prefix", B=4, H=12, Hkv=12, T=1, P=512, S=33, D=64, dtype="fp16"),
        # 64 samples of one long prompt, one token each.
        dict(name="prefix_token_long", op="prefix", B=64, H=32, Hkv=8, T=1, P=16384, S=512, D=128, dtype="bf16"),
        # Several tokens at once (a drafted continuation, a short question) behind a shared document.
        dict(name="prefix_chunk", op="prefix", B=8, H=32, Hkv=8, T=64, P=4096, S=256, D=128, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_any(rng):
    op = rng.choice(("cross", "cross", "bias", "bias", "prefix"))
    D = rng.choice((64, 128))
    dtype = rng.choice(("fp16", "bf16"))
    Hkv = rng.choice((1, 2, 4, 8, 12))
    if op == "prefix":
        G = rng.choice((1, 1, 2, 3, 4, 8))
        T = rng.choice((1, 1, 1, _log_int(rng, 2, 64)))
        return dict(op=op, B=_log_int(rng, 2, 64), H=Hkv * G, Hkv=Hkv, T=T, P=_log_int(rng, 64, 16384),
                    S=T + _log_int(rng, 1, 512), D=D, dtype=dtype)
    train = rng.random() < 0.5
    token = not train and rng.random() < 0.4
    B = _log_int(rng, 1, 32)
    layout = rng.choice(("bhnd", "bnhd"))
    if op == "cross":
        G = rng.choice((1, 1, 2, 4))
        Nq = 1 if token else _log_int(rng, 16, 1024)
        Nk = _log_int(rng, 64, 8192) if token else _log_int(rng, 64, 2048)
        mask = rng.choice(("none", "padding")) if token else rng.choice(("none", "padding", "bernoulli", "block"))
        return dict(op=op, B=B, H=Hkv * G, Hkv=Hkv, Nq=Nq, Nk=Nk, D=D, dtype=dtype, mask=mask, train=train,
                    layout=layout)
    G = rng.choice((1, 1, 1, 4))
    Nk = _log_int(rng, 64, 4096) if token else _log_int(rng, 64, 1024)
    Nq = 1 if token else Nk
    two_sided = not token and rng.random() < 0.5
    mask = rng.choice(("none", "padding")) if token else rng.choice(("padding", "bernoulli") if two_sided else ("causal",))
    return dict(op=op, B=B, H=Hkv * G, Hkv=Hkv, Nq=Nq, Nk=Nk, D=D, dtype=dtype, mask=mask, train=train, layout=layout,
                buckets=rng.choice((16, 32, 64)), distance=rng.choice((64, 128, 256)), two_sided=two_sided,
                offset=Nk - 1 if token else 0)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw_any(rng)
        if _cost(c) <= most:
            return c


# ------------------------------------------------------------------ work

# Share of the (query, key) pairs that a mask leaves, where whole keys or blocks fall away.  A random mask leaves no
# block out, so all pairs of it are computed.
_SHARE = {"none": 1.0, "padding": 0.75, "causal": 0.5, "bernoulli": 1.0, "block": 0.3}


def _mask_bytes(c):
    B, H, Nq, Nk = c["B"], c["H"], c["Nq"], c["Nk"]
    return {"none": 0, "padding": B * Nk, "causal": Nq * Nk, "bernoulli": B * H * Nq * Nk, "block": B * Nq * Nk}[c["mask"]]


def work(case):
    c = case
    if c["op"] == "prefix":
        q = c["B"] * c["H"] * c["T"] * c["D"]
        kv = 2 * c["Hkv"] * c["D"] * (c["P"] + c["B"] * c["S"] // 2)
        pairs = c["B"] * c["H"] * c["T"] * (c["P"] + c["S"] / 2)
        return {"bytes": 2 * (2 * q + kv), "flops": 4.0 * pairs * c["D"]}
    q = c["B"] * c["H"] * c["Nq"] * c["D"]
    share = _SHARE[c["mask"]]
    kv = 2 * c["B"] * c["Hkv"] * c["Nk"] * c["D"] * (share if c["mask"] == "padding" else 1.0)
    pairs = c["B"] * c["H"] * c["Nq"] * c["Nk"] * share
    table = c.get("buckets", 0) * c["H"]
    if c["train"]:  # q, dout, out, dq; k, v, dk, dv
        return {"bytes": 2 * (4 * q + 2 * kv + 2 * table) + _mask_bytes(c), "flops": 14.0 * pairs * c["D"]}
    return {"bytes": 2 * (2 * q + kv + table) + _mask_bytes(c), "flops": 4.0 * pairs * c["D"]}


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


# ------------------------------------------------------------------ inputs


def _heads(gen, B, H, N, D, dtype, layout):
    """Projections [B, H, N, D], as laid out by a projection: either contiguous, or a view of [B, N, H, D]."""
    if layout == "bnhd":
        return torch.randn(B, N, H, D, generator=gen, device=DEVICE).to(dtype).transpose(1, 2)
    return torch.randn(B, H, N, D, generator=gen, device=DEVICE).to(dtype)


def _mask(gen, c):
    B, H, Nq, Nk, kind = c["B"], c["H"], c["Nq"], c["Nk"], c["mask"]
    if kind == "none":
        return None
    if kind == "padding":
        lengths = torch.randint(max(1, Nk // 2), Nk + 1, (B,), generator=gen, device=DEVICE)
        return (torch.arange(Nk, device=DEVICE)[None] < lengths[:, None]).view(B, 1, 1, Nk)
    if kind == "causal":
        return torch.ones(Nq, Nk, dtype=torch.bool, device=DEVICE).tril().view(1, 1, Nq, Nk)
    if kind == "bernoulli":
        return torch.rand(B, H, Nq, Nk, generator=gen, device=DEVICE) < 0.25
    alive = torch.rand(B, 1, -(-Nq // 64), -(-Nk // 64), generator=gen, device=DEVICE) < 0.3
    rows = torch.arange(alive.shape[2], device=DEVICE)
    alive[:, :, rows, rows * alive.shape[3] // alive.shape[2]] = True  # every block of queries keeps a block of keys
    alive = alive.repeat_interleave(64, 2).repeat_interleave(64, 3)[:, :, :Nq, :Nk]
    return alive & (torch.rand(B, 1, Nq, Nk, generator=gen, device=DEVICE) < 0.5)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))
    dtype = DTYPES[c["dtype"]]
    s = {"case": c}
    if c["op"] == "prefix":
        B, H, Hkv, T, P, S, D = (c[x] for x in ("B", "H", "Hkv", "T", "P", "S", "D"))
        s["q"] = _heads(gen, B, H, T, D, dtype, "bhnd")
        s["kp"], s["vp"] = (_heads(gen, 1, Hkv, P, D, dtype, "bhnd")[0] for _ in range(2))
        s["k"], s["v"] = (_heads(gen, B, Hkv, S, D, dtype, "bhnd") for _ in range(2))
        s["lengths"] = torch.randint(T, S + 1, (B,), generator=gen, device=DEVICE, dtype=torch.int32)
        return s
    s["q"] = _heads(gen, c["B"], c["H"], c["Nq"], c["D"], dtype, c["layout"])
    s["k"], s["v"] = (_heads(gen, c["B"], c["Hkv"], c["Nk"], c["D"], dtype, c["layout"]) for _ in range(2))
    s["mask"] = _mask(gen, c)
    if c["op"] == "bias":
        s["table"] = torch.randn(c["buckets"], c["H"], generator=gen, device=DEVICE).to(dtype)
    if c["train"]:
        s["dout"] = torch.randn(c["B"], c["H"], c["Nq"], c["D"], generator=gen, device=DEVICE).to(dtype)
        for x in ("q", "k", "v", "table"):
            if x in s:
                s[x].requires_grad_(True)
    return s


# ------------------------------------------------------------------ plain forms


def _starts(buckets, distance):
    """Smallest distance of every bucket of one side: one bucket for each of the first buckets // 2 distances, then
    buckets whose bounds grow geometrically up to `distance`; compared in whole numbers, so no bound is off by a
    rounding of the logarithm."""
    exact_n = buckets // 2
    rest = buckets - exact_n
    starts = list(range(exact_n))
    d = exact_n
    for j in range(rest):  # bucket exact_n + j starts where (d / exact_n) ** rest >= (distance / exact_n) ** j
        while d ** rest * exact_n ** j < distance ** j * exact_n ** rest:
            d += 1
        starts.append(d)
    return starts


def _buckets(c):
    """Bucket of every (query, key) pair's relative position, [Nq, Nk]."""
    rel = torch.arange(c["Nk"], device=DEVICE)[None] - (torch.arange(c["Nq"], device=DEVICE)[:, None] + c["offset"])
    side = c["buckets"] // 2 if c["two_sided"] else c["buckets"]
    starts = torch.tensor(_starts(side, c["distance"]), device=DEVICE)
    far = rel.abs() if c["two_sided"] else (-rel).clamp_min(0)
    bucket = torch.searchsorted(starts, far.contiguous(), right=True) - 1
    return bucket + (rel > 0) * side if c["two_sided"] else bucket


def _softmax(s, keep):
    """Softmax of the kept scores; a row that keeps nothing is 0."""
    if keep is not None:
        s = s.masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / total.masked_fill(total == 0, 1.0)


def _plain_attention(s):
    c = s["case"]
    B, H, Hkv, Nq, Nk, D = (c[x] for x in ("B", "H", "Hkv", "Nq", "Nk", "D"))
    scale = 1.0 / math.sqrt(D)
    rows = (H // Hkv) * Nq
    dtype = s["q"].dtype
    with torch.no_grad():
        q = s["q"].float().reshape(B, Hkv, rows, D)
        k, v = s["k"].float(), s["v"].float()
        scores = torch.matmul(q, k.transpose(2, 3)).view(B, H, Nq, Nk) * scale
        if c["op"] == "bias":
            bucket = _buckets(c)
            scores = scores + s["table"].float().t()[:, bucket]
        p = _softmax(scores, s["mask"])
        del scores
        out = torch.matmul(p.view(B, Hkv, rows, Nk), v)
        if not c["train"]:
            return out.view(B, H, Nq, D).to(dtype)
        dout = s["dout"].float().reshape(B, Hkv, rows, D)
        delta = (dout * out).sum(-1, keepdim=True)
        ds = torch.matmul(dout, v.transpose(2, 3)) - delta
        p = p.view(B, Hkv, rows, Nk)
        dv = torch.matmul(p.transpose(2, 3), dout)
        ds = ds.mul_(p)
        del p
        got = {"out": out.view(B, H, Nq, D).to(dtype), "dv": dv.to(dtype)}
        got["dq"] = (torch.matmul(ds, k) * scale).view(B, H, Nq, D).to(dtype)
        got["dk"] = (torch.matmul(ds.transpose(2, 3), q) * scale).to(dtype)
        if c["op"] == "bias":
            # Sums along the diagonals (all pairs of one relative position), then over each bucket's diagonals.
            by_pair = ds.view(B, H, Nq, Nk).sum(0).flip(1)
            skewed = torch.nn.functional.pad(by_pair, (0, Nq)).view(H, -1)[:, : Nq * (Nq + Nk - 1)]
            diagonals = skewed.reshape(H, Nq, Nq + Nk - 1).sum(1, dtype=torch.float64)
            of_diagonal = torch.cat([bucket[1:, 0].flip(0), bucket[0]])
            member = of_diagonal[:, None] == torch.arange(c["buckets"], device=DEVICE)
            got["dtable"] = torch.matmul(diagonals, member.double()).t().contiguous().to(dtype)
        return got


def _plain_prefix(s):
    c = s["case"]
    B, H, Hkv, T, P, S, D = (c[x] for x in ("B", "H", "Hkv", "T", "P", "S", "D"))
    G = H // Hkv
    scale = 1.0 / math.sqrt(D)
    q = s["q"].float().view(B, Hkv, G * T, D)
    shared = torch.matmul(q.transpose(0, 1).reshape(Hkv, B * G * T, D), s["kp"].float().transpose(1, 2))
    shared = shared.view(Hkv, B, G * T, P).transpose(0, 1)
    mine = torch.matmul(q, s["k"].float().transpose(2, 3))
    # The T queries are the last T of each sequence's own tokens; each sees its own keys up to itself.
    last = s["lengths"].long()[:, None] - T + 1 + torch.arange(T, device=DEVICE)
    keep = torch.arange(S, device=DEVICE) < last[:, :, None]
    mine = mine.view(B, H, T, S).masked_fill(~keep[:, None], -math.inf)
    p = _softmax(torch.cat([shared.reshape(B, H, T, P), mine], -1) * scale, None)
    pp = p[..., :P].reshape(B, Hkv, G * T, P).transpose(0, 1).reshape(Hkv, B * G * T, P)
    out = torch.matmul(pp, s["vp"].float()).view(Hkv, B, G * T, D).transpose(0, 1)
    out = out + torch.matmul(p[..., P:].reshape(B, Hkv, G * T, S), s["v"].float())
    return out.reshape(B, H, T, D).to(s["q"].dtype)


# ------------------------------------------------------------------ the library's calls


def _library():
    if "python" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "sparse-mask-attention-auto-research_b200"))
    import python

    return python


def _own_attention(s):
    lib, c = _library(), s["case"]
    if c["op"] == "bias":
        out = lib.relative_bias_attention(s["q"], s["k"], s["v"], s["table"], s["mask"], bidirectional=c["two_sided"],
                                          max_distance=c["distance"], query_offset=c["offset"])
    else:
        out = lib.cross_attention(s["q"], s["k"], s["v"], s["mask"])
    if not c["train"]:
        return out
    names = ("q", "k", "v", "table") if c["op"] == "bias" else ("q", "k", "v")
    grads = torch.autograd.grad(out, [s[x] for x in names], s["dout"])
    return {"out": out.detach(), **{"d" + x: g for x, g in zip(names, grads)}}


def run(state):
    if state["case"]["op"] == "prefix":
        if own:
            return _library().shared_prefix_attention(state["q"], state["kp"], state["vp"], state["k"], state["v"],
                                                      state["lengths"])
        return _plain_prefix(state)
    return _own_attention(state) if own else _plain_attention(state)


# ------------------------------------------------------------------ the definition in 64 bits


def _bucket_of(d, c):
    """Bucket of relative position d (key - query), from the definition, in whole numbers."""
    side, base = c["buckets"], 0
    if c["two_sided"]:
        side //= 2
        base = side if d > 0 else 0
        d = abs(d)
    else:
        d = max(-d, 0)
    small = side // 2
    if d < small:
        return base + d
    j = 0
    while j + 1 < side - small and d ** (side - small) * small ** (j + 1) >= c["distance"] ** (j + 1) * small ** (side - small):
        j += 1
    return base + small + j


def _exact_rows(q, k, v, add, keep):
    """Rows [R, D] over keys [N, D]; add and keep are [R, N] or None."""
    x = torch.einsum("rd,nd->rn", q, k) / math.sqrt(q.shape[-1])
    if add is not None:
        x = x + add
    if keep is not None:
        x = torch.where(keep, x, torch.full_like(x, -1e300))
    w = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
    if keep is not None:
        w = torch.where(keep, w, torch.zeros_like(w))
    return torch.einsum("rn,nd->rd", w, v)


def _exact_prefix(s):
    c = s["case"]
    B, H, Hkv, T, S = (c[x] for x in ("B", "H", "Hkv", "T", "S"))
    G = H // Hkv
    out = torch.empty(B, H, T, c["D"], dtype=torch.float64, device=DEVICE)
    lengths = s["lengths"].tolist()
    t = torch.arange(T, device=DEVICE).repeat(G)[:, None]
    for g in range(Hkv):
        kp, vp = s["kp"][g].double(), s["vp"][g].double()
        for b in range(B):
            n = lengths[b]
            keys, values = torch.cat([kp, s["k"][b, g, :n].double()]), torch.cat([vp, s["v"][b, g, :n].double()])
            keep = torch.arange(keys.shape[0], device=DEVICE)[None] <= c["P"] + n - T + t
            rows = s["q"][b, g * G : (g + 1) * G].double().reshape(G * T, -1)
            out[b, g * G : (g + 1) * G] = _exact_rows(rows, keys, values, None, keep).view(G, T, -1)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "prefix":
        return _exact_prefix(s)
    B, H, Hkv, Nq, Nk, D = (c[x] for x in ("B", "H", "Hkv", "Nq", "Nk", "D"))
    G = H // Hkv
    keep_all = None if s["mask"] is None else s["mask"].expand(B, H, Nq, Nk)
    bucket = None
    if c["op"] == "bias":
        by_distance = torch.tensor([_bucket_of(d, c) for d in range(-(Nq - 1) - c["offset"], Nk - c["offset"])],
                                   device=DEVICE)
        at = torch.arange(Nk, device=DEVICE)[None] - torch.arange(Nq, device=DEVICE)[:, None] + Nq - 1
        bucket = by_distance[at]
    leaves = {x: s[x].detach().double().contiguous() for x in ("q", "k", "v", "table") if x in s}
    out = torch.empty(B, H, Nq, D, dtype=torch.float64, device=DEVICE)
    grads = {x: torch.zeros_like(t) for x, t in leaves.items()}
    for b in range(B):
        for g in range(Hkv):
            heads = slice(g * G, (g + 1) * G)
            part = {"q": leaves["q"][b, heads], "k": leaves["k"][b, g], "v": leaves["v"][b, g]}
            if bucket is not None:
                part["table"] = leaves["table"][:, heads]
            part = {x: t.clone().requires_grad_(c["train"]) for x, t in part.items()}
            add = None if bucket is None else part["table"].t()[:, bucket].reshape(G * Nq, Nk)
            keep = None if keep_all is None else keep_all[b, heads].reshape(G * Nq, Nk)
            o = _exact_rows(part["q"].reshape(G * Nq, D), part["k"], part["v"], add, keep).view(G, Nq, D)
            out[b, heads] = o.detach()
            if c["train"]:
                got = torch.autograd.grad(o, list(part.values()), s["dout"][b, heads].double())
                for x, t in zip(part, got):
                    if x == "table":
                        grads[x][:, heads] += t
                    elif x == "q":
                        grads[x][b, heads] += t
                    else:
                        grads[x][b, g] += t
    if not c["train"]:
        return out
    return {"out": out, **{"d" + x: t for x, t in grads.items()}}
