"""The decode operators around a key/value cache, as cases that can be timed and compared.

Three operators of the talker's decode path:

  shared    one decode step of a batch of requests whose caches continue one shared prefix: the prefix's
            keys and values are read once for all of them, each request's own rows once for it
  weighted  the same step that also adds every attended row's weight to the request's running total
  evict     a cache brought down to a budget of rows by those totals, the kept rows in their order

`run` computes them in elementary torch operations in 32 bits, or, with `own` set, through this package.
"""

import math
import random

import torch

own = False

# Talker sizes (28 layers, 16 query heads over 8 key/value heads of 128, prompts of 96 rows, caches of 1536
# rows, 16 decode slots) are this package's own serving configuration; the others are generic.
_LISTED = [
    # the serving default: 16 slots decoding behind one 96-row voice prompt, at ragged lengths
    dict(name="shared slots16 prompt96", op="shared", R=16, P=96, lo=1, hi=1404, M=1536, nq=16, nkv=8, hd=128,
         cache="bf16", io="f32", idle=0, gone=0, mix=1),
    # the smallest call: two talkers just started behind a short prompt, where latency counts
    dict(name="shared two short", op="shared", R=2, P=96, lo=0, hi=24, M=256, nq=16, nkv=8, hd=128,
         cache="bf16", io="f32", idle=0, gone=0, mix=2),
    # a full server: 64 requests behind a long conditioning prefix, a few slots idle
    dict(name="shared 64 prefix8192", op="shared", R=64, P=8192, lo=1, hi=1404, M=1536, nq=16, nkv=8, hd=128,
         cache="bf16", io="bf16", idle=3, gone=0, mix=3),
    # few requests, a very long prefix: the split over the long axis
    dict(name="shared 3 prefix40001", op="shared", R=3, P=40001, lo=100, hi=700, M=1024, nq=16, nkv=8, hd=128,
         cache="bf16", io="f32", idle=0, gone=0, mix=4),
    # more query rows than one tile holds, heads of 64, four query heads a group, odd sizes, 16-bit activations
    dict(name="shared 45 heads64 odd", op="shared", R=45, P=1001, lo=0, hi=333, M=391, nq=28, nkv=7, hd=64,
         cache="bf16", io="bf16", idle=1, gone=0, mix=5),
    # the 32-bit parity mode
    dict(name="shared f32 cache", op="shared", R=8, P=500, lo=1, hi=600, M=640, nq=16, nkv=8, hd=128,
         cache="f32", io="f32", idle=0, gone=0, mix=6),
    # one stream with its weights tracked, no prefix: every step of a bounded cache
    dict(name="weighted one stream", op="weighted", R=1, P=0, lo=1119, hi=1119, M=1536, nq=16, nkv=8, hd=128,
         cache="bf16", io="f32", idle=0, gone=0, mix=7),
    # 16 bounded streams behind a prompt whose caches have been evicted before (position past the rows held)
    dict(name="weighted slots16 bounded", op="weighted", R=16, P=96, lo=700, hi=1500, M=1536, nq=16, nkv=8, hd=128,
         cache="bf16", io="f32", idle=2, gone=2500, mix=8),
    # one layer of one stream: the smallest eviction
    dict(name="evict one layer", op="evict", N=1, R=1, lo=1536, hi=1536, M=1536, nkv=8, hd=128, cache="bf16",
         keep=1024, first=96, recent=256, mix=9),
    # every layer of one stream, as a bounded stream does each time its cache is full
    dict(name="evict 28 layers", op="evict", N=28, R=1, lo=1536, hi=1536, M=1536, nkv=8, hd=128, cache="bf16",
         keep=768, first=4, recent=128, mix=10),
    # every layer of four streams with longer caches at ragged lengths, one of them below its budget
    dict(name="evict 28 layers x4", op="evict", N=28, R=4, lo=1900, hi=4096, M=4096, nkv=8, hd=128, cache="bf16",
         keep=2000, first=96, recent=500, mix=11),
    # 32-bit caches, heads of 64, odd sizes
    dict(name="evict f32 odd", op="evict", N=5, R=3, lo=200, hi=1001, M=1001, nkv=3, hd=64, cache="f32",
         keep=333, first=1, recent=37, mix=12),
]

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}
_EPS, _THETA = 1e-6, 1e6


def listed():
    return [dict(c) for c in _LISTED]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: any operator, sizes over the ranges that the listed cases span."""
    op = rng.choice(["shared", "shared", "weighted", "evict"])
    mix = rng.randrange(1 << 20)
    cache = "f32" if rng.random() < 0.2 else "bf16"
    if op == "evict":
        big = _spread(rng, 64, 4096)
        keep = rng.randint(max(1, big // 4), max(1, big - 1))
        first = rng.randint(0, keep // 4)
        recent = rng.randint(0, (keep - first) // 2)
        nkv, hd = rng.choice([(8, 128), (8, 128), (4, 128), (3, 64)])
        return dict(op=op, N=_spread(rng, 1, 28), R=rng.randint(1, 4), lo=rng.randint(max(1, big // 3), big), hi=big,
                    M=big + rng.choice([0, 0, 1, 7, 64]), nkv=nkv, hd=hd, cache=cache, keep=keep, first=first,
                    recent=recent, mix=mix)
    nkv, g, hd = rng.choice([(8, 2, 128), (8, 2, 128), (8, 2, 128), (4, 8, 128), (7, 4, 64), (5, 3, 128), (8, 1, 64)])
    f32 = cache == "f32"
    R = _spread(rng, 1, 16 if f32 else 64)
    P = _spread(rng, 1, 1000 if f32 else 8192) if op == "shared" or rng.random() < 0.5 else 0
    hi = _spread(rng, 1, 600 if f32 else 1404)
    return dict(op=op, R=R, P=P, lo=rng.randint(0, hi), hi=hi, M=hi + rng.randint(1, 200), nq=nkv * g, nkv=nkv, hd=hd,
                cache=cache, io="f32" if f32 or rng.random() < 0.6 else "bf16", idle=rng.randint(0, R // 4),
                gone=rng.choice([0, 0, 1000]) if op == "weighted" else 0, mix=mix)


def _lens(case):
    """Rows that each request's cache holds before the call; -1: an idle slot."""
    r = random.Random(case["mix"])
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["R"])]
    if case["R"] > 1:
        lens[0] = case["hi"]
    for i in r.sample(range(case["R"]), case.get("idle", 0)):
        lens[i] = -1
    return lens


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _TYPES[case["cache"]]
    normal = lambda *shape: torch.randn(shape, device=dev, generator=g)  # noqa: E731
    R, M, nkv, hd = case["R"], case["M"], case["nkv"], case["hd"]
    lens = _lens(case)
    s = {"case": case, "lens": lens, "rows": torch.tensor(lens, device=dev, dtype=torch.int64)}

    def keys(*shape):  # keys arrive normalised, one unit of power per element
        x = normal(*shape)
        return (x * torch.rsqrt((x * x).mean(-1, keepdim=True))).to(dt)

    if case["op"] == "evict":
        shape = (case["N"], R, nkv, M, hd)
        s["K"], s["V"] = torch.empty(shape, device=dev, dtype=dt), torch.empty(shape, device=dev, dtype=dt)
        for n in range(case["N"]):
            s["K"][n], s["V"][n] = keys(*shape[1:]), normal(*shape[1:]).to(dt)
        # totals of attention weight: a few rows hold most of it; a row's total also grows with its age
        s["mass"] = torch.exp(1.5 * normal(*shape[:4])) * torch.linspace(2, 0.1, M, device=dev)
        s["to"] = (torch.zeros(shape, device=dev, dtype=dt), torch.zeros(shape, device=dev, dtype=dt),
                   torch.zeros(shape[:4], device=dev), torch.zeros_like(s["rows"]))
        if own:
            from sokutou_b200 import ops
            s["plan"] = ops.cache_evict_plan(s["K"], s["V"], s["mass"], s["rows"], case["keep"], case["first"],
                                             case["recent"], out=s["to"])
        return s
    nq, P = case["nq"], case["P"]
    io = _TYPES[case["io"]]
    n_pos = P + M + case["gone"]
    inv = _THETA ** (-torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd)
    ang = torch.arange(n_pos, device=dev, dtype=torch.float64)[:, None] * inv
    s["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float()
    s["pos"] = torch.where(s["rows"] < 0, -1, s["rows"] + P + case["gone"])
    s["rows"] = s["rows"].clamp(min=0)
    s["Kp"], s["Vp"] = keys(nkv, P, hd), normal(nkv, P, hd).to(dt)
    s["K"], s["V"] = keys(R, nkv, M, hd), normal(R, nkv, M, hd).to(dt)
    s["qkv"] = normal(R, (nq + 2 * nkv) * hd).to(io)
    s["qn"], s["kn"] = 1 + 0.02 * normal(hd), 1 + 0.02 * normal(hd)
    s["out"] = torch.zeros(R, nq * hd, device=dev, dtype=io)
    s["mass"] = normal(R, nkv, M).abs() if case["op"] == "weighted" else None
    if own:
        from sokutou_b200 import ops
        s["plan"] = ops.shared_decode_plan(s["K"], s["V"], s["pos"], s["rope"], nq, _EPS, rows=s["rows"],
                                           Kp=s["Kp"], Vp=s["Vp"], mass=s["mass"], qkv_dtype=io, out_dtype=io)
    return s


def _head_norm(x, w):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_decode(s):
    c = s["case"]
    R, P, M, nq, nkv, hd = c["R"], c["P"], c["M"], c["nq"], c["nkv"], c["hd"]
    g = nq // nkv
    live = s["pos"] >= 0
    q, k, v = s["qkv"].float().view(R, nq + 2 * nkv, hd).split([nq, nkv, nkv], 1)
    cos, sin = s["rope"][s["pos"].clamp(min=0)].unsqueeze(1).chunk(2, -1)
    q = _rotate(_head_norm(q, s["qn"]), cos, sin) / math.sqrt(hd)
    k = _rotate(_head_norm(k, s["kn"]), cos, sin)
    at, who = s["rows"], torch.arange(R, device=q.device)  # the new row, then read back as the cache holds it
    keep = live[:, None, None]
    s["K"][who, :, at] = torch.where(keep, k.to(s["K"].dtype), s["K"][who, :, at])
    s["V"][who, :, at] = torch.where(keep, v.to(s["V"].dtype), s["V"][who, :, at])
    q = q.view(R, nkv, g, hd)
    over_prefix = torch.matmul(q.transpose(0, 1).reshape(nkv, R * g, hd), s["Kp"].float().transpose(1, 2))
    over_prefix = over_prefix.view(nkv, R, g, P).transpose(0, 1)
    over_own = torch.matmul(q, s["K"].float().transpose(2, 3))
    seen = torch.arange(M, device=q.device) <= at[:, None]
    over_own = over_own.masked_fill(~seen[:, None, None], -math.inf)
    m = over_own.amax(-1, keepdim=True)
    if P:
        m = torch.maximum(m, over_prefix.amax(-1, keepdim=True))
    ep, eo = torch.exp(over_prefix - m), torch.exp(over_own - m)
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    from_prefix = torch.matmul(ep.transpose(0, 1).reshape(nkv, R * g, P), s["Vp"].float())
    from_prefix = from_prefix.view(nkv, R, g, hd).transpose(0, 1)
    o = (from_prefix + torch.matmul(eo, s["V"].float())) / total
    s["out"].copy_(torch.where(live[:, None], o.reshape(R, nq * hd).to(s["out"].dtype), s["out"]))
    if s["mass"] is not None:
        w = (eo / total).sum(2)
        new = torch.arange(M, device=q.device) == at[:, None]
        grown = torch.where(new[:, None], w, s["mass"] + w)
        s["mass"].copy_(torch.where(keep, grown, s["mass"]))


def _plain_evict(s):
    c = s["case"]
    N, R, nkv, M, hd = s["K"].shape
    keep = c["keep"]
    j = torch.arange(M, device=s["K"].device)
    n = s["rows"][:, None]
    held = (j < n)[:, None]  # (R, 1, M)
    always = ((j < c["first"]) | (j >= n - c["recent"]))[:, None] & held
    key = torch.where(always, math.inf, torch.where(held, s["mass"], -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    order = torch.where(torch.arange(keep, device=j.device) < n[:, None], order, M)  # short caches keep what they hold
    order = torch.sort(order, dim=-1).values
    kept = order < M
    src = order.clamp(max=M - 1)
    Kt, Vt, mt, rt = s["to"]
    at = src.unsqueeze(-1).expand(N, R, nkv, keep, hd)
    for_rows = kept.unsqueeze(-1)
    Kt[..., :keep, :] = torch.where(for_rows, torch.gather(s["K"], 3, at), Kt[..., :keep, :])
    Vt[..., :keep, :] = torch.where(for_rows, torch.gather(s["V"], 3, at), Vt[..., :keep, :])
    mt[..., :keep] = torch.where(kept, torch.gather(s["mass"], 3, src), mt[..., :keep])
    rt.copy_(s["rows"].clamp(max=keep))


def run(s):
    c = s["case"]
    if c["op"] == "evict":
        if own:
            from sokutou_b200 import ops
            ops.cache_evict(s["plan"])
        else:
            _plain_evict(s)
        Kt, Vt, mt, rt = s["to"]
        return {"K": Kt, "V": Vt, "mass": mt, "rows": rt}
    if own:
        from sokutou_b200 import ops
        ops.decode_attention_shared(s["plan"], s["qkv"], s["qn"], s["kn"], out=s["out"])
    else:
        _plain_decode(s)
    got = {"out": s["out"], "K": s["K"], "V": s["V"]}
    if s["mass"] is not None:
        got["mass"] = s["mass"]
    return got


def work(case):
    b, hd, nkv, lens = _BYTES[case["cache"]], case["hd"], case["nkv"], _lens(case)
    if case["op"] == "evict":
        kept = sum(min(n, case["keep"]) for n in lens)
        heads = case["N"] * nkv
        # every total read once, each kept row read and written
        return {"bytes": heads * (4 * sum(lens) + kept * 2 * (2 * hd * b + 4)), "flops": heads * sum(lens)}
    io, g = _BYTES[case["io"]], case["nq"] // nkv
    live = [n for n in lens if n >= 0]
    rows = case["P"] + sum(live)  # the prefix once for all
    per = (case["nq"] + 2 * nkv) * hd * io + case["nq"] * hd * io + 2 * nkv * hd * b
    size = 2 * nkv * rows * hd * b + len(live) * per
    if case["op"] == "weighted":
        size += 8 * nkv * sum(live)
    return {"bytes": size, "flops": 4 * nkv * g * hd * (len(live) * (case["P"] + 1) + sum(live))}


def exact(case, seed):
    """The definitions in 64 bits, one request or one cache after another."""
    s = prepare(case, seed)
    K, V, mass = s["K"].double(), s["V"].double(), None if s["mass"] is None else s["mass"].double()
    if case["op"] == "evict":
        Kt, Vt, mt, rt = (t.clone() for t in s["to"])
        Kt, Vt, mt = Kt.double(), Vt.double(), mt.double()
        for r, n in enumerate(s["lens"]):
            n_kept = min(n, case["keep"])
            rt[r] = n_kept
            a, z = case["first"], n - case["recent"]
            if n <= case["keep"]:
                Kt[:, r, :, :n], Vt[:, r, :, :n], mt[:, r, :, :n] = K[:, r, :, :n], V[:, r, :, :n], mass[:, r, :, :n]
                continue
            middle = mass[:, r, :, a:z]  # distinct with near certainty; the lowest index first where not
            best = torch.argsort(-middle, dim=-1, stable=True)[..., :n_kept - a - case["recent"]] + a
            ends = torch.cat([torch.arange(a), torch.arange(z, n)]).to(best.device).expand(*best.shape[:2], -1)
            rows = torch.cat([best, ends], -1).sort(-1).values
            for i in range(case["N"]):
                for h in range(case["nkv"]):
                    Kt[i, r, h, :n_kept], Vt[i, r, h, :n_kept] = K[i, r, h, rows[i, h]], V[i, r, h, rows[i, h]]
                    mt[i, r, h, :n_kept] = mass[i, r, h, rows[i, h]]
        return {"K": Kt, "V": Vt, "mass": mt, "rows": rt}
    P, nq, nkv, hd = case["P"], case["nq"], case["nkv"], case["hd"]
    g = nq // nkv
    out = s["out"].double()
    dt = s["K"].dtype
    w_q, w_k = s["qn"].double(), s["kn"].double()
    for r, n in enumerate(s["lens"]):
        if n < 0:
            continue
        x = s["qkv"][r].double().view(nq + 2 * nkv, hd)
        x[:nq] = x[:nq] / (x[:nq].pow(2).mean(1, keepdim=True) + _EPS).sqrt() * w_q
        x[nq:nq + nkv] = x[nq:nq + nkv] / (x[nq:nq + nkv].pow(2).mean(1, keepdim=True) + _EPS).sqrt() * w_k
        turn = s["rope"][P + n + case["gone"]].double()
        z = torch.view_as_complex(torch.stack([x[:nq + nkv, :hd // 2], x[:nq + nkv, hd // 2:]], -1).contiguous())
        z = z * torch.complex(turn[:hd // 2], turn[hd // 2:])
        x[:nq + nkv] = torch.cat([z.real, z.imag], -1)
        K[r, :, n], V[r, :, n] = x[nq:nq + nkv].to(dt).double(), x[nq + nkv:].to(dt).double()
        for h in range(nkv):
            kk = torch.cat([s["Kp"][h].double(), K[r, h, :n + 1]])
            vv = torch.cat([s["Vp"][h].double(), V[r, h, :n + 1]])
            p = torch.softmax(x[h * g:(h + 1) * g] @ kk.T * hd ** -0.5, -1)
            out[r].view(nq, hd)[h * g:(h + 1) * g] = p @ vv
            if mass is not None:
                grown = p[:, P:].sum(0)
                mass[r, h, :n] += grown[:n]
                mass[r, h, n] = grown[n]
    got = {"out": out, "K": K, "V": V}
    if mass is not None:
        got["mass"] = mass
    return got
