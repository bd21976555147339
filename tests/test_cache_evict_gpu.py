"""sk_cache_evict (ops.cache_evict): the kept rows, their order and every byte against a plain restatement —
nothing is computed, so everything has to be equal, rows past the kept ones and NaN payloads included. And the
bounded stream as a whole: weighted decode steps with evictions between them, against float64."""

import math

import numpy as np
import pytest
import torch

from conftest import rel_l2
from sokutou_b200 import ops

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def bits(t):
    t = t.detach().contiguous()
    return t.view({2: torch.int16, 4: torch.int32, 8: torch.int64}[t.element_size()]).cpu().numpy()


def kept_rows(mass, n, keep, first, recent):
    if n <= keep:
        return np.arange(max(n, 0))
    mid = np.arange(first, n - recent)
    x = mass[mid].astype(np.float64)
    x[np.isnan(x)] = -np.inf
    below = np.isnan(mass[mid])  # a NaN ranks below -inf
    best = mid[np.lexsort((mid, below, -x))][:keep - first - recent]
    return np.sort(np.concatenate([np.arange(first), best, np.arange(n - recent, n)])).astype(int)


def make(dev, N, lens, nkv, M, hd, dt, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    R = len(lens)
    K, V = (torch.randn(N, R, nkv, M, hd, generator=g).to(dt) for _ in range(2))
    K[..., ::7, 3] = math.nan  # payloads are moved, not looked at
    mass = torch.rand(N, R, nkv, M, generator=g)
    if kind == "ties":
        mass = (mass * 4).floor()
    elif kind == "one value":
        mass.fill_(0.25)
    elif kind == "special":
        pick = torch.randint(0, 8, mass.shape, generator=g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, 1e-42, -1.0)):
            mass[pick == i] = x
    elif kind == "close":  # neighbours in the last bits
        mass = torch.nextafter(torch.ones_like(mass), mass * 9) + torch.randint(0, 5, mass.shape, generator=g) * 2.0 ** -23
    elif kind == "spread":
        mass = torch.exp(20 * torch.randn(mass.shape, generator=g))
    rows = torch.tensor(lens, dtype=torch.int64)
    return [t.to(dev) for t in (K, V, mass, rows)]


def check(src, dst, was, keep, first, recent):
    """src: K, V, mass, rows before the call; was: the destination before it; dst: after it."""
    K, V, mass, rows = src
    m, lens = mass.cpu().numpy(), rows.cpu().numpy()
    want = [bits(t).copy() for t in was]
    from_ = [bits(t) for t in src]
    for r, n in enumerate(lens):
        if n < 0:
            want[3][r] = n
            continue
        want[3][r] = min(n, keep)
        for i in range(K.shape[0]):
            for h in range(K.shape[2]):
                at = kept_rows(m[i, r, h], int(n), keep, first, recent)
                for x in range(3):
                    want[x][i, r, h, :len(at)] = from_[x][i, r, h, at]
    for w, t in zip(want, dst):
        assert np.array_equal(w, bits(t))
    assert ops.device_error() == 0


CASES = {
    "plain": dict(N=2, lens=[100, 77, 60], nkv=3, M=100, keep=60, first=4, recent=16),
    "one row more than the budget": dict(N=1, lens=[65, 64], nkv=2, M=65, keep=64, first=0, recent=0),
    "keep one": dict(N=1, lens=[2, 1, 300], nkv=2, M=300, keep=1, first=0, recent=0),
    "only the ends": dict(N=2, lens=[500, 40], nkv=2, M=512, keep=40, first=8, recent=32),
    "only the recent": dict(N=1, lens=[500], nkv=2, M=512, keep=40, first=0, recent=40),
    "only the first": dict(N=1, lens=[500], nkv=2, M=512, keep=40, first=40, recent=0),
    "idle and empty": dict(N=2, lens=[-1, 0, 333, -5], nkv=2, M=333, keep=100, first=1, recent=1),
    "more than a pass of every kind": dict(N=1, lens=[5000, 4097], nkv=2, M=5003, keep=3001, first=96, recent=256),
    "long": dict(N=1, lens=[40000], nkv=1, M=40000, keep=20001, first=3, recent=1001),
    "almost all kept": dict(N=1, lens=[2000], nkv=2, M=2000, keep=1999, first=96, recent=256),
    "keep all but the buffer": dict(N=1, lens=[700, 701], nkv=2, M=701, keep=700, first=0, recent=5),
    "many heads": dict(N=28, lens=[90] * 4, nkv=8, M=96, keep=64, first=4, recent=8),
}
KINDS = ["random", "ties", "one value", "special", "close", "spread"]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", CASES)
def test_evict(cuda, case, kind, in_place):
    c = dict(CASES[case])
    keep, first, recent = c.pop("keep"), c.pop("first"), c.pop("recent")
    dt, hd = (BF, 128) if len(case) % 2 else (F32, 64)
    src = make(cuda, hd=hd, dt=dt, kind=kind, seed=len(case), **c)
    keepsake = [t.clone() for t in src]
    if in_place:
        got = ops.cache_evict(ops.cache_evict_plan(*src, keep, first, recent))
        assert got[0] is src[0] and got[3] is src[3]
        check(keepsake, src, keepsake, keep, first, recent)
        return
    g = torch.Generator(device=cuda).manual_seed(1)
    shape = list(src[0].shape)
    shape[3] = keep + 3
    dst = [torch.randn(shape, device=cuda, generator=g).to(dt) for _ in range(2)]
    dst += [torch.rand(shape[:4], device=cuda, generator=g), torch.full_like(src[3], 99)]
    was = [t.clone() for t in dst]
    ops.cache_evict(ops.cache_evict_plan(*src, keep, first, recent, out=tuple(dst)))
    check(keepsake, dst, was, keep, first, recent)
    for a, b in zip(src, keepsake):  # the source is only read
        assert np.array_equal(bits(a), bits(b))


@pytest.mark.parametrize("hd,dt", [(64, BF), (128, BF), (64, F32), (128, F32)])
@pytest.mark.parametrize("in_place", [False, True])
def test_layouts(cuda, hd, dt, in_place):
    """Four-dimensional caches, slices of wider ones, rows of all heads side by side; rows shared with the source."""
    K, V, mass, rows = make(cuda, 3, [200, 150], 4, 210, hd, dt, "ties", seed=hd)
    wide = [torch.zeros(3, 2, 210, 5, hd, dtype=dt, device=cuda)[:, :, :, 1:].transpose(2, 3) for _ in range(2)]
    for w, t in zip(wide, (K, V)):
        w.copy_(t)
    m = torch.zeros(2, 4, 3, 230, device=cuda)[..., 10:220].permute(2, 0, 1, 3)
    m.copy_(mass)
    for layers in (slice(None), 1):
        src = [wide[0][layers], wide[1][layers], m[layers], rows.clone()]
        five = [t if t.dim() == d else t.unsqueeze(0) for t, d in zip(src, (5, 5, 4, 1))]
        before = [t.clone() for t in five]
        if in_place:
            ops.cache_evict(ops.cache_evict_plan(*src, 70, 5, 9))
            check(before, five, before, 70, 5, 9)
            for w, t in zip(wide, (K, V)):
                w.copy_(t)
            m.copy_(mass)
        else:
            dst = [torch.zeros_like(before[0]), torch.zeros_like(before[1]), torch.zeros_like(before[2])]
            was = [t.clone() for t in dst] + [before[3]]
            ops.cache_evict(ops.cache_evict_plan(*src, 70, 5, 9, out=(*dst, src[3])))
            check(before, [*dst, src[3]], was, 70, 5, 9)


def test_more_rows_than_the_cache(cuda):
    src = make(cuda, 1, [100, 300, 90], 2, 100, 64, BF, "random")
    before = [t.clone() for t in src]
    ops.cache_evict(ops.cache_evict_plan(*src, 50, 0, 0))
    assert ops.device_error() == 1
    assert src[3].tolist() == [50, 300, 50]
    assert np.array_equal(bits(src[0][:, 1]), bits(before[0][:, 1]))


def test_offsets_past_32_bits(cuda):
    M, stride = 70, (1 << 31) // 60 // 8 * 8
    big = [torch.zeros(M * stride, dtype=BF, device=cuda).as_strided((1, 1, 1, M, 128), (8, 8, 8, stride, 1))
           for _ in range(2)]
    K, V, mass, rows = make(cuda, 1, [70], 1, M, 128, BF, "random")
    for b, t in zip(big, (K, V)):
        b.copy_(t)
    before = [K, V, mass.clone(), rows.clone()]
    ops.cache_evict(ops.cache_evict_plan(*big, mass, rows, 66, 1, 1))
    check(before, [*big, mass, rows], before, 66, 1, 1)


def test_graph_replay_and_two_streams(cuda):
    sets = [make(cuda, 4, [900, 300, 511], 8, 900, 128, BF, "random", seed=s) for s in (1, 2)]
    before = [[t.clone() for t in s] for s in sets]
    plans = [ops.cache_evict_plan(*s, 400, 16, 64) for s in sets]
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        ops.cache_evict(plans[0])
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        for s, b in zip(sets, before):
            for t, o in zip(s, b):
                t.copy_(o)
        torch.cuda.synchronize()
        gr.replay()
        with torch.cuda.stream(other):
            ops.cache_evict(plans[1])
        torch.cuda.synchronize()
        for s, b in zip(sets, before):
            check(b, s, b, 400, 16, 64)
    del gr


def test_refusals(cuda):
    K, V, mass, rows = make(cuda, 2, [50, 50], 2, 50, 64, BF, "random")
    ok = dict(K=K, V=V, mass=mass, rows=rows, keep=20)
    short = (K[..., :10, :].clone(), V[..., :10, :].clone(), mass[..., :10].clone(), rows.clone())
    for kw in (dict(keep=0), dict(keep=51), dict(first=11, recent=10), dict(first=-1), dict(recent=-1), dict(V=V.float()),
               dict(mass=mass.double()), dict(mass=mass[..., :9]), dict(rows=rows.int()), dict(rows=rows[:1]), dict(out=short),
               dict(K=K.cpu(), V=V.cpu()), dict(K=K[..., :32], V=V[..., :32]), dict(K=K.half(), V=V.half())):
        with pytest.raises((ValueError, TypeError)):
            ops.cache_evict_plan(**(ok | kw))
    p = ops.cache_evict_plan(**ok, workspace=torch.empty(16, dtype=torch.uint8, device=cuda))
    with pytest.raises(ops._lib.SokutouError):
        ops.cache_evict(p)
    # in place for one buffer and not for another, or over itself at other strides
    for out in ((K, V.clone(), mass.clone(), rows), (K[:, :, :, 1:], V[:, :, :, 1:], mass[..., 1:], rows),):
        p = ops.cache_evict_plan(K, V, mass, rows, 20, out=out)
        with pytest.raises(ops._lib.SokutouError):
            ops.cache_evict(p)
    assert ops.device_error() == 0


@pytest.mark.parametrize("cdt", [BF, F32])
def test_bounded_streams_against_float64(cuda, cdt):
    """The operators as they are used together: talkers behind a shared prompt (taken once by the single-request
    kernels), decoding with their weights kept, evicted whenever their caches are full. Every output against a
    float64 restatement that attends the rows kept; the choice of rows is checked to follow from the masses.
    fp32 activations: relative L2 1e-5 (as the step's own tests); after an eviction both sides go on from the
    same rows, so errors do not build up but through the caches' own rounding."""
    from sokutou_b200.qwen3 import TalkerAttention, TalkerGroup

    L, R, nq, nkv, hd, P, M, steps = 2, 3, 4, 2, 128, 40, 96, 150
    dev = cuda
    g = torch.Generator(device=dev).manual_seed(4)
    ta = TalkerAttention(L, nq, nkv, P + 8, 1e6, 1e-6, dev, cdt)
    w = [1 + 0.02 * torch.randn(2, hd, device=dev, generator=g) for _ in range(L)]
    att = torch.empty(nq * hd, device=dev)
    for _ in range(P):
        for i in range(L):
            ta.attn(i, torch.randn((nq + 2 * nkv) * hd, device=dev, generator=g), w[i][0], w[i][1], att)
        ta.pos.add_(1)
    tg = TalkerGroup(L, R, nq, nkv, M, 1e6, 1e-6, dev, prefix=(ta.k[:, :, :P], ta.v[:, :, :P]), cache_dtype=cdt,
                     n_pos=P + steps + 1, track_mass=True)
    tg.start(0)
    tg.start(2)
    keep, first, recent = 64, 8, 16
    own = {(i, r, h): ([], [], []) for i in range(L) for r in range(R) for h in range(nkv)}  # k, v, mass kept
    d = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    rope, kp, vp = d(tg.rope), d(ta.k), d(ta.v)
    live = {0: 0, 2: 0}  # slot -> position past the prompt
    for step in range(steps):
        if step == 30:
            tg.start(1)
            live[1] = 0
        if step == 110:
            tg.stop(2)
            del live[2]
        for i in range(L):
            qkv = torch.randn(R, (nq + 2 * nkv) * hd, device=dev, generator=g)
            out = tg.attn(i, qkv, w[i][0], w[i][1])
            x, o, wn = d(qkv), d(out), d(w[i])
            for r, at in live.items():
                head = x[r].reshape(-1, hd)
                c, s = np.split(rope[P + at], 2)

                def turn(y, wt):
                    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + 1e-6) * wt
                    a, b = np.split(y, 2, -1)
                    return np.concatenate([a * c - b * s, b * c + a * s], -1)

                q, k = turn(head[:nq], wn[0]), turn(head[nq:nq + nkv], wn[1])
                n = len(own[i, r, 0][0])
                # the appended rows as the caches hold them (their rounding is tested in the step's own tests)
                for h in range(nkv):
                    ks, vs, ms = own[i, r, h]
                    k_row = d(tg.k[i, r, h, n])
                    assert np.abs(k_row - k[h]).max() <= (2.0 ** -7 if cdt == BF else 1e-5) * np.abs(k[h]).max()
                    ks.append(k_row)
                    vs.append(d(tg.v[i, r, h, n]))
                    ms.append(0.0)
                    for e in range(nq // nkv):
                        qi = h * (nq // nkv) + e
                        sc = np.concatenate([kp[i, h, :P], np.array(ks)]) @ q[qi] * hd ** -0.5
                        p = np.exp(sc - sc.max())
                        p /= p.sum()
                        ref = p @ np.concatenate([vp[i, h, :P], np.array(vs)])
                        assert rel_l2(o[r, qi * hd:(qi + 1) * hd], ref) <= 1e-5
                        for j in range(n + 1):
                            ms[j] += p[P + j]
        tg.advance()
        for r in live:
            live[r] += 1
        if int(tg.rows.max()) >= M - 1:
            mass, n = d(tg.mass), tg.rows.tolist()
            tg.evict(keep, first, recent)
            assert tg.rows.tolist() == [min(x, keep) for x in n]
            for (i, r, h), (ks, vs, ms) in own.items():
                if r not in live:
                    continue
                assert rel_l2(mass[i, r, h, :n[r]], np.array(ms)) <= 1e-5
                at = kept_rows(mass[i, r, h].astype(np.float32), n[r], keep, first, recent)
                for t in (ks, vs, ms):
                    t[:] = [t[j] for j in at]
    assert ops.device_error() == 0


def test_group_slots_taken_again_and_budgets_changed(cuda):
    """A slot's next request does not inherit the weights of the last one, and budgets share one workspace."""
    from sokutou_b200.qwen3 import TalkerGroup

    tg = TalkerGroup(2, 3, 4, 2, 64, 1e6, 1e-6, cuda, track_mass=True)
    tg.mass.fill_(5.0)
    tg.start(1, rows=40)
    assert (tg.mass[:, 1, :, :40] == 0).all() and (tg.mass[:, 0] == 5).all() and (tg.mass[:, 1, :, 40:] == 5).all()
    tg.mass.copy_(torch.rand(tg.mass.shape, device=cuda))
    for keep in (30, 20, 10):
        before, k = tg.mass.clone(), tg.k.normal_().clone()
        n = int(tg.rows[1])
        tg.evict(keep, 2, 3)
        assert tg.rows.tolist() == [0, keep, 0] and tg.pos.tolist() == [-1, 40, -1]
        for i in range(2):
            for h in range(2):
                at = kept_rows(before[i, 1, h].cpu().numpy(), n, keep, 2, 3)
                assert torch.equal(tg.mass[i, 1, h, :keep], before[i, 1, h][at])
                assert torch.equal(tg.k[i, 1, h, :keep], k[i, 1, h][at])
    assert len({p.workspace.data_ptr() for p in tg._evict_plans.values()}) == 1 and ops.device_error() == 0
    with pytest.raises(ValueError):
        tg.start(3)
    with pytest.raises(ValueError):
        tg.start(0, rows=64)
    with pytest.raises(ValueError):
        TalkerGroup(1, 1, 4, 2, 64, 1e6, 1e-6, cuda).evict(10)
