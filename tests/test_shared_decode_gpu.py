"""sk_decode_attention_shared (ops.decode_attention_shared): one decode step of R requests behind one shared
prefix, against a float64 restatement. The caches behind the rows in use, the prefix's buffer past its length
and the masses of unused rows hold NaN throughout, so nothing may come from there.

Bars (relative L2). fp32 activations out of fp32 caches: 1e-5, the package's parity bar. fp32 activations out
of bf16 caches: q and the weights are split into two bf16 terms at least (each rounding at most 2^-8 of what it
rounds: 2^-16 of the number together, three leave 2^-24), rms errors 2^-16 / sqrt(3) = 8.8e-6 of a score of about 1
and of a weight, independent over the keys, so their average over the keys is below 1e-5 as well. bf16 activations: the result
(2^-8) and the weights (2^-8, averaged over keys) are each rounded once: 2^-7. Masses: a weight's error as
above, 1e-5. Appended rows: one rounding to the cache dtype of a value computed in fp32 (bf16: one step, 2^-7
of the element, where fp32 and float64 fall on two sides of a border, and 2e-6 where the rotation's two products,
up to about 4 each, nearly cancel: 3 roundings of 2^-24 of 8; fp32: 1e-5 of the row's largest).
"""

import math

import numpy as np
import pytest
import torch

from conftest import rel_l2
from sokutou_b200 import ops

pytestmark = pytest.mark.gpu

EPS = 1e-6
BF, F32 = torch.bfloat16, torch.float32


def host(t):
    return t.detach().double().cpu().numpy()


def rope_table(n, hd):
    inv = 1e6 ** (-np.arange(0, hd, 2) / hd)
    a = np.arange(n)[:, None] * inv
    return torch.from_numpy(np.concatenate([np.cos(a), np.sin(a)], 1)).float()


class Step:
    """The tensors of one call, on the GPU."""

    def __init__(self, dev, lens, P, nq, nkv, hd, cdt=BF, io=F32, mass=False, gone=0, slack=9, seed=0, strided=0):
        g = torch.Generator().manual_seed(seed)
        R, M = len(lens), max(max(lens) + 1, 1) + slack
        self.nq, self.nkv, self.hd, self.P, self.io, self.lens, self.R, self.M = nq, nkv, hd, P, io, lens, R, M

        def cache(n, rows, used):  # (n, nkv, rows, hd) with NaN where nothing is held
            x = torch.randn(n, nkv, rows, hd, generator=g)
            for i in range(n):
                x[i, :, max(used[i], 0):] = math.nan
            x = x.to(cdt)
            if strided:  # rows of all heads side by side, a gap of `strided` elements after each head's part
                y = torch.full((n, rows, nkv, hd + strided), math.nan, dtype=cdt).to(dev)[..., :hd].permute(0, 2, 1, 3)
                y.copy_(x)
                return y
            return x.to(dev)

        self.K, self.V = cache(R, M, lens), cache(R, M, lens)
        kp, vp = cache(1, P + slack, [P])[0], cache(1, P + slack, [P])[0]
        self.Kp, self.Vp = kp[:, :P], vp[:, :P]
        self.rows = torch.tensor([max(n, 0) for n in lens], device=dev)
        self.pos = torch.tensor([n + P + gone if n >= 0 else -1 for n in lens], device=dev)
        self.rope = rope_table(P + M + gone, hd).to(dev)
        self.qkv = torch.randn(R, (nq + 2 * nkv) * hd, generator=g).to(io).to(dev)
        for r, n in enumerate(lens):
            if n < 0:
                self.qkv[r] = math.nan
        self.qn = (1 + 0.02 * torch.randn(hd, generator=g)).to(dev)
        self.kn = (1 + 0.02 * torch.randn(hd, generator=g)).to(dev)
        self.mass = None
        if mass:
            self.mass = torch.rand(R, nkv, M, generator=g)
            for r, n in enumerate(lens):
                self.mass[r, :, max(n, 0):] = math.nan
            self.mass = self.mass.to(dev)
        self.out = torch.full((R, nq * hd), 7.0, device=dev, dtype=io)

    def plan(self, **kw):
        return ops.shared_decode_plan(self.K, self.V, self.pos, self.rope, self.nq, EPS, rows=self.rows, Kp=self.Kp,
                                      Vp=self.Vp, mass=self.mass, qkv_dtype=self.io, out_dtype=self.io, **kw)

    def want(self, scale=None):
        """out, the appended k and v rows and the masses, in float64."""
        nq, nkv, hd, g = self.nq, self.nkv, self.hd, self.nq // self.nkv
        out, mass = host(self.out), None if self.mass is None else host(self.mass)
        K, V, Kp, Vp, x, pos = (host(t) for t in (self.K, self.V, self.Kp, self.Vp, self.qkv, self.pos))
        rope, qn, kn = host(self.rope), host(self.qn), host(self.kn)
        dt = self.K.dtype
        new = {}
        for r, n in enumerate(self.lens):
            if n < 0:
                continue
            h = x[r].reshape(-1, hd)
            c, s = np.split(rope[int(pos[r])], 2)

            def turn(y, w):
                y = y / np.sqrt((y * y).mean(-1, keepdims=True) + EPS) * w
                a, b = np.split(y, 2, -1)
                return np.concatenate([a * c - b * s, b * c + a * s], -1)

            q, k, v = turn(h[:nq], qn), turn(h[nq:nq + nkv], kn), h[nq + nkv:]
            stored = lambda y: torch.from_numpy(y).float().to(dt).double().numpy()  # noqa: E731
            new[r] = (k, v)
            K[r, :, n], V[r, :, n] = stored(k), stored(v)
            for i in range(nq):
                kv = i // g
                kk = np.concatenate([Kp[kv], K[r, kv, :n + 1]])
                vv = np.concatenate([Vp[kv], V[r, kv, :n + 1]])
                sc = kk @ q[i] * (scale or hd ** -0.5)
                p = np.exp(sc - sc.max())
                p /= p.sum()
                out[r, i * hd:(i + 1) * hd] = p @ vv
                if mass is not None:
                    if i % g == 0:
                        mass[r, kv, n] = 0
                    mass[r, kv, :n + 1] += p[self.P:]
        return out, new, mass

    def check(self, want, before):
        out, new, mass = want
        live = [r for r, n in enumerate(self.lens) if n >= 0]
        tol = 2.0 ** -7 if self.io == BF else 1e-5
        got = host(self.out)
        for r in range(self.R):
            if r not in live:
                assert np.array_equal(got[r], host(before["out"])[r])  # an idle slot's row stays as it was
            else:
                assert rel_l2(got[r], out[r]) <= tol, (r, rel_l2(got[r], out[r]))
        for name, t, i in (("K", self.K, 0), ("V", self.V, 1)):
            a, b = host(t), host(before[name])
            for r in live:
                row, ref = a[r, :, self.lens[r]].copy(), new[r][i]
                a[r, :, self.lens[r]] = b[r, :, self.lens[r]]
                step = 2.0 ** -7 * np.abs(ref) + 2e-6 if t.dtype == BF else 1e-5 * np.abs(ref).max()
                assert (np.abs(row - ref) <= step).all()
            assert np.array_equal(a, b, equal_nan=True)  # nothing else was written
        if mass is not None:
            got = host(self.mass)
            for r, n in enumerate(self.lens):
                assert np.array_equal(got[r, :, n + 1:], mass[r, :, n + 1:], equal_nan=True)
                if n >= 0:
                    assert rel_l2(got[r, :, :n + 1], mass[r, :, :n + 1]) <= 1e-5
        assert ops.device_error() == 0

    def before(self):
        return {"out": self.out.clone(), "K": self.K.clone(), "V": self.V.clone()}

    def run(self, **kw):
        want, before = self.want(kw.get("scale")), self.before()
        ops.decode_attention_shared(self.plan(**kw), self.qkv, self.qn, self.kn, out=self.out)
        self.check(want, before)


EDGES = [0, 1, 63, 64, 65, 127, 128, 129, 255, 256, 257]
CASES = {
    "one token, nothing before it": dict(lens=[0], P=0, nq=16, nkv=8, hd=128),
    "one prefix row": dict(lens=[0, 0], P=1, nq=2, nkv=1, hd=128),
    "tile edges": dict(lens=EDGES, P=96, nq=16, nkv=8, hd=128),
    "tile edges, no prefix": dict(lens=EDGES, P=0, nq=4, nkv=2, hd=128),
    "tile edges, heads of 64": dict(lens=EDGES, P=129, nq=4, nkv=2, hd=64),
    "prefix only": dict(lens=[0] * 5, P=777, nq=16, nkv=8, hd=128),
    "prefix of one tile": dict(lens=[3] * 4, P=128, nq=16, nkv=8, hd=128),
    "33 query rows": dict(lens=[11] * 33, P=300, nq=3, nkv=3, hd=128),
    "two tiles of query rows": dict(lens=[5 + 3 * (i % 7) for i in range(70)], P=200, nq=4, nkv=2, hd=128),
    "three heads a group, over a tile's edge": dict(lens=[i for i in range(47)], P=130, nq=6, nkv=2, hd=128),
    "five heads a group": dict(lens=[40, 0, 260], P=65, nq=5, nkv=1, hd=64),
    "eight heads a group": dict(lens=[300, 20, 131, 2] * 5, P=150, nq=16, nkv=2, hd=128),
    "seven heads of 64": dict(lens=[300, 20, 131, 2] * 5, P=15, nq=7, nkv=1, hd=64),
    "idle slots": dict(lens=[-1, 200, -1, -1, 0, 77, -1], P=140, nq=16, nkv=8, hd=128),
    "all idle": dict(lens=[-1, -1], P=140, nq=16, nkv=8, hd=128),
    "long prefix, few requests": dict(lens=[100, 300, 0], P=20011, nq=4, nkv=2, hd=128),
    "long own rows": dict(lens=[9000, 17], P=33, nq=4, nkv=2, hd=128),
    "many short requests": dict(lens=[(7 * i) % 50 for i in range(400)], P=40, nq=2, nkv=1, hd=64),
    "the most requests": dict(lens=[(3 * i) % 5 for i in range(1024)], P=5, nq=2, nkv=1, hd=64),
    "evicted before": dict(lens=[500, 131], P=96, nq=16, nkv=8, hd=128, gone=4000),
    "strided caches": dict(lens=[500, 131, 0], P=96, nq=6, nkv=3, hd=128, strided=16),
    "rows on 16 bytes only": dict(lens=[500, 131, 0], P=96, nq=6, nkv=3, hd=128, strided=8),
    "strided caches of 64": dict(lens=[500, 131, 0], P=96, nq=6, nkv=3, hd=64, strided=24),
}
TYPES = {"bf16 cache, f32 io": (BF, F32), "bf16 cache, bf16 io": (BF, BF), "f32 cache": (F32, F32)}


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_step_against_float64(cuda, case, types, mass):
    cdt, io = TYPES[types]
    Step(cuda, cdt=cdt, io=io, mass=mass, seed=len(case), **CASES[case]).run()


# Prefixes long enough that the requests share their tiles instead of reading them each (bf16 caches:
# R * nkv * P rows of K and V past 12 MB + R * nkv / 3 MB), by query rows n of a key/value head.
TILED = {
    "n = 2": dict(lens=[150], P=4801, nq=16, nkv=8, hd=128),
    "n = 8, the most of the short form": dict(lens=[40, 0, 129, 3], P=3900, nq=4, nkv=2, hd=128),
    "n = 9, the least of the long form": dict(lens=[0, 1, 2, 3, 127, 128, 129, 255, 256], P=3500, nq=1, nkv=1, hd=128),
    "n = 10, an idle slot among them": dict(lens=[40, -1, 0, 129, 3], P=3201, nq=4, nkv=2, hd=128),
    "n = 96, groups of eight": dict(lens=[(29 * i) % 300 for i in range(12)], P=1801, nq=16, nkv=2, hd=128),
    "n = 128": dict(lens=[(7 * i) % 60 for i in range(64)], P=1152, nq=4, nkv=2, hd=128),
    "n = 140, two row tiles": dict(lens=[5 + 3 * (i % 7) for i in range(70)], P=899, nq=4, nkv=2, hd=128),
    "n = 141, a group over a row tile's edge": dict(lens=[i for i in range(47)], P=1000, nq=6, nkv=2, hd=128),
    "n = 300, three row tiles, groups of five": dict(lens=[(11 * i) % 200 for i in range(60)], P=1201, nq=5, nkv=1, hd=128),
    "heads of 64, groups of five": dict(lens=[(41 * i) % 333 for i in range(24)], P=1701, nq=35, nkv=7, hd=64),
    "heads of 64, n = 3": dict(lens=[17, 500, 0], P=18001, nq=1, nkv=1, hd=64),
    "strided caches": dict(lens=[40, 0, 129, 3, 9], P=3301, nq=6, nkv=3, hd=128, strided=8),
    "evicted before": dict(lens=[500, 131, 7], P=2801, nq=16, nkv=8, hd=128, gone=4000),
    "all idle": dict(lens=[-1, -1], P=4001, nq=16, nkv=8, hd=128),
}


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("io", [F32, BF])
@pytest.mark.parametrize("case", TILED)
def test_shared_tiles_against_float64(cuda, case, io, mass):
    a = TILED[case]
    heads = len(a["lens"]) * a["nkv"]
    assert heads * a["P"] * 4 * a["hd"] > (12 << 20) + heads * (1 << 20) // 3
    Step(cuda, io=io, mass=mass, seed=len(case), **a).run()


@pytest.mark.parametrize("mass", [False, True])
@pytest.mark.parametrize("R,P,nq,nkv,hd", [(1024, 2100, 2, 1, 64), (300, 900, 4, 4, 128), (100, 10601, 3, 1, 128)])
def test_shared_tiles_of_fp32_caches_against_float64(cuda, R, P, nq, nkv, hd, mass):
    """More than 1 GB of rows if every request read the prefix for itself."""
    assert R * nkv * P * 8 * hd > 1 << 30
    lens = [-1 if i % 19 == 5 else (7 * i) % 67 for i in range(R)]
    Step(cuda, lens, P, nq, nkv, hd, cdt=F32, mass=mass, seed=R).run()


@pytest.mark.parametrize("R,P,nq,nkv,hd,own", [(1, 300001, 16, 8, 128, 40), (8, 200001, 16, 8, 128, 3), (2, 500001, 3, 3, 64, 0),
                                               (2, 100, 8, 8, 128, 150001), (1, 96, 16, 8, 128, 8183), (1, 96, 16, 8, 128, 8185)])
def test_long_sums_stay_within_the_bar(cuda, R, P, nq, nkv, hd, own):
    """Hundreds of tiles for every CTA: sums over them in tensor memory, whose additions cut off what does not fit,
    have to be short (a tile of 128 keys takes 8 additions of 2^-24 of the sum per term and product, so the 40 tiles of
    a partial take 40 * 8 * 2^-25 on the average, 9.5e-6, if every one of them cuts off half of a last place). The float64
    restatement runs on the GPU."""
    s = Step(cuda, [1] * R, 2, nq, nkv, hd, seed=30)  # small tensors of the right kinds, then the long ones
    g = torch.Generator(device=cuda).manual_seed(31)
    M = own + 8
    s.K, s.V = (torch.randn(R, nkv, M, hd, device=cuda, generator=g, dtype=F32).to(BF) for _ in range(2))
    s.Kp, s.Vp = (torch.randn(nkv, P, hd, device=cuda, generator=g, dtype=F32).to(BF) for _ in range(2))
    s.rope = rope_table(P + M, hd).to(cuda)
    s.rows.fill_(own)
    s.pos.fill_(P + own)
    ops.decode_attention_shared(s.plan(), s.qkv, s.qn, s.kn, out=s.out)
    assert ops.device_error() == 0
    d = lambda t: t.double()  # noqa: E731
    c, sn = d(s.rope[P + own]).chunk(2)
    for r in range(R):
        x = d(s.qkv[r]).view(-1, hd)[:nq]
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * d(s.qn)
        a, b = x.chunk(2, -1)
        q = torch.cat([a * c - b * sn, b * c + a * sn], -1)
        for h in range(nkv):
            K = torch.cat([d(s.Kp[h]), d(s.K[r, h, :own + 1])])  # (the row appended as the cache holds it)
            V = torch.cat([d(s.Vp[h]), d(s.V[r, h, :own + 1])])
            for i in range(h * nq // nkv, (h + 1) * nq // nkv):
                ref = torch.softmax(K @ q[i] * hd ** -0.5, 0) @ V
                got = d(s.out[r, i * hd:(i + 1) * hd])
                assert ((got - ref).norm() / ref.norm()).item() <= 1e-5, (r, i)


@pytest.mark.parametrize("io", [F32, BF])
def test_shared_tiles_captured_twice_with_one_workspace(cuda, io):
    """Two captured steps and an eager one, all of one plan's workspace, in turn on one stream."""
    s = Step(cuda, [(31 * i) % 400 for i in range(12)], 1500, 16, 8, 128, io=io, mass=True, seed=24)
    want, before, m0, plan = s.want(), s.before(), s.mass.clone(), s.plan()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.decode_attention_shared(plan, s.qkv, s.qn, s.kn, out=s.out)
        graphs.append(g)
    run = [graphs[0].replay, graphs[1].replay, lambda: ops.decode_attention_shared(plan, s.qkv, s.qn, s.kn, out=s.out)]
    for i in range(9):
        s.out.fill_(7.0)
        s.mass.copy_(m0)
        run[i % 3]()
    s.check(want, before)


def test_shared_tiles_on_two_streams(cuda):
    steps = [Step(cuda, [(31 * i) % 300 for i in range(12)], 1500, 16, 8, 128, mass=True, seed=s) for s in (26, 27)]
    want, before = [s.want() for s in steps], [s.before() for s in steps]
    plans, m0 = [s.plan() for s in steps], [s.mass.clone() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(20):
        for s, p, st, m in zip(steps, plans, streams, m0):
            with torch.cuda.stream(st):
                s.mass.copy_(m)
                ops.decode_attention_shared(p, s.qkv, s.qn, s.kn, out=s.out)
    torch.cuda.synchronize()
    for s, w, b in zip(steps, want, before):
        s.check(w, b)


@pytest.mark.parametrize("cdt", [BF, F32])
def test_softmax_scale(cuda, cdt):
    Step(cuda, [300, 3], 170, 4, 2, 128, cdt=cdt, mass=True).run(scale=0.31)


@pytest.mark.parametrize("cdt", [BF, F32])
def test_scores_far_apart(cuda, cdt):
    """Keys whose scores span hundreds: the running maximum moves up late in the prefix and in the own rows,
    and all but a few weights underflow."""
    s = Step(cuda, [400, 130], 700, 4, 2, 128, cdt=cdt, mass=True, seed=3)
    for x, n in ((s.Kp, 700), (s.K[0], 400), (s.K[1], 130)):
        x[:, :n] *= torch.linspace(0.05, 12, n, device=cuda)[:, None].to(cdt)
    want, before = s.want(), s.before()
    ops.decode_attention_shared(s.plan(), s.qkv, s.qn, s.kn, out=s.out)
    # scores up to about 12 * 4: an error of 2^-16 / sqrt(3) of one (in natural units) is 48 times the bar's
    # share of a score of 1, in every weight
    for r in range(2):
        tol = 48 * 1e-5 if cdt == BF else 5e-5
        assert rel_l2(host(s.out)[r], want[0][r]) <= tol
        assert rel_l2(host(s.mass)[r, :, :s.lens[r] + 1], want[2][r, :, :s.lens[r] + 1]) <= tol
    assert torch.equal(before["K"][0, :, :400], s.K[0, :, :400])


@pytest.mark.parametrize("cdt", [BF, F32])
def test_nan_and_infinity_stay_with_their_request(cuda, cdt):
    """A NaN in one request's own rows, or in its q, makes that request's heads NaN and nobody else's; an
    infinite value row makes the columns of its head infinite or NaN for everyone who attends it."""
    s = Step(cuda, [200, 150, 140], 90, 4, 2, 128, cdt=cdt, mass=True, seed=5)
    clean = Step(cuda, [200, 150, 140], 90, 4, 2, 128, cdt=cdt, mass=True, seed=5)
    s.K[1, 0, 17, 3] = math.nan
    s.qkv[2, 3 * 128] = math.nan  # head 3 of request 2
    for x in (s, clean):
        ops.decode_attention_shared(x.plan(), x.qkv, x.qn, x.kn, out=x.out)
    got, ref = s.out.view(3, 4, 128), clean.out.view(3, 4, 128)
    assert torch.isnan(got[1, :2]).all() and torch.isnan(got[2, 3]).all()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1, 2:], ref[1, 2:]) and torch.equal(got[2, :3], ref[2, :3])
    s.Vp[1, 50, 7] = math.inf
    ops.decode_attention_shared(s.plan(), s.qkv, s.qn, s.kn, out=s.out)
    assert not torch.isfinite(s.out.view(3, 4, 128)[:, 2:, 7]).any()
    assert torch.isfinite(s.out.view(3, 4, 128)[0, :2]).all()


@pytest.mark.parametrize("cdt", [BF, F32])
def test_position_or_row_out_of_range(cuda, cdt):
    """Records SK_DEVERR_POS_RANGE and leaves that request alone; the others are served."""
    for field, value in (("pos", 10 ** 6), ("rows", 10 ** 6), ("rows", -3)):
        s = Step(cuda, [200, 150, 140], 90, 4, 2, 128, cdt=cdt, mass=True, seed=6)
        want, before = s.want(), s.before()
        m1 = s.mass[1].clone()
        getattr(s, field)[1] = value
        ops.decode_attention_shared(s.plan(), s.qkv, s.qn, s.kn, out=s.out)
        assert ops.device_error() == 1
        assert torch.equal(s.out[1], before["out"][1]) and torch.equal(s.mass[1].isnan(), m1.isnan())
        assert np.array_equal(host(s.K[1]), host(before["K"][1]), equal_nan=True)
        for r in (0, 2):
            assert rel_l2(host(s.out)[r], want[0][r]) <= 1e-5


def test_rows_default_to_the_position(cuda):
    s = Step(cuda, [200, 0, -1, 140], 90, 4, 2, 128, mass=True, seed=7)
    want, before = s.want(), s.before()
    p = ops.shared_decode_plan(s.K, s.V, s.pos, s.rope, s.nq, EPS, Kp=s.Kp, Vp=s.Vp, mass=s.mass)
    ops.decode_attention_shared(p, s.qkv, s.qn, s.kn, out=s.out)
    s.check(want, before)


@pytest.mark.parametrize("cdt", [BF, F32])
@pytest.mark.parametrize("R,P,nkv,g,hd", [(24, 1111, 8, 2, 128), (24, 2500, 8, 2, 128), (40, 900, 8, 4, 64), (70, 700, 8, 2, 128)])
def test_same_bits_every_time(cuda, cdt, R, P, nkv, g, hd):
    """Shares that hold segments of both kinds (many query rows, few), again and again."""
    s = Step(cuda, [(37 * i) % 900 for i in range(R)], P, nkv * g, nkv, hd, cdt=cdt, mass=True, seed=8)
    plan, m0 = s.plan(), s.mass.clone()
    first = None
    for _ in range(60):
        s.mass.copy_(m0)
        ops.decode_attention_shared(plan, s.qkv, s.qn, s.kn, out=s.out)
        got = (s.out.clone(), s.mass.nan_to_num(0))
        first = first or got
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])


@pytest.mark.parametrize("cdt", [BF, F32])
def test_padded_activations_and_new_output(cuda, cdt):
    """qkv and out with a stride between rows; out allocated by the call; one request whose row stride is moot."""
    s = Step(cuda, [200, 3, 140], 90, 4, 2, 128, cdt=cdt, seed=9)
    want, _ = s.want(), s.before()
    wide = torch.full((3, 8 * 128 + 64), math.nan, device=cuda)
    wide[:, :8 * 128] = s.qkv
    o = torch.zeros(3, 4 * 128 + 8, device=cuda)
    p = s.plan(qkv_stride=8 * 128 + 64, out_stride=4 * 128 + 8)
    ops.decode_attention_shared(p, wide[:, :8 * 128], s.qn, s.kn, out=o[:, :512])
    assert rel_l2(host(o[:, :512]), want[0]) <= 1e-5 and (o[:, 512:] == 0).all()
    got = ops.decode_attention_shared(s.plan(), s.qkv, s.qn, s.kn)
    assert rel_l2(host(got), want[0]) <= 1e-5
    one = Step(cuda, [77], 90, 4, 2, 128, cdt=cdt, seed=10)
    want = one.want()
    got = ops.decode_attention_shared(one.plan(), torch.cat([one.qkv, one.qkv], 1)[:, :8 * 128], one.qn, one.kn)
    assert rel_l2(host(got), want[0]) <= 1e-5


@pytest.mark.parametrize("cdt", [BF, F32])
def test_offsets_past_32_bits(cuda, cdt):
    """Rows, heads and requests whose element offsets pass 2^31."""
    hd, stride = 128, (1 << 31) // 60 // 8 * 8
    s = Step(cuda, [65, 40], 70, 2, 1, hd, cdt=cdt, mass=True, slack=4, seed=11)
    M = s.M
    big = [torch.empty(M * stride, dtype=cdt, device=cuda).as_strided((2, 1, M, hd), (4 * hd, 2 * hd, stride, 1)) for _ in range(2)]
    assert M * stride > 1 << 31
    for b, t in zip(big, (s.K, s.V)):
        b.copy_(t)
    s.K, s.V = big
    want = s.want()
    ops.decode_attention_shared(s.plan(), s.qkv, s.qn, s.kn, out=s.out)
    assert rel_l2(host(s.out), want[0]) <= 1e-5 and ops.device_error() == 0


@pytest.mark.parametrize("cdt", [BF, F32])
def test_graph_replay_reads_lengths_on_the_device(cuda, cdt):
    """One captured step replayed while positions advance, a slot goes idle and another joins: as eager steps."""
    mk = lambda: Step(cuda, [120, 63, -1, 0], 100, 4, 2, 128, cdt=cdt, mass=True, slack=40, seed=12)  # noqa: E731
    a, b = mk(), mk()
    plan_a, plan_b = a.plan(), b.plan()
    step = torch.tensor([1, 1, 0, 1], device=cuda)
    for x in (a, b):
        x.step = step.clone()
    def one(x, plan):
        ops.decode_attention_shared(plan, x.qkv, x.qn, x.kn, out=x.out)
        x.pos.add_(x.step)
        x.rows.add_(x.step)
    snap = [t.clone() for t in (a.K, a.V, a.mass, a.pos, a.rows)]
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        one(a, plan_a)
    torch.cuda.current_stream().wait_stream(st)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        one(a, plan_a)
    for t, old in zip((a.K, a.V, a.mass, a.pos, a.rows), snap):
        t.copy_(old)
    a.out.fill_(7.0)
    g = torch.Generator(device=cuda).manual_seed(1)
    for i in range(12):
        x = torch.randn(a.qkv.shape, device=cuda, generator=g)
        for s in (a, b):
            s.qkv.copy_(x)
            if i == 5:  # slot 1 ends, slot 2 begins
                s.pos[1], s.rows[1], s.step[1] = -1, 0, 0
                s.pos[2], s.rows[2], s.step[2] = s.P, 0, 1
        gr.replay()
        one(b, plan_b)
    torch.cuda.synchronize()
    assert torch.equal(a.out, b.out)
    for x, y in ((a.K, b.K), (a.V, b.V), (a.mass, b.mass)):
        assert torch.equal(x.nan_to_num(0), y.nan_to_num(0))
    del gr
    assert ops.device_error() == 0


def test_two_streams_with_their_own_workspaces(cuda):
    steps = [Step(cuda, [(31 * i) % 700 for i in range(12)], 900, 16, 8, 128, mass=True, seed=s) for s in (20, 21)]
    want = [s.want() for s in steps]
    before = [s.before() for s in steps]
    plans = [s.plan() for s in steps]
    m0 = [s.mass.clone() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(20):
        for s, p, st, m in zip(steps, plans, streams, m0):
            with torch.cuda.stream(st):
                s.mass.copy_(m)
                ops.decode_attention_shared(p, s.qkv, s.qn, s.kn, out=s.out)
    torch.cuda.synchronize()
    for s, w, b in zip(steps, want, before):
        s.check(w, b)


def test_follows_and_precedes_other_kernels_on_the_stream(cuda):
    """The activations written by the kernel just before and the outputs read by the one just after."""
    s = Step(cuda, [300, 200], 500, 16, 8, 128, seed=22)
    want, before = s.want(), s.before()
    x, plan = s.qkv.clone(), s.plan()
    for _ in range(30):
        s.qkv.fill_(math.nan)
        s.qkv.copy_(x)
        ops.decode_attention_shared(plan, s.qkv, s.qn, s.kn, out=s.out)
        got = s.out * 1.0
        s.out.fill_(3.0)
        assert rel_l2(host(got), want[0]) <= 1e-5
    s.out.copy_(got)
    s.check(want, before)


def test_refusals(cuda):
    s = Step(cuda, [30, 20], 50, 4, 2, 128, mass=True)
    ok = s.plan()
    bad = [dict(K=s.K[0]), dict(V=s.V.float()), dict(pos=s.pos.int()), dict(pos=s.pos[:1]), dict(rope=s.rope[:, :64]),
           dict(rope=s.rope.double()), dict(Kp=None), dict(Kp=s.Kp[:, :9]), dict(Kp=s.Kp.float(), Vp=s.Vp.float()),
           dict(mass=s.mass[:, :, :3]), dict(mass=s.mass.double()), dict(rows=s.rows.cpu()), dict(nq=5), dict(nq=18),
           dict(K=s.K.half(), V=s.V.half())]
    for kw in bad:
        a = dict(K=s.K, V=s.V, pos=s.pos, rope=s.rope, nq=s.nq, eps=EPS, rows=s.rows, Kp=s.Kp, Vp=s.Vp, mass=s.mass) | kw
        with pytest.raises((ValueError, TypeError)):
            ops.shared_decode_plan(**a)
    for kw in (dict(qkv=s.qkv[:1]), dict(qkv=s.qkv.bfloat16()), dict(qkv=s.qkv.cpu()), dict(qkv=s.qkv.t().contiguous().t()),
               dict(qn=s.qn[:64]), dict(kn=s.kn.double()), dict(out=s.out[:, :5]), dict(out=s.out.bfloat16())):
        a = dict(qkv=s.qkv, qn=s.qn, kn=s.kn, out=s.out) | kw
        with pytest.raises(ValueError):
            ops.decode_attention_shared(ok, **a)
    small = ops.shared_decode_plan(s.K, s.V, s.pos, s.rope, s.nq, EPS, rows=s.rows, Kp=s.Kp, Vp=s.Vp,
                                   workspace=torch.empty(256, dtype=torch.uint8, device=cuda))
    with pytest.raises(ops._lib.SokutouError):
        ops.decode_attention_shared(small, s.qkv, s.qn, s.kn, out=s.out)
    odd = torch.zeros(2, 2, 40, 129, device=cuda, dtype=BF)[..., :128]  # rows not 16-byte aligned
    p = ops.shared_decode_plan(odd, odd, s.pos, s.rope, s.nq, EPS, rows=s.rows)
    with pytest.raises(ops._lib.SokutouError):
        ops.decode_attention_shared(p, s.qkv, s.qn, s.kn, out=s.out)
    assert (s.out == 7.0).all() and ops.device_error() == 0
