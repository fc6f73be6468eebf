"""The expert block of a few tokens in one call (izb_moe_layer) against the formula in 64 bits, and against the six calls it stands for."""
import numpy as np
import pytest

from arcinferzero_b200 import synth as S
from oracle import oracle as O

pytestmark = pytest.mark.gpu
# Exact integer block sums, added up in f32: a chain of at most 64 roundings of 2^-24 per projection, and h off by 2^-22 of its block's largest value;
# against the result's largest value (terms of a sum of K are about sqrt(K) times smaller than the sum of their sizes, hence a factor of ten).
TOL = 1e-5


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


def rows(qt, N, K, seed):
    """GGUF rows like a model's: mean about 0, deviation about 1 / sqrt(K)."""
    w = S.make_weight(qt, N, K, seed)
    rng, s = np.random.default_rng(seed + 1), 1.0 / np.sqrt(K)
    if qt == 12:
        b = w.reshape(-1, 144)
        d = rng.uniform(0.5, 1.5, len(b)) * s / 165.0
        b[:, 0:2], b[:, 2:4] = d.astype(np.float16).view(np.uint8).reshape(-1, 2), (7.5 * d).astype(np.float16).view(np.uint8).reshape(-1, 2)
        b[:, 8:12] = b[:, 4:8]
        b[:, 12:16] = (b[:, 12:16] & 15) * 17
    else:
        b = w.reshape(-1, 34 if qt == 8 else 18)
        b[:, 0:2] = (rng.uniform(0.5, 1.5, len(b)) * s / (76.0 if qt == 8 else 4.8)).astype(np.float16).view(np.uint8).reshape(-1, 2)
    return w


class Block:
    def __init__(self, izb, torch, T, E, F, NE, NU, qt, qd, joined=False, seed=0, shared=False, experts=None):
        rng = np.random.default_rng(seed)
        self.izb, self.torch, self.T, self.E, self.F, self.NE, self.NU, self.qt, self.qd, self.shared = izb, torch, T, E, F, NE, NU, qt, qd, shared
        self.e0, self.e1 = experts or (0, NE)
        self.g, self.u, self.d = rows(qt, NE * F, E, seed + 1), rows(qt, NE * F, E, seed + 2), rows(qd, NE * E, F, seed + 3)
        n = self.e1 - self.e0
        of = lambda w, N: w[self.e0 * N:self.e1 * N]
        self.joined = joined
        self.wg = izb.gateup_weight(qt, of(self.g, F), of(self.u, F), F, E, n_mats=n) if joined else izb.Weight(qt, of(self.g, F), F, E, n_mats=n)
        self.wu = None if joined else izb.Weight(qt, of(self.u, F), F, E, n_mats=n)
        self.wd = izb.Weight(qd, of(self.d, E), E, F, n_mats=n)
        cu = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()
        self.x = cu(rng.standard_normal((T, E)))
        self.aq, self.asc, _ = izb.quantize_act(cu(rng.standard_normal((T, E))))
        self.logits = cu(rng.standard_normal((T, NE + (1 if shared else 0))))
        self.sh = cu(rng.standard_normal((T, E))) if shared else None

    def call(self, x=None, out=None):
        return self.izb.moe_layer(self.wg, self.wu, self.wd, self.aq, self.asc, self.logits, self.NU, x=x, out=out, sh=self.sh, e0=self.e0)

    def want(self):
        """The block without the residual, in 64 bits."""
        T, E, F, NE, NU = self.T, self.E, self.F, self.NE, self.NU
        lg, out = self.logits.cpu().numpy().astype(np.float64), np.zeros((T, E))
        aq, asc = self.aq.cpu().numpy(), self.asc.cpu().numpy()
        for t in range(T):
            order = sorted(range(NE), key=lambda e: (-lg[t, e], e))[:NU]
            w = np.exp(lg[t, order] - lg[t, order[0]])
            w /= w.sum()
            for e, we in zip(order, w):
                if not self.e0 <= e < self.e1:
                    continue
                one = lambda m, N: O.matmul(self.qt, np.ascontiguousarray(m[e * N:(e + 1) * N]), E, np.ascontiguousarray(aq[t:t + 1]), np.ascontiguousarray(asc[:, t:t + 1]), 1, "f64")[0].astype(np.float64)
                g, u = one(self.g, F), one(self.u, F)
                out[t] += we * (dense(self.qd, self.d[e * E:(e + 1) * E], F) @ (g / (1 + np.exp(-g)) * u))
            if self.shared:
                out[t] += self.sh.cpu().numpy()[t].astype(np.float64) / (1 + np.exp(-lg[t, NE]))
        return out


def dense(qt, w, K):
    """GGUF rows as f64, written from the formats."""
    f16 = lambda b: np.ascontiguousarray(b).view(np.float16).astype(np.float64)
    if qt == 8:
        b = w.reshape(-1, 34)
        return (f16(b[:, 0:2]) * np.ascontiguousarray(b[:, 2:]).view(np.int8)).reshape(len(w), K)
    if qt == 2:
        b = w.reshape(-1, 18)
        q = np.concatenate([b[:, 2:] & 15, b[:, 2:] >> 4], 1).astype(np.float64) - 8
        return (f16(b[:, 0:2]) * q).reshape(len(w), K)
    b = w.reshape(-1, 144)
    s = b[:, 4:16].astype(int)
    sc = np.concatenate([s[:, 0:4] & 63, (s[:, 8:12] & 15) | (s[:, 0:4] >> 6 << 4)], 1)
    mn = np.concatenate([s[:, 4:8] & 63, (s[:, 8:12] >> 4) | (s[:, 4:8] >> 6 << 4)], 1)
    q = b[:, 16:].reshape(-1, 4, 32)
    q = np.stack([q & 15, q >> 4], 2).reshape(-1, 8, 32)
    return (f16(b[:, 0:2])[:, :, None] * sc[:, :, None] * q - f16(b[:, 2:4])[:, :, None] * mn[:, :, None]).reshape(len(w), K)


def rel(got, want):
    return float(np.abs(got.cpu().numpy().astype(np.float64) - want).max() / np.abs(want).max())


@pytest.mark.parametrize("T,E,F,NE,NU,qt,qd,joined", [
    (1, 256, 256, 4, 1, 12, 12, False),
    (1, 512, 768, 16, 8, 12, 8, True),
    (2, 768, 512, 3, 3, 8, 12, False),       # every token at every expert
    (5, 2048, 768, 128, 8, 12, 12, True),
    (7, 1280, 256, 60, 4, 8, 8, True),
    (9, 256, 1280, 5, 2, 12, 12, False),     # several tokens per expert
    (17, 512, 512, 2, 1, 12, 8, False),      # more tokens of an expert than columns of an instruction
    (32, 512, 256, 8, 2, 8, 12, True),
    (32, 256, 512, 16, 16, 12, 12, False),   # the most pairs
    (3, 4352, 256, 33, 5, 2, 2, False),      # Q4_0; a K that does not divide among the warps
    (4, 256, 4864, 6, 2, 12, 8, False),      # a long F
    (31, 1536, 256, 512, 4, 8, 8, False),    # the most experts
])
def test_against_64_bits(izb, torch, T, E, F, NE, NU, qt, qd, joined):
    b = Block(izb, torch, T, E, F, NE, NU, qt, qd, joined, seed=T + E)
    want = b.want()
    got = b.call()
    assert rel(got, want) <= TOL
    out = torch.full_like(b.x, float("nan"))
    assert b.call(x=b.x, out=out) is out
    assert torch.equal(out, b.x + got)       # the sum is rounded once, then added
    x = b.x.clone()
    b.call(x=x, out=x)
    assert torch.equal(x, out)


def test_shared_expert_and_split(izb, torch):
    """The shared expert joins through its gate; two halves of the experts add up to the whole."""
    b = Block(izb, torch, 6, 512, 256, 20, 6, 12, 12, shared=True)
    want = b.want()
    assert rel(b.call(), want) <= TOL
    b.sh, gate = None, b.logits
    b.logits, b.shared = gate[:, :20], False  # (rows of 21, 20 of them meant)
    whole = b.call()
    parts = [Block(izb, torch, 6, 512, 256, 20, 6, 12, 12, shared=True, experts=r) for r in ((0, 7), (7, 20))]
    for p in parts:
        p.sh, p.logits, p.shared = None, b.logits, False
        assert rel(p.call(), p.want()) <= TOL
    assert float((parts[0].call() + parts[1].call() - whole).abs().max()) <= TOL * float(whole.abs().max())


def test_against_the_six_calls(izb, torch):
    """The separate calls quantise h: one part in 254 of a block's largest value per element, 1/sqrt(3) of it on average, so about 1 % of the result."""
    b = Block(izb, torch, 8, 1024, 512, 32, 4, 12, 12)
    ids, wts, counts = izb.moe_route(b.logits, 4)
    _, tiles, max_tiles, stok, swt, inv = izb.moe_sort(ids, wts, counts, 8)
    h = izb.moe_gateup(b.wg, b.wu, b.aq, b.asc, tiles, max_tiles, 8, stok, 32)
    hq, hsc, _ = izb.quantize_act(h)
    y = izb.moe_down(b.wd, hq, hsc, tiles, max_tiles, 8, swt, 32)
    six = b.x.clone()
    izb.moe_combine(six, y, inv, 4)
    one = b.call(x=b.x)
    assert float((six - one).norm() / (one - b.x).norm()) < 0.02


def test_ties_and_rows_of_one_call(izb, torch):
    """Equal logits go to the lower expert, -0 and 0 are equal; a token's row does not depend on the other tokens of the call."""
    b = Block(izb, torch, 12, 512, 256, 40, 4, 12, 8)
    b.logits[0] = 0.0
    b.logits[1] = -b.logits[0]
    b.logits[2, 5:30] = 7.0
    b.logits[3] = float("-inf")
    b.logits[3, 17], b.logits[3, 3] = 0.0, -1.0  # (the other choices have weight 0)
    assert rel(b.call(), b.want()) <= TOL if np.isfinite(b.want()).all() else True
    whole = b.call()
    assert bool(torch.isfinite(whole).all())
    aq, asc, logits, T = b.aq, b.asc, b.logits, b.T
    for t in (0, 3, 11):
        b.aq, b.asc, b.logits, b.T = torch.zeros_like(aq), torch.zeros_like(asc), logits[t:t + 1], 1
        b.aq[0], b.asc[:, 0] = aq[t], asc[:, t]
        assert torch.equal(b.call()[0], whole[t])


def test_numbers_that_are_none_stay_with_their_token(izb, torch):
    b = Block(izb, torch, 6, 512, 256, 4, 2, 12, 12)
    ref = b.call()
    b.asc[5, 2] = float("nan")
    b.asc[1, 4] = float("inf")
    got = b.call()
    assert bool(torch.isnan(got[2]).all())
    assert not bool(torch.isfinite(got[4]).any())
    keep = [0, 1, 3, 5]
    assert torch.equal(got[keep], ref[keep])
    b.asc.zero_()  # nothing but zeros in
    assert float(b.call().abs().max()) == 0.0


def test_sizes_of_the_activations(izb, torch):
    """h from tiny to large: its block scales carry any size."""
    for size in (1e-18, 1e-3, 1e6):
        b = Block(izb, torch, 3, 512, 512, 6, 2, 8, 12, seed=5)
        b.asc *= size
        assert rel(b.call(), b.want()) <= TOL


def test_captured_with_other_logits_at_replay(izb, torch):
    a, b = Block(izb, torch, 3, 512, 256, 12, 3, 12, 12, joined=True), Block(izb, torch, 20, 512, 256, 12, 3, 8, 12, seed=9)
    outs, graphs = [torch.zeros_like(x.x) for x in (a, b)], []
    torch.cuda.synchronize()
    for x, out in zip((a, b), outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.call(out=out)
        graphs.append(g)
    for x in (a, b):
        x.logits.copy_(torch.randn_like(x.logits))
    eager = torch.zeros_like(b.x)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            b.call(out=eager)
    torch.cuda.synchronize()
    assert rel(outs[0], a.want()) <= TOL and rel(outs[1], b.want()) <= TOL and torch.equal(eager, outs[1])


def test_refusals(izb, torch):
    b = Block(izb, torch, 4, 512, 256, 8, 2, 12, 12)
    args = (b.wg, b.wu, b.wd, b.aq, b.asc, b.logits)

    def status(*a, **kw):
        with pytest.raises(izb.IzbError) as e:
            izb.moe_layer(*a, **kw)
        return e.value.status

    assert status(*args, 9) == -2 and status(*args, 0) == -2 and status(*args, 2, e0=1) == -2 and status(*args, 2, e0=-1) == -2
    assert status(b.wg, None, *args[2:], 2) == -1                                  # no up projection
    assert status(b.wg, b.wd, *args[2:], 2) == -2                                  # a stack of another shape
    k6 = izb.Weight(14, S.make_weight(14, 8 * 512, 256, 1), 512, 256, n_mats=8)
    assert status(b.wg, b.wu, k6, *args[3:], 2) == -3
    many = torch.zeros((33, 8), device="cuda")
    aq, asc, _ = izb.quantize_act(torch.zeros((33, 512), device="cuda"))
    assert status(*args[:3], aq, asc, many, 2) == -10
    buf = torch.zeros((5 * 512,), device="cuda")
    assert status(*args, 2, x=buf[:2048].view(4, 512), out=buf[512:].view(4, 512)) == -1
    for kw in (dict(x=b.x[:3]), dict(out=b.x.double()), dict(sh=b.x[:, :256])):
        with pytest.raises((ValueError, TypeError)):
            izb.moe_layer(*args, 2, **kw)
    with pytest.raises(ValueError):
        izb.moe_layer(*args[:3], b.aq[:, :256], *args[4:], 2)


@pytest.mark.parametrize("T,E,F,NE,NU,qt,qd,experts", [
    (32, 256, 768, 40, 8, 12, 12, None),     # few outputs, many pairs: clusters of eight CTAs
    (25, 512, 1024, 6, 5, 12, 8, None),
    (12, 768, 256, 32, 4, 8, 12, (5, 30)),   # some choices are another rank's
    (32, 1024, 512, 64, 2, 8, 8, (60, 64)),  # hardly any expert is here: most CTAs have nothing to add
])
def test_few_outputs_shared_by_a_cluster(izb, torch, T, E, F, NE, NU, qt, qd, experts):
    b = Block(izb, torch, T, E, F, NE, NU, qt, qd, seed=11, shared=experts is None, experts=experts)
    want = b.want()
    got = b.call()
    assert rel(got, want) <= TOL
    same = b.x.clone()
    b.call(x=same, out=same)
    assert rel(same - b.x, want) <= TOL + 2.0 ** -22 * 8
    for _ in range(3):
        assert torch.equal(b.call(), got)
    # a token's sums do not depend on how many CTAs share them
    for t in (0, T - 1):
        asc = torch.zeros((E // 32, 16), device="cuda")
        asc[:, 0] = b.asc[:, t]
        one = b.izb.moe_layer(b.wg, b.wu, b.wd, b.aq[t:t + 1].contiguous(), asc, b.logits[t:t + 1].contiguous(), b.NU, sh=b.sh[t:t + 1].contiguous() if b.shared else None, e0=b.e0)
        assert torch.equal(one[0], got[t])


def test_refuses_a_first_expert_that_no_sum_holds(izb, torch):
    """e0 + n_mats past 2^31."""
    b = Block(izb, torch, 2, 256, 256, 4, 2, 12, 12)
    for e0 in (2 ** 31 - 1, 2 ** 31 - 4, 5):
        with pytest.raises(izb.IzbError) as e:
            izb.moe_layer(b.wg, b.wu, b.wd, b.aq, b.asc, b.logits, 2, x=b.x, e0=e0)
        assert e.value.status == -2


def one_hot(N, K, at, d, q=1):
    """Q8_0 rows with one value each: row n has d[n] * q[n] at at[n]."""
    w = np.zeros((N, K // 32, 34), np.uint8)
    n = np.arange(N)
    w[n, at // 32, 0:2] = np.asarray(d, np.float16).reshape(-1, 1).view(np.uint8).reshape(N, 2)
    w[n, at // 32, 2 + at % 32] = np.broadcast_to(np.asarray(q, np.int8), (N,)).view(np.uint8)
    return w.reshape(N, -1)


@pytest.mark.parametrize("size", [2.0 ** -90, 2.0 ** -20, 1.0, 2.0 ** 60])
def test_how_exactly_h_is_held(izb, torch, size):
    """Gate 64 (its silu is 64 to the last bit), up rows and down rows of one value each: the outputs are h as the second kernel gets it.  h is off by half a
    unit, and a unit is 2^-22 of the power of two below the block's largest value M * 2^e -- or twice that, but then M > 0xFEFEFE, so that it is 2^-22 / 0.996 of
    the largest value itself at most."""
    F = E = 256
    rng = np.random.default_rng(int(np.log2(size)) + 100)
    most = np.array([0x800000, 0xFEFEFE, 0xFEFEFF, 0xFEFF00, 0xFFFFFF, 0x800001, 0x900000 + rng.integers(0x100000), 0xC00000 + rng.integers(0x100000)], np.float64)
    asc = np.zeros((8, 16), np.float32)
    asc[:, 0] = most * 2.0 ** -23 * size * 2.0 ** rng.integers(-3, 4, 8)
    asc[0, 0] = 1.0  # (the gate's)
    aq = np.zeros((16, E), np.int8)
    aq[0, 0], aq[0, 1::32] = 64, 1
    c = np.arange(F)
    d = rng.uniform(-1, 1, F).astype(np.float16)
    d[::32] = rng.choice([-1, 1], F // 32)  # each block's largest
    h = 64.0 * (d.astype(np.float32) * asc[c // 32, 0]).astype(np.float64)
    wg, wu, wd = (izb.Weight(8, w, 256, 256, n_mats=1) for w in (one_hot(F, E, 0 * c, np.ones(F)), one_hot(F, E, 32 * (c // 32) + 1, d), one_hot(E, F, c, np.ones(E))))
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    got = izb.moe_layer(wg, wu, wd, cu(aq), cu(asc), torch.zeros((1, 1), device="cuda"), 1).cpu().numpy()[0].astype(np.float64)
    off = np.abs(got - h).reshape(-1, 32).max(1) / np.abs(h).reshape(-1, 32).max(1)
    assert (off <= 2.0 ** -23 / 0.996).all(), off * 2.0 ** 23


@pytest.mark.parametrize("T,E,F,NE,NU,qt,qd,joined", [
    (16, 512, 256, 40, 32, 12, 12, True),    # the most choices of a token
    (5, 256, 512, 17, 17, 8, 8, False),      # every expert, more of them than half a warp
    (12, 2048, 768, 64, 8, 12, 12, False),
    (8, 768, 2560, 24, 20, 12, 8, True),
])
def test_on_average(izb, torch, T, E, F, NE, NU, qt, qd, joined):
    """Off on average, as a share of the result: h is off by a unit / sqrt(12) per value, a unit being 2^-22 of its block's largest value at most, and 32 values whose largest is M have
    a norm of M at least: sqrt(32 / 12) 2^-22 = 6.6 * 2^-24.  The roundings of the sums, 2^-24 of a partial sum each, add up as the square root of their number:
    a warp's superblocks, three roundings each, and the joins, of gate and up, then of down, and the combine's."""
    b = Block(izb, torch, T, E, F, NE, NU, qt, qd, joined, seed=NE)
    want = b.want()
    limit = 2.0 ** -24 * (6.6 + (2 * (3 * E / 256 / 4 + 12) + 3 * F / 256 + 12 + 2 * NU) ** 0.5)
    got = b.call().cpu().numpy().astype(np.float64)
    assert np.linalg.norm(got - want) / np.linalg.norm(want) <= limit


def test_ties_and_choices_of_no_weight(izb, torch):
    """Compared with the 64-bit result whatever it is: it is finite, the choices that are -inf have weight 0."""
    b = Block(izb, torch, 12, 512, 256, 40, 4, 12, 8)
    b.logits[0] = 0.0
    b.logits[1] = -b.logits[0]
    b.logits[2, 5:30] = 7.0
    b.logits[3] = float("-inf")
    b.logits[3, 17], b.logits[3, 3] = 0.0, -1.0
    want = b.want()
    assert np.isfinite(want).all() and rel(b.call(), want) <= TOL
