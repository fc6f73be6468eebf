"""Adapters of many requests beside a projection (izb_lora_add) against the formula in 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


class Case:
    def __init__(self, izb, torch, lens, adapters, ranks, N, K, dtype, seed=0, first=0, behind=0, R=None):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed + 7)
        rn = lambda *s: torch.randn(s, generator=gen, device="cuda")
        self.torch, self.lens, self.adapters, self.ranks, self.N, self.K = torch, lens, adapters, ranks, N, K
        self.first, self.T = first, first + sum(lens) + behind
        self.R, n = R or (max(ranks) + 15) // 16 * 16, len(ranks)
        self.aq, self.asc, _ = izb.quantize_act(rn(self.T, K))
        self.A, self.B = torch.zeros((n, self.R, K), device="cuda"), torch.zeros((n, N, self.R), device="cuda")
        for a, r in enumerate(ranks):
            self.A[a, :r], self.B[a, :, :r] = rn(r, K) / K ** 0.5, rn(N, r)
        dt = torch.float16 if dtype == "f16" else torch.bfloat16
        self.A, self.B = self.A.to(dt), self.B.to(dt)
        self.scales = 0.5 + torch.rand((n,), generator=gen, device="cuda")
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        self.seg, self.adapter = i32(np.cumsum([first] + list(lens)).tolist()), i32(adapters)
        self.rk = i32(ranks)
        self.base = rn(self.T, N)

    def args(self):
        return self.A, self.B, self.scales, self.aq, self.asc, self.T, self.seg, self.adapter

    def want(self, base):
        """The result in 64 bits, and what its 32-bit sums may be off by: every sum is a chain of at most 128 roundings (32 products of a block, at most 32
        blocks of a warp, 64 partial sums) of terms whose absolute values add up to at most the sums below; an operand held in pieces is off by 2^-21 of the
        largest value of its row."""
        f8 = self.torch.float64
        out, room, t = base.to(f8).clone(), base.to(f8).abs() * 2.0 ** -23, self.first
        for n, a in zip(self.lens, self.adapters):
            if n and 0 <= a < len(self.ranks):
                x = self.aq[t:t + n].to(f8) * self.asc[:, t:t + n].to(f8).repeat_interleave(32, 0).t()
                A, B, s = self.A[a].to(f8), self.B[a].to(f8), float(self.scales[a])
                u = x @ A.t()
                out[t:t + n] += s * (u @ B.t())
                du = 128 * 2.0 ** -24 * (x.abs() @ A.abs().t()) + 2.0 ** -21 * u.abs().amax(1, keepdim=True)
                room[t:t + n] += s * (du @ B.abs().t() + 128 * 2.0 ** -24 * (u.abs() @ B.abs().t()))
            t += n
        return out, room


def off(got, want, room):
    return float(((got.double() - want).abs() / (room + 1e-30)).max())


CASES = [
    # lens, adapters, ranks, N, K, type
    ([1], [0], [16], 64, 256, "f16"),
    ([1], [1], [16, 16], 5120, 5120, "bf16"),
    ([1, 1, 1, 1, 1], [0, -1, 2, 0, 5], [16, 8, 4], 1000, 512, "f16"),           # no adapter, one that is not there
    ([0, 3, 0, 0, 8, 9, 0], [0, 1, 0, 1, 0, 1, 1], [16, 32], 48, 768, "bf16"),   # empty segments
    ([1] * 40, [i % 7 for i in range(40)], [1, 16, 17, 64, 128, 33, 5], 257, 1280, "f16"),
    ([70, 1, 33, 64, 65, 128], [0, 1, 2, 1, 0, 2], [64, 16, 48], 777, 512, "bf16"),
    ([300], [0], [256], 129, 256, "f16"),                                        # the largest rank
    ([17, 200], [0, 1], [256, 240], 36, 2304, "bf16"),
    ([513, 2], [0, 1], [16, 32], 2048, 5120, "f16"),
    ([40, 40, 40], [2, 2, 2], [16, 16, 32], 1, 256, "f16"),                      # one output column
    ([129, 31], [0, 1], [80, 112], 15, 1024, "bf16"),
    ([2000, 48], [0, 1], [32, 96], 640, 17408, "f16"),                           # a long K
    ([3, 2], [1, 0], [128, 112], 100, 512, "f16"),                               # few segments of a few rows: the widest clusters
    ([8, 7], [0, 1], [256, 16], 64, 768, "bf16"),
    ([1, 1], [0, 1], [256, 128], 333, 1280, "f16"),                              # single rows of high rank
    ([1, 1, 1], [0, 1, 0], [48, 80], 70, 512, "bf16"),
    ([4] * 9, [0, 1, 2] * 3, [16, 32, 64], 200, 512, "f16"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}-r{max(c[2])}-{c[3]}x{c[4]}-{c[5]}")
def test_against_64_bits(izb, torch, case):
    c = Case(izb, torch, *case, first=2, behind=5)
    N, T, last = c.N, c.T, c.first + sum(c.lens)
    want, room = c.want(c.base)
    # another buffer for the base, outputs at a column of a wider buffer of odd stride: nothing beside them is written
    for c_off, pad in ((0, 0), (3, 5), (16, 16)):
        out = torch.full((T, c_off + N + pad), float("nan"), device="cuda")
        izb.lora_add(*c.args(), out, base=c.base, c_off=c_off, ranks=c.rk)
        got = out[:, c_off:c_off + N]
        assert off(got[c.first:last], want[c.first:last], room[c.first:last]) <= 1
        assert bool(torch.isnan(out[:c.first]).all() and torch.isnan(out[last:]).all() and torch.isnan(out[:, :c_off]).all() and torch.isnan(out[:, c_off + N:]).all())
    # in place, every rank taken as R (the rows past a rank are zeros)
    same = c.base.clone()
    izb.lora_add(*c.args(), same)
    assert off(same[c.first:last], want[c.first:last], room[c.first:last]) <= 1
    assert torch.equal(same[:c.first], c.base[:c.first]) and torch.equal(same[last:], c.base[last:])
    again = c.base.clone()
    izb.lora_add(*c.args(), again)
    assert torch.equal(again, same)  # no order of its own from run to run


def test_without_a_base(izb, torch):
    """The C entry with base = NULL: the adapters' part alone, zeros where a segment has none."""
    import ctypes as C
    c = Case(izb, torch, [3, 2, 70], [1, -1, 0], [16, 16], 100, 512, "f16")
    out = torch.full((c.T, 100), float("nan"), device="cuda")
    q = lambda t: C.c_void_p(t.data_ptr())
    izb.lib().izb_lora_scratch.restype = C.c_size_t
    scratch = torch.empty(izb.lib().izb_lora_scratch(1, 16, c.T, 3), dtype=torch.uint8, device="cuda")
    rc = izb.lib().izb_lora_add(1, q(c.A), q(c.B), 2, 16, None, q(c.scales), 100, 512, q(c.aq), q(c.asc), c.T, c.asc.shape[1], q(c.seg), q(c.adapter), 3, None, 0, q(out), 100, 0, q(scratch),
                                C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    want, room = c.want(torch.zeros_like(c.base))
    assert off(out, want, room) <= 1 and float(out[3:5].abs().max()) == 0.0


def test_numbers_that_are_none_stay_in_their_row(izb, torch):
    for lens in ([1, 1, 1, 1], [40, 41]):
        c = Case(izb, torch, lens, [0, 1, 0, 1][:len(lens)], [16, 32], 65, 512, "f16")
        ref = c.base.clone()
        izb.lora_add(*c.args(), ref)
        c.asc[3, 1] = float("nan")
        got = c.base.clone()
        izb.lora_add(*c.args(), got)
        assert bool(torch.isnan(got[1]).all())
        keep = [t for t in range(c.T) if t != 1]
        assert torch.equal(got[keep], ref[keep])
        got = c.base.clone()
        got[2, 7] = float("inf")
        izb.lora_add(*c.args(), got)
        assert float(got[2, 7]) == float("inf") and int(torch.isinf(got).sum()) == 1


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e4, 1e30])
def test_sizes_of_the_activations(izb, torch, size):
    """Inner sums far from 1 (past what 16 bits hold) keep their precision."""
    for lens in ([1, 2], [64, 9]):
        c = Case(izb, torch, lens, [0, 1], [16, 32], 80, 512, "f16")
        c.asc *= size
        c.base *= size
        want, room = c.want(c.base)
        got = c.base.clone()
        izb.lora_add(*c.args(), got)
        assert off(got, want, room) <= 1


def test_offsets_and_ranks_out_of_range_are_cut(izb, torch):
    c = Case(izb, torch, [5, 6, 7], [0, 1, 0], [16, 32], 64, 512, "bf16")
    ref = c.base.clone()
    izb.lora_add(*c.args(), ref)
    c.seg[0], c.seg[3] = -5, 1000
    c.rk[0], c.rk[1] = 1000, -3  # (cut to R and to 0)
    got = c.base.clone()
    izb.lora_add(*c.args(), got, ranks=c.rk)
    assert torch.equal(got[:5], ref[:5]) and torch.equal(got[11:], ref[11:]) and torch.equal(got[5:11], c.base[5:11])
    c.seg[1] = 900  # (then decreasing: what comes after is empty or cut)
    izb.lora_add(*c.args(), c.base.clone())
    torch.cuda.synchronize()


def test_captured_with_other_requests_at_replay(izb, torch):
    """A captured call reads segments, adapters and activations at replay; two graphs and an eager call beside them on other streams."""
    c = Case(izb, torch, [1] * 6, [0, 1, 2, 0, 1, 2], [16, 16, 32], 300, 512, "f16")
    d = Case(izb, torch, [70, 30], [1, 0], [64, 16], 300, 512, "bf16", seed=1)
    outs = [torch.zeros((x.T, 300), device="cuda") for x in (c, d)]
    graphs = []
    torch.cuda.synchronize()
    for x, out in zip((c, d), outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            izb.lora_add(*x.args(), out, base=x.base)
        graphs.append(g)
    c.seg.copy_(torch.tensor([0, 0, 2, 3, 3, 3, 6], dtype=torch.int32))
    c.lens = [0, 2, 1, 0, 0, 3]
    d.adapter.copy_(torch.tensor([-1, 1], dtype=torch.int32))
    d.adapters = [-1, 1]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    eager = torch.zeros_like(outs[1])
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            izb.lora_add(*d.args(), eager, base=d.base)
    torch.cuda.synchronize()
    for x, out in zip((c, d, d), (*outs, eager)):
        want, room = x.want(x.base)
        assert off(out, want, room) <= 1


def test_refused_by_the_binding(izb, torch):
    c = Case(izb, torch, [1, 2], [0, 1], [16, 32], 64, 512, "f16")
    out = c.base.clone()
    bad = lambda **kw: izb.lora_add(*[kw.get(n, v) for n, v in zip(("A", "B", "scales", "aq", "asc", "T", "seg", "adapter"), c.args())], kw.get("out", out), base=kw.get("base"))
    for kw in (dict(A=c.A[:1]), dict(A=c.A.transpose(1, 2)), dict(scales=c.scales[:1]), dict(aq=c.aq[:, :256]), dict(T=99), dict(seg=c.seg[:2]), dict(adapter=c.adapter.long()), dict(out=out[:, :63]),
               dict(out=out.t()), dict(base=c.base[:2]), dict(base=c.base.double()), dict(A=c.A.bfloat16())):
        with pytest.raises((ValueError, TypeError)):
            bad(**kw)
    with pytest.raises(izb.IzbError):
        bad(A=c.A[:, :8].contiguous(), B=c.B[:, :, :8].contiguous())


@pytest.mark.parametrize("lens,adapters,ranks,N,K,dtype", [
    ([70, 1, 33, 64, 65, 128], [0, 1, 2, -1, 0, 2], [64, 16, 48], 777, 512, "bf16"),
    ([700, 90], [0, 1], [32, 80], 1001, 256, "f16"),
    ([640], [0], [256], 1499, 256, "bf16"),
    ([64, 9, 130], [0, 0, 0], [16], 67, 256, "f16"),
    ([20], [0], [128], 3, 256, "f16")])
def test_prompts_rows_wherever_they_start(izb, torch, lens, adapters, ranks, N, K, dtype):
    """Base and outputs in windows of wider buffers: the bits are those of rows on 16-byte boundaries, and what is beside the windows stays."""
    c = Case(izb, torch, lens, adapters, ranks, N, K, dtype, first=1, behind=3)
    T, last = c.T, c.first + sum(lens)
    lines = torch.empty((T, (N + 3) // 4 * 4), device="cuda")[:, :N]
    on = torch.zeros((T, (N + 3) // 4 * 4), device="cuda")[:, :N]
    lines.copy_(c.base)
    izb.lora_add(*c.args(), on, base=lines, ranks=c.rk)
    want, room = c.want(c.base)
    assert off(on[c.first:last], want[c.first:last], room[c.first:last]) <= 1
    #            columns before and behind, of the outputs and of the base (None: in place)
    for c0, c1, b0, b1 in ((0, 1, None, 0), (1, 2, None, 0), (3, 0, None, 0), (2, 5, None, 0), (1, 4, 5, 4), (2, 3, 2, 3), (3, 3, 7, 3), (1, 1, 0, 2), (0, 3, 1, 1)):
        wide = torch.full((T, c0 + N + c1), 7.0, device="cuda")
        if b0 is None:
            wide[:, c0:c0 + N] = c.base
            izb.lora_add(*c.args(), wide, c_off=c0, ranks=c.rk)
            rest = c.base
        else:
            base = torch.full((T, b0 + N + b1), float("nan"), device="cuda")
            base[:, b0:b0 + N] = c.base
            izb.lora_add(*c.args(), wide, base=base[:, b0:b0 + N], c_off=c0, ranks=c.rk)
            rest = torch.full((T, N), 7.0, device="cuda")
        got = wide[:, c0:c0 + N]
        assert torch.equal(got[c.first:last], on[c.first:last]), (c0, c1, b0, b1)
        assert torch.equal(got[:c.first], rest[:c.first]) and torch.equal(got[last:], rest[last:])
        assert bool((wide[:, :c0] == 7.0).all() and (wide[:, c0 + N:] == 7.0).all())
