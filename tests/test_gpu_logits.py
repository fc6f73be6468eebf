"""Each request's rules on its row of logits (izb_logits_process): the new logits bit for bit against the same operations in numpy's f32, the best token
exact, log(sum(exp)) against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
f4 = np.float32


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


def want(l, params=None, hist=None, bias=None, mask=None, mask_row=None):
    """hist: a list of token lists per row; bias: a list of (id, value) lists per row."""
    out = l.astype(f4).copy()
    rows, V = out.shape
    with np.errstate(all="ignore"):
        for r in range(rows):
            o = out[r]
            rep, pres, freq, temp = params[r] if params is not None else (f4(1), f4(0), f4(0), f4(0))
            if params is not None and hist is not None:
                h = np.array([v for v in hist[r] if 0 <= v < V], np.int64)
                v, c = np.unique(h, return_counts=True)
                s = o[v]
                s = np.where(s > 0, s / rep, s * rep).astype(f4)
                o[v] = s - ((freq * c.astype(f4)).astype(f4) + pres).astype(f4)
            if bias is not None:
                last = {i: b for i, b in bias[r] if 0 <= i < V}
                for i, b in last.items():
                    o[i] = o[i] + f4(b)
            m = -1 if mask is None else r if mask_row is None else int(mask_row[r])
            if mask is not None and 0 <= m < len(mask):
                bits = (mask[m].view(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1
                o[bits.reshape(-1)[:V] == 0] = -np.inf
            if temp > 0:
                o[:] = o / temp
    best, logz = [], []
    for r in range(rows):
        o = out[r].astype(np.float64)
        top = np.nanmax(np.where(np.isnan(o), -np.inf, o))
        best.append(int(np.flatnonzero(out[r] == top)[0]) if top > -np.inf else 0)
        with np.errstate(all="ignore"):
            logz.append(np.nan if np.isnan(o).any() else top if np.isinf(top) else top + np.log(np.exp(o - top).sum()))
    return out, np.array(best), np.array(logz)


def same_bits(a, b):
    a, b = np.ascontiguousarray(a, f4), np.ascontiguousarray(b, f4)
    return bool((np.isnan(a) == np.isnan(b)).all() and (a.view(np.uint32)[~np.isnan(a)] == b.view(np.uint32)[~np.isnan(b)]).all())


def ragged(torch, lists, dtype=np.int32):
    off = np.cumsum([0] + [len(x) for x in lists]).astype(np.int32)
    flat = np.array([v for x in lists for v in x], dtype)
    return torch.from_numpy(flat).cuda(), torch.from_numpy(off).cuda()


def run(izb, torch, l, params=None, hist=None, bias=None, mask=None, mask_row=None, pad=(0, 0), skip=0):
    """Through a padded input and output, NaN between the rows; `skip`: floats before the first."""
    rows, V = l.shape
    cu = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()
    def buffer(p):
        return torch.full((rows * (V + p) + skip,), float("nan"), device="cuda")
    bi, bo = buffer(pad[0]), buffer(pad[1])
    li, lo = bi[skip:].view(rows, V + pad[0])[:, :V], bo[skip:].view(rows, V + pad[1])[:, :V]
    li.copy_(cu(l))
    kw = dict(params=cu(params), mask=cu(mask), mask_row=cu(mask_row))
    if hist is not None:
        kw["hist"] = ragged(torch, hist)
    if bias is not None:
        ids, off = ragged(torch, [[i for i, _ in b] for b in bias])
        kw["bias"] = (ids, ragged(torch, [[v for _, v in b] for b in bias], f4)[0], off)
    out, best, logz = izb.logits_process(li, out=lo, **kw)
    assert out is lo and bool(torch.isnan(bo[skip:].view(rows, V + pad[1])[:, V:]).all() and torch.isnan(bo[:skip]).all())
    w, wb, wz = want(l, params, hist, bias, mask, mask_row)
    assert same_bits(out.cpu().numpy(), w)
    assert (best.cpu().numpy() == wb).all()
    z = logz.cpu().numpy().astype(np.float64)
    # a sum of V positive f32 terms in chains of at most V / 512 + 64, each term's exp within a few units of its last place, its argument within
    # 2^-24 of its size (weighted by the term, at most log V), and the logarithm's and the sum's own rounding
    room = (V / 512 + 128) * 2.0 ** -24 + 2.0 ** -23 * np.abs(np.where(np.isfinite(wz), wz, 0))
    fin = np.isfinite(wz)
    assert (np.isnan(z) == np.isnan(wz)).all() and (z[np.isinf(wz)] == wz[np.isinf(wz)]).all() and (np.abs(z[fin] - wz[fin]) <= room[fin]).all(), np.abs(z[fin] - wz[fin]) / room[fin]
    # in place the same
    izb.logits_process(li, **kw)
    assert same_bits(li.cpu().numpy(), w)


def setup(rows, V, seed, hist=50, bias=8):
    rng = np.random.default_rng(seed)
    l = (rng.standard_normal((rows, V)) * 3).astype(f4)
    params = np.stack([rng.uniform(1, 1.6, rows), rng.uniform(0, 1, rows), rng.uniform(0, 0.5, rows), np.where(rng.random(rows) < 0.3, 0, rng.uniform(0.3, 1.5, rows))], 1).astype(f4)
    hists = [(rng.random(rng.integers(0, hist + 1)) ** 3 * V).astype(int).tolist() for _ in range(rows)]
    biases = [[(int(i), float(rng.standard_normal() * 4)) for i in rng.integers(0, V, rng.integers(0, bias + 1))] for _ in range(rows)]
    words = (V + 31) // 32
    mask = rng.integers(0, 2 ** 32, (rows, words), dtype=np.uint64).astype(np.uint32).view(np.int32)
    mask_row = rng.integers(-1, rows, rows).astype(np.int32)
    return l, params, hists, biases, mask, mask_row


@pytest.mark.parametrize("rows,V,pad,skip", [(1, 1, (0, 0), 0), (1, 5, (0, 3), 1), (3, 33, (0, 0), 0), (2, 1000, (4, 8), 0), (4, 4096, (0, 0), 0), (5, 4097, (0, 0), 0), (3, 32003, (1, 2), 3),
                                             (2, 151936, (0, 0), 0), (1, 152065, (0, 0), 2), (9, 65536, (0, 1), 0), (300, 777, (3, 0), 0), (2, 600000, (0, 0), 0)])
def test_all_rules(izb, torch, rows, V, pad, skip):
    l, params, hist, bias, mask, mask_row = setup(rows, V, V + rows, hist=700)
    run(izb, torch, l, params, hist, bias, mask, mask_row, pad, skip)


@pytest.mark.parametrize("which", ["none", "params", "hist", "bias", "mask", "mask_row"])
def test_one_rule_at_a_time(izb, torch, which):
    l, params, hist, bias, mask, mask_row = setup(6, 9001, 3)
    kw = {"none": {}, "params": dict(params=params), "hist": dict(params=params, hist=hist), "bias": dict(bias=bias), "mask": dict(mask=mask), "mask_row": dict(mask=mask, mask_row=mask_row)}[which]
    run(izb, torch, l, **kw)


def test_rows_that_nothing_is_left_of_and_infinities(izb, torch):
    V = 5000
    l, params, hist, bias, mask, mask_row = setup(8, V, 4)
    params[:, 3] = [0, 0.5, 0, 2, 0, 1, 0, 1]
    mask[:] = -1
    mask[0] = 0                                    # nothing allowed
    mask[1], l[1] = 0, np.nan                      # NaN behind the mask
    mask[1, 3], l[1, 96:128] = 1 << 30, 2.0        # one token left
    l[2] = -np.inf
    l[3, 17] = np.inf
    l[4, 9], l[4, 4321] = np.nan, 50.0             # NaN is never the best
    l[5] = np.finfo(f4).min
    l[6] = 1.25                                    # all equal: the lowest index
    bias[6], hist[6] = [], []
    bias[7] = [(4999, -np.inf), (3, np.inf), (3, 1.0)]  # the last entry counts
    run(izb, torch, l, params, hist, bias, mask)


def test_tokens_that_come_often_or_are_none(izb, torch):
    V = 20000
    l, params, _, _, _, _ = setup(3, V, 5)
    hist = [[7] * 70000 + [V - 1] * 3, [-1, V, 2 ** 31 - 1, -2 ** 31, 5, 5], []]
    bias = [[(5, 1.0), (5, 2.0), (5, 3.0)], [(-1, 9.0), (V, 9.0), (4, -2.0)], []]
    run(izb, torch, l, params, hist, bias)


def test_offsets_past_the_arrays_are_cut(izb, torch):
    V = 3000
    l, params, _, _, _, _ = setup(2, V, 6)
    cu = lambda a, d=np.int32: torch.from_numpy(np.array(a, d)).cuda()
    for off in ([-3, 2, 1000], [0, 5, 2], [9, 9, 9]):
        out, _, _ = izb.logits_process(cu(l, f4), out=torch.empty((2, V), device="cuda"), params=cu(params, f4), hist=(cu([1, 2, 3, 4]), cu(off)))
        lo, hi = np.clip(off[:2], 0, 4), np.clip(off[1:], 0, 4)
        w, _, _ = want(l, params, [[1, 2, 3, 4][a:max(a, b)] for a, b in zip(lo, hi)])
        assert same_bits(out.cpu().numpy(), w)


def test_captured_with_other_histories_at_replay(izb, torch):
    V, rows = 40000, 3
    l, params, hist, _, mask, _ = setup(rows, V, 8)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    li, lo, pd, md, mr = cu(l), torch.zeros((rows, V), device="cuda"), cu(params), cu(mask), torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    tok, off = torch.zeros(64, dtype=torch.int32, device="cuda"), torch.zeros(rows + 1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, best, logz = izb.logits_process(li, out=lo, params=pd, hist=(tok, off), mask=md, mask_row=mr)
    for step in range(3):
        h = [np.random.default_rng(step + r).integers(0, V, 20 * step % 21).tolist() for r in range(rows)]
        flat, o = ragged(torch, h)
        tok[:flat.numel()] = flat
        off.copy_(o)
        mr.copy_(torch.tensor([step - 1, -1, 2], dtype=torch.int32))
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.replay()
        torch.cuda.synchronize()
        w, wb, _ = want(l, params, h, None, mask, np.array([step - 1, -1, 2]))
        assert same_bits(lo.cpu().numpy(), w) and (best.cpu().numpy() == wb).all()


def test_refused_by_the_binding(izb, torch):
    l = torch.zeros((3, 100), device="cuda")
    i = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")
    for kw in (dict(out=l[:2]), dict(out=l.double()), dict(params=torch.zeros((3, 3), device="cuda")), dict(hist=(i(4), i(3)), params=torch.zeros((3, 4), device="cuda")),
               dict(bias=(i(4), torch.zeros(3, device="cuda"), i(4))), dict(mask=i(4)), dict(mask=i(12).view(3, 4), mask_row=i(2)), dict(hist=(i(4).long(), i(4)))):
        with pytest.raises((ValueError, TypeError)):
            izb.logits_process(l, **kw)
    for kw in (dict(hist=(i(4), i(4))), dict(mask=i(9).view(3, 3)), dict(mask=i(8).view(2, 4))):
        with pytest.raises(izb.IzbError):
            izb.logits_process(l, **kw)
    with pytest.raises(ValueError):
        izb.logits_process(l.t())
