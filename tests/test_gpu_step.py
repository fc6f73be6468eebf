"""A decode step's new parts together, as a server would run them: a projection with each request's adapter, the expert block, the head with each request's
rules on its logits -- eager and captured, against the same steps in 64 bits."""
import numpy as np
import pytest

from arcinferzero_b200 import synth as S
from oracle import oracle as O
from tests.test_gpu_moe_layer import dense, rows

pytestmark = pytest.mark.gpu


def test_decode_step(izb):
    import torch
    T, E, F, NE, NU, V, R = 6, 512, 256, 16, 4, 5003, 16
    rng = np.random.default_rng(11)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    wo, wg, wu, wd, wr, wh = rows(12, E, E, 1), rows(12, NE * F, E, 2), rows(12, NE * F, E, 3), rows(8, NE * E, F, 4), rows(8, NE, E, 5), rows(8, V, E, 6)
    Wo, Wr, Wh = izb.Weight(12, wo, E, E), izb.Weight(8, wr, NE, E), izb.Weight(8, wh, V, E)
    Wgu, Wd = izb.gateup_weight(12, wg, wu, F, E, n_mats=NE), izb.Weight(8, wd, E, F, n_mats=NE)
    A, B = (rng.standard_normal((3, R, E)) / E ** 0.5).astype(np.float16), rng.standard_normal((3, E, R)).astype(np.float16)
    scales, adapter = np.array([0.5, 1.0, 2.0], np.float32), np.array([0, -1, 2, 1, 0, 2], np.int32)
    norm = (1 + 0.1 * rng.standard_normal(E)).astype(np.float32)
    x0, a0 = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((T, E)).astype(np.float32)
    params = np.tile(np.array([[1.2, 0.3, 0.1, 0.8]], np.float32), (T, 1))
    hist, off = rng.integers(0, V, 5 * T).astype(np.int32), np.arange(0, 5 * T + 1, 5).astype(np.int32)
    mask = rng.integers(0, 2 ** 32, (T, (V + 31) // 32), dtype=np.uint64).astype(np.uint32).view(np.int32)
    d = {k: cu(v) for k, v in dict(A=A, B=B, scales=scales, adapter=adapter, norm=norm, a0=a0, params=params, hist=hist, off=off, mask=mask, seg=np.arange(T + 1, dtype=np.int32)).items()}
    x = cu(x0)

    def step():
        aq, asc, _ = izb.quantize_act(d["a0"])
        izb.matmul(Wo, aq, asc, T, out=x, acc=1)
        izb.lora_add(d["A"], d["B"], d["scales"], aq, asc, T, d["seg"], d["adapter"], x)
        mid = x.clone()
        aq2, asc2, _ = izb.rmsnorm_quant(x, d["norm"], 1e-6)
        router = izb.matmul(Wr, aq2, asc2, T)[:T]
        izb.moe_layer(Wgu, None, Wd, aq2, asc2, router, NU, x=x, out=x)
        aq3, asc3, _ = izb.rmsnorm_quant(x, d["norm"], 1e-6)
        logits = izb.matmul(Wh, aq3, asc3, T)[:T]
        raw = logits.clone()
        _, best, logz = izb.logits_process(logits, params=d["params"], hist=(d["hist"], d["off"]), mask=d["mask"])
        return aq, asc, mid, aq2, asc2, router.clone(), x.clone(), raw, logits.clone(), best, logz

    first = step()
    x.copy_(cu(x0))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again = step()
    x.copy_(cu(x0))
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))

    aq, asc, mid, aq2, asc2, router, after, raw, logits, best, logz = (t.cpu().numpy() for t in first)
    # each part from the inputs it had (an int8 rounding that goes the other way would move everything after it): 1e-5 of the largest value, as the products' tests
    near = lambda got, ref: float(np.abs(got - ref).max() / np.abs(ref).max()) <= 1e-5
    deq = lambda q, s: q[:T].astype(np.float64) * np.repeat(s[:, :T].astype(np.float64), 32, 0).T
    v = deq(aq, asc)
    ref = x0.astype(np.float64) + O.matmul(12, wo, E, aq, asc, T, "f64")[:T]
    for t, a in enumerate(adapter):
        if a >= 0:
            ref[t] += scales[a] * ((v[t] @ A[a].astype(np.float64).T) @ B[a].astype(np.float64).T)
    assert near(mid, ref)
    v, ref = deq(aq2, asc2), mid.astype(np.float64)
    for t in range(T):
        order = sorted(range(NE), key=lambda e: (-router[t, e], e))[:NU]
        w = np.exp(router[t, order].astype(np.float64) - router[t, order[0]])
        for e, we in zip(order, w / w.sum()):
            gate, up = (dense(12, m[e * F:(e + 1) * F], E) @ v[t] for m in (wg, wu))
            ref[t] += we * (dense(8, wd[e * E:(e + 1) * E], F) @ (gate / (1 + np.exp(-gate)) * up))
    assert near(after, ref)
    from tests.test_gpu_logits import same_bits, want
    w, wb, wz = want(raw, params, [hist[5 * t:5 * t + 5].tolist() for t in range(T)], None, mask)
    assert same_bits(logits, w) and (best == wb).all() and np.abs(logz - wz).max() <= 1e-4
