"""Adapters (izb_lora_add): the three forms one by one, in both types, with bounds that an operand of fewer pieces does not meet."""
import numpy as np
import pytest

from tests.test_gpu_lora import Case, off

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as t
    assert t.cuda.is_available()
    return t


def spread(case):
    """What the adapters' part alone may be off by on average, as a share of its own norm.  A matrix instruction's f32 sums need not be rounded to the nearest: cut off, a
    sum is short by half a unit, 2^-24 of itself, on average, and always to the same side, so that n of them in a row add up.  The norm of the sum after i of n
    like terms is sqrt(i / n) of the last one's, hence at most 2/3 n 2^-24 for the second product's n = pieces * R / 16, and 2 more for a block of the first one.  Other sums
    are rounded, and independent roundings add up as the square root of their number: a warp's blocks of K (a fourth of all of them at most), the joins of
    warps and CTAs (24), the pieces' own and the outputs' (16, generously)."""
    pieces = 0 if case.T <= len(case.lens) else 2 if case.A.dtype == case.torch.float16 else 3  # (single rows: f32 throughout)
    n = pieces * case.R / 16
    limit = 2.0 ** -24 * (2 + 2 / 3 * n + (case.K / 128 + 40) ** 0.5)
    assert limit < 2.0 ** -24 * 41 or case.R > 128  # (what u in two bf16 pieces instead of three is off by, see below)
    return limit


def check(izb, torch, c):
    N, T, last = c.N, c.T, c.first + sum(c.lens)
    want, room = c.want(c.base)
    got = c.base.clone()
    izb.lora_add(*c.args(), got, ranks=c.rk)
    assert off(got[c.first:last], want[c.first:last], room[c.first:last]) <= 1
    assert torch.equal(got[:c.first], c.base[:c.first]) and torch.equal(got[last:], c.base[last:])
    alone, _ = c.want(torch.zeros_like(c.base))
    part = torch.zeros((T, N + 3), device="cuda")  # (rows that start anywhere)
    izb.lora_add(*c.args(), part, c_off=1)
    if float(alone.norm()):
        assert float((part[:, 1:N + 1].double() - alone).norm() / alone.norm()) <= spread(c)
    assert float(part[:, 0].abs().max()) == 0.0 and float(part[:, N + 1:].abs().max()) == 0.0
    lines = torch.zeros((T, (N + 3) // 4 * 4), device="cuda")[:, :N]
    izb.lora_add(*c.args(), lines)
    assert torch.equal(lines, part[:, 1:N + 1])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,ranks,N,K,empty", [
    (1, [256], 133, 1024, 0),
    (2, [8, 24], 1000, 768, 1),
    (5, [17, 64, 33], 515, 256, 0),                 # fewer blocks of K than warps
    (28, [80, 16, 128, 1], 321, 2304, 3),           # clusters of fifteen CTAs
    (40, [16, 32], 77, 5120, 0),                    # eleven
    (64, [8, 16, 32, 64], 700, 1280, 0),            # six
    (100, [256, 240, 48], 65, 512, 20),             # four
    (300, [64, 5], 40, 512, 0),                     # more segments than threads, more rows than places for clusters
])
def test_one_row_per_request(izb, torch, T, ranks, N, K, empty, dtype):
    """T <= segments: the form of decode steps.  Every third request has another adapter, every seventh none."""
    lens = [1] * T + [0] * empty
    check(izb, torch, Case(izb, torch, lens, [-1 if i % 7 == 6 else i % len(ranks) for i in range(len(lens))], ranks, N, K, dtype, seed=T))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,ranks,N,K", [
    ([3, 8, 1, 0, 5], [128, 16], 203, 768),
    ([8] * 5, [256], 50, 1280),
    ([2, 1] * 200, [16, 48], 36, 256),              # more segments than threads
])
def test_a_few_rows_per_request(izb, torch, lens, ranks, N, K, dtype):
    check(izb, torch, Case(izb, torch, lens, [i % (len(ranks) + 1) - 1 for i in range(1, len(lens) + 1)], ranks, N, K, dtype, seed=3, behind=2))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,ranks,N,K", [
    ([9, 64, 65, 20], [16, 64], 300, 512),
    ([130, 33], [256, 112], 130, 768),
    ([9, 0, 10, 8, 11] * 120, [32, 80, 16], 36, 256),  # more segments than threads
    ([700], [48], 2100, 5120),
])
def test_prompts(izb, torch, lens, ranks, N, K, dtype):
    check(izb, torch, Case(izb, torch, lens, [i % (len(ranks) + 1) - 1 if len(lens) > 4 else i % len(ranks) for i in range(len(lens))], ranks, N, K, dtype, seed=9, first=1, behind=4))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[64] + [0] * 63, [0] * 63 + [64], [437] + [1] * 63, [1] * 63 + [450]], ids=["64 and none", "none and 64", "437 and 63", "63 and 450"])
def test_tables_of_one_size(izb, torch, lens, dtype):
    """A step's table of 64 segments: prompts beside empty segments and decode rows, in whichever form the averages pick."""
    check(izb, torch, Case(izb, torch, lens, [i % 3 for i in range(len(lens))], [16, 64, 32], 150, 512, dtype, seed=5))


def pieces_of(u, count):
    """u rounded to `count` bf16 pieces, one after the other."""
    left, out = u.astype(np.float32), np.zeros(u.shape)
    for _ in range(count):
        b = left.view(np.uint32)
        h = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
        out += h
        left = left - h
    return out


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens,R", [([1, 1, 1], 16), ([1, 1], 64), ([1], 112), ([8, 5, 3], 16), ([7, 8], 48), ([8], 256), ([64, 9], 32), ([40], 80), ([17, 70], 256)])
def test_numbers_that_need_every_bit(izb, torch, lens, R, dtype):
    """u of 24 bits, each the sum of two activations times powers of two; every output is one of them times a power of two.  bf16 pieces hold them exactly (24 bits in
    three), f16 pieces to 2^-23 of the row's largest (that one is 2^13 and more after its power of two, what the first piece leaves of it is 4 at most, and the
    second piece is off by 2^-10 at most); single rows are f32 throughout.  Two bf16 pieces alone, in the oracle, miss most outputs (a single row has as few as 25 values of u, some of them short)."""
    K, rng = 512, np.random.default_rng(R + len(lens))
    T, N = sum(lens), 2 * R + 3
    asc = np.zeros((K // 32, (T + 15) // 16 * 16), np.float32)
    aq = np.zeros((asc.shape[1], K), np.int8)
    k1, k2 = rng.integers(0, K // 2, T), rng.integers(K // 2, K, T)
    for t in range(T):
        aq[t, k1[t]], aq[t, k2[t]] = 1, -1
        asc[k1[t] // 32, t], asc[k2[t] // 32, t] = rng.uniform(1, 2, 2).astype(np.float32)
    a1, a2 = 2.0 ** rng.integers(-2, 3, R), 2.0 ** rng.integers(-4, 1, R) * rng.choice([-1, 1], R)
    A = np.where(np.arange(K) < K // 2, a1[:, None], a2[:, None])
    of = rng.permutation(np.arange(N) % R)
    B = np.zeros((N, R))
    B[np.arange(N), of] = 2.0 ** rng.integers(-3, 4, N)
    x1, x2 = asc[k1 // 32, np.arange(T)].astype(np.float64), asc[k2 // 32, np.arange(T)].astype(np.float64)
    u = (x1[:, None] * a1 - x2[:, None] * a2).astype(np.float32)  # (rounded once; each product is exact)
    scale = B[np.arange(N), of]
    want = (u.astype(np.float64)[:, of] * scale).astype(np.float32)
    dt = torch.float16 if dtype == "f16" else torch.bfloat16
    cu = lambda v: torch.from_numpy(np.ascontiguousarray(v)).cuda()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    out = torch.zeros((T, N), device="cuda")
    izb.lora_add(cu(A[None]).to(dt), cu(B[None]).to(dt), torch.ones(1, device="cuda"), cu(aq), cu(asc), T, i32(np.cumsum([0] + lens).tolist()), i32([0] * len(lens)), out)
    got = out.cpu().numpy()
    if dtype == "bf16" or T <= len(lens):
        assert (got == want).all(), float(np.abs(got - want).max())
    else:
        assert (np.abs(got.astype(np.float64) - want) <= 2.0 ** -23 * np.abs(u).max(1, keepdims=True) * scale).all()
    z = rng.standard_normal(100000).astype(np.float32)
    assert 40 < np.linalg.norm(pieces_of(z, 2) - z) / np.linalg.norm(z) * 2.0 ** 24 < 42
    assert ((pieces_of(u, 2)[:, of] * scale).astype(np.float32) == want).mean() < 0.5 and ((pieces_of(u, 3)[:, of] * scale).astype(np.float32) == want).all()
