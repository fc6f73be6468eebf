"""The per-request operators of a decode step and of prompt chunks: low-rank adapters beside a shared projection, the whole
mixture-of-experts block of a few tokens, and the rules on the output head's logits.

    listed()             the cases; draw(rng) one more case of the same ranges
    prepare(case, seed)  the inputs on the GPU and the handles a program keeps
    run(state)           one pass: the plain torch form, or with own = True the library's call
    exact(case, seed)    the same results in 64 bits
    work(case)           bytes and operations a pass cannot do without
"""
import math

import torch

own = False

Q8_0, Q4_K = 8, 12
FILE_BYTES = {Q8_0: 272, Q4_K: 144}  # per 256 weights, as in the file


# ------------------------------------------------------------------------------------------------ cases
def _lora(name, lens, adapters, ranks, N, K, dtype, pad=0):
    """Segments of `lens` rows with the adapters named beside them (-1: none); ranks: one per adapter; pad: floats between rows."""
    t = lambda v: ",".join(str(x) for x in v)  # noqa: E731
    c = {"op": "lora", "lens": t(lens), "adapters": t(adapters), "ranks": t(ranks), "N": N, "K": K, "dtype": dtype, "pad": pad}
    return {"name": name, **c} if name else c


def _moe(name, T, E, F, NE, NU, gate, down, joined=False, shared=False):
    """joined: gate and up rows in one interleaved stack; shared: a shared expert's output joins through its gate."""
    c = {"op": "moe", "T": T, "E": E, "F": F, "NE": NE, "NU": NU, "gate": gate, "down": down, "joined": joined, "shared": shared}
    return {"name": name, **c} if name else c


def _logits(name, rows, V, hist, bias, masked, pad=0):
    """hist, bias: the longest history and bias list of a row; masked: the share of the rows with a grammar mask, in percent."""
    c = {"op": "logits", "rows": rows, "V": V, "hist": hist, "bias": bias, "masked": masked, "pad": pad}
    return {"name": name, **c} if name else c


def listed():
    return [
        # One request decodes: the attention output projection of a 5120-wide model with a small adapter.  All latency.
        _lora("lora_one_token", [1], [2], [16] * 4, 5120, 5120, "f16"),
        # A decode step of 64 requests on 32 adapters of unlike ranks, some requests without one: the gate or up projection.
        _lora("lora_decode_64", [1] * 64, [(7 * i) % 36 if (7 * i) % 36 < 32 else -1 for i in range(64)], [(8, 16, 32, 64)[i % 4] for i in range(32)], 17408, 5120, "bf16"),
        # Prompt chunks of unlike lengths (one of a single token, one empty) beside a few decoding requests, an odd output width.
        _lora("lora_ragged_prompts", [611, 1, 0, 333, 1, 1, 1, 900, 47, 129], [0, 1, 2, 3, 0, -1, 1, 2, 3, 1], [64, 16, 64, 32], 2055, 2048, "f16"),
        # Long prompts through the down projection's neighbour: 8192 rows of 17408 outputs, bound by the outputs' bytes.
        _lora("lora_long_prompts", [4096, 2500, 1596], [0, 1, 0], [64, 32], 17408, 5120, "bf16"),
        # A single request decodes through a fine-grained mixture of experts (hidden 2048, 128 experts of 768, top 8).
        _moe("moe_one_token", 1, 2048, 768, 128, 8, Q4_K, Q4_K),
        # Eight requests: most tokens have most of their experts for themselves.
        _moe("moe_8_tokens", 8, 2048, 768, 128, 8, Q4_K, Q4_K),
        # 32 requests: nearly every expert is read, each for about two tokens; gate and up in the one stack the prompts use.
        _moe("moe_32_tokens_joined", 32, 2048, 768, 128, 8, Q4_K, Q4_K, joined=True),
        # A wider model with fewer experts, 8-bit weights below 4-bit ones, and a shared expert; an odd number of tokens.
        _moe("moe_5_tokens_shared", 5, 4096, 1280, 60, 4, Q4_K, Q8_0, shared=True),
        # One request's logits over the largest vocabulary, with its history and a grammar.
        _logits("logits_one_row", 1, 151936, 2048, 64, 100),
        # A small decode batch over an odd vocabulary: rows that start anywhere.
        _logits("logits_8_rows_odd", 8, 32003, 1024, 16, 50, pad=2),
        # A decode batch with long histories and some grammars.
        _logits("logits_64_rows", 64, 151936, 8192, 300, 25),
        # A large batch without much to do per row: bound by the logits' bytes.
        _logits("logits_256_rows", 256, 128256, 512, 4, 10),
    ]


def _ints(text):
    return [int(v) for v in text.split(",")]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _draw(rng):
    op = rng.choice(("lora", "moe", "logits"))
    if op == "lora":
        n_seg, T = _log_int(rng, 1, 64), _log_int(rng, 1, 8192)
        cuts = sorted(rng.randint(0, T) for _ in range(n_seg - 1))
        lens = [b - a for a, b in zip([0] + cuts, cuts + [T])]
        n_ad = _log_int(rng, 1, 32)
        return _lora(None, lens, [rng.randint(-1, n_ad - 1) for _ in lens], [rng.choice((4, 8, 16, 16, 32, 64, 128)) for _ in range(n_ad)],
                     _log_int(rng, 100, 17408), 256 * _log_int(rng, 1, 68), rng.choice(("f16", "bf16")), rng.choice((0, 0, 4, 3)))
    if op == "moe":
        NE = _log_int(rng, 4, 128)
        joined = rng.random() < 0.4
        return _moe(None, rng.randint(1, 32), 256 * _log_int(rng, 2, 16), 256 * _log_int(rng, 1, 6), NE, rng.randint(1, min(8, NE)),
                    rng.choice((Q4_K, Q8_0)), rng.choice((Q4_K, Q8_0)), joined, rng.random() < 0.3)
    return _logits(None, _log_int(rng, 1, 256), _log_int(rng, 1000, 152000), _log_int(rng, 1, 8192), _log_int(rng, 1, 300), rng.choice((0, 25, 100)), rng.choice((0, 0, 1, 4)))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["op"], {"bytes": 0.0, "flops": 0.0})
        for k in m:
            m[k] = max(m[k], w[k])
    while True:
        c = _draw(rng)
        w = work(c)
        stack = c["NE"] * c["E"] * c["F"] if c["op"] == "moe" else 0  # (what the handles of a state take to make)
        if all(w[k] <= most[c["op"]][k] for k in w) and stack <= 128 * 2048 * 768:
            return c


def work(case):
    c = case
    if c["op"] == "lora":
        rows, ranks = list(zip(_ints(c["lens"]), _ints(c["adapters"]))), _ints(c["ranks"])
        T, N, K = sum(n for n, _ in rows), c["N"], c["K"]
        with_one = [(n, ranks[a]) for n, a in rows if a >= 0]
        used = {a for n, a in rows if a >= 0 and n}
        # quantised rows with their scales, the adapters that are used, the base in and the outputs
        return {"bytes": sum(n for n, _ in with_one) * K * 1.125 + 2.0 * sum(ranks[a] for a in used) * (K + N) + 8.0 * T * N,
                "flops": 2.0 * sum(n * r for n, r in with_one) * (K + N)}
    if c["op"] == "moe":
        T, E, F, NE, NU = (c[k] for k in ("T", "E", "F", "NE", "NU"))
        experts = NE * (1.0 - (1.0 - NU / NE) ** T)  # expected, every token picking NU of NE
        weights = experts * E * F * (2 * FILE_BYTES[c["gate"]] + FILE_BYTES[c["down"]]) / 256
        return {"bytes": weights + T * (1.125 * E + 8.0 * E + 4.0 * NE + (4.0 * E if c["shared"] else 0.0)), "flops": 6.0 * T * NU * E * F}
    rows, V = c["rows"], c["V"]
    return {"bytes": rows * (8.0 * V + c["masked"] / 100 * V / 8 + 4.0 * (c["hist"] / 2) + 8.0 * (c["bias"] / 2)), "flops": 6.0 * rows * V}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _randint(gen, lo, hi, *shape, dtype=torch.int64):
    return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=dtype)


def _quantised(x):
    """int8 rows and one scale per 32 values, [rows][K] and [K/32][rows], the rows padded as the library's GEMM wants them."""
    T, K = x.shape
    Mp = (T + 127) // 128 * 128 if T >= 128 else (T + 15) // 16 * 16
    b = x.view(T, K // 32, 32)
    s = b.abs().amax(2) / 127.0
    aq, asc = torch.zeros((Mp, K), dtype=torch.int8, device="cuda"), torch.zeros((K // 32, Mp), device="cuda")
    aq[:T] = torch.round(b / s[:, :, None].clamp_min(1e-30)).to(torch.int8).view(T, K)
    asc[:, :T] = s.t()
    return aq, asc


def _gguf_rows(gen, qt, rows, K):
    """Random rows in the file's block form, scaled to weights of mean 0 and deviation about 1 / sqrt(K)."""
    R, s = rows * (K // 256), 1.0 / math.sqrt(K)
    b = _randint(gen, 0, 256, R, FILE_BYTES[qt], dtype=torch.uint8)
    half = lambda v: v.half().view(torch.uint8)  # noqa: E731
    if qt == Q4_K:  # fp16 d, dmin | 6-bit scales and mins (scale = min here, so that q - 7.5 is what counts) | 4-bit quants
        d = (0.5 + torch.rand((R, 1), generator=gen, device="cuda")) * (s / 165.0)
        b[:, 0:2], b[:, 2:4] = half(d), half(d * 7.5)
        b[:, 8:12] = b[:, 4:8]
        b[:, 12:16] = (b[:, 12:16] & 15) * 17
    else:  # eight blocks of fp16 d | 32 int8
        v = b.view(R, 8, 34)
        v[:, :, 0:2] = half((0.5 + torch.rand((R, 8, 1), generator=gen, device="cuda")) * (s / 76.0))
    return b.view(rows, -1)


def prepare(case, seed):
    return {"lora": _prepare_lora, "moe": _prepare_moe, "logits": _prepare_logits}[case["op"]](case, _generator(seed))


def _prepare_lora(c, gen):
    lens, ranks, N, K = _ints(c["lens"]), _ints(c["ranks"]), c["N"], c["K"]
    T, n_ad, R = sum(lens), len(ranks), (max(ranks) + 15) // 16 * 16
    dtype = torch.float16 if c["dtype"] == "f16" else torch.bfloat16
    st = {"op": "lora", "T": T, "N": N, "K": K}
    st["aq"], st["asc"] = _quantised(_randn(gen, T, K))
    st["ranks"] = torch.tensor(ranks, dtype=torch.int32, device="cuda")
    there = torch.arange(R, device="cuda")[None, :] < st["ranks"][:, None]  # rows past an adapter's rank are zeros
    st["A"] = (_randn(gen, n_ad, R, K) * there[:, :, None] / math.sqrt(K)).to(dtype)
    st["B"] = (_randn(gen, n_ad, N, R) * there[:, None, :] / math.sqrt(R)).to(dtype)
    st["scales"] = 0.5 + torch.rand((n_ad,), generator=gen, device="cuda")
    st["seg"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
    st["adapter"] = torch.tensor(_ints(c["adapters"]), dtype=torch.int32, device="cuda")
    st["base"] = _randn(gen, T, N + c["pad"])[:, :N]
    st["out"] = torch.zeros((T, N + c["pad"]), device="cuda")[:, :N]
    return st


def _prepare_moe(c, gen):
    T, E, F, NE, NU = (c[k] for k in ("T", "E", "F", "NE", "NU"))
    st = {"op": "moe", "T": T, "E": E, "F": F, "NE": NE, "NU": NU, "gate": c["gate"], "down": c["down"]}
    st["aq"], st["asc"] = _quantised(_randn(gen, T, E))
    st["logits"] = _randn(gen, T, NE + (1 if c["shared"] else 0))
    st["x"] = _randn(gen, T, E)
    st["sh"] = _randn(gen, T, E) if c["shared"] else None
    st["out"] = torch.zeros((T, E), device="cuda")
    g, u, d = _gguf_rows(gen, c["gate"], NE * F, E), _gguf_rows(gen, c["gate"], NE * F, E), _gguf_rows(gen, c["down"], NE * E, F)
    if own:  # the handles of the same bytes
        import arcinferzero_b200 as izb
        g, u, d = g.cpu().numpy(), u.cpu().numpy(), d.cpu().numpy()
        if c["joined"]:
            st["wg"], st["wu"] = izb.gateup_weight(c["gate"], g, u, F, E, n_mats=NE), None
        else:
            st["wg"], st["wu"] = izb.Weight(c["gate"], g, F, E, n_mats=NE), izb.Weight(c["gate"], u, F, E, n_mats=NE)
        st["wd"] = izb.Weight(c["down"], d, E, F, n_mats=NE)
    else:
        st["wg"], st["wu"], st["wd"] = g.view(NE, F, -1), u.view(NE, F, -1), d.view(NE, E, -1)
    return st


def _prepare_logits(c, gen):
    rows, V = c["rows"], c["V"]
    st = {"op": "logits", "V": V}
    st["logits"] = (_randn(gen, rows, V + c["pad"]) * 3.0)[:, :V]
    st["out"] = torch.zeros((rows, V + c["pad"]), device="cuda")[:, :V]
    # repetition, presence, frequency, temperature; every third row is greedy (temperature 0: logits as they are)
    p = torch.rand((rows, 4), generator=gen, device="cuda") * torch.tensor([0.5, 1.0, 0.5, 1.0], device="cuda") + torch.tensor([1.0, 0.0, 0.0, 0.3], device="cuda")
    p[::3, 3] = 0.0
    st["params"] = p
    def ragged(most):
        n = _randint(gen, 0, most + 1, rows)
        n[-1] = most
        off = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
        off[1:] = n.cumsum(0)
        return off.to(torch.int32), int(off[-1])
    st["hist_off"], n = ragged(c["hist"])
    u = torch.rand((n,), generator=gen, device="cuda")
    st["hist"] = (u * u * u * V).to(torch.int32).clamp_max(V - 1)  # (some tokens come often)
    st["bias_off"], n = ragged(c["bias"])
    first = _randint(gen, 0, V, rows).repeat_interleave((st["bias_off"][1:] - st["bias_off"][:-1]).long(), output_size=n)
    at = torch.arange(n, device="cuda") - st["bias_off"][:-1].long().repeat_interleave((st["bias_off"][1:] - st["bias_off"][:-1]).long(), output_size=n)
    st["bias_ids"] = ((first + at * (V // (c["bias"] + 1))) % V).to(torch.int32)  # (no token twice in a row's list)
    st["bias"] = _randn(gen, n) * 5.0
    words = (V + 31) // 32
    n_masks = max(1, rows * c["masked"] // 100)
    st["mask"] = torch.bitwise_and(_randint(gen, -2 ** 31, 2 ** 31, n_masks, words, dtype=torch.int32), _randint(gen, -2 ** 31, 2 ** 31, n_masks, words, dtype=torch.int32))
    st["mask_row"] = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    if c["masked"]:
        st["mask_row"][torch.arange(n_masks, device="cuda") * rows // n_masks] = torch.arange(n_masks, dtype=torch.int32, device="cuda")
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    return {"lora": _run_lora, "moe": _run_moe, "logits": _run_logits}[st["op"]](st)


def _run_lora(st):
    if own:
        import arcinferzero_b200 as izb
        return izb.lora_add(st["A"], st["B"], st["scales"], st["aq"], st["asc"], st["T"], st["seg"], st["adapter"], st["out"], base=st["base"], ranks=st["ranks"])
    T, N, K = st["T"], st["N"], st["K"]
    n_ad, R = st["A"].shape[:2]
    x = (st["aq"][:T].float().view(T, K // 32, 32) * st["asc"][:, :T].t()[:, :, None]).view(T, K)
    # every row against every adapter, then only its own kept
    at = torch.searchsorted(st["seg"][1:].contiguous(), torch.arange(T, dtype=torch.int32, device="cuda"), right=True)
    mine = st["adapter"][at]
    u = (x @ st["A"].float().view(n_ad * R, K).t()).view(T, n_ad, R)
    keep = (torch.arange(n_ad, device="cuda")[None, :] == mine[:, None]).float() * st["scales"][None, :]
    u = u * keep[:, :, None] * (torch.arange(R, device="cuda")[None, :] < st["ranks"][:, None]).float()[None]
    return st["base"] + u.view(T, n_ad * R) @ st["B"].float().permute(0, 2, 1).reshape(n_ad * R, N)


def _decoded(qt, b):
    """[..., bytes of a row] in the file's form -> [..., K] f32."""
    lead = b.shape[:-1]
    b = b.reshape(-1, FILE_BYTES[qt])
    if qt == Q8_0:
        v = b.view(-1, 34)
        return (v[:, 0:2].contiguous().view(torch.float16).float() * v[:, 2:].contiguous().view(torch.int8).float()).view(*lead, -1)
    d, dmin = b[:, 0:2].contiguous().view(torch.float16).float(), b[:, 2:4].contiguous().view(torch.float16).float()
    s = b[:, 4:16].to(torch.int32)
    a, m, t = s[:, 0:4], s[:, 4:8], s[:, 8:12]
    sc = torch.cat([a & 63, (t & 15) | ((a >> 6) << 4)], 1).float()
    mn = torch.cat([m & 63, (t >> 4) | ((m >> 6) << 4)], 1).float()
    q = b[:, 16:144].view(-1, 4, 32)
    q = torch.stack([q & 15, q >> 4], 2).view(-1, 8, 32).float()
    return ((d * sc)[:, :, None] * q - (dmin * mn)[:, :, None]).view(*lead, -1)


def _run_moe(st):
    if own:
        import arcinferzero_b200 as izb
        return izb.moe_layer(st["wg"], st["wu"], st["wd"], st["aq"], st["asc"], st["logits"], st["NU"], x=st["x"], out=st["out"], sh=st["sh"])
    T, E, F, NE, NU = (st[k] for k in ("T", "E", "F", "NE", "NU"))
    top, ids = st["logits"][:, :NE].sort(dim=1, descending=True, stable=True)
    top, ids = top[:, :NU], ids[:, :NU].reshape(-1)
    p = (top - top[:, :1]).exp()
    w = p / p.sum(1, keepdim=True)
    x = (st["aq"][:T].float().view(T, E // 32, 32) * st["asc"][:, :T].t()[:, :, None]).view(T, 1, E, 1).expand(T, NU, E, 1).reshape(T * NU, E, 1)
    g = (_decoded(st["gate"], st["wg"][ids]) @ x)[:, :, 0]
    u = (_decoded(st["gate"], st["wu"][ids]) @ x)[:, :, 0]
    h = g / (1.0 + (-g).exp()) * u
    y = (_decoded(st["down"], st["wd"][ids]) @ h[:, :, None]).view(T, NU, E)
    out = st["x"] + (y * w[:, :, None]).sum(1)
    if st["sh"] is not None:
        out = out + st["sh"] / (1.0 + (-st["logits"][:, NE:]).exp())
    return out


def _run_logits(st):
    if own:
        import arcinferzero_b200 as izb
        out, best, logz = izb.logits_process(st["logits"], out=st["out"], params=st["params"], hist=(st["hist"], st["hist_off"]),
                                             bias=(st["bias_ids"], st["bias"], st["bias_off"]), mask=st["mask"], mask_row=st["mask_row"])
        return {"logits": out, "best": best, "logz": logz}
    l, V = st["logits"], st["V"]
    rows = l.shape[0]
    rep, pres, freq, temp = (st["params"][:, i:i + 1] for i in range(4))
    r = torch.arange(rows, device="cuda")

    def of_row(off, n):
        return r.repeat_interleave((off[1:] - off[:-1]).long(), output_size=n)

    n = st["hist"].numel()
    c = torch.zeros(rows * V, device="cuda").index_add_(0, of_row(st["hist_off"], n) * V + st["hist"], torch.ones(n, device="cuda")).view(rows, V)
    l = torch.where(c > 0, torch.where(l > 0, l / rep, l * rep) - (freq * c + pres), l)
    n = st["bias"].numel()
    add = torch.zeros(rows * V, device="cuda")
    add[of_row(st["bias_off"], n) * V + st["bias_ids"]] = st["bias"]
    l = l + add.view(rows, V)
    v = torch.arange(V, device="cuda")
    allowed = (st["mask"][st["mask_row"].clamp_min(0).long()][:, v >> 5] >> (v & 31).to(torch.int32)) & 1
    l = torch.where((allowed == 0) & (st["mask_row"] >= 0)[:, None], -math.inf, l)
    l = torch.where(temp > 0, l / torch.where(temp > 0, temp, 1.0), l)
    top = l.amax(1, keepdim=True)
    best = torch.where(l == top, v[None, :], V).amin(1)
    # (100000 terms: their sum in 64 bits)
    logz = ((l - top).exp().double().sum(1).log() + top[:, 0].double()).float()
    return {"logits": l, "best": best.to(torch.int32), "logz": torch.where(top[:, 0] == -math.inf, -math.inf, logz)}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    c, f8 = case, torch.float64
    st = _prepare_lora(c, _generator(seed)) if c["op"] == "lora" else _prepare_logits(c, _generator(seed)) if c["op"] == "logits" else None
    if c["op"] == "lora":
        out, first = st["base"].to(f8).clone(), 0
        for n, a in zip(_ints(c["lens"]), _ints(c["adapters"])):
            if n and a >= 0:
                r = _ints(c["ranks"])[a]
                x = st["aq"][first:first + n].to(f8) * st["asc"][:, first:first + n].to(f8).repeat_interleave(32, 0).t()
                out[first:first + n] += st["scales"][a].to(f8) * ((x @ st["A"][a, :r].to(f8).t()) @ st["B"][a, :, :r].to(f8).t())
            first += n
        return out
    if c["op"] == "logits":
        out, logz = st["logits"].to(f8).clone(), []
        for r in range(c["rows"]):
            rep, pres, freq, temp = (float(v) for v in st["params"][r].to(f8))
            row = out[r]
            seen, times = st["hist"][int(st["hist_off"][r]):int(st["hist_off"][r + 1])].long().unique(return_counts=True)
            l = row[seen]
            row[seen] = torch.where(l > 0, l / rep, l * rep) - freq * times.to(f8) - pres
            some = slice(int(st["bias_off"][r]), int(st["bias_off"][r + 1]))
            row[st["bias_ids"][some].long()] += st["bias"][some].to(f8)
            m = int(st["mask_row"][r])
            if m >= 0:
                bits = (st["mask"][m][:, None] >> torch.arange(32, dtype=torch.int32, device="cuda")[None, :]) & 1
                row[bits.reshape(-1)[:c["V"]] == 0] = -math.inf
            if temp > 0:
                row /= temp
            logz.append(torch.logsumexp(row, 0))
        return {"logits": out, "best": None, "logz": torch.stack(logz)}
    global own
    kept, own = own, False
    try:
        st = _prepare_moe(c, _generator(seed))
    finally:
        own = kept
    T, E, NE, NU = (c[k] for k in ("T", "E", "NE", "NU"))
    out, logits = st["x"].to(f8).clone(), st["logits"].to(f8)

    def weights(qt, rows):
        b = rows.reshape(-1, 34) if qt == Q8_0 else rows.reshape(-1, 144)
        two = b[:, 0:4].contiguous().view(torch.float16).to(f8)
        if qt == Q8_0:
            return (two[:, 0:1] * b[:, 2:].contiguous().view(torch.int8).to(f8)).reshape(rows.shape[0], -1)
        blocks = []
        for j in range(8):  # 6-bit scale and min of block j
            lo, hi = b[:, 4 + j % 4].long(), b[:, 8 + j % 4].long()
            s, m = (lo & 63, hi & 63) if j < 4 else ((b[:, 8 + j].long() & 15) + 16 * (lo >> 6), (b[:, 8 + j].long() >> 4) + 16 * (hi >> 6))
            q = b[:, 16 + 32 * (j // 2):48 + 32 * (j // 2)]
            q = (q >> 4 if j % 2 else q & 15).to(f8)
            blocks.append(two[:, 0:1] * s.to(f8)[:, None] * q - two[:, 1:2] * m.to(f8)[:, None])
        return torch.stack(blocks, 1).reshape(rows.shape[0], -1)

    for t in range(T):
        l = logits[t, :NE].tolist()
        chosen = sorted(range(NE), key=lambda e: (-l[e], e))[:NU]
        p = [math.exp(l[e] - l[chosen[0]]) for e in chosen]
        x = st["aq"][t].to(f8) * st["asc"][:, t].to(f8).repeat_interleave(32)
        for e, w in zip(chosen, p):
            g, u = weights(c["gate"], st["wg"][e]) @ x, weights(c["gate"], st["wu"][e]) @ x
            out[t] += w / sum(p) * (weights(c["down"], st["wd"][e]) @ (g / (1.0 + torch.exp(-g)) * u))
        if st["sh"] is not None:
            out[t] += st["sh"][t].to(f8) / (1.0 + torch.exp(-logits[t, NE]))
    return out
