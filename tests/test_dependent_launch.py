"""Dependent launch.  A kernel that lets the next one in early (griddepcontrol.launch_dependents) makes none of its writes, nor those of the kernels before it,
visible to that one: only griddepcontrol.wait does.  Kernels of the per-request operators may touch the library's weights ahead of it, and nothing else.
The sources are checked for that on the CPU; on the GPU a chain of calls that feed one another is compared with one that waits in between."""
import os
import re

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "arcinferzero_b200", "csrc")
# what the kernels read or write that another kernel may have written or may still read
FIELDS = {
    "izb_moe_layer.cu": ("logits", "x", "sh", "aq", "asc", "hq", "hs", "hsum", "out", "routes"),
    "izb_lora.cu": ("A", "B", "ranks", "seg", "adapter", "scales", "asc", "aq", "base", "C"),
    "izb_logits.cu": ("in", "out", "params", "hist", "hist_off", "bias_ids", "bias", "bias_off", "mask", "mask_row", "best", "logz"),
}


def functions(text):
    """name -> body, of everything that looks like a function definition at the start of a line"""
    out = {}
    for m in re.finditer(r"^(?:__global__|__device__|template)[^;{]*?(\w+)\((?:[^;{}]|\{\})*?\)\s*(?:const )?\{", text, re.M):
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        out[m.group(1)] = text[m.end():i], "__global__" in m.group(0)
    return out


@pytest.mark.parametrize("name", sorted(FIELDS))
def test_nothing_but_weights_ahead_of_the_wait(name):
    text = "\n".join(re.sub(r"//.*", "", line) for line in open(os.path.join(CSRC, name)).read().split("\n"))
    text = re.sub(r"__launch_bounds__\([^)]*\) ", "", text)
    found = functions(text)
    kernels = {k: body for k, (body, is_kernel) in found.items() if is_kernel}
    assert kernels and len(kernels) == len(re.findall(r"^(?:template <[^>]*>\s*)?__global__", text, re.M))
    field = re.compile(r"\bp\.(?:%s)\b" % "|".join(FIELDS[name]))
    touching = {k for k, (body, is_kernel) in found.items() if not is_kernel and field.search(body)}
    for _ in found:  # (functions that call such functions)
        touching |= {k for k, (body, is_kernel) in found.items() if not is_kernel and any(re.search(r"\b%s\b[<(]" % t, body) for t in touching)}
    for kernel, body in kernels.items():
        assert "pdl_wait();" in body, kernel
        head = body[:body.index("pdl_wait();")].replace("p.base == p.C", "")  # (addresses, of which nothing is read)
        assert not field.search(head), (kernel, field.search(head).group(0))
        for t in touching:
            assert not re.search(r"\b%s\b[<(]" % t, head), (kernel, t)
        assert not re.search(r"\breturn\b", head), kernel  # (completion is passed on along the stream: every path waits)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,F,NE,NU", [(1, 512, 256, 16, 4), (6, 768, 512, 64, 8), (32, 512, 768, 32, 6)])
def test_calls_that_feed_one_another(izb, T, E, F, NE, NU):
    """Norm, router, expert block in place, again and again: the logits and the residual of every call come from the kernels right before it."""
    import torch

    from tests.test_gpu_moe_layer import rows
    rng = np.random.default_rng(T)
    cu = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda()
    Wr, Wd = izb.Weight(8, rows(8, NE, E, 1), NE, E), izb.Weight(12, rows(12, NE * E, F, 2), E, F, n_mats=NE)
    Wgu = izb.gateup_weight(12, rows(12, NE * F, E, 3), rows(12, NE * F, E, 4), F, E, n_mats=NE)
    norm, x0 = cu(np.ones(E)), cu(rng.standard_normal((T, E)))

    def steps(wait):
        x, seen = x0.clone(), []
        router = torch.zeros((T, NE), device="cuda")
        for _ in range(60):
            aq, asc, _ = izb.rmsnorm_quant(x, norm, 1e-6)
            izb.matmul(Wr, aq, asc, T, out=router)
            if wait:
                torch.cuda.synchronize()
            izb.moe_layer(Wgu, None, Wd, aq, asc, router, NU, x=x, out=x)
            if wait:
                torch.cuda.synchronize()
            seen.append(x.clone())
        return torch.stack(seen)

    want = steps(True)
    assert bool(torch.isfinite(want).all()) and not torch.equal(want[-1], want[-2])
    for _ in range(3):
        assert torch.equal(steps(False), want)
