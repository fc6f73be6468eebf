"""What the adapters, the expert block and the logit rules refuse, before anything is launched (no GPU needed)."""
import ctypes as C

import numpy as np
import pytest
import torch

import arcinferzero_b200 as izb

ARG, SHAPE, TYPE, ALIGN, LIMIT = -1, -2, -3, -4, -10


def p(a, byte=0):
    return C.c_void_p(a.ctypes.data + byte)


def aligned(n, dtype=np.float32):
    raw = np.zeros(n * np.dtype(dtype).itemsize + 16, np.uint8)
    first = -raw.ctypes.data % 16
    return raw[first:first + n * np.dtype(dtype).itemsize].view(dtype)


def lora(**kw):
    b = aligned(65536)
    a = dict(dtype=1, A=p(b), B=p(b), n=2, R=16, ranks=None, scales=p(b), N=32, K=256, aq=p(b), asc=p(b), T=3, Mp=16, seg=p(b), adapter=p(b), n_seg=1, base=None, ldb=32,
             C=p(b), ldc=32, c_off=0, scratch=None)
    a.update(kw)
    return izb.lib().izb_lora_add(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(A=None), ARG), (dict(B=None), ARG), (dict(scales=None), ARG), (dict(aq=None), ARG), (dict(asc=None), ARG), (dict(seg=None), ARG), (dict(adapter=None), ARG),
    (dict(C=None), ARG), (dict(dtype=0), TYPE), (dict(dtype=8), TYPE), (dict(n=0), SHAPE), (dict(R=8), SHAPE), (dict(R=24), SHAPE), (dict(R=272), SHAPE),
    (dict(N=0), SHAPE), (dict(K=0), SHAPE), (dict(K=288), SHAPE), (dict(T=0), SHAPE), (dict(T=17), SHAPE), (dict(Mp=24), SHAPE), (dict(n_seg=0), SHAPE),
    (dict(ldc=31), SHAPE), (dict(c_off=1), SHAPE), (dict(c_off=-1), SHAPE),
])
def test_lora_add_refuses(kw, status):
    assert lora(**kw) == status, izb.lib().izb_last_error()


def test_lora_add_refuses_addresses():
    b = aligned(65536)
    for name in ("A", "B", "aq", "asc"):
        assert lora(**{name: p(b, 8)}) == ALIGN
    assert lora(C=p(b, 2)) == ALIGN and lora(base=p(b, 2)) == ALIGN
    assert lora(base=p(b), C=p(b), ldb=31) == SHAPE
    assert lora(base=p(b), C=p(b, 4)) == ARG                    # shifted by a column
    assert lora(base=p(b), C=p(b), ldb=32, ldc=33) == ARG       # the same first row, then apart
    assert lora(base=p(b), C=p(b, 16), ldb=64, ldc=64) == ARG   # windows that overlap


def logits(**kw):
    b = aligned(65536)
    a = dict(l=p(b), ldl=100, out=p(b), ldo=100, rows=3, V=100, params=None, hist=None, hist_off=None, n_hist=0, bias_ids=None, bias=None, bias_off=None, n_bias=0, mask=None,
             words=0, n_masks=0, mask_row=None, best=None, logz=None)
    a.update(kw)
    return izb.lib().izb_logits_process(*a.values(), None)


def test_logits_process_refuses():
    b = aligned(65536)
    q = p(b)
    for kw, status in ((dict(l=None), ARG), (dict(out=None), ARG), (dict(rows=0), SHAPE), (dict(V=0), SHAPE), (dict(ldl=99), SHAPE), (dict(ldo=99), SHAPE),
                       (dict(n_hist=1, params=q, hist=q), ARG), (dict(n_hist=1, params=q, hist_off=q), ARG), (dict(n_hist=-1), ARG), (dict(n_hist=1, hist=q, hist_off=q), ARG),
                       (dict(n_bias=1, bias_ids=q, bias=q), ARG), (dict(n_bias=1, bias_ids=q, bias_off=q), ARG), (dict(n_bias=1, bias=q, bias_off=q), ARG), (dict(n_bias=-1), ARG),
                       (dict(mask=q, words=3, n_masks=3), SHAPE), (dict(mask=q, words=4, n_masks=2), SHAPE), (dict(mask=q, words=4, n_masks=0, mask_row=q), SHAPE), (dict(mask_row=q), ARG),
                       (dict(l=p(b, 2), out=p(b, 2)), ALIGN), (dict(l=q, out=p(b, 4)), ARG), (dict(l=q, out=q, ldo=101), ARG), (dict(l=q, out=p(b, 400 * 2)), ARG)):
        assert logits(**kw) == status, (kw, izb.lib().izb_last_error())


def test_logits_process_refuses_arrays_past_its_numbers():
    """Positions in the arrays are 32-bit numbers that the kernel adds strides to."""
    q = p(aligned(65536))
    for n, status in (((1 << 30) + 1, LIMIT), (2 ** 31 - 1, LIMIT)):
        assert logits(n_hist=n, params=q, hist=q, hist_off=q) == status
        assert logits(n_bias=n, bias_ids=q, bias=q, bias_off=q) == status
    assert logits(V=(1 << 30) + 1, ldl=(1 << 30) + 1, ldo=(1 << 30) + 1) == SHAPE


def test_moe_layer_refuses_without_weights():
    L = izb.lib()
    q = p(aligned(64))
    assert L.izb_moe_layer(None, None, None, q, q, 1, 16, q, 8, 8, 2, 0, None, None, q, q, None) == ARG
    L.izb_moe_layer_scratch.restype = C.c_size_t
    assert L.izb_moe_layer_scratch(0, 8, 768) == 0 and L.izb_moe_layer_scratch(3, 8, 768) >= 3 * 8 * 768 * 3


def test_binding_refuses_tensors_of_the_host():
    """A tensor of the wrong place, type or form is named before its address reaches a kernel."""
    f, i = lambda *s: torch.zeros(s), lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(ValueError, match="logits: a tensor on the GPU"):
        izb.logits_process(f(2, 8))
    with pytest.raises(TypeError, match="logits"):
        izb.logits_process(f(2, 8).double())
    with pytest.raises(ValueError, match="logits: 2 dimensions"):
        izb.logits_process(f(8))
    A, B = torch.zeros((2, 16, 256), dtype=torch.float16), torch.zeros((2, 32, 16), dtype=torch.float16)
    args = (f(2), torch.zeros((16, 256), dtype=torch.int8), f(8, 16), 3, i(2), i(1), f(3, 32))
    with pytest.raises(ValueError, match="A: a tensor on the GPU"):
        izb.lora_add(A, B, *args)
    with pytest.raises(TypeError, match="A"):
        izb.lora_add(A.float(), B, *args)
    W = izb.Weight.__new__(izb.Weight)
    W.handle, W.N, W.K = C.c_void_p(0), 256, 256
    with pytest.raises(ValueError, match="logits: a tensor on the GPU"):
        izb.moe_layer(W, W, W, args[1], args[2], f(1, 4), 2)
