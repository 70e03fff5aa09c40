"""The transformer-training entries without a GPU: refusals of the C ABI and
of the layers, and calls with nothing to do."""
from __future__ import annotations

import ctypes as C
import math

import pytest

from rushlite_b200 import capi


def test_layer_norm_refusals():
    L = capi.lib()
    assert L.lmpb_layer_norm(capi.INT32, None, None, None, 1, 1, 1e-5, None, None, None, None) == 1
    assert L.lmpb_layer_norm(capi.FLOAT32, None, None, None, -1, 1, 1e-5, None, None, None, None) == 1
    assert L.lmpb_layer_norm(capi.FLOAT32, None, None, None, 1, 0, 1e-5, None, None, None, None) == 1
    assert L.lmpb_layer_norm(capi.FLOAT32, None, None, None, 1, 8, -1.0, None, None, None, None) == 1
    assert L.lmpb_layer_norm(capi.FLOAT32, None, None, None, 1, 8, 1e-5, None, None, None, None) == 1
    assert L.lmpb_layer_norm(capi.FLOAT32, 16, None, None, 1, 8, 1e-5, 16, 16, None, None) == 1
    assert b"lmpb_layer_norm" in L.lmpb_last_error()
    assert L.lmpb_layer_norm(capi.FLOAT32, None, None, None, 0, 8, 1e-5, None, None, None, None) == 0
    assert L.lmpb_layer_norm_backward(capi.BOOL, None, None, None, None, None, 1, 1, None, None, None, None) == 1
    assert L.lmpb_layer_norm_backward(capi.FLOAT32, None, None, None, None, None, 1, 1, 16, None, None, None) == 1
    assert L.lmpb_layer_norm_backward(capi.FLOAT32, None, None, None, None, None, 4, 8, None, None, None, None) == 0


def test_adamw_refusals():
    L = capi.lib()
    ok = dict(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.1, step=16)

    def call(dt=capi.FLOAT32, tensors=(), count=None, **kw):
        a = {**ok, **kw}
        ts = (capi.AdamWTensor * max(1, len(tensors)))(*[capi.AdamWTensor(*t) for t in tensors])
        return L.lmpb_adamw(dt, ts, len(tensors) if count is None else count, a["lr"], a["b1"], a["b2"], a["eps"],
                            a["wd"], a["step"], None)

    assert call(capi.INT64) == 1 and call(count=-1) == 1 and call(step=None) == 1
    for kw in (dict(lr=-1.0), dict(lr=math.inf), dict(b1=1.0), dict(b2=math.nan), dict(eps=-1e-8), dict(wd=-1.0)):
        assert call(**kw) == 1, kw
    assert call(tensors=[(None, 16, 16, 16, 4)]) == 1
    assert call(tensors=[(16, 16, 16, 16, -4)]) == 1
    assert b"lmpb_adamw" in L.lmpb_last_error()


def test_sequences_and_attention_refusals():
    L = capi.lib()
    with pytest.raises(capi.LmpbError, match="negative"):
        capi.Sequences([4, -1])
    with pytest.raises(capi.LmpbError, match="2\\^30"):
        capi.Sequences([1 << 30, 1 << 30])
    with pytest.raises(capi.LmpbError, match="2\\^30"):
        capi.Sequences([1 << 62])
    assert L.lmpb_sequences_create(None, 2, C.byref(C.c_void_p())) == 1
    assert L.lmpb_sequences_create(None, 0, None) == 1
    assert L.lmpb_sequences_release(None) == 0
    empty = capi.Sequences([])
    zeros = capi.Sequences([0, 0])

    def call(seqs=empty.h, tokens=0, heads=4, kv=2, dim=8, scale=1.0):
        return L.lmpb_attention(None, None, None, None, None, tokens, heads, kv, dim, scale, seqs, None)

    assert call() == 0 and call(zeros.h) == 0
    for kw in (dict(seqs=None), dict(tokens=-1), dict(heads=0), dict(kv=3), dict(dim=0), dict(dim=129), dict(scale=0.0),
               dict(scale=math.nan), dict(tokens=5), dict(heads=131072, kv=1)):
        assert call(**kw) == 1, kw
    assert L.lmpb_attention_backward(None, None, None, None, None, None, None, None, None, 0, 4, 2, 8, 1.0, empty.h, None) == 0
    assert L.lmpb_attention_backward(*[16] * 7, None, 16, 0, 4, 2, 8, 1.0, empty.h, None) == 1
    assert L.lmpb_attention_backward(*[None] * 9, 5, 4, 2, 8, 1.0, None, None) == 1


def test_layers_check_their_arguments():
    from rushlite_b200.nets import layers

    for args in ((10, 3), (12, 0), (12, 4, 3), (12, 4, 0)):
        with pytest.raises(ValueError):
            layers.CausalSelfAttention(*args)


def test_layers_refuse_what_they_cannot_compute():
    import rushlite_b200 as rsl
    from rushlite_b200.nets import layers

    cpu = rsl.device.cpu  # construction alone needs no GPU
    for kw in (dict(dtype=rsl.dtype.float64), dict(dtype=rsl.dtype.int32)):
        with pytest.raises(ValueError, match="float32"):
            layers.CausalSelfAttention(64, 4, device=cpu, **kw)
    with pytest.raises(ValueError, match="multiple"):
        layers.CausalSelfAttention(0, 4, device=cpu)
    for args in ((1024, 4), (129, 1), (516, 4, 2)):
        with pytest.raises(ValueError, match="128"):
            layers.CausalSelfAttention(*args, device=cpu)
    for args in ((512, 4), (128, 1), (64, 4, 2)):
        for dtype in (None, rsl.dtype.float32):
            layers.CausalSelfAttention(*args, device=cpu, dtype=dtype)
    for kw in (dict(features=0), dict(features=8, eps=-1e-5), dict(features=8, eps=math.nan), dict(features=8, eps=math.inf),
               dict(features=8, dtype=rsl.dtype.int64)):
        with pytest.raises(ValueError):
            layers.LayerNorm(**kw, device=cpu)
    for dtype in (None, rsl.dtype.float32, rsl.dtype.float64):
        layers.LayerNorm(8, 0.0, device=cpu, dtype=dtype)
