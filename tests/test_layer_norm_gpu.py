"""Layer norm against the formula in more bits, its gradients against
differences, and its refusals.

Tolerances: u is half a step of the type.  A row's sums are chains of at most
32 additions in a thread and 13 across threads, so a mean is off by at most
45 u of the row's mean magnitude and rstd by under 30 u; C = 64 covers these
with the last few roundings.  A sum over rows adds at most one rounding per
row.  Every bound multiplies the magnitudes of what was added, elementwise."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SHAPES = [(1, 1), (1, 7), (3, 64), (32, 256), (9, 100), (5, 129), (17, 513), (40, 1001), (33, 1024), (7, 1025),
          (300, 2048), (4, 2052), (19, 4096), (3, 4099), (2, 8192), (3, 8193), (2, 20000), (1500, 32),
          (310, 5001), (700, 1030), (330, 6144)]
HALF = {"float32": 2.0 ** -24, "float64": 2.0 ** -53}
C = 64


def _reference(x, w, b, g, eps):
    """Values and the magnitudes their roundings scale with, in 80 bits."""
    x, w, b, g = (None if t is None else t.astype(np.longdouble) for t in (x, w, b, g))
    f = x.shape[-1]
    mean = x.sum(-1, keepdims=True) / f
    c = x - mean
    rstd = 1 / np.sqrt((c * c).sum(-1, keepdims=True) / f + np.longdouble(eps))
    h = c * rstd
    w1 = np.ones(f, np.longdouble) if w is None else w
    y = h * w1 + (0 if b is None else b)
    hm = rstd * np.abs(x).mean(-1, keepdims=True) + np.abs(h)  # what h's roundings scale with
    a = g * w1
    dx = rstd * (a - a.mean(-1, keepdims=True) - h * (a * h).mean(-1, keepdims=True))
    am = np.abs(a)
    dxm = rstd * (am + am.mean(-1, keepdims=True) + hm * (am * np.abs(h)).mean(-1, keepdims=True)
                  + np.abs(h) * (am * hm).mean(-1, keepdims=True)) + np.abs(dx)
    axes = tuple(range(x.ndim - 1))
    return {"y": (y, hm * np.abs(w1) + np.abs(y), C), "dx": (dx, dxm, 2 * C),
            "dw": ((g * h).sum(axes), (np.abs(g) * hm).sum(axes), C + x[..., 0].size),
            "db": (g.sum(axes), np.abs(g).sum(axes), C + x[..., 0].size)}


def _check(name, got, ref, u):
    want, mag, count = ref
    got = np.asarray(got, np.longdouble)
    assert got.shape == want.shape, name
    off = np.abs(got - want) - count * u * mag
    assert not (off > 0).any() and np.isfinite(got).all(), (name, float(off.max()))


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("rows,features", SHAPES)
def test_forward_and_backward(cuda, rows, features, dtype):
    import rushlite_b200 as rsl

    rng = np.random.default_rng(rows * 10007 + features)
    kind = getattr(rsl.dtype, dtype)
    x = (rng.standard_normal((rows, features)) * 1.5 + 3).astype(dtype)
    w, b, g = (rng.standard_normal(s).astype(dtype) for s in ((features,), (features,), (rows, features)))
    for uw, ub in ((True, True), (True, False), (False, True), (False, False)):
        ref = _reference(x, w if uw else None, b if ub else None, g, 1e-5)
        vx = rsl.Variable(x, True, dtype=kind)
        vw = rsl.Variable(w, True, dtype=kind) if uw else None
        vb = rsl.Variable(b, True, dtype=kind) if ub else None
        y = rsl.layer_norm(vx, vw, vb, 1e-5)
        y.backward(rsl.Variable(g, dtype=kind))
        _check("y", y.numpy(), ref["y"], HALF[dtype])
        _check("dx", vx.grad.numpy(), ref["dx"], HALF[dtype])
        if uw:
            _check("dw", vw.grad.numpy(), ref["dw"], HALF[dtype])
        if ub:
            _check("db", vb.grad.numpy(), ref["db"], HALF[dtype])


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("rows,features", [(64, 64), (65, 64), (512, 16), (8192, 1), (1000, 8), (8, 1024), (9, 900)])
def test_few_and_many_narrow_rows(cuda, rows, features, dtype):
    """Both sides of where one CTA takes all rows."""
    test_forward_and_backward(cuda, rows, features, dtype)


def test_dimensions_before_the_last_are_rows(cuda):
    import rushlite_b200 as rsl

    rng = np.random.default_rng(1)
    x, w = rng.standard_normal((3, 5, 36)).astype(np.float32), rng.standard_normal(36).astype(np.float32)
    g = rng.standard_normal((3, 5, 36)).astype(np.float32)
    vx, vw = rsl.Variable(x, True), rsl.Variable(w, True)
    y = rsl.layer_norm(vx, vw)
    y.backward(rsl.Variable(g))
    ref = _reference(x, w, None, g, 1e-5)
    _check("y", y.numpy(), ref["y"], HALF["float32"])
    _check("dx", vx.grad.numpy(), ref["dx"], HALF["float32"])
    _check("dw", vw.grad.numpy(), ref["dw"], HALF["float32"])


@pytest.mark.parametrize("rows,features", [(4, 24), (3, 1500)])
def test_gradients_are_the_differences(cuda, rows, features):
    """Central differences in float64 with step h: their own error is h^2 times
    a third derivative (below 100 of the terms here) plus 2^-53 / h."""
    import rushlite_b200 as rsl

    rng = np.random.default_rng(features)
    f64 = rsl.dtype.float64
    vals = {"x": rng.standard_normal((rows, features)), "w": rng.standard_normal(features), "b": rng.standard_normal(features)}
    g = rng.standard_normal((rows, features))
    h = 1e-5

    def value(v):
        y = rsl.layer_norm(*(rsl.Variable(v[k], dtype=f64) for k in "xwb")).numpy()
        return float((y.astype(np.longdouble) * g).sum())

    var = {k: rsl.Variable(v, True, dtype=f64) for k, v in vals.items()}
    rsl.layer_norm(var["x"], var["w"], var["b"]).backward(rsl.Variable(g, dtype=f64))
    for k in "xwb":
        d = rng.standard_normal(vals[k].shape)
        slope = (value({**vals, k: vals[k] + h * d}) - value({**vals, k: vals[k] - h * d})) / (2 * h)
        got = float((var[k].grad.numpy() * d).sum())
        size = float(np.abs(g).sum() * np.abs(d).max())
        assert abs(got - slope) <= (100 * h * h + 64 * 2.0 ** -53 / h) * size, k


def test_zero_variance_large_mean_and_special_values(cuda):
    import rushlite_b200 as rsl

    x = np.full((4, 96), 7.25, np.float32)  # sums of it are exact
    y = rsl.layer_norm(rsl.Variable(x)).numpy()
    assert (y == 0).all()
    z = rsl.layer_norm(rsl.Variable(x), eps=0.0).numpy()  # 0 / 0
    assert np.isnan(z).all()
    rng = np.random.default_rng(2)
    x = (rng.standard_normal((8, 300)) + 1e4).astype(np.float32)
    ref = _reference(x, None, None, np.ones_like(x), 1e-5)
    _check("y", rsl.layer_norm(rsl.Variable(x)).numpy(), ref["y"], HALF["float32"])
    x[3, 5], x[6, 7] = np.nan, np.inf
    y = rsl.layer_norm(rsl.Variable(x)).numpy()
    bad = np.isnan(y).any(1)
    assert bad.tolist() == [i in (3, 6) for i in range(8)]  # other rows keep their values
    _check("y", y[:3], tuple(t[:3] if isinstance(t, np.ndarray) else t for t in ref["y"]), HALF["float32"])


def test_gradients_accumulate_and_repeat_to_the_bit(cuda):
    import rushlite_b200 as rsl

    rng = np.random.default_rng(3)
    x, w, b = rng.standard_normal((700, 384)), rng.standard_normal(384), rng.standard_normal(384)
    g = rsl.Variable(rng.standard_normal((700, 384)).astype(np.float32))
    v = [rsl.Variable(t.astype(np.float32), True) for t in (x, w, b)]
    runs = []
    for _ in range(2):
        for t in v:
            t.zero_grad()
        rsl.layer_norm(*v).backward(g)
        runs.append([t.grad.numpy() for t in v])
    assert all((p == q).all() for p, q in zip(*runs))
    rsl.layer_norm(*v).backward(g)  # on top
    for t, p in zip(v, runs[0]):
        assert (t.grad.numpy() == p + p).all()


def test_one_variable_as_weight_and_bias(cuda):
    import rushlite_b200 as rsl

    rng = np.random.default_rng(4)
    x, w, g = (rng.standard_normal(s).astype(np.float32) for s in ((6, 40), (40,), (6, 40)))
    vw = rsl.Variable(w, True)
    rsl.layer_norm(rsl.Variable(x), vw, vw).backward(rsl.Variable(g))
    ref = _reference(x, w, w, g, 1e-5)
    total = ref["dw"][0] + ref["db"][0]
    _check("dw + db", vw.grad.numpy(), (total, ref["dw"][1] + ref["db"][1] + np.abs(total), C + 6), HALF["float32"])


def test_empty_batch(cuda):
    import rushlite_b200 as rsl

    x, w, b = rsl.Variable(np.zeros((0, 12), np.float32), True), rsl.ones([12], True), rsl.zeros([12], True)
    y = rsl.layer_norm(x, w, b)
    assert y.shape == [0, 12]
    y.backward(rsl.Variable(np.zeros((0, 12), np.float32)))
    assert (w.grad.numpy() == 0).all() and (b.grad.numpy() == 0).all() and x.grad.shape == [0, 12]


def test_unaligned_rows_through_the_c_entry(cuda):
    """Buffers one element off a 16-byte boundary."""
    from rushlite_b200 import capi

    torch = cuda
    for f in (64, 1000, 1028):
        x = torch.randn(5 * f + 1, device="cuda")[1:]
        y = torch.full((5 * f + 2,), 7.0, device="cuda")
        capi.layer_norm(capi.FLOAT32, x.data_ptr(), None, None, 5, f, 1e-5, y[1:].data_ptr())
        torch.cuda.synchronize()
        ref = _reference(x.cpu().numpy().reshape(5, f), None, None, np.ones((5, f), np.float32), 1e-5)
        _check("y", y[1:-1].cpu().numpy().reshape(5, f), ref["y"], HALF["float32"])
        assert y[0] == 7 and y[-1] == 7  # nothing outside


def test_refusals(cuda):
    import rushlite_b200 as rsl

    x = rsl.ones([4, 8])
    for args, text in (((rsl.ones([4, 8], dtype=rsl.dtype.int32),), "float32 or float64"),
                       ((rsl.ones([4, 8], device=rsl.device.cpu),), "CUDA"),
                       ((x, rsl.ones([7])), "shape"), ((x, rsl.ones([4, 8])), "shape"),
                       ((x, rsl.ones([8], dtype=rsl.dtype.float64)), "dtype"),
                       ((x, None, rsl.ones([9])), "bias"), ((x, None, None, -1.0), "eps"),
                       ((x, None, None, float("nan")), "eps"), ((rsl.Variable(np.zeros((4, 0), np.float32)),), "at least 1")):
        with pytest.raises(RuntimeError, match=text):
            rsl.layer_norm(*args)
    y = rsl.layer_norm(rsl.ones([4, 8], True))
    with pytest.raises(RuntimeError, match="shape"):
        y.backward(rsl.ones([8, 4]))


@pytest.mark.parametrize("rows,features", [(4, 64), (700, 1030), (60, 9000)])
def test_recorded_passes_give_the_same_bits(cuda, rows, features):
    """Eager, recorded and replayed, on another stream too: one CTA, tiles with the fold behind them, long rows."""
    import rushlite_b200 as rsl

    rng = np.random.default_rng(rows)
    val = {"x": (rows, features), "w": (features,), "b": (features,), "g": (rows, features)}
    val = {n: rng.standard_normal(s).astype(np.float32) for n, s in val.items()}
    var = {n: rsl.Variable(a, n != "g") for n, a in val.items()}

    def step():
        for n in "xwb":
            var[n].zero_grad()
        y = rsl.layer_norm(var["x"], var["w"], var["b"])
        y.backward(var["g"])
        return y

    y = step()
    want = [y.numpy()] + [var[n].grad.numpy() for n in "xwb"]
    s = cuda.cuda.Stream()
    try:
        rsl.cuda.set_stream(s.cuda_stream)
        graph = rsl.cuda.Graph()
        with graph:
            y = step()
        for _ in range(3):
            graph.replay()
        got = [y.numpy()] + [var[n].grad.numpy() for n in "xwb"]
    finally:
        rsl.cuda.synchronize()
        rsl.cuda.set_stream(0)
    for a, b in zip(got, want):
        assert (a == b).all()
