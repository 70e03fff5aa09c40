"""The AdamW step against its formula in more bits.

Tolerances: u is half a step of the type.  Each moment has 4 roundings, two of
them of constants; the update has those of both moments (half of the second's,
under the root), the rates, a root, a product, a sum, a quotient: under 16; the
parameter keeps two more of its own."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = {"float32": 2.0 ** -24, "float64": 2.0 ** -53}
HP = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def _formula(p, g, m, v, t, lr, betas, eps, weight_decay):
    p, g, m, v = (a.astype(np.longdouble) for a in (p, g, m, v))
    b1, b2 = (np.longdouble(b) for b in betas)
    lr, eps, wd = np.longdouble(lr), np.longdouble(eps), np.longdouble(weight_decay)
    mm, vv = np.abs(b1 * m) + np.abs((1 - b1) * g), b2 * v + (1 - b2) * g * g
    m = b1 * m + (1 - b1) * g
    step = lr / (1 - b1 ** t) / (np.sqrt(vv) / np.sqrt(1 - b2 ** t) + eps)
    new = p - lr * wd * p - step * m
    return {"p": (new, 3 * np.abs(p) + 16 * step * mm), "m": (m, 4 * mm), "v": (vv, 4 * vv)}


def _random(rng, shape, dtype):
    return [(rng.standard_normal(shape) * s).astype(dtype) for s in (0.05, 1e-3, 1e-4)] + [
        (np.square(rng.standard_normal(shape)) * 1e-6).astype(dtype)]


def _optimizer(rsl, sets, dtype, step=0, **hp):
    kind = getattr(rsl.dtype, dtype)
    params = [rsl.Variable(p, True, dtype=kind) for p, _, _, _ in sets]
    opt = rsl.optim.AdamW(params, **{**HP, **hp})
    opt.load_state_dict({"step": step, "exp_avg": [s[2] for s in sets], "exp_avg_sq": [s[3] for s in sets]})
    for p, (_, g, _, _) in zip(params, sets):
        p.grad.copy(rsl.Variable(g, dtype=kind).data)
    return opt


def _check(opt, sets, t, dtype, **hp):
    state = opt.state_dict()
    assert state["step"] == t
    for i, (p, g, m, v) in enumerate(sets):
        ref = _formula(p, g, m, v, t, **{**HP, **hp})
        for name, got in (("p", opt.params[i].numpy()), ("m", state["exp_avg"][i]), ("v", state["exp_avg_sq"][i])):
            want, mag = ref[name]
            assert got.shape == want.shape
            assert (np.abs(got - want) <= HALF[dtype] * mag + np.finfo(dtype).tiny).all(), (i, name)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("shapes", [[(1,)], [(256, 64), (64,), (64, 10), (10,)], [(4096,), (4097,), (4095,), (3,)],
                                    [(2048, 3), (0,), (5, 0, 2), (17,)], [(7, 1001)] * 3,
                                    [(n + 1,) for n in range(130)], [(1 << 20,), (1,)]])
def test_one_step(cuda, shapes, dtype):
    import rushlite_b200 as rsl

    rng = np.random.default_rng(len(shapes))
    sets = [_random(rng, s, dtype) for s in shapes]
    for step in (0, 999):
        opt = _optimizer(rsl, sets, dtype, step)
        opt.step()
        _check(opt, sets, step + 1, dtype)


@pytest.mark.parametrize("hp", [dict(betas=(0.0, 0.0)), dict(weight_decay=0.0), dict(lr=0.0), dict(eps=0.5)])
def test_edges_of_the_rates(cuda, hp):
    import rushlite_b200 as rsl

    sets = [_random(np.random.default_rng(1), (300,), "float32")]
    opt = _optimizer(rsl, sets, "float32", 4, **hp)
    opt.step()
    _check(opt, sets, 5, "float32", **hp)


def test_steps_count_and_the_state_is_carried(cuda):
    """Three steps, each from the values that the one before left."""
    import rushlite_b200 as rsl

    sets = [_random(np.random.default_rng(2), (77, 5), "float32")]
    opt = _optimizer(rsl, sets, "float32")
    for t in (1, 2, 3):
        opt.step()
        _check(opt, sets, t, "float32")
        state = opt.state_dict()
        sets = [[opt.params[0].numpy(), sets[0][1], state["exp_avg"][0], state["exp_avg_sq"][0]]]


def test_no_gradient_is_a_gradient_of_zero(cuda):
    import rushlite_b200 as rsl

    p = np.linspace(-1, 1, 50).astype(np.float32)
    opt = rsl.optim.AdamW([rsl.Variable(p, True)], lr=0.1, weight_decay=0.5)
    opt.step()
    z = np.zeros_like(p)
    _check(opt, [[p, z, z, z]], 1, "float32", lr=0.1, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.5)


def test_recorded_step_counts_its_replays(cuda):
    import rushlite_b200 as rsl

    sets = [_random(np.random.default_rng(3), (129, 3), "float32"), _random(np.random.default_rng(4), (65,), "float32")]
    a, b = _optimizer(rsl, sets, "float32"), _optimizer(rsl, sets, "float32")
    for _ in range(4):
        a.step()
    graph = rsl.cuda.Graph()
    b.step()
    with graph:
        b.step()
    for _ in range(3):
        graph.replay()
    assert b.state_dict()["step"] == a.state_dict()["step"] == 4
    for p, q in zip(a.params, b.params):
        assert (p.numpy() == q.numpy()).all()


def test_recorded_step_outlives_the_optimizer(cuda):
    import rushlite_b200 as rsl

    rng = np.random.default_rng(6)
    sets = [_random(rng, (300, 100), "float32")]
    opt, twin = _optimizer(rsl, sets, "float32"), _optimizer(rsl, sets, "float32")
    param, graph = opt.params[0], rsl.cuda.Graph()
    with graph:
        opt.step()
    del opt
    junk = [rsl.Variable(np.full((300, 100), 1e9, np.float32)) for _ in range(8)]  # over any memory given back
    for _ in range(3):
        graph.replay()
        twin.step()
    assert (param.numpy() == twin.params[0].numpy()).all()
    assert all((j.numpy() == 1e9).all() for j in junk)


@pytest.mark.parametrize("shape", [(300, 100), (5,)])
def test_recorded_step_keeps_its_gradients(cuda, shape):
    """A replay reads the gradients of the capture, also after zero_grad() gave the parameters others."""
    import rushlite_b200 as rsl

    rng = np.random.default_rng(8)
    sets = [_random(rng, shape, "float32")]
    opt, twin = _optimizer(rsl, sets, "float32"), _optimizer(rsl, sets, "float32")
    graph = rsl.cuda.Graph()
    with graph:
        opt.step()
    opt.zero_grad()
    junk = [rsl.Variable(np.full(shape, 1e9, np.float32)) for _ in range(8)]  # over any memory given back
    for _ in range(3):
        graph.replay()
        twin.step()
    assert (opt.params[0].numpy() == twin.params[0].numpy()).all()
    assert (opt.params[0].grad.numpy() == 0).all() and all((j.numpy() == 1e9).all() for j in junk)


def test_special_values_stay_where_they_are(cuda):
    import rushlite_b200 as rsl

    s = _random(np.random.default_rng(5), (5000,), "float32")
    s[1][17], s[1][4999] = np.nan, np.inf
    opt = _optimizer(rsl, [s], "float32")
    opt.step()
    got = opt.params[0].numpy()
    assert np.flatnonzero(~np.isfinite(got)).tolist() == [17, 4999]


def test_unaligned_buffers_through_the_c_entry(cuda):
    from rushlite_b200 import capi

    torch = cuda
    n = 9001
    sets = _random(np.random.default_rng(6), (n,), "float32")
    bufs = [torch.full((n + 2,), 7.0, device="cuda") for _ in sets]
    for t, a in zip(bufs, sets):
        t[1:-1] = torch.from_numpy(a).cuda()
    step = torch.zeros(2, dtype=torch.int64, device="cuda")
    capi.adamw(capi.FLOAT32, [(*(t[1:].data_ptr() for t in bufs), n)], 3e-3, 0.9, 0.999, 1e-8, 0.1, step.data_ptr())
    torch.cuda.synchronize()
    ref = _formula(*sets, 1, **HP)
    for t, name in ((bufs[0], "p"), (bufs[2], "m"), (bufs[3], "v")):
        assert (np.abs(t[1:-1].cpu().numpy() - ref[name][0]) <= HALF["float32"] * ref[name][1]).all()
        assert t[0] == 7 and t[-1] == 7
    assert step.tolist() == [1, 0]


def test_refusals(cuda):
    import rushlite_b200 as rsl

    p = rsl.ones([3], True)
    for bad in ([], [p, p], [rsl.ones([3])], [rsl.ones([3], True, device=rsl.device.cpu)],
                [rsl.ones([3], True, dtype=rsl.dtype.int32)], [p, rsl.ones([3], True, dtype=rsl.dtype.float64)]):
        with pytest.raises(ValueError, match="AdamW"):
            rsl.optim.AdamW(bad)
    for hp in (dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0),
               dict(weight_decay=-0.1)):
        with pytest.raises(RuntimeError, match="adamw"):
            rsl.optim.AdamW([p], **hp).step()
    opt = rsl.optim.AdamW([p])
    with pytest.raises(ValueError, match="shapes"):
        opt.load_state_dict({"step": 0, "exp_avg": [np.zeros(4)], "exp_avg_sq": [np.zeros(3)]})
    with pytest.raises(ValueError, match="negative"):
        opt.load_state_dict({"step": -1, "exp_avg": [np.zeros(3)], "exp_avg_sq": [np.zeros(3)]})
    view = rsl.Variable(p.data, True)  # the same memory under another name
    with pytest.raises(RuntimeError, match="twice"):
        rsl.optim.AdamW([p, view]).step()
    assert opt.state_dict()["step"] == 0 and (p.numpy() == 1).all()
