"""Causal attention over packed sequences against the formula in 64 bits, its
gradients against differences, and its refusals.

Tolerances, per element, from what is added (magnitudes M below):
* a score is a sum of D products.  On the tensor cores each operand is two
  fp16 parts, together within 2^-22 of it, and the product of the two small
  parts is left out (2^-22): 3 * 2^-22 of each product; the accumulator may
  lose a step of 2^-23 of the sum of magnitudes at each addition of a product,
  D * 2^-23 at most.  Plain fp32 loses at most D * 2^-24.  So a score is within
  E = (3 + D / 2) * 2^-22 * scale * |q| . |k|.
* a weight P is exp of a difference of two such scores (or score and lse, whose
  value is rounded to fp32, as a base-2 logarithm): within 2 E + 2^-23 |lse| +
  2^-21 of itself.
* what sums weights times values has the same 3 * 2^-22 a product, and at most
  2^-23 a product and block of additions that follow one another: L 2^-23.
* the fp16 parts have a smallest step of 2^-24, so of an operand scaled to have
  its largest value (of a 128-row tile), a weight 1, or dS its bound
  B = max|g| max|v| + max|delta| at 2^14 or more, the two parts are within
  max(2^-22 |x|, 2^-25) of x in that scale: an absolute 2^-39 of that largest
  value.  Where all of a sum's terms are tiny against it, this is what is left.
Each bound is the sum of these times the magnitudes added, in 64 bits."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

CASES = [  # lengths, heads, kv_heads, head_dim, rows behind the last sequence
    ([1], 1, 1, 1, 0), ([7], 4, 4, 64, 0), ([1, 2, 3, 0, 5], 2, 1, 8, 2), ([63, 64, 65], 4, 2, 33, 0),
    ([128, 127, 129, 1], 4, 1, 128, 5), ([300, 17, 513], 6, 2, 80, 0), ([0, 0], 2, 2, 16, 3), ([], 2, 1, 4, 4),
    ([1030], 3, 3, 96, 1), ([255, 256, 257], 8, 1, 16, 0), ([2049], 4, 2, 128, 0), ([1500, 31, 700, 1], 4, 2, 64, 0),
    ([1] * 40, 3, 1, 31, 0), ([640] * 3, 2, 2, 65, 130),
    ([5, 60, 30, 40, 1, 0, 128, 3, 127, 1, 64, 64, 2, 70], 4, 2, 64, 0),  # several sequences in a 128-row tile
    ([90, 20, 18, 90, 38, 0, 0, 1, 300, 5], 6, 1, 128, 9),
]


FLOOR = 2.0 ** -39


def _inputs(torch, rng, case, scale=1.0):
    lengths, hq, hkv, d, tail = case
    t = sum(lengths) + tail
    x = {"q": (t, hq, d), "k": (t, hkv, d), "v": (t, hkv, d), "g": (t, hq, d)}
    x = {n: torch.from_numpy((rng.standard_normal(s) * scale).astype(np.float32)) for n, s in x.items()}
    if tail:  # rows of no sequence: never read
        for a in x.values():
            a[t - tail:] = math.nan
    return x


def _reference(torch, x, lengths, scale=None):
    """{name: (value, tolerance)}, rows behind the last sequence 0."""
    x = {n: a.cuda().double() for n, a in x.items()}
    q, k, v, g = (x[n] for n in "qkvg")
    t, hq, d = q.shape
    hkv = k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    zero = lambda a: [torch.zeros_like(a), torch.zeros_like(a)]  # noqa: E731
    out = {"out": zero(q), "dq": zero(q), "dk": zero(k), "dv": zero(v)}
    w = 2.0 ** -22
    start = 0
    for n in lengths:
        rows = slice(start, start + n)
        start += n
        if n == 0:
            continue
        for h in range(hq):
            j = h * hkv // hq
            Q, K, V, G = q[rows, h], k[rows, j], v[rows, j], g[rows, h]
            mask = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            S = (scale * Q @ K.T).masked_fill(~mask, -math.inf)
            lse = torch.logsumexp(S, 1, keepdim=True)
            P = torch.exp(S - lse)
            top = {a: float(b.abs().max()) for a, b in (("q", Q), ("k", K), ("v", V), ("g", G))}
            q1, k1, v1, g1 = (a.abs().sum(1) for a in (Q, K, V, G))
            E = (3 + d / 2) * w * scale * (Q.abs() @ K.abs().T) + scale * FLOOR * (top["k"] * q1[:, None] + top["q"] * k1)
            E = E.masked_fill(~mask, 0)
            rel = 2 * E.amax(1, keepdim=True) + w * (lse.abs() / 2 + 2)  # of a weight
            sums = (3 + n / 2) * w
            O = P @ V
            seen = mask.double()
            out["out"][0][rows, h] = O
            out["out"][1][rows, h] = (rel + sums) * (P @ V.abs()) + FLOOR * (seen @ V.abs() + top["v"])
            dP = G @ V.T
            delta = (G * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            # dP and delta: D products each, delta with the output's own error
            size = (G.abs() @ V.abs().T) + (G.abs() * (P @ V.abs())).sum(1, keepdim=True)
            dSt = (rel + (3 + d / 2) * w + sums) * P * size + rel * dS.abs()
            dSt = dSt + P * FLOOR * (top["v"] * g1[:, None] + top["g"] * v1 + (G.abs() @ V.abs().sum(0)[:, None] + top["v"] * g1[:, None]))
            bound = float(G.norm(dim=1).max() * V.norm(dim=1).max() + delta.abs().max())
            dSt = dSt + FLOOR * bound * seen
            dSm = P * size
            out["dq"][0][rows, h] = scale * dS @ K
            out["dq"][1][rows, h] = scale * (dSt @ K.abs() + sums * (dSm @ K.abs()) + FLOOR * top["k"] * dSm.sum(1, keepdim=True))
            out["dk"][0][rows, j] += scale * dS.T @ Q
            out["dk"][1][rows, j] += scale * (dSt.T @ Q.abs() + sums * (dSm.T @ Q.abs()) + FLOOR * top["q"] * dSm.sum(0)[:, None])
            out["dv"][0][rows, j] += P.T @ G
            out["dv"][1][rows, j] += (rel * P).T @ G.abs() + sums * (P.T @ G.abs())
            out["dv"][1][rows, j] += FLOOR * (seen.T @ G.abs() + top["g"] * P.sum(0)[:, None])
    return {n: (a.cpu().numpy(), b.cpu().numpy()) for n, (a, b) in out.items()}


def _check(name, got, ref):
    want, tol = ref
    assert got.shape == want.shape, name
    assert np.isfinite(got).all(), (name, np.argwhere(~np.isfinite(got))[:3])
    worst = np.abs(got - want) - tol - 1e-37
    assert (worst <= 0).all(), (name, np.argwhere(worst > 0)[:3], float(worst.max()))


def _run(rsl, x, lengths, scale=None, seqs=None):
    var = {n: rsl.Variable(x[n].numpy(), n != "g") for n in "qkvg"}
    o = rsl.causal_attention(var["q"], var["k"], var["v"], seqs or rsl.Sequences(lengths), scale)
    o.backward(var["g"])
    return {"out": o.numpy(), **{"d" + n: var[n].grad.numpy() for n in "qkv"}}


@pytest.mark.parametrize("case", CASES, ids=lambda c: "%s-%d-%d-%d-%d" % ("_".join(map(str, c[0][:5])), *c[1:]))
def test_forward_and_backward(cuda, case):
    import rushlite_b200 as rsl

    x = _inputs(cuda, np.random.default_rng(sum(case[0]) + case[3]), case)
    got = _run(rsl, x, case[0])
    ref = _reference(cuda, x, case[0])
    for name in got:
        _check(name, got[name], ref[name])
    # and as a whole, for inputs of unit size, where roundings average out: 2^-18 (forward) and 2^-17
    for name in got:
        norm = np.linalg.norm(ref[name][0])
        if norm > 1e-3 * np.linalg.norm(ref[name][1]) / 2.0 ** -22:
            assert np.linalg.norm(got[name] - ref[name][0]) <= 2.0 ** (-18 if name == "out" else -17) * norm, name


def _results(x, lengths, scale=None):
    import rushlite_b200 as rsl

    return _run(rsl, x, lengths, scale)


def _rows_reference(torch, x, lengths, scale):
    """As _reference, for gradients whose rows differ in size: what is left
    where terms are tiny counts against the largest term of the result's own
    row, not of its sequence or tile.

    A row of grad has its own scale, its largest value g* at 2^14 or more, so
    its parts are within 2^-39 g* (FLOOR).  Scaled rows are at most 2^15
    sqrt(D) long and dP - delta of them at most 2^15 R with R = sqrt(D) max|v| +
    max(|delta| / g*).  dq: a row's bound is then 2 sqrt(D) g* max|v| + |delta|,
    and dS is within 2^-39 of it.  dk, dv: the weights of key j, P_ij over the
    scale of row i, are scaled to have the largest between 2^13 and 2^14, so
    with T_j = max(P_ij g*_i) a step of 2^-25 is at most
    2^-25 2 T_j / 2^28 of a weight: 2^-37 T_j sum(|g| / g*) of dv, and with dS's
    own step as much again times R, 2^-36 T_j R of dS.  T_j counts as 2^-98 at
    least (the scale ends at 2^112)."""
    x = {n: a.cuda().double() for n, a in x.items()}
    q, k, v, g = (x[n] for n in "qkvg")
    hq, d, hkv = q.shape[1], q.shape[2], k.shape[1]
    zero = lambda a: [torch.zeros_like(a), torch.zeros_like(a)]  # noqa: E731
    out = {"dq": zero(q), "dk": zero(k), "dv": zero(v)}
    w = 2.0 ** -22
    top = {n: float(x[n].abs().max()) for n in "qkv"}
    vnorm = float(v.norm(dim=2).max())
    start, parts = 0, []
    for n in lengths:
        rows = slice(start, start + n)
        start += n
        for h in range(hq if n else 0):
            j = h * hkv // hq
            Q, K, V, G = q[rows, h], k[rows, j], v[rows, j], g[rows, h]
            mask = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
            S = (scale * Q @ K.T).masked_fill(~mask, -math.inf)
            lse = torch.logsumexp(S, 1, keepdim=True)
            P = torch.exp(S - lse)
            O = P @ V
            delta = (G * O).sum(1, keepdim=True)
            big = G.abs().amax(1, keepdim=True)
            parts.append((rows, h, j, Q, K, V, G, mask, S, lse, P, O, delta, big))
    ratio = max(float((p[-2].abs() / p[-1].clamp_min(1e-300)).max()) for p in parts)
    R = math.sqrt(d) * vnorm + ratio
    for rows, h, j, Q, K, V, G, mask, S, lse, P, O, delta, big in parts:
        n = len(Q)
        g1, v1, k1, q1 = (a.abs().sum(1) for a in (G, V, K, Q))
        E = (3 + d / 2) * w * scale * (Q.abs() @ K.abs().T) + scale * FLOOR * (top["k"] * q1[:, None] + top["q"] * k1)
        rel = 2 * E.masked_fill(~mask, 0).amax(1, keepdim=True) + w * (lse.abs() / 2 + 2)
        sums, seen = (3 + n / 2) * w, mask.double()
        dP = G @ V.T
        dS = P * (dP - delta)
        size = (G.abs() @ V.abs().T) + (G.abs() * (P @ V.abs())).sum(1, keepdim=True)
        dSm = P * size
        dSt = (rel + (3 + d / 2) * w + sums) * dSm + rel * dS.abs()
        dSt = dSt + P * FLOOR * (2 * top["v"] * g1[:, None] + big * v1 + G.abs() @ V.abs().sum(0)[:, None])
        own = FLOOR * (2 * math.sqrt(d) * big * vnorm + delta.abs()) * seen
        T = (P * big).amax(0).clamp_min(2.0 ** -98)
        key = 2.0 ** -36 * R * T * seen
        unit = G.abs() / big.clamp_min(1e-300)
        out["dq"][0][rows, h] = scale * dS @ K
        out["dq"][1][rows, h] = scale * ((dSt + own) @ K.abs() + sums * (dSm @ K.abs()) + FLOOR * top["k"] * dSm.sum(1, keepdim=True))
        out["dk"][0][rows, j] += scale * dS.T @ Q
        out["dk"][1][rows, j] += scale * ((dSt + key).T @ Q.abs() + sums * (dSm.T @ Q.abs()) + FLOOR * top["q"] * dSm.sum(0)[:, None])
        out["dv"][0][rows, j] += P.T @ G
        out["dv"][1][rows, j] += (rel * P).T @ G.abs() + sums * (P.T @ G.abs())
        out["dv"][1][rows, j] += 2.0 ** -37 * T[:, None] * (seen.T @ unit) + FLOOR * (P.T @ big)
    return {n: (a.cpu().numpy(), b.cpu().numpy()) for n, (a, b) in out.items()}


SMALL_ROWS = [(case, where) for case in (([300], 2, 1, 64, 0), ([300], 2, 2, 128, 0), ([2049], 1, 1, 64, 0),
                                         ([1000, 64, 64, 40, 40, 7], 2, 1, 33, 0), ([40] * 6 + [600], 4, 2, 96, 3))
              for where in ("every other row", "few large rows", "every other sequence")
              if where != "every other sequence" or len(case[0]) > 1]


@pytest.mark.parametrize("case,where", SMALL_ROWS, ids=lambda a: a if isinstance(a, str) else
                         "%s-%d" % ("_".join(map(str, a[0][:3])), a[3]))
@pytest.mark.parametrize("bits", [8, 14, 20, 26, 40, 80])
def test_rows_with_small_gradients(cuda, case, where, bits):
    """A row whose gradient is far below its neighbours' keeps its own accuracy, alone and where sequences share a tile."""
    lengths, hq, _, d, tail = case
    x = _inputs(cuda, np.random.default_rng(bits + d), case)
    t = sum(lengths)
    if where == "every other row":
        small = np.arange(t) % 2 == 1
    elif where == "few large rows":
        small = np.arange(t) % 50 != 20
    else:
        small = np.concatenate([np.full(n, i % 2 == 1) for i, n in enumerate(lengths)])
    x["g"][:t][cuda.from_numpy(small)] *= 2.0 ** -bits
    got = _results(x, lengths)
    ref = _rows_reference(cuda, {n: a[:t] for n, a in x.items()}, lengths, 1 / math.sqrt(d))
    for name in ("dq", "dk", "dv"):
        _check(name, got[name][:t], ref[name])
        assert not got[name][t:].any()
    for rows in (small, ~small):  # the bar of test_forward_and_backward, for each size of its own
        err, value = (got["dq"][:t] - ref["dq"][0])[rows], ref["dq"][0][rows]
        assert np.linalg.norm(err) <= 2.0 ** -17 * np.linalg.norm(value)
    if where == "every other sequence":
        for name in ("dk", "dv"):
            err, value = (got[name][:t] - ref[name][0])[small], ref[name][0][small]
            assert np.linalg.norm(err) <= 2.0 ** -17 * np.linalg.norm(value), name


@pytest.mark.parametrize("dim", [64, 128])
def test_sequences_of_very_different_gradients_share_a_tile(cuda, dim):
    lengths = [31, 30, 33, 34, 200]
    x = _inputs(cuda, np.random.default_rng(3 + dim), (lengths, 2, 1, dim, 0))
    start = 0
    for n, f in zip(lengths, (1.0, 1e-6, 1e-10, 1e-13, 1e-20)):
        x["g"][start:start + n] *= f
        start += n
    got = _results(x, lengths)
    ref = _rows_reference(cuda, x, lengths, 1 / math.sqrt(dim))
    start = 0
    for name in ("dq", "dk", "dv"):
        _check(name, got[name], ref[name])
    for n in lengths:
        rows = slice(start, start + n)
        start += n
        for name in ("dq", "dk", "dv"):
            value = ref[name][0][rows]
            assert np.linalg.norm(got[name][rows] - value) <= 2.0 ** -17 * np.linalg.norm(value), (name, n)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits", [0, 20, 40])
def test_small_gradients_with_sharp_weights(cuda, dim, bits):
    """Scores with a deviation of 8 and more: keys that hardly a row looks at, seen by rows with large and small gradients."""
    lengths = [500, 60, 60]
    x = _inputs(cuda, np.random.default_rng(5 + dim), (lengths, 2, 1, dim, 0))
    x["g"][::2] *= 2.0 ** -bits
    got = _results(x, lengths, 1.0)
    ref = _rows_reference(cuda, x, lengths, 1.0)
    for name in ("dq", "dk", "dv"):
        _check(name, got[name], ref[name])


def _tiles_reference(torch, x, scale):
    """_rows_reference for one sequence whose 128-row tiles differ in size: what
    is left where terms are tiny counts against the largest term of the
    result's row in the same tile of keys (of queries, for dk and dv), 2^-39
    of it and for powers of two between twice that."""
    x = {n: a.cuda().double() for n, a in x.items()}
    Q, K, V, G = (x[n][:, 0] for n in "qkvg")
    n, d = Q.shape
    w, sums = 2.0 ** -22, (3 + n / 2) * 2.0 ** -22
    tiles = [slice(b, min(b + 128, n)) for b in range(0, n, 128)]
    mask = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    S = (scale * Q @ K.T).masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(S, 1, keepdim=True)
    P = torch.exp(S - lse)
    O, dP = P @ V, G @ V.T
    delta = (G * O).sum(1, keepdim=True)
    dS = P * (dP - delta)
    big = G.abs().amax(1, keepdim=True)
    full = lambda: torch.zeros(n, n, dtype=torch.float64, device="cuda")  # noqa: E731
    e, own, key, wrow, wcol, parts = full(), full(), full(), full(), full(), full()
    least = min(float(V[c].norm(dim=1).max()) or math.inf for c in tiles)
    for c in tiles:
        kt, vt, vn = float(K[c].abs().max()), float(V[c].abs().max()), float(V[c].norm(dim=1).max())
        top = P[:, c].amax(1, keepdim=True)
        e[:, c] = FLOOR * kt * Q.abs().sum(1)[:, None]
        wrow[:, c] = FLOOR * top
        own[:, c] = 2 * FLOOR * top * (2 * math.sqrt(d) * big * vn + delta.abs())
        parts[:, c] = FLOOR * (vt * G.abs().sum(1)[:, None] + big * V[c].abs().sum(1))
        for r in tiles:
            e[r, c] += FLOOR * float(Q[r].abs().max()) * K[c].abs().sum(1)
            ratio = float((delta[r].abs() / big[r]).max())
            T = (P[r, c] * big[r]).amax(0)
            wcol[r, c] = 2.0 ** -37 * T
            if ratio <= 2.0 ** 19 * math.sqrt(d) * (vn or least):  # else the fp32 kernels' result
                key[r, c] = 2.0 ** -36 * (math.sqrt(d) * vn + ratio) * T
    E = (3 + d / 2) * w * scale * (Q.abs() @ K.abs().T) + scale * e
    rel = 2 * E.masked_fill(~mask, 0).amax(1, keepdim=True) + w * (lse.abs() / 2 + 2)
    seen = mask.double()
    size = (G.abs() @ V.abs().T) + (G.abs() * (P @ V.abs())).sum(1, keepdim=True)
    tv, tk, tq = (torch.cat([a[b].abs().max().expand(b.stop - b.start) for b in tiles])[:, None] for a in (V, K, Q))
    # delta: the products, the weights' steps and v's parts of out
    left = (G.abs() * ((wrow * seen) @ V.abs() + FLOOR * P @ tv)).sum(1, keepdim=True)
    dSm = P * size
    dSt = (rel + (3 + d / 2) * w + sums) * dSm + rel * dS.abs() + P * (parts + left)
    out = {"out": (O, (rel + sums) * (P @ V.abs()) + (wrow * seen) @ V.abs() + FLOOR * (P @ tv)),
           "dq": (scale * dS @ K, scale * ((dSt + own * seen) @ K.abs() + sums * (dSm @ K.abs()) + FLOOR * (dSm @ tk))),
           "dk": (scale * dS.T @ Q, scale * ((dSt + key * seen).T @ Q.abs() + sums * (dSm.T @ Q.abs()) + FLOOR * (dSm.T @ tq))),
           "dv": (P.T @ G, (rel * P).T @ G.abs() + sums * (P.T @ G.abs()) + (wcol * seen).T @ (G.abs() / big) + FLOOR * (P.T @ big))}
    return {n: tuple(b.cpu().numpy()[:, None] for b in a) for n, a in out.items()}


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("what", ["v", "k", "vk", "q", "g"])
@pytest.mark.parametrize("bits", [(25, 0, 0, 0), (0, 20, 0, 30), (0, 0, 30, 10), (-25, 0, -10, 0)])
@pytest.mark.parametrize("scale", [1.0, 2.0])
def test_tiles_of_very_different_size(cuda, dim, what, bits, scale):
    """Tiles of 128 tokens whose values lie powers of two apart, under sharp weights: a row that hardly looks
    at a tile of large values keeps its accuracy.  The size of k and q stands in a column where the other is 0."""
    n = 450
    x = _inputs(cuda, np.random.default_rng(31 + dim), ([n], 1, 1, dim, 0))
    f = cuda.tensor([2.0 ** b for b in bits]).repeat_interleave(128)[:n, None]
    x["k"][:, :, 0] = x["q"][:, :, 0] = 0
    if "q" in what:
        x["q"][:, :, 0] = f
    if "k" in what:
        x["k"][:, :, 0] = f
    for name in set(what) & set("vg"):
        x[name] *= f[:, :, None]
    got, ref = _results(x, [n], scale), _tiles_reference(cuda, x, scale)
    for name in got:
        _check(name, got[name], ref[name])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("sizes", [(1.0, 0.0, 1.0, 1.0), (0.0, 1.0, 0.0, 2.0 ** -25), (2.0 ** 22, 0.0, 1.0, 1.0)])
def test_tiles_without_values(cuda, dim, sizes):
    """Tiles of 128 tokens whose v is 0, as a program that masks keys may leave them."""
    n = 500
    x = _inputs(cuda, np.random.default_rng(35 + dim), ([n], 1, 1, dim, 0))
    x["v"] *= cuda.tensor(sizes).repeat_interleave(128)[:n, None, None]
    got, ref = _results(x, [n], 1.0), _tiles_reference(cuda, x, 1.0)
    for name in got:
        _check(name, got[name], ref[name])


@pytest.mark.parametrize("dim", [33, 64, 128])
@pytest.mark.parametrize("bits", [dict(v=16, k=10), dict(v=14, k=14), dict(v=16, q=10), dict(v=12, q=16), dict(v=15, q=10, k=10)],
                         ids=lambda b: "-".join(n + str(a) for n, a in b.items()))
def test_two_operands_with_rows_far_apart(cuda, dim, bits):
    """A gradient's weight follows the size of v and is multiplied by q or k.  Where rows of both differ, terms of
    small rows stand next to large ones of little weight.  Each row against the magnitudes of its terms: the roundings
    of scores (up to 60 here, 2^-24 of them twice) move weights by 2^-17 at most, and sums average out: 2^-16."""
    lengths = [5, 20, 50, 33, 20, 12, 48, 47, 70, 9, 60, 60, 41, 80, 128, 200, 300] * 4
    t = sum(lengths)
    x = _inputs(cuda, np.random.default_rng(37 + dim), (lengths, 2, 1, dim, 0))
    for name, b in bits.items():
        x[name] *= 2.0 ** -(b * (cuda.arange(t) % 2).float())[:, None, None]
    scale = float(np.float32(10 / math.sqrt(dim)))
    got = _results(x, lengths, scale)
    ref = _reference(cuda, x, lengths, scale)
    x = {n: a.cuda().double() for n, a in x.items()}
    size = {"dq": cuda.zeros_like(x["q"]), "dk": cuda.zeros_like(x["k"])}
    start = 0
    for n in lengths:
        r = slice(start, start + n)
        start += n
        for h in range(2):
            Q, K, V, G = x["q"][r, h], x["k"][r, 0], x["v"][r, 0], x["g"][r, h]
            P = (scale * Q @ K.T).masked_fill(~cuda.ones(n, n, dtype=cuda.bool, device="cuda").tril(), -math.inf).softmax(1)
            A = scale * P * (G.abs() @ V.abs().T + (G.abs() * (P @ V.abs())).sum(1, keepdim=True))
            size["dq"][r, h] = A @ K.abs()
            size["dk"][r, 0] += A.T @ Q.abs()
    for name in size:
        off = np.linalg.norm(got[name] - ref[name][0], axis=-1) / size[name].norm(dim=-1).cpu().numpy()
        assert off.max() <= 2.0 ** -16, (name, off.argmax(), math.log2(off.max()))


@pytest.mark.parametrize("size", [1e-30, 1e-33, 1e-35, 1e-37])
def test_gradients_next_to_underflow(cuda, size):
    """The bar of test_forward_and_backward where the results' own steps, 2^-149, still pass it."""
    lengths = [40, 40, 40]
    x = _inputs(cuda, np.random.default_rng(36), (lengths, 2, 1, 64, 0))
    x["g"] *= size
    got, ref = _results(x, lengths), _reference(cuda, x, lengths)
    for name in ("dq", "dk", "dv"):
        want = ref[name][0]
        assert np.linalg.norm((got[name] - want) / size) <= 2.0 ** -17 * np.linalg.norm(want / size), name


def test_rows_without_a_gradient(cuda):
    """Rows that a loss leaves out: their dq is 0, and they change nobody's results."""
    lengths = [200, 50, 60]
    x = _inputs(cuda, np.random.default_rng(6), (lengths, 2, 1, 64, 0))
    x["g"] *= 1e-12
    out = np.arange(310) % 3 != 0
    x["g"][cuda.from_numpy(out)] = 0
    x["g"][250:] = 0  # a whole sequence
    got = _results(x, lengths)
    ref = _rows_reference(cuda, x, lengths, 1 / 8)
    for name in ("dq", "dk", "dv"):
        _check(name, got[name], ref[name])
    assert not got["dq"][out].any() and not got["dk"][250:].any() and not got["dv"][250:].any()


@pytest.mark.parametrize("scale", [1e-3, 0.7, 3.0])
def test_scale(cuda, scale):
    import rushlite_b200 as rsl

    case = ([200, 9], 2, 1, 40, 0)
    x = _inputs(cuda, np.random.default_rng(7), case)
    got, ref = _run(rsl, x, case[0], scale), _reference(cuda, x, case[0], float(np.float32(scale)))
    for name in got:
        _check(name, got[name], ref[name])


@pytest.mark.parametrize("size", [1e-20, 1e-6, 30.0])
def test_sizes_of_values(cuda, size):
    """Products of tiny values underflow to 0, which the formula's are too within fp32's smallest steps."""
    import rushlite_b200 as rsl

    case = ([300, 40], 2, 2, 64, 0)
    x = _inputs(cuda, np.random.default_rng(8), case, size)
    if size == 1e-20:  # gradients of it underflow: the forward alone
        got = rsl.causal_attention(*(rsl.Variable(x[n].numpy()) for n in "qkv"), rsl.Sequences(case[0])).numpy()
        return _check("out", got, _reference(cuda, x, case[0])["out"])
    got, ref = _run(rsl, x, case[0]), _reference(cuda, x, case[0])
    for name in got:
        _check(name, got[name], ref[name])


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf, 3e38, 1e30])
@pytest.mark.parametrize("dim", [48, 128])
def test_what_a_row_does_not_see_does_not_reach_it(cuda, bad, dim):
    """Values behind the diagonal, in another sequence and in another group's
    heads: rows before them and the other heads keep results within tolerance."""
    import rushlite_b200 as rsl

    lengths, t = [400, 300, 5], 705
    x = _inputs(cuda, np.random.default_rng(9), (lengths, 4, 2, dim, 0))
    ref = _reference(cuda, x, lengths)
    p = 190  # in the first sequence
    x["k"][p, 1, 3] = bad
    x["v"][p + 1, 1, 0] = bad
    got = {n: a for n, a in _run(rsl, x, lengths).items()}
    for name in ("out", "dq"):  # group 0's heads; group 1's rows of the first sequence before p; the other sequences
        for rows, heads in ((slice(0, t), slice(0, 2)), (slice(0, p), slice(2, 4)), (slice(400, t), slice(2, 4))):
            _check(name, got[name][rows, heads], tuple(a[rows, heads] for a in ref[name]))
    for name in ("dk", "dv"):  # keys of group 1's first sequence hear from rows behind p
        for rows, heads in ((slice(0, t), slice(0, 1)), (slice(400, t), slice(1, 2))):
            _check(name, got[name][rows, heads], tuple(a[rows, heads] for a in ref[name]))
    if not math.isfinite(bad):
        assert not np.isfinite(got["out"][p + 1:400, 2:]).any(axis=-1).all()
    # a query's own values reach its row alone, and the keys it sees
    x = _inputs(cuda, np.random.default_rng(9), (lengths, 4, 2, dim, 0))
    x["q"][p, 3, 1] = bad
    x["g"][p, 3, 2] = bad
    got = _run(rsl, x, lengths)
    keep = np.ones(t, bool)
    keep[p] = False
    for name in ("out", "dq"):
        _check(name, got[name][keep], tuple(a[keep] for a in ref[name]))
    for name in ("dk", "dv"):
        _check(name, got[name][:, 0], tuple(a[:, 0] for a in ref[name]))
        _check(name, got[name][p + 1:, 1], tuple(a[p + 1:, 1] for a in ref[name]))


@pytest.mark.parametrize("lengths", [[20, 7], [300, 9, 100]])
@pytest.mark.parametrize("size", [2.0 ** 5, 2.0 ** 12, 2.0 ** 30])
def test_scores_far_apart_pick_one_key(cuda, lengths, size):
    """Keys that are powers-of-two multiples of each other's direction: every row's
    largest score is its own key's and the next one at least size^2 / 4 below,
    so its weight is 1 exactly and the gradients through the weights are 0."""
    import rushlite_b200 as rsl

    t, d = sum(lengths), 16
    rng = np.random.default_rng(21)
    v, g = (rng.standard_normal((t, 1, d)).astype(np.float32) for _ in range(2))
    at = np.concatenate([np.arange(n) for n in lengths])
    k = np.zeros((t, 1, d), np.float32)
    k[:, 0, 0] = size * (1 + at / 4)  # exact
    q = np.zeros((t, 1, d), np.float32)
    q[:, 0, 0] = size
    x = {"q": q, "k": k, "v": v, "g": g}
    got = _run(rsl, {n: cuda.from_numpy(a) for n, a in x.items()}, lengths, 1.0)
    tol = 2.0 ** -20 * np.abs(v).max()
    assert (np.abs(got["out"] - v) <= tol).all()
    assert (np.abs(got["dv"] - g) <= 2.0 ** -20 * np.abs(g).max()).all()
    # dS = P (dP - delta) with P = 1: what is left is roundings of dP and delta, D products each
    left = 2 * (d + 24) * 2.0 ** -22 * float((np.abs(g) @ np.abs(v).swapaxes(1, 2)).max()) * d
    assert (np.abs(got["dq"][:, 0, 0]) <= left * np.abs(k).max() * max(lengths)).all()
    assert np.isfinite(got["dk"]).all() and (np.abs(got["dk"]) <= left * size * max(lengths)).all()


@pytest.mark.parametrize("size", [300.0, 3e4, 1e8])
def test_large_values_stay_finite(cuda, size):
    """Scores whose own rounding passes 1: weights are between 0 and 1 all the same."""
    import rushlite_b200 as rsl

    lengths = [260, 30]
    x = _inputs(cuda, np.random.default_rng(22), (lengths, 2, 1, 64, 0))
    x["q"] *= size
    x["k"] *= size
    got = _run(rsl, x, lengths)
    assert all(np.isfinite(a).all() for a in got.values())
    assert (np.abs(got["out"]) <= float(x["v"].abs().max()) * (1 + 2.0 ** -18)).all()


def test_repeated_backward_of_one_graph(cuda):
    import rushlite_b200 as rsl

    lengths = [140, 20]
    x = _inputs(cuda, np.random.default_rng(23), (lengths, 2, 1, 64, 0))
    once = _run(rsl, x, lengths)
    var = {n: rsl.Variable(x[n].numpy(), n != "g") for n in "qkvg"}
    o = rsl.causal_attention(var["q"], var["k"], var["v"], rsl.Sequences(lengths))
    for _ in range(3):
        o.backward(var["g"])
    for n in "qkv":
        d = once["d" + n]
        assert (var[n].grad.numpy() == (d + d) + d).all(), n


def test_a_score_of_minus_infinity_has_no_weight(cuda):
    import rushlite_b200 as rsl

    lengths = [150]
    x = _inputs(cuda, np.random.default_rng(10), (lengths, 1, 1, 32, 0))
    x["q"][:, :, 0] = 1.0
    x["k"][70, 0, 0] = -math.inf
    got = rsl.causal_attention(*(rsl.Variable(x[n].numpy()) for n in "qkv"), rsl.Sequences(lengths)).numpy()
    want = _reference(cuda, {**x, "k": x["k"].clone().nan_to_num_(neginf=-1e30)}, lengths)["out"]
    want = (want[0], _reference(cuda, {**x, "k": x["k"].clone().nan_to_num_(neginf=0.0)}, lengths)["out"][1])
    _check("out", got, want)


def test_lowest_values_as_a_mask(cuda):
    """A program that masks keys by fp32's lowest value in k: those keys weigh nothing."""
    import rushlite_b200 as rsl

    lengths = [260]
    x = _inputs(cuda, np.random.default_rng(11), (lengths, 2, 1, 64, 0))
    x["q"][:, :, 0] = 1.0
    x["k"][100:180, 0] = 0.0
    x["k"][100:180, 0, 0] = float(np.finfo(np.float32).min)
    got = _run(rsl, x, lengths)
    soft = {**x, "k": x["k"].clone()}
    soft["k"][100:180, 0, 0] = -1e4
    ref, tol = _reference(cuda, soft, lengths), _reference(cuda, {**x, "k": x["k"].clone().clamp_(min=-50)}, lengths)
    for name in ("out", "dv"):
        _check(name, got[name], (ref[name][0], tol[name][1]))


def test_gradients_are_the_differences(cuda):
    """A directional difference of the formula in 64 bits; its own error is
    h^2 times a third derivative of terms of size 1, below 1e-6 here."""
    import rushlite_b200 as rsl

    torch = cuda
    lengths = [90, 200]
    x = _inputs(torch, np.random.default_rng(12), (lengths, 4, 2, 24, 0))
    got = _run(rsl, x, lengths)
    ref = _reference(torch, x, lengths)
    h = 1e-4
    for n in "qkv":
        d = torch.randn(x[n].shape, dtype=torch.float64)
        value = [float((torch.from_numpy(_reference(torch, {**x, n: x[n].double() + s * h * d}, lengths)["out"][0])
                        * x["g"].double()).sum()) for s in (1, -1)]
        slope = (value[0] - value[1]) / (2 * h)
        mine = float((torch.from_numpy(got["d" + n]).double() * d).sum())
        room = float((torch.from_numpy(ref["d" + n][1]) * d.abs()).sum()) + 1e-6 * float(x["g"].abs().sum())
        assert abs(mine - slope) <= room, n


def test_repeats_to_the_bit_and_accumulates(cuda):
    import rushlite_b200 as rsl

    lengths = [700, 129]
    x = _inputs(cuda, np.random.default_rng(13), (lengths, 4, 1, 64, 0))
    seqs = rsl.Sequences(lengths)
    assert seqs.lengths == lengths and seqs.tokens == 829
    a, b = _run(rsl, x, lengths, seqs=seqs), _run(rsl, x, lengths, seqs=seqs)
    assert all((a[n] == b[n]).all() for n in a)
    var = {n: rsl.Variable(x[n].numpy(), n != "g") for n in "qkvg"}
    for _ in range(2):
        rsl.causal_attention(var["q"], var["k"], var["v"], seqs).backward(var["g"])
    for n in "qkv":
        assert (var[n].grad.numpy() == a["d" + n] + a["d" + n]).all()


def test_gradients_of_some_inputs(cuda):
    import rushlite_b200 as rsl

    lengths = [200]
    x = _inputs(cuda, np.random.default_rng(14), (lengths, 2, 2, 64, 0))
    full = _run(rsl, x, lengths)
    for want in ("q", "k", "v", "qv"):
        var = {n: rsl.Variable(x[n].numpy(), n in want) for n in "qkvg"}
        rsl.causal_attention(var["q"], var["k"], var["v"], rsl.Sequences(lengths)).backward(var["g"])
        for n in want:
            assert (var[n].grad.numpy() == full["d" + n]).all(), (want, n)
    with rsl.no_grad():
        assert not rsl.causal_attention(*(rsl.Variable(x[n].numpy(), True) for n in "qkv"), rsl.Sequences(lengths)).requires_grad


def test_one_variable_in_all_places(cuda):
    import rushlite_b200 as rsl

    lengths = [140, 3]
    x = _inputs(cuda, np.random.default_rng(15), (lengths, 2, 2, 32, 0))
    x["k"] = x["v"] = x["q"]
    ref = _reference(cuda, x, lengths)
    q, g = rsl.Variable(x["q"].numpy(), True), rsl.Variable(x["g"].numpy())
    rsl.causal_attention(q, q, q, rsl.Sequences(lengths)).backward(g)
    total, tol = (sum(ref[n][i] for n in ("dq", "dk", "dv")) for i in (0, 1))
    _check("sum", q.grad.numpy(), (total, tol + 2.0 ** -22 * (sum(np.abs(ref[n][0]) for n in ("dq", "dk", "dv")))))


def test_other_streams_and_sequences_outlive_their_handle(cuda):
    import rushlite_b200 as rsl

    torch = cuda
    lengths = [300, 200]
    x = _inputs(torch, np.random.default_rng(16), (lengths, 2, 1, 64, 0))
    want = _run(rsl, x, lengths)
    s = torch.cuda.Stream()
    try:
        rsl.cuda.set_stream(s.cuda_stream)
        got = _run(rsl, x, lengths)
        var = {n: rsl.Variable(x[n].numpy(), n != "g") for n in "qkvg"}
        graph, seqs = rsl.cuda.Graph(), rsl.Sequences(lengths)
        with graph:
            o = rsl.causal_attention(var["q"], var["k"], var["v"], seqs)
            o.backward(var["g"])
        del seqs  # the graph keeps it
        junk = [rsl.Sequences([5] * 50) for _ in range(4)]
        graph.replay()
        rec = {"out": o.numpy(), **{"d" + n: var[n].grad.numpy() for n in "qkv"}}
        del junk
    finally:
        rsl.cuda.synchronize()
        rsl.cuda.set_stream(0)
    for name in want:
        assert (got[name] == want[name]).all() and (rec[name] == want[name]).all(), name


def test_two_graphs_in_turn(cuda):
    """Each recorded call has a workspace of its own."""
    import rushlite_b200 as rsl

    recs = []
    for seed, lengths in ((17, [400]), (18, [130, 260])):
        x = _inputs(cuda, np.random.default_rng(seed), (lengths, 2, 2, 64, 0))
        want = _run(rsl, x, lengths)
        var = {n: rsl.Variable(x[n].numpy(), n != "g") for n in "qkvg"}
        g, seqs = rsl.cuda.Graph(), rsl.Sequences(lengths)
        with g:
            o = rsl.causal_attention(var["q"], var["k"], var["v"], seqs)
            o.backward(var["g"])
        recs.append((g, o, var, want))
    for _ in range(3):
        for g, *_ in recs:
            g.replay()
    for g, o, var, want in recs:
        g.replay()
        assert (o.numpy() == want["out"]).all()
        for n in "qkv":
            assert (var[n].grad.numpy() == want["d" + n]).all(), n


def test_two_streams_at_once(cuda):
    """Calls on two streams share nothing but the sequences, which are there as soon as they are made."""
    from rushlite_b200 import capi

    torch = cuda
    lengths, h, kv, d = [700, 1, 129, 40, 500], 4, 2, 64
    n = sum(lengths)
    gen = torch.Generator(device="cuda").manual_seed(2)
    sets = []
    for _ in range(2):
        x = [torch.randn(n, m, d, device="cuda", generator=gen) for m in (h, kv, kv, h)]  # q, k, v, grad
        sets.append((x, [torch.full_like(x[i], math.nan) for i in (0, 0, 1, 2)], torch.empty(h, n, device="cuda")))

    def call(x, y, lse, seqs, stream):
        p = [a.data_ptr() for a in (*x, *y, lse)]
        capi.attention(p[0], p[1], p[2], p[4], p[8], n, h, kv, d, 0.125, seqs, stream)
        capi.attention_backward(p[0], p[1], p[2], p[4], p[8], p[3], p[5], p[6], p[7], n, h, kv, d, 0.125, seqs, stream)

    want = []
    for x, y, lse in sets:
        call(x, y, lse, capi.Sequences(lengths), 0)
        torch.cuda.synchronize()
        want.append([a.clone() for a in (*y, lse)])
        for a in (*y, lse):
            a.fill_(math.nan)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    seqs = capi.Sequences(lengths)
    for _ in range(20):
        for s, (x, y, lse) in zip(streams, sets):
            call(x, y, lse, seqs, s.cuda_stream)
    torch.cuda.synchronize()
    for (x, y, lse), w in zip(sets, want):
        for a, b in zip((*y, lse), w):
            assert torch.equal(a, b)
    capi.device_error()


def test_offsets_past_32_bits(cuda):
    """q, out and their gradients hold over 2^31 values."""
    from rushlite_b200 import capi

    torch = cuda
    heads, d, n, count = 256, 128, 300, 220
    t = n * count
    assert t * heads * d > 2 ** 31
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("not enough free memory")
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, g = (torch.randn(t, heads, d, device="cuda", generator=gen) for _ in range(2))
    k, v = (torch.randn(t, 1, d, device="cuda", generator=gen) for _ in range(2))
    out, dq = torch.empty_like(q), torch.empty_like(q)
    dk, dv, lse = torch.empty_like(k), torch.empty_like(v), torch.empty(heads, t, device="cuda")
    seqs = capi.Sequences([n] * count)
    args = (t, heads, 1, d, 1 / math.sqrt(d), seqs)
    ptr = lambda *ts: [a.data_ptr() for a in ts]  # noqa: E731
    capi.attention(*ptr(q, k, v, out, lse), *args)
    capi.attention_backward(*ptr(q, k, v, out, lse, g, dq, dk, dv), *args)
    torch.cuda.synchronize()
    for i in (0, count - 1):
        rows = slice(i * n, (i + 1) * n)
        ref = _reference(torch, {"q": q[rows].cpu(), "k": k[rows].cpu(), "v": v[rows].cpu(), "g": g[rows].cpu()}, [n])
        for name, a in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
            _check(name, a[rows].cpu().numpy(), ref[name])


def test_unaligned_buffers_through_the_c_entry(cuda):
    from rushlite_b200 import capi

    torch = cuda
    lengths, hq, hkv, d = [150, 40], 2, 1, 64
    x = _inputs(torch, np.random.default_rng(19), (lengths, hq, hkv, d, 0))
    t = sum(lengths)

    def off(a):
        b = torch.full((a.numel() + 2,), 7.0, device="cuda")
        b[1:-1] = a.reshape(-1).cuda()
        return b

    ins = {n: off(a) for n, a in x.items()}
    outs = {n: off(torch.zeros_like(x[s])) for n, s in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    lse = torch.empty(hq * t + 1, device="cuda")
    p = {n: b[1:].data_ptr() for n, b in {**ins, **outs, "lse": lse}.items()}
    args = (t, hq, hkv, d, 1 / math.sqrt(d), capi.Sequences(lengths))
    capi.attention(p["q"], p["k"], p["v"], p["out"], p["lse"], *args)
    capi.attention_backward(p["q"], p["k"], p["v"], p["out"], p["lse"], p["g"], p["dq"], p["dk"], p["dv"], *args)
    torch.cuda.synchronize()
    ref = _reference(torch, x, lengths)
    for n, b in outs.items():
        _check(n, b[1:-1].cpu().numpy().reshape(ref[n][0].shape), ref[n])
        assert b[0] == 7 and b[-1] == 7, n


@pytest.mark.parametrize("heads,kv_heads", [(16400, 16400), (32768, 16384)])
def test_more_heads_than_the_tensor_core_kernels_take(cuda, heads, kv_heads):
    """The plain fp32 kernels on their own; some groups of heads against the formula."""
    lengths, dim, group = [41, 1, 0, 70], 3, heads // kv_heads
    x = _inputs(cuda, np.random.default_rng(33), (lengths, heads, kv_heads, dim, 2))
    got = _results(x, lengths)
    for j in (0, 1, 8191, kv_heads - 1):
        h = slice(j * group, (j + 1) * group)
        part = {"q": x["q"][:, h], "k": x["k"][:, j:j + 1], "v": x["v"][:, j:j + 1], "g": x["g"][:, h]}
        ref = _reference(cuda, part, lengths)
        for name in got:
            _check(name, got[name][:, h if name in ("out", "dq") else slice(j, j + 1)], ref[name])


def test_plain_fp32_kernels_on_every_case(cuda):
    """The cases above, in a process that takes the plain fp32 kernels for all of them."""
    import os
    import subprocess
    import sys

    names = ("test_forward_and_backward or test_scale or test_rows_with_small_gradients or test_scores_far_apart "
             "or test_repeats_to_the_bit or test_tiles_of_very_different_size or does_not_see")
    r = subprocess.run([sys.executable, "-m", "pytest", "-m", "gpu", "-x", "-q", "-p", "no:cacheprovider", "-k", names,
                        os.path.abspath(__file__)], env={**os.environ, "LMPB_ATTENTION": "simt"}, capture_output=True,
                       text=True, timeout=600)
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:]


def test_refusals(cuda):
    import rushlite_b200 as rsl

    q, kv, s = rsl.ones([6, 4, 8]), rsl.ones([6, 2, 8]), rsl.Sequences([2, 4])
    bad = [((rsl.ones([6, 4, 8], dtype=rsl.dtype.float64), kv, kv, s), "float32"),
           ((rsl.ones([6, 4, 8], device=rsl.device.cpu), kv, kv, s), "CUDA"), ((rsl.ones([6, 32]), kv, kv, s), "head_dim"),
           ((q, kv, rsl.ones([6, 2, 4]), s), "same shape"), ((q, rsl.ones([6, 3, 8]), rsl.ones([6, 3, 8]), s), "multiple"),
           ((q, rsl.ones([5, 2, 8]), rsl.ones([5, 2, 8]), s), "tokens"), ((q, kv, kv, rsl.Sequences([7])), "tokens"),
           ((rsl.ones([6, 2, 129]),) * 3 + (s,), "128"), ((q, kv, kv, s, 0.0), "scale"), ((q, kv, kv, s, -1.0), "scale"),
           ((q, kv, kv, s, float("nan")), "scale"), ((q, kv, kv, s, float("inf")), "scale"), ((q, kv, kv, s, 1e20), "scale")]
    for args, text in bad:
        with pytest.raises(RuntimeError, match=text):
            rsl.causal_attention(*args)
    with pytest.raises(RuntimeError, match="negative"):
        rsl.Sequences([3, -1])
    g = rsl.cuda.Graph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with g:
            rsl.Sequences([3])
    with pytest.raises(TypeError):
        rsl.causal_attention(q, kv, kv, [2, 4])
    assert rsl.causal_attention(q, kv, kv, s).shape == [6, 4, 8]  # still usable
