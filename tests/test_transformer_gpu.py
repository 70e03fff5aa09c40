"""A transformer block's training step with everything that it uses together:
layer norm, attention over packed sequences, Linear, ReLU, the softmax loss and
AdamW, against a plain version in 64 bits and its automatic gradients; and the
same step recorded as a CUDA graph."""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F, HEADS, KV, HIDDEN, CLASSES = 64, 4, 2, 96, 10
LENGTHS = [70, 1, 0, 129, 40]


def _block(rsl):
    from rushlite_b200.nets import layers

    class Block(rsl.Module):
        def __init__(self):
            super().__init__()
            self.norm1 = layers.LayerNorm(F)
            self.attention = layers.CausalSelfAttention(F, HEADS, KV)
            self.norm2 = layers.LayerNorm(F, bias=False)
            self.up = layers.Linear(F, HIDDEN)
            self.relu = layers.ReLU()
            self.down = layers.Linear(HIDDEN, F)
            self.head = layers.Linear(F, CLASSES)
            self.softmax = layers.Softmax(-1)

        def forward(self, x, sequences):
            x = x + self.attention(self.norm1(x), sequences)
            x = x + self.down(self.relu(self.up(self.norm2(x))))
            return self.softmax(self.head(x))

    return Block()


def _weights(model, rng):
    """The initial values of every parameter, scaled by its inputs."""
    out = {}
    for name, p in model.named_parameters():
        s = p.shape
        if name.startswith("norm"):
            out[name] = ((1 if name.endswith("weights") else 0) + 0.1 * rng.standard_normal(s)).astype(np.float32)
        else:
            out[name] = (rng.standard_normal(s) / math.sqrt(s[0])).astype(np.float32)
    return out


def _load(rsl, model, weights):
    for name, p in model.named_parameters():
        p.data.copy(rsl.Variable(weights[name]).data)


def _step(rsl, model, x, y, seqs):
    with rsl.capture_on():
        loss = (-y * rsl.log(model(x, seqs) + 1e-3)).sum(1).sum(0)
    loss.backward()
    return loss


def _plain(torch, w, x, y):
    """The same loss and gradients in 64 bits by torch's autograd."""
    w = {n: torch.from_numpy(a).cuda().double().requires_grad_() for n, a in w.items()}
    x, y = torch.from_numpy(x).cuda().double(), torch.from_numpy(y).cuda().double()

    def norm(x, name):
        c = x - x.mean(1, keepdim=True)
        h = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-5) * w[name + ".weights"]
        return h + w[name + ".bias"] if name + ".bias" in w else h

    def linear(x, name):
        return x @ w[name + ".weights"] + w[name + ".bias"]

    h = norm(x, "norm1")
    q, k, v = (linear(h, "attention." + n).view(len(x), -1, F // HEADS) for n in ("query", "key", "value"))
    seq = torch.repeat_interleave(torch.arange(len(LENGTHS), device="cuda"), torch.tensor(LENGTHS, device="cuda"))
    at = torch.arange(len(x), device="cuda")
    mask = (seq[:, None] == seq) & (at[:, None] >= at)
    k, v = (a.repeat_interleave(HEADS // KV, 1) for a in (k, v))
    s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(F // HEADS)
    p = torch.softmax(s.masked_fill(~mask, -math.inf), -1)
    x = x + linear(torch.einsum("hij,jhd->ihd", p, v).reshape(len(x), F), "attention.out")
    z = linear(norm(x, "norm2"), "up")
    x = x + linear(torch.relu(z), "down")
    loss = -(y * torch.log(torch.softmax(linear(x, "head"), -1) + 1e-3)).sum()
    loss.backward()
    return float(loss.detach()), {n: a.grad.cpu().numpy() for n, a in w.items()}


def _batch(rng):
    t = sum(LENGTHS)
    y = np.zeros((t, CLASSES), np.float32)
    y[np.arange(t), rng.integers(0, CLASSES, t)] = 1
    return rng.standard_normal((t, F)).astype(np.float32), y


def test_training_steps(cuda):
    """Each step's gradients against the plain version's on the same weights,
    and the weights after it against AdamW's formula on its gradients.  The
    gradients end a chain of a dozen products and sums of fp32 (each within
    1e-5 of its result's largest, the matmul's bar): 1.2e-4."""
    import rushlite_b200 as rsl

    rng = np.random.default_rng(0)
    model = _block(rsl)
    w = _weights(model, rng)
    _load(rsl, model, w)
    params = dict(model.named_parameters())
    opt = rsl.optim.AdamW(params.values(), lr=1e-2, weight_decay=0.01)
    m, v = ({n: np.zeros(a.shape) for n, a in w.items()} for _ in range(2))
    xs, ys = _batch(rng)
    x, y, seqs = rsl.Variable(xs), rsl.Variable(ys), rsl.Sequences(LENGTHS)
    for t in (1, 2, 3):
        opt.zero_grad()
        loss = _step(rsl, model, x, y, seqs)
        want, grads = _plain(cuda, w, xs, ys)
        assert abs(loss.tolist()[0] - want) <= 1e-5 * abs(want)
        for n, p in params.items():
            g = p.grad.numpy().astype(np.float64)
            big = np.abs(grads[n]).max()
            if n == "attention.key.bias":  # a shift of all keys changes no weight: 0 but for roundings of its terms
                big = np.abs(grads["attention.key.weights"]).max()
            assert np.abs(g - grads[n]).max() <= 1.2e-4 * big, (t, n)
            m[n] = 0.9 * m[n] + 0.1 * g
            v[n] = 0.999 * v[n] + 0.001 * g * g
            w[n] = w[n] * (1 - 1e-4) - 1e-2 / (1 - 0.9 ** t) * m[n] / (np.sqrt(v[n] / (1 - 0.999 ** t)) + 1e-8)
        opt.step()
        for n, p in params.items():  # m and v of the formula are in 64 bits: cancelling moments lose a few more bits
            assert np.abs(p.numpy() - w[n]).max() <= 1e-6, (t, n)
            w[n] = p.numpy()


def test_recorded_step_equals_the_eager_one(cuda):
    """Bit for bit over four steps, with an eager graph of the same parameters alive during the capture."""
    import rushlite_b200 as rsl

    rng = np.random.default_rng(1)
    xs, ys = _batch(rng)
    results = []
    init = None
    for recorded in (False, True):
        model = _block(rsl)
        init = init or _weights(model, np.random.default_rng(2))
        _load(rsl, model, init)
        opt = rsl.optim.AdamW(model.parameters(), lr=1e-2)
        x, y, seqs = rsl.Variable(xs), rsl.Variable(ys), rsl.Sequences(LENGTHS)

        def step():
            opt.zero_grad()
            loss = _step(rsl, model, x, y, seqs)
            opt.step()
            return loss

        losses = []
        if recorded:
            losses.append(step().tolist()[0])
            alive = model(x, seqs)  # an eager graph of the same leaves
            graph = rsl.cuda.Graph()
            with graph:
                loss = step()
            for _ in range(3):
                graph.replay()
                losses.append(loss.tolist()[0])
            assert alive.shape == [sum(LENGTHS), CLASSES]
        else:
            losses = [step().tolist()[0] for _ in range(4)]
        results.append((losses, [p.numpy() for p in model.parameters()], opt.state_dict()["step"]))
    assert results[0][0] == results[1][0] and results[0][2] == results[1][2] == 4
    assert all((a == b).all() for a, b in zip(results[0][1], results[1][1]))


def test_backward_from_a_given_gradient(cuda):
    import rushlite_b200 as rsl

    rng = np.random.default_rng(3)
    a, g = (rng.standard_normal((4, 6)).astype(np.float32) for _ in range(2))
    for variable in (True, False):
        v = rsl.Variable(a, True)
        seed = rsl.Variable(g)
        out = v * v
        out.backward(seed)
        assert (v.grad.numpy() == a * g + a * g).all()
        out.backward(seed)  # the seed again: the intermediate's gradient is the given one, the leaf's accumulates
        assert (v.grad.numpy() == (a * g + a * g) + a * g + a * g).all()
        assert (seed.numpy() == g).all()  # untouched
    leaf = rsl.Variable(a, True)
    leaf.backward(rsl.Variable(g))
    assert (leaf.grad.numpy() == g).all()
    seed = rsl.Variable(g)
    leaf.zero_grad()
    leaf.backward(seed)
    (leaf * 2.0).backward()
    assert (leaf.grad.numpy() == g + 2).all() and (seed.numpy() == g).all()
    with pytest.raises(RuntimeError, match="dtype"):
        leaf.backward(rsl.Variable(g, dtype=rsl.dtype.float64))


_FAILING = r"""
#include <dlfcn.h>
#include <stdlib.h>
#include "lmpb.h"
static int calls;
static void* real(const char* name) { return dlsym(dlopen(getenv("REAL_LMPB"), RTLD_NOW | RTLD_NOLOAD), name); }
lmpb_status lmpb_attention_backward(const float* q, const float* k, const float* v, const float* out, const float* lse,
                                    const float* grad, float* dq, float* dk, float* dv, int64_t tokens, int heads,
                                    int kv_heads, int head_dim, float scale, lmpb_sequences s, void* stream) {
  if (calls++ % 2 == 0) return LMPB_ERR_CUDA;
  lmpb_status (*f)() = (lmpb_status (*)())real("lmpb_attention_backward");
  return ((lmpb_status (*)(const float*, const float*, const float*, const float*, const float*, const float*, float*, float*,
                           float*, int64_t, int, int, int, float, lmpb_sequences, void*))f)(
      q, k, v, out, lse, grad, dq, dk, dv, tokens, heads, kv_heads, head_dim, scale, s, stream);
}
lmpb_status lmpb_layer_norm_backward(int dtype, const void* x, const void* w, const void* mean, const void* rstd,
                                     const void* grad, int64_t rows, int64_t features, void* dx, void* dw, void* db,
                                     void* stream) {
  if (calls++ % 2 == 0) return LMPB_ERR_CUDA;
  lmpb_status (*f)() = (lmpb_status (*)())real("lmpb_layer_norm_backward");
  return ((lmpb_status (*)(int, const void*, const void*, const void*, const void*, const void*, int64_t, int64_t, void*,
                           void*, void*, void*))f)(dtype, x, w, mean, rstd, grad, rows, features, dx, dw, db, stream);
}
"""

_AFTER_FAILURE = r"""
import numpy as np
import rushlite_b200 as rsl

def run(fail):
    rng = np.random.default_rng(0)
    q, k, v, g = (rsl.Variable(rng.standard_normal((50, 2, 8)).astype(np.float32), i < 3) for i in range(4))
    x = rsl.Variable(rng.standard_normal((9, 40)).astype(np.float32), True)
    w = rsl.Variable(rng.standard_normal(40).astype(np.float32), True)
    b, gy = rsl.zeros([40], True), rsl.Variable(rng.standard_normal((9, 40)).astype(np.float32))
    junk = [rsl.Variable(np.full((50, 2, 8), 1e9, np.float32)) for _ in range(8)]  # what fresh memory may hold
    del junk
    for make, seed in ((lambda: rsl.causal_attention(q, q, v, rsl.Sequences([50])), g),
                       (lambda: rsl.causal_attention(q, k, v, rsl.Sequences([50])), g), (lambda: rsl.layer_norm(x, w, b), gy)):
        for attempt in range(2):
            try:
                make().backward(seed)
                assert attempt or not fail, "the call was to fail"
                if not fail:
                    break
            except RuntimeError:
                assert fail and attempt == 0
    return [a.grad.numpy() for a in (q, k, v, x, w, b)]

import os, sys
np.save(sys.argv[2], np.concatenate([a.ravel() for a in run(sys.argv[1] == "fail")]))
"""


def test_gradients_after_a_failed_backward(cuda, tmp_path):
    """A backward call that fails (a fake of the C entries returns an error
    every other time) leaves the gradients as they were: tried again, it gives
    what it gives without a failure."""
    import os
    import subprocess
    import sys

    from rushlite_b200 import capi

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "fake.c").write_text(_FAILING)
    subprocess.run(["gcc", "-shared", "-fPIC", "-I", os.path.join(root, "include"), "-o", str(tmp_path / "fake.so"),
                    str(tmp_path / "fake.c"), "-ldl"], check=True)
    env = {**os.environ, "REAL_LMPB": os.path.abspath(capi.LIB_PATH), "PYTHONPATH": root}
    got = {}
    for what in ("pass", "fail"):
        if what == "fail":
            env["LD_PRELOAD"] = str(tmp_path / "fake.so")
        r = subprocess.run([sys.executable, "-c", _AFTER_FAILURE, what, str(tmp_path / what)], env=env, cwd=root,
                           capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        got[what] = np.load(str(tmp_path / what) + ".npy")
    assert np.isfinite(got["pass"]).all() and (got["pass"] == got["fail"]).all()
