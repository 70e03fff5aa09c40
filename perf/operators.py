"""Cases that measure the transformer-training operators: layer norm, causal attention over packed
sequences and the AdamW step.

``run`` computes a case in plain torch operations, or, where ``own`` is true, through rushlite_b200's
public calls on the same values.
"""
import math

import torch

own = False

# The tensors of two models: the README's MLP (256-64-10) and the data-parallel MLP (4 x 4096 wide, 1000 classes).
_README_MLP = "256x64,64,64x10,10"
_WIDE_MLP = ",".join(["4096x4096,4096"] * 4 + ["4096x1000,1000"])


def listed():
    return [
        # a few tokens through one small head group: what an interactive fine-tuning step on one line of text costs
        dict(name="attention_tiny", op="attention", lengths="7", heads=4, kv_heads=4, dim=64, train=True),
        # a batch of sentences, many of them short, packed without padding
        dict(name="attention_sentences", op="attention", train=True, heads=8, kv_heads=8, dim=64,
             lengths=",".join(str(1 + (37 * i) % 96) for i in range(96))),
        # documents of very different lengths in one training batch, grouped heads
        dict(name="attention_documents", op="attention", train=True, heads=16, kv_heads=4, dim=128,
             lengths="1500,31,700,1,1865"),
        # one key/value head for all query heads, a head size that is no power of two, odd lengths
        dict(name="attention_one_kv_head", op="attention", train=True, heads=6, kv_heads=1, dim=80, lengths="777,1234"),
        # evaluating a long prompt: forward only
        dict(name="attention_prompt", op="attention", train=False, heads=16, kv_heads=4, dim=64, lengths="8192"),
        # long-context training
        dict(name="attention_long", op="attention", train=True, heads=8, kv_heads=2, dim=128, lengths="16384"),
        # the README MLP's batch and width: latency
        dict(name="layer_norm_readme", op="layer_norm", rows=32, features=256, dtype="float32", affine=True, train=True),
        # evaluation over an odd width, no 16-byte alignment from row to row
        dict(name="layer_norm_odd", op="layer_norm", rows=1023, features=1001, dtype="float32", affine=True, train=False),
        # double precision training at a wide layer
        dict(name="layer_norm_double", op="layer_norm", rows=2048, features=4096, dtype="float64", affine=True, train=True),
        # the data-parallel MLP's batch and width
        dict(name="layer_norm_wide", op="layer_norm", rows=8192, features=4096, dtype="float32", affine=True, train=True),
        # the README MLP's four parameters: latency
        dict(name="adamw_readme", op="adamw", tensors=_README_MLP, dtype="float32"),
        # the data-parallel MLP's ten parameters, 71 M values
        dict(name="adamw_wide", op="adamw", tensors=_WIDE_MLP, dtype="float32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "layer_norm", "layer_norm", "adamw"])
    if op == "attention":
        kv = rng.choice([1, 1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4])
        dim = rng.choice([rng.randint(1, 128), 64, 128, 8 * rng.randint(2, 16)])
        longest = _log_int(rng, 1, 16384)
        # no more visible pairs than the longest listed case, and no more padded scores in the plain form
        longest = min(longest, int(16380 * math.sqrt(8 / heads)) if heads > 8 else 16384)
        lengths = [longest]
        for _ in range(rng.choice([0, 0, 1, 3, 7, 40])):
            n = _log_int(rng, 1, longest)
            if heads * (len(lengths) + 1) * longest ** 2 <= 8 * 16384 ** 2 and sum(lengths) + n <= 32768:
                lengths.append(n)
        rng.shuffle(lengths)
        return dict(op=op, lengths=",".join(map(str, lengths)), heads=heads, kv_heads=kv, dim=dim,
                    train=rng.random() < 0.6)
    if op == "layer_norm":
        features = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(65536, 8192 * 4096 // features))
        dtype = rng.choice(["float32", "float32", "float64"])
        if dtype == "float64":
            rows = max(1, rows // 2)
        return dict(op=op, rows=rows, features=features, dtype=dtype, affine=rng.random() < 0.9,
                    train=rng.random() < 0.7)
    dtype = rng.choice(["float32", "float32", "float64"])
    left = 70_000_000 if dtype == "float32" else 35_000_000
    shapes = []
    for _ in range(_log_int(rng, 1, 20)):
        n = _log_int(rng, 1, min(left, 16_000_000))
        if n > 4096 and rng.random() < 0.5:
            c = rng.randint(2, 4096)
            shapes.append("%dx%d" % (n // c, c))
            n = n // c * c
        else:
            shapes.append(str(n))
        left -= n
        if left < 1000:
            break
    return dict(op=op, tensors=",".join(shapes), dtype=dtype)


def _shapes(case):
    return [tuple(int(n) for n in t.split("x")) for t in case["tensors"].split(",")]


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def work(case):
    if case["op"] == "attention":
        lengths, hq, hkv, d = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
        tokens, pairs = sum(lengths), sum(n * (n + 1) // 2 for n in lengths) * hq
        q, kv = tokens * hq * d * 4, 2 * tokens * hkv * d * 4
        if case["train"]:  # q, k, v and the output's gradient in; output and three gradients out
            return {"bytes": 4 * q + 2 * kv, "flops": 14 * d * pairs}
        return {"bytes": 2 * q + kv, "flops": 4 * d * pairs}
    size = 8 if case["dtype"] == "float64" else 4
    if case["op"] == "layer_norm":
        n, f = case["rows"] * case["features"], case["features"]
        affine = 2 * f if case["affine"] else 0
        if case["train"]:  # x, gradient, weight, bias in; y, dx, dw, db out
            return {"bytes": size * (4 * n + 2 * affine), "flops": 20 * n}
        return {"bytes": size * (2 * n + affine), "flops": 8 * n}
    n = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": 7 * size * n, "flops": 15 * n}


_LR, _BETAS, _EPS, _DECAY, _STEP, _NORM_EPS = 1e-3, (0.9, 0.999), 1e-8, 0.01, 10, 1e-5


def _inputs(case, seed):
    """The case's input values, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    if case["op"] == "attention":
        t, hq, hkv, d = sum(_lengths(case)), case["heads"], case["kv_heads"], case["dim"]
        x = {"q": normal(t, hq, d), "k": normal(t, hkv, d), "v": normal(t, hkv, d)}
        if case["train"]:
            x["grad"] = normal(t, hq, d) * 0.1
        return x
    dtype = getattr(torch, case["dtype"])
    if case["op"] == "layer_norm":
        rows, f = case["rows"], case["features"]
        x = {"x": normal(rows, f, dtype=dtype) * 1.5 + 0.5}  # activations away from zero mean and unit variance
        if case["affine"]:
            x["weight"], x["bias"] = 1 + 0.1 * normal(f, dtype=dtype), 0.1 * normal(f, dtype=dtype)
        if case["train"]:
            x["grad"] = normal(rows, f, dtype=dtype) * 0.1
        return x
    shapes = _shapes(case)
    # parameters, gradients and moments in the middle of a training
    return {"p": [0.02 * normal(*s, dtype=dtype) for s in shapes],
            "g": [1e-3 * normal(*s, dtype=dtype) for s in shapes],
            "m": [1e-4 * normal(*s, dtype=dtype) for s in shapes],
            "v": [1e-6 * normal(*s, dtype=dtype).square() for s in shapes]}


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["op"] == "attention":
        # where each token of each sequence is, for a batch padded to the longest
        lengths = torch.tensor(_lengths(case), device="cuda")
        starts = torch.cumsum(lengths, 0) - lengths
        at = torch.arange(int(lengths.max()), device="cuda")
        state["inside"] = at < lengths[:, None]
        state["index"] = torch.where(state["inside"], starts[:, None] + at, 0)
    if case["op"] == "adamw":
        state["step"] = _STEP
    if own:  # the same values as the framework's own tensors, and the handles that its user keeps
        import rushlite_b200 as rsl

        kind = {torch.float32: rsl.dtype.float32, torch.float64: rsl.dtype.float64}

        def var(t, requires_grad=False):
            return rsl.Variable(t.cpu().numpy(), requires_grad, dtype=kind[t.dtype])

        if case["op"] == "adamw":
            state["params"] = [var(t, True) for t in state["p"]]
            for p, t in zip(state["params"], state["g"]):
                p.grad.copy(var(t).data)
            opt = rsl.optim.AdamW(state["params"], lr=_LR, betas=_BETAS, eps=_EPS, weight_decay=_DECAY)
            opt.load_state_dict({"step": _STEP, "exp_avg": [t.cpu().numpy() for t in state["m"]],
                                 "exp_avg_sq": [t.cpu().numpy() for t in state["v"]]})
            state["optimizer"] = opt
            state["out"] = [[_view(x) for x in (p.data, m.data, v.data)]
                            for p, m, v in zip(state["params"], opt.exp_avg, opt.exp_avg_sq)]
        else:
            for key in ("x", "weight", "bias", "q", "k", "v", "grad"):
                if key in state:
                    state[key] = var(state[key], case["train"] and key != "grad")
            if case["op"] == "attention":
                state["sequences"] = rsl.Sequences(_lengths(case))
    return state


def _view(t):
    """A torch tensor on the memory of one of the framework's tensors."""
    return torch.as_tensor(t, device="cuda")


def run(state):
    return {"attention": _attention, "layer_norm": _layer_norm, "adamw": _adamw}[state["case"]["op"]](state)


def _attention(s):
    if own:
        import rushlite_b200 as rsl

        if not s["case"]["train"]:
            return {"out": _view(rsl.causal_attention(s["q"], s["k"], s["v"], s["sequences"]).data)}
        s["q"].zero_grad(), s["k"].zero_grad(), s["v"].zero_grad()
        o = rsl.causal_attention(s["q"], s["k"], s["v"], s["sequences"])
        o.backward(s["grad"])
        return {"out": _view(o.data), "dq": _view(s["q"].grad), "dk": _view(s["k"].grad), "dv": _view(s["v"].grad)}
    index, inside = s["index"], s["inside"]
    n, longest = index.shape
    hq, hkv, d = s["case"]["heads"], s["case"]["kv_heads"], s["case"]["dim"]
    scale = 1 / math.sqrt(d)

    def padded(x, h):  # [sequence, kv head, query head of it, token, dim]
        x = torch.where(inside[:, :, None, None], x[index], 0)
        return x.view(n, longest, hkv, h // hkv, d).permute(0, 2, 3, 1, 4)

    def packed(x, h):
        return x.permute(0, 3, 1, 2, 4).reshape(n, longest, h, d)[inside]

    q, k, v = padded(s["q"], hq), padded(s["k"], hkv), padded(s["v"], hkv)
    at = torch.arange(longest, device="cuda")
    p = torch.matmul(q, k.transpose(-1, -2))
    p.mul_(scale).masked_fill_(at > at[:, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p, v)
    if not s["case"]["train"]:
        return {"out": packed(o, hq)}
    g = padded(s["grad"], hq)
    dv = torch.matmul(p.transpose(-1, -2), g).sum(2, keepdim=True)
    ds = torch.matmul(g, v.transpose(-1, -2)).sub_((g * o).sum(-1, keepdim=True)).mul_(p)
    dq = torch.matmul(ds, k).mul_(scale)
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True).mul_(scale)
    return {"out": packed(o, hq), "dq": packed(dq, hq), "dk": packed(dk, hkv), "dv": packed(dv, hkv)}


def _layer_norm(s):
    train = s["case"]["train"]
    if own:
        import rushlite_b200 as rsl

        x, w, b = s["x"], s.get("weight"), s.get("bias")
        if not train:
            return {"y": _view(rsl.layer_norm(x, w, b, _NORM_EPS).data)}
        leaves = [("dx", x)] + ([("dw", w), ("db", b)] if w is not None else [])
        for _, leaf in leaves:
            leaf.zero_grad()
        y = rsl.layer_norm(x, w, b, _NORM_EPS)
        y.backward(s["grad"])
        return {"y": _view(y.data), **{name: _view(leaf.grad) for name, leaf in leaves}}
    x, w = s["x"], s.get("weight")
    c = x - x.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + _NORM_EPS).rsqrt()
    h = c * rstd
    y = h * w + s["bias"] if w is not None else h
    if not train:
        return {"y": y}
    g = s["grad"]
    a = g * w if w is not None else g
    dx = rstd * (a - a.mean(-1, keepdim=True) - h * (a * h).mean(-1, keepdim=True))
    out = {"y": y, "dx": dx}
    if w is not None:
        out["dw"], out["db"] = (g * h).sum(0), g.sum(0)
    return out


def _adamw(s):
    if own:
        s["optimizer"].step()
        return s["out"]
    s["step"] += 1
    return _adamw_formula(s["p"], s["g"], s["m"], s["v"], s["step"])


def _adamw_formula(params, grads, first, second, step):
    b1, b2 = _BETAS
    rate, root = _LR / (1 - b1 ** step), math.sqrt(1 - b2 ** step)

    def one(p, g, m, v):
        m.mul_(b1).add_(g * (1 - b1))
        v.mul_(b2).add_(g * g * (1 - b2))
        p.mul_(1 - _LR * _DECAY).sub_(m / (v.sqrt() / root + _EPS) * rate)
        return [p, m, v]

    return [one(*t) for t in zip(params, grads, first, second)]


def exact(case, seed):
    x = _inputs(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, x)
    if case["op"] == "layer_norm":
        up = {key: t.double() for key, t in x.items()}
        mean = up["x"].sum(1, keepdim=True) / case["features"]
        var = ((up["x"] - mean) ** 2).sum(1, keepdim=True) / case["features"]
        sigma = torch.sqrt(var + _NORM_EPS)
        w, b = up.get("weight", torch.ones(1, device="cuda")), up.get("bias", torch.zeros(1, device="cuda"))
        h = (up["x"] - mean) / sigma
        out = {"y": h * w + b}
        if case["train"]:
            a, f = up["grad"] * w, case["features"]
            out["dx"] = (f * a - a.sum(1, keepdim=True) - h * (a * h).sum(1, keepdim=True)) / (f * sigma)
            if case["affine"]:
                out["dw"], out["db"] = (up["grad"] * h).sum(0), up["grad"].sum(0)
        return out
    out = []
    t, (b1, b2) = _STEP + 1, _BETAS
    for p, g, m, v in zip(x["p"], x["g"], x["m"], x["v"]):
        p, g, m, v = p.double(), g.double(), m.double(), v.double()
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        out.append([p - _LR * _DECAY * p - _LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)) ** 0.5 + _EPS), m, v])
    return out


def _exact_attention(case, x):
    lengths, hq, hkv, d = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
    if 14 * d * hq * sum(n * n for n in lengths) > 6e12:  # over about 20 seconds in 64 bits
        return None
    out = {"out": torch.zeros(*x["q"].shape, dtype=torch.float64, device="cuda")}
    if case["train"]:
        out.update({key: torch.zeros(*x[key[1]].shape, dtype=torch.float64, device="cuda") for key in ("dq", "dk", "dv")})
    start = 0
    for n in lengths:
        rows = slice(start, start + n)
        start += n
        for h in range(hq):
            j = h * hkv // hq
            k, v = x["k"][rows, j].double(), x["v"][rows, j].double()
            for a in range(0, n, 2048):  # rows a..b see keys 0..b
                b = min(n, a + 2048)
                part = slice(rows.start + a, rows.start + b)
                q = x["q"][part, h].double()
                z = (q @ k[:b].T) / math.sqrt(d)
                z = z.masked_fill(torch.ones(b - a, b, dtype=torch.bool, device="cuda").triu(a + 1), -math.inf)
                p = torch.softmax(z, 1)
                out["out"][part, h] = p @ v[:b]
                if case["train"]:
                    g = x["grad"][part, h].double()
                    dp = g @ v[:b].T
                    dz = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                    out["dq"][part, h] = dz @ k[:b]
                    out["dk"][rows, j][:b] += dz.T @ q
                    out["dv"][rows, j][:b] += p.T @ g
    return out
