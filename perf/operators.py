"""The layer operators as they are measured: the fused linear layer and the table lookup, with their gradients.

``own = False`` computes them in elementary torch operations (32 bits inside, rounded once at the end); ``own = True`` calls
``nrhints_amd.ops``.  Sizes: the networks of this repository are 256 wide with inputs of 39 to 361 columns and heads of 1 and 3, over
64 to 1 024 rays of 128 or 160 samples in training and up to 655 360 rays at once in evaluation; its tables hold one row per training
view.  The rest of the range is generic.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTIVATIONS = ("none", "relu", "softplus", "sigmoid", "silu", "gelu")


def _linear(name, m, k, n, dtype, act, *, train=False, bias=True, residual=False, pad=0, beta=100.0):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "train": train, "bias": bias,
            "residual": residual, "pad": pad, "beta": beta}


def _lookup(name, v, d, n, dtype, *, train=False, scale=1.0, index="int64", spread="even", absent=0.0):
    return {"name": name, "op": "embedding", "v": v, "d": d, "n": n, "dtype": dtype, "train": train, "scale": scale, "index": index,
            "spread": spread, "absent": absent}


def listed():
    return [
        # one query point through a hidden layer: an interactive probe of the field, nothing but latency
        _linear("point_f32", 1, 256, 256, "f32", "softplus"),
        # a handful of query vectors against a wide layer: the weights are all there is to read
        _linear("few_bf16", 5, 1024, 1024, "bf16", "silu", residual=True),
        # the colour head of a 64-ray batch at 160 samples: three columns out, an odd width to write
        _linear("head_f32", 64 * 160, 128, 3, "f32", "sigmoid"),
        # a hidden layer of the background network, 1 024 rays x 160 samples, in the framework's own type
        _linear("hidden_f32", 1024 * 160, 256, 256, "f32", "relu"),
        # its skip layer (84 encoded inputs beside 256 hidden ones) in training: forward, input, weight and bias gradients
        _linear("skip_train_f32", 1024 * 160, 340, 256, "f32", "silu", train=True),
        # a small training batch, 64 rays x 128 samples, 16-bit, ReLU as in the reflectance network
        _linear("small_train_bf16", 64 * 128, 256, 256, "bf16", "relu", train=True),
        # encoded positions that start off a 16-byte boundary inside a wider buffer; every size odd
        _linear("ragged_train_f16", 20011, 63, 129, "f16", "gelu", train=True, pad=3),
        # one sample per ray of a whole frame through a residual layer, 16-bit
        _linear("frame_bf16", 655360, 256, 256, "bf16", "relu", residual=True),
        # a wide residual block in training: the large matrix products
        _linear("wide_train_bf16", 16384, 1024, 1024, "bf16", "gelu", train=True, residual=True),
        # the 3 x 4 pose deltas of 100 views, looked up for a batch of 1 024 rays
        _lookup("views_f32", 100, 12, 1024, "f32"),
        # ... and their gradient for a chunk of 131 072 rays: every row is hit about 1 300 times
        _lookup("views_train_f32", 100, 12, 131072, "f32", train=True),
        # a vocabulary of codes with uneven use, scaled, some slots empty: lookup and gradient
        _lookup("codes_train_bf16", 50000, 1024, 16384, "bf16", train=True, scale=32.0, index="int32", spread="uneven", absent=0.03),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    dtype = rng.choice(("f32", "f16", "bf16"))
    train = rng.random() < 0.5
    if rng.random() < 0.6:
        cap_bytes = 1.0e9                                          # of the largest listed case
        cap_macs = 4.0e10 if dtype == "f32" else 5.0e10
        while True:
            m, k, n = _log_int(rng, 1, 655360), _log_int(rng, 1, 1024), _log_int(rng, 1, 1024)
            case = _linear("", m, k, n, dtype, rng.choice(ACTIVATIONS), train=train, bias=rng.random() < 0.8, residual=rng.random() < 0.4,
                           pad=rng.choice((0, 0, 0, 1, 3, 8)), beta=rng.choice((1.0, 100.0)))
            if train and case["act"] == "softplus":
                case["beta"] = 1.0
            w = work(case)
            if w["bytes"] <= cap_bytes and w["flops"] <= 2.0 * cap_macs:
                break
    else:
        while True:
            case = _lookup("", _log_int(rng, 1, 200000), _log_int(rng, 1, 2048), _log_int(rng, 1, 200000), dtype, train=train,
                           scale=rng.choice((1.0, 0.125, 32.0, round(rng.uniform(0.1, 30.0), 3))), index=rng.choice(("int64", "int32")),
                           spread=rng.choice(("even", "uneven", "one")), absent=rng.choice((0.0, 0.0, 0.1)))
            if work(case)["bytes"] <= 1.0e9:
                break
    del case["name"]
    return case


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        fwd = m * k + n * k + m * n + (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        if not case["train"]:
            return {"bytes": e * fwd, "flops": 2 * m * k * n}
        bwd = m * n + m * k + n * k + (n if case["bias"] else 0)   # the incoming gradient; the three outgoing ones
        return {"bytes": e * (fwd + bwd), "flops": 6 * m * k * n}
    v, d, n = case["v"], case["d"], case["n"]
    ib = 8 if case["index"] == "int64" else 4
    rows = min(v, n)
    fwd = e * (rows * d + n * d) + ib * n
    if not case["train"]:
        return {"bytes": fwd, "flops": n * d}
    return {"bytes": fwd + e * (n * d + v * d), "flops": 3 * n * d}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _gen(seed)
    dt = DTYPES[case["dtype"]]
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    if case["op"] == "linear":
        m, k, n, pad = case["m"], case["k"], case["n"], case["pad"]
        x, w, b = rnd(m, k + pad), rnd(n, k) / math.sqrt(k), 0.1 * rnd(n)
        if case["train"] and case["act"] == "relu":
            # the sign of x w + b decides which gradients pass: on a grid whose sums are exact in 32 bits (steps of 2^-5 and 2^-9,
            # magnitudes below 2^3 and 2^2) it does not hang on the order of summation
            x = (x.clamp(-3.9, 3.9) * 32.0).round() / 32.0
            w = (w.clamp(-0.24, 0.24) * 512.0).round() / 512.0
            b = (b.clamp(-0.24, 0.24) * 512.0).round() / 512.0
        st = {"case": case, "x": x.to(dt)[:, pad:], "w": w.to(dt), "b": b.to(dt) if case["bias"] else None,
              "r": rnd(m, n).to(dt) if case["residual"] else None}
        if case["train"]:
            st["yb"] = rnd(m, n).to(dt)
        return st
    v, d, n = case["v"], case["d"], case["n"]
    if case["spread"] == "one":
        idx = torch.full((n,), int(seed) % v, device="cuda", dtype=torch.int64)
    else:
        u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
        idx = ((u ** 6 if case["spread"] == "uneven" else u) * v).long().clamp_(max=v - 1)
        if case["spread"] == "uneven":       # the frequent rows lie anywhere in the table
            idx = torch.randperm(v, generator=g, device="cuda")[idx]
    if case["absent"] > 0.0:                 # padded slots carry no row
        idx = torch.where(torch.rand(n, generator=g, device="cuda") < case["absent"], torch.full_like(idx, -1), idx)
    st = {"case": case, "table": (0.02 * rnd(v, d)).to(dt), "idx": idx.to(getattr(torch, case["index"]))}
    if case["train"]:
        st["yb"] = rnd(n, d).to(dt)
    return st


def _act(z, act, beta):
    """act(z) and act'(z)."""
    if act == "none":
        return z, None
    if act == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if act == "softplus":
        e = torch.exp(-(beta * z).abs())
        return torch.clamp(z, min=0.0) + torch.log1p(e) / beta, torch.where(z > 0, torch.ones_like(z), e) / (1.0 + e)
    e = torch.exp(-z.abs())
    s = torch.where(z > 0, torch.ones_like(z), e) / (1.0 + e)
    if act == "sigmoid":
        return s, s * torch.where(z > 0, e, torch.ones_like(z)) / (1.0 + e)
    if act == "silu":
        return z * s, s * (1.0 + z * (1.0 - s))
    phi = 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))


def _run_plain(st):
    case = st["case"]
    dt = DTYPES[case["dtype"]]
    if case["op"] == "linear":
        x, w = st["x"].float(), st["w"].float()
        z = x @ w.t()
        if st["b"] is not None:
            z = z + st["b"].float()
        y, d = _act(z, case["act"], case["beta"])
        if st["r"] is not None:
            y = y + st["r"].float()
        out = {"y": y.to(dt)}
        if case["train"]:
            zb = st["yb"].float() if d is None else st["yb"].float() * d
            out["x_bar"] = (zb @ w).to(dt)
            out["w_bar"] = (zb.t() @ x).to(dt)
            if st["b"] is not None:
                out["b_bar"] = zb.sum(0).to(dt)
        return out
    idx = st["idx"].long()
    live = idx >= 0
    safe = torch.clamp(idx, min=0)
    rows = st["table"][safe].float() * case["scale"]
    out = {"rows": (rows * live[:, None]).to(dt)}
    if case["train"]:
        g = st["yb"].float() * live[:, None]
        acc = torch.zeros(case["v"], case["d"], dtype=torch.float32, device=g.device)
        acc.index_add_(0, safe, g)
        out["table_bar"] = (acc * case["scale"]).to(dt)
    return out


def _run_own(st):
    from nrhints_amd import ops
    case = st["case"]
    if case["op"] == "linear":
        x, w, b, r, act, beta = st["x"], st["w"], st["b"], st["r"], case["act"], case["beta"]
        if not case["train"]:
            return {"y": ops.linear(x, w, b, r, activation=act, beta=beta)}
        y, saved = ops.linear_train_forward(x, w, b, r, activation=act, beta=beta)
        xb, wb, bb = ops.linear_backward(st["yb"], x, w, saved, activation=act, want_bias=b is not None)
        return {"y": y, "x_bar": xb, "w_bar": wb} if bb is None else {"y": y, "x_bar": xb, "w_bar": wb, "b_bar": bb}
    out = {"rows": ops.embedding(st["table"], st["idx"], scale=case["scale"])}
    if case["train"]:
        out["table_bar"] = ops.embedding_backward(st["yb"], st["idx"], case["v"], scale=case["scale"])
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


def exact(case, seed):
    """The definitions in float64: the layer through autograd, the table's gradient as an accumulating assignment."""
    st = prepare(case, seed)
    if case["op"] == "linear":
        F = torch.nn.functional
        leaf = lambda t: None if t is None else t.double().requires_grad_(case["train"])
        x, w, b = leaf(st["x"]), leaf(st["w"]), leaf(st["b"])
        z = F.linear(x, w, b)
        y = {"none": lambda t: t, "relu": F.relu, "sigmoid": torch.sigmoid, "silu": F.silu, "gelu": F.gelu,
             "softplus": lambda t: torch.logaddexp(case["beta"] * t, torch.zeros_like(t)) / case["beta"]}[case["act"]](z)
        if st["r"] is not None:
            y = y + st["r"].double()
        out = {"y": y.detach()}
        if case["train"]:
            grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], st["yb"].double())
            out.update(zip(("x_bar", "w_bar", "b_bar"), grads))
        return out
    idx, scale = st["idx"].long(), float(case["scale"])
    hit = (idx >= 0).nonzero()[:, 0]
    rows = torch.zeros(case["n"], case["d"], dtype=torch.float64, device=idx.device)
    rows[hit] = st["table"].double().index_select(0, idx[hit]) * scale
    out = {"rows": rows}
    if case["train"]:
        tb = torch.zeros(case["v"], case["d"], dtype=torch.float64, device=idx.device)
        out["table_bar"] = tb.index_put_((idx[hit],), st["yb"].double()[hit] * scale, accumulate=True)
    return out
