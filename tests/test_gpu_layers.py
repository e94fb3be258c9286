"""Layer operators (nrhints_amd/ops.py: linear*, embedding*; layers.py) against their definitions in float64.

Tolerances are bounds, computed element by element from the operands (u32 = 2^-24, uT = half a step of the tensor's type):
  * a float32 sum of R products differs from the exact one by at most (R + 8) u32 sum |a b| (any order; the 8 covers the three-way
    bfloat16 split of float32 operands, whose left-out products are below 2 u32 |a b|, bias and residual);
  * an activation is evaluated to 8 u32 of its value and passes the argument's error on with its Lipschitz constant;
  * every output is rounded once: uT |value| (float16: at least half a subnormal step, 2^-25); in the backward of a 16-bit type
    ybar act' is rounded once (not for "none" and "relu", where it is exact), and act' once to the wider type it is kept in.
ReLU's gradient is tested on operands whose sums are exact in float32, so that the sign of an argument is no matter of rounding."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

from nrhints_amd import _lib, layers, ops  # noqa: E402

U32 = 2.0 ** -24
LIPSCHITZ = {"none": 1.0, "relu": 1.0, "softplus": 1.0, "sigmoid": 0.25, "silu": 1.1, "gelu": 1.13}
CURVATURE = {"none": 0.0, "relu": 0.0, "softplus": 0.25, "sigmoid": 0.1, "silu": 0.5, "gelu": 0.8}     # times beta for softplus
DT = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]


def ut(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return {torch.float32: 1e-37, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-37}[dtype]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def act64(z, act, beta):
    return {"none": lambda t: t, "relu": F.relu, "sigmoid": torch.sigmoid, "silu": F.silu, "gelu": F.gelu,
            "softplus": lambda t: torch.logaddexp(beta * t, torch.zeros_like(t)) / beta}[act](z)


def operands(m, k, n, dtype, act, seed, bias=True, residual=False, pad=0, wide=0):
    g = gen(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, w, b = rnd(m, k + pad + wide), rnd(n, k + wide) / math.sqrt(k), 0.1 * rnd(n)
    if act == "relu":
        x, w, b = (x.clamp(-3.9, 3.9) * 32).round() / 32, (w.clamp(-0.24, 0.24) * 512).round() / 512, (b.clamp(-0.24, 0.24) * 512).round() / 512
    cut = lambda t, lo, hi: t.to(dtype)[:, lo:hi]
    return (cut(x, pad, pad + k), cut(w, 0, k), b.to(dtype) if bias else None, rnd(m, n).to(dtype) if residual else None, rnd(m, n).to(dtype))


def check_linear(x, w, b, r, yb, act, beta, train=True):
    dtype, (m, k), n = x.dtype, x.shape, w.shape[0]
    X, W, B, R, YB = (None if t is None else t.double() for t in (x, w, b, r, yb))
    leaves = [t.requires_grad_(True) for t in (X, W, B) if t is not None]
    z = F.linear(X, W, B)
    a = act64(z, act, beta)
    want = a if R is None else a + R
    with torch.no_grad():
        size = X.abs() @ W.abs().t() + (0 if B is None else B.abs())
        ez = (k + 8) * U32 * size
        bound = LIPSCHITZ[act] * ez + 8 * U32 * a.abs() + (0 if R is None else U32 * (a.abs() + R.abs())) + ut(dtype) * want.abs() * (1 + 2 * U32) + tiny(dtype)
        got = ops.linear(x, w, b, r, activation=act, beta=beta)
        assert got.dtype == dtype and got.shape == want.shape
        assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())
    if not train:
        return
    y, dact = ops.linear_train_forward(x, w, b, r, activation=act, beta=beta)
    assert torch.equal(y, got)
    grads = torch.autograd.grad(want, leaves, YB)
    xb, wb, bb = ops.linear_backward(yb, x, w, dact, activation=act, want_bias=b is not None)
    zl = z.detach().requires_grad_(True)
    d = torch.autograd.grad(act64(zl, act, beta).sum(), zl)[0]
    with torch.no_grad():
        curve = CURVATURE[act] * (beta if act == "softplus" else 1.0)
        # (|d| + 1: act' is a sum of terms of size up to 1 + |z| that may cancel)
        ed = curve * ez + 16 * U32 * (1.0 + (z.abs() if act in ("silu", "gelu") else 0.0)) if act not in ("none", "relu") else torch.zeros_like(z)
        exact_zb = dtype == torch.float32 or act in ("none", "relu")
        kept = {torch.float32: 0.0, torch.float16: 0.0, torch.bfloat16: ut(torch.float16)}[dtype]      # the rounding of act'
        ezb = YB.abs() * (ed * (1 + 4 * ut(dtype)) + (0.0 if exact_zb else 1.0) * ((1.01 * ut(dtype) + kept) * d.abs() + 2.0 ** -25))
        ezb = ezb + (U32 * (YB * d).abs() if not act == "none" else 0.0) + (0.0 if exact_zb else tiny(dtype))
        zb = (YB * d).abs()
        ex = ezb @ W.abs() + (n + 8) * U32 * (zb @ W.abs()) + 1.01 * ut(dtype) * grads[0].abs() + tiny(dtype)
        ew = ezb.t() @ X.abs() + (m + 8) * U32 * (zb.t() @ X.abs()) + 1.01 * ut(dtype) * grads[1].abs() + tiny(dtype)
        for name, g, want_g, e in (("x", xb, grads[0], ex), ("w", wb, grads[1], ew)) + \
                ((("b", bb, grads[2], ezb.sum(0) + (m + 8) * U32 * zb.sum(0) + 1.01 * ut(dtype) * grads[2].abs() + tiny(dtype)),) if b is not None else ()):
            assert g.dtype == dtype and g.shape == want_g.shape
            err = (g.double() - want_g).abs()
            assert bool((err <= e).all()), (name, float((err / e).max()))


SIZES = [(1, 1, 1), (1, 256, 256), (2, 7, 3), (5, 1024, 513), (16, 40, 8), (31, 256, 1), (33, 33, 33), (64, 64, 64), (65, 129, 63), (127, 84, 256),
         (128, 128, 128), (129, 340, 256), (300, 361, 255), (1000, 63, 129), (4099, 256, 3), (8192, 256, 256), (20000, 39, 217), (16500, 1000, 1030), (3000, 2050, 2000),
         (517, 3, 70), (9, 7, 2), (1030, 1, 5), (16, 1, 16), (3, 5, 3), (2, 3, 400), (40, 15, 1), (700, 9, 7), (9, 8, 8), (17, 16, 1), (70000, 3, 2), (2, 7001, 3), (3, 2, 7001)]


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_sizes(m, k, n, dtype):
    act = ops.ACTIVATIONS[(m + k + n) % 6]
    beta = 100.0 if (m + n) % 2 else 1.0
    check_linear(*operands(m, k, n, dtype, act, m * 7 + k, bias=k % 2 == 0 or n % 2 == 0, residual=m % 2 == 1), act, beta)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("act", ops.ACTIVATIONS)
def test_linear_activations(act, dtype):
    for bias, residual in ((True, False), (False, True), (True, True)):
        check_linear(*operands(301, 70, 130, dtype, act, 5, bias, residual), act, 3.0)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("pad,wide", [(1, 0), (3, 5), (8, 8), (4, 4)])
def test_linear_strided_operands(pad, wide, dtype):
    """x and weight as column blocks of wider buffers, aligned and not, and tensors with other strides (copied)."""
    x, w, b, r, yb = operands(700, 96, 160, dtype, "silu", 9, True, True, pad, wide)
    assert x.stride(0) == 96 + pad + wide and not x.is_contiguous()
    check_linear(x, w, b, r, yb, "silu", 1.0)
    xt = x.t().contiguous().t()
    ybw = torch.cat([yb, yb], dim=1)[:, :160]
    assert torch.equal(ops.linear(xt, w, b, r, "silu"), ops.linear(x, w, b, r, "silu"))
    _, d = ops.linear_train_forward(x, w, b, r, "silu")
    for p, q in zip(ops.linear_backward(yb, x, w, d, "silu"), ops.linear_backward(ybw, xt, w.contiguous(), d, "silu")):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
def test_linear_leading_dimensions_and_empty_batches(dtype):
    x, w, b, r, yb = operands(60, 24, 40, dtype, "gelu", 2, True, True)
    y2 = ops.linear(x, w, b, r, "gelu")
    assert torch.equal(ops.linear(x.reshape(3, 4, 5, 24), w, b, r.reshape(3, 4, 5, 40), "gelu"), y2.reshape(3, 4, 5, 40))
    assert torch.equal(ops.linear(x[0], w, b, r[0], "gelu").double(), ops.linear(x[:1], w, b, r[:1], "gelu")[0].double())
    empty = ops.linear(x[:0], w, b, None, "gelu")
    assert empty.shape == (0, 40)
    xb, wb, bb = ops.linear_backward(yb[:0], x[:0], w, ops.linear_train_forward(x[:0], w, b, None, "gelu")[1], "gelu")
    assert xb.shape == (0, 24) and not wb.any() and not bb.any() and wb.shape == (40, 24) and bb.shape == (40,)


@pytest.mark.parametrize("scale", [1e-30, 1e-12, 1e15])
def test_linear_float32_has_no_preferred_magnitude(scale):
    x, w, b, r, yb = operands(200, 300, 140, torch.float32, "none", 3, False, False)
    check_linear(x * scale, w, None, None, yb * scale if scale < 1 else yb, "none", 1.0)


def test_linear_float32_infinities_and_nan_stay_in_their_rows():
    """A row that holds an infinity, a NaN or values whose bfloat16 part overflows gives what float32 arithmetic gives; the other rows of
    the tile stay within the bound."""
    x, w, b, r, yb = operands(300, 130, 150, torch.float32, "none", 4)
    clean = ops.linear(x, w, b)
    x = x.clone()
    x[3, 5], x[77, 0], x[130, 129], x[200, 64] = float("inf"), float("nan"), -float("inf"), 3.4e38
    w = w.clone()
    w[10, 5] = 0.0
    got = ops.linear(x, w, b)
    want = F.linear(x.double(), w.double(), b.double())
    bad = [3, 77, 130]
    assert torch.isnan(got[77]).all() and torch.isnan(got[3, 10]) and torch.equal(torch.isnan(got[bad]), torch.isnan(want[bad]))
    fin = [i for i in range(150) if i != 10]
    assert torch.equal(got[3, fin].double(), want[3, fin]) and torch.equal(got[130].double(), want[130])
    in32 = want[200].abs() < 3.3e38
    assert bool(in32.any()) and bool(((got[200].double() - want[200]).abs()[in32] <= 140 * U32 * (x[200].double().abs() @ w.double().abs().t())[in32]).all())
    keep = [i for i in range(300) if i not in (3, 77, 130, 200)]
    cols = [i for i in range(150) if i != 10]
    size = x.double().abs() @ w.double().abs().t()
    assert bool(((got.double() - clean.double()).abs()[keep][:, cols] <= 2 * 140 * U32 * (size + 1)[keep][:, cols]).all())
    # ... and gradients
    yb = yb.clone()
    yb[7, 3] = float("inf")
    x0 = x.nan_to_num(0.0, 0.0, 0.0)
    xb, wb, bb = ops.linear_backward(yb, x0, w, None)
    assert not torch.isfinite(xb[7]).any() and torch.isfinite(xb[:7]).all() and torch.isfinite(xb[8:]).all()
    # column 64 of x holds 3.4e38 once: times |ybar| > 1.0009 that is past float32, as float64 followed by one rounding says
    want_w = (yb.double().t() @ x0.double()).float()
    assert torch.equal(torch.isfinite(wb), torch.isfinite(want_w)) and not torch.isfinite(wb[3]).all() and not torch.isfinite(wb[:, 64]).all()
    other = [j for j in range(130) if j != 64]
    assert torch.isfinite(wb[:3][:, other]).all() and torch.isfinite(wb[4:][:, other]).all() and torch.isinf(bb[3]) and torch.isfinite(bb[:3]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_linear_16_bit_infinities(dtype):
    x, w, b, r, yb = operands(70, 64, 64, dtype, "none", 4)
    x = x.clone()
    x[3, 5], x[40, 2] = float("inf"), float("nan")
    got, want = ops.linear(x, w, b, activation="relu"), F.relu(F.linear(x.double(), w.double(), b.double()))
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want.to(dtype)))


@pytest.mark.parametrize("dtype", DT, ids=IDS)
def test_linear_extreme_arguments_of_the_activations(dtype):
    """z of every magnitude through every activation: finite, and act' stays within [-0.2, 1.2]."""
    z = torch.tensor([0.0, -0.0, 1e-7, -1e-7, 1.0, -1.0, 30.0, -30.0, 88.0, -88.0, 200.0, -200.0, 6e4, -6e4], device="cuda", dtype=dtype)[:, None]
    one = torch.ones(1, 1, device="cuda", dtype=dtype)
    for act in ops.ACTIVATIONS:
        y, d = ops.linear_train_forward(z, one, None, None, act, beta=100.0)
        want = act64(z.double(), act, 100.0)
        err = (y.double() - want).abs()
        assert bool((err <= 16 * U32 * want.abs() + ut(dtype) * want.abs() + 32 * tiny(dtype) + (1e-9 if act in ("softplus", "sigmoid", "silu", "gelu") else 0)).all()), (act, err)
        if d is not None and act != "relu":
            assert torch.isfinite(d).all() and float(d.min()) > -0.2 and float(d.max()) < 1.2


def test_linear_gradient_against_differences():
    """d/dt of sum(ybar y(x + t v)) by central differences of the kernel's own float32 values: the difference quotient is exact to
    h^2 / 6 max|y'''| |v|^3 plus 2 bound(y) / h, summed over the outputs."""
    for act in ("silu", "gelu", "softplus", "sigmoid"):
        x, w, b, r, yb = operands(40, 24, 30, torch.float32, act, 8)
        y, d = ops.linear_train_forward(x, w, b, None, act, 1.0)
        xb, wb, bb = ops.linear_backward(yb, x, w, d, act)
        h = 2.0 ** -7
        loss = lambda x_, w_, b_: (ops.linear(x_, w_, b_, None, act, 1.0).double() * yb.double()).sum()
        g = gen(11)
        vx, vw, vb = (torch.randn(t.shape, generator=g, device="cuda") * 0.3 for t in (x, w, b))
        vx, vw, vb = [(v * 128).round() / 128 for v in (vx, vw, vb)]
        for t, v, gr in ((0, vx, xb), (1, vw, wb), (2, vb, bb)):
            plus, minus = [x, w, b], [x, w, b]
            plus[t], minus[t] = plus[t] + h * v, minus[t] - h * v
            num = float((loss(*plus) - loss(*minus)) / (2 * h))
            dz = (vx.double() @ w.double().t(), x.double() @ vw.double().t(), vb.double()[None, :].expand(40, 30))[t].abs()
            size = x.double().abs() @ w.double().abs().t() + b.double().abs() + 1.0
            bound = float((yb.double().abs() * (h * h / 6 * 2.0 * dz ** 3 + 2 * (24 + 16) * U32 * size / h)).sum())
            assert abs(num - float((gr.double() * v.double()).sum())) <= bound, (act, t)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
def test_linear_writes_only_its_own_columns(dtype):
    """The C entries with row strides wider than the rows: what lies between the rows stays."""
    lib = _lib.load()
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    m, k, n = 200, 72, 100
    x, w, b, r, yb = operands(m, k, n, dtype, "silu", 6)
    P = lambda t: None if t is None else t.data_ptr()
    for ldy in (n, n + 1, n + 8):
        buf = torch.full((m + 2, ldy), 7.0, dtype=dtype, device="cuda")
        rc = lib.nrh_linear_forward(code, P(x), k, P(w), k, P(b), None, 0, 4, 1.0, m, n, k, buf[1:].data_ptr(), ldy, None, None, 0, _lib.stream_handle())
        assert rc == 0
        assert torch.equal(buf[1:m + 1, :n], ops.linear(x, w, b, None, "silu")) and bool((buf[:, n:] == 7).all()) and bool((buf[0] == 7).all()) and bool((buf[m + 1] == 7).all())
    for ldx in (k, k + 3):
        bx = torch.full((m, ldx), 7.0, dtype=dtype, device="cuda")
        bw = torch.full((n, ldx), 7.0, dtype=dtype, device="cuda")
        ws = [torch.empty(max(1, lib.nrh_linear_workspace_bytes(op, code, 0, m, n, k)), dtype=torch.uint8, device="cuda") for op in (1, 2)]
        assert lib.nrh_linear_backward_data(code, P(yb), n, None, 0, 0, P(w), k, m, n, k, P(bx), ldx, P(ws[0]), ws[0].numel(), _lib.stream_handle()) == 0
        assert lib.nrh_linear_backward_weight(code, P(yb), n, None, 0, 0, P(x), k, m, n, k, P(bw), ldx, None, P(ws[1]), ws[1].numel(), _lib.stream_handle()) == 0
        xb, wb, _ = ops.linear_backward(yb, x, w, None)
        assert torch.equal(bx[:, :k], xb) and torch.equal(bw[:, :k], wb) and bool((bx[:, k:] == 7).all()) and bool((bw[:, k:] == 7).all())


def test_linear_offsets_past_32_bits():
    """2^31 elements and more behind one operand: the last rows are right (16-bit rows of 4 100 elements, 600 000 of them)."""
    m, ld, k, n = 600000, 4100, 96, 40
    big = torch.zeros(m, ld, dtype=torch.bfloat16, device="cuda")
    assert big.numel() > 2 ** 31
    x = big[:, 2000:2000 + k]
    g = gen(1)
    x.copy_(torch.randn(m, k, generator=g, device="cuda"))
    w = torch.randn(n, k, generator=g, device="cuda").bfloat16()
    y = ops.linear(x, w)
    assert torch.equal(y[-300:], ops.linear(x[-300:].contiguous(), w)) or float((y[-300:].double() - x[-300:].double() @ w.double().t()).abs().max()) < 0.3
    tail = y[-300:].double() - x[-300:].double() @ w.double().t()
    bound = (k + 8) * U32 * (x[-300:].double().abs() @ w.double().abs().t()) + ut(torch.bfloat16) * y[-300:].double().abs() * 1.01
    assert bool((tail.abs() <= bound).all())


# ---- embedding ---------------------------------------------------------------------------------------------------------------
def indices(n, v, spread, seed, dtype=torch.int64, absent=0.0):
    g = gen(seed)
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    idx = {"even": lambda: (u * v).long(), "uneven": lambda: ((u ** 6) * v).long(), "one": lambda: torch.full((n,), v - 1, device="cuda"),
           "sorted": lambda: (u * v).long().sort()[0]}[spread]().clamp_(0, v - 1)
    if absent:
        a = torch.rand(n, generator=g, device="cuda") < absent
        idx[a] = torch.where(torch.rand(int(a.sum()), generator=g, device="cuda") < 0.5, -1, v)
    return idx.to(dtype)


def check_embedding(v, d, n, dtype, spread, index_dtype, absent, scale, seed=0):
    """Integer gradients small enough that every order of summation is exact: equality up to the one rounding."""
    idx = indices(n, v, spread, seed + n, index_dtype, absent)
    g = gen(seed + 1)
    table = torch.randn(v, d, generator=g, device="cuda").to(dtype)
    live = (idx >= 0) & (idx < v)
    safe = torch.where(live, idx, torch.zeros_like(idx)).long()
    rows = ops.embedding(table, idx, scale)
    want = torch.where(live[:, None], (table[safe].float() * scale).to(dtype), torch.zeros((), dtype=dtype, device="cuda"))
    assert rows.dtype == dtype and torch.equal(rows, want)
    gb = torch.randint(-8, 9, (n, d), generator=g, device="cuda").to(dtype)
    got = ops.embedding_backward(gb, idx, v, scale)
    acc = torch.zeros(v, d, dtype=torch.float64, device="cuda")
    if spread == "one":
        acc[v - 1] = (gb.double() * live[:, None]).sum(0)
    else:
        acc.index_add_(0, safe, gb.double() * live[:, None])
    assert float(acc.abs().max() if acc.numel() else 0) < 2 ** 24
    assert torch.equal(got, (acc.float() * scale).to(dtype)), (v, d, n)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 64, 65, 511, 512, 513, 1000, 2047, 2048, 2049, 5000, 70001, 140000])
def test_embedding_tokens(n, dtype):
    for v, d, spread in ((1, 3, "even"), (100, 12, "uneven"), (70000, 64, "even"), (300, 5, "one"), (255, 260, "even"), (40, 9, "one")):
        check_embedding(v, d, n, dtype, spread, torch.int64 if n % 2 else torch.int32, 0.1, 1.0)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("v", [1, 2, 255, 256, 257, 65535, 65536, 300000])
def test_embedding_table_heights(v, dtype):
    for n, d, spread in ((3000, 8, "even"), (777, 33, "sorted")):
        check_embedding(v, d, n, dtype, spread, torch.int64, 0.0, 2.0)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("d", [1, 2, 4, 7, 8, 12, 48, 100, 256, 513, 1030, 4096])
def test_embedding_row_lengths(d, dtype):
    for n, spread in ((400, "uneven"), (2500, "one")):
        check_embedding(50, d, n, dtype, spread, torch.int32, 0.3, 0.5)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
def test_embedding_values(dtype):
    """Real-valued gradients: a float32 sum of c terms is exact to c u32 sum|.|, then the scale and one rounding; shapes, views."""
    v, d, n = 90, 40, 6000
    idx = indices(n, v, "uneven", 3)
    big = torch.randn(n, d + 3, generator=gen(2), device="cuda").to(dtype)
    gb = big[:, 3:]
    got = ops.embedding_backward(gb.reshape(60, 100, d), idx.reshape(60, 100), v, 0.37)
    acc = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_add_(0, idx, gb.double())
    mag = torch.zeros(v, d, dtype=torch.float64, device="cuda").index_add_(0, idx, gb.double().abs())
    cnt = torch.bincount(idx, minlength=v)[:, None].double()
    scale = float(torch.tensor(0.37))
    bound = scale * ((cnt + 2) * U32 * mag) + (ut(dtype) * 1.01 + U32) * (scale * acc).abs() + tiny(dtype)
    assert bool(((got.double() - scale * acc).abs() <= bound).all())
    assert torch.equal(got, ops.embedding_backward(gb, idx, v, 0.37))
    table = torch.randn(v, d + 5, generator=gen(4), device="cuda").to(dtype)[:, 2:d + 2]
    # the product is rounded to the type from float32 or at once (v_fma_mixlo_f16): uT (1 + u32) + u32 of the value either way
    rows, exact = ops.embedding(table, idx.reshape(60, 100), 0.37), (table.double()[idx] * scale).reshape(60, 100, d)
    assert bool(((rows.double() - exact).abs() <= (ut(dtype) * 1.01 + U32) * exact.abs() + tiny(dtype)).all())
    bad = gb.clone()
    bad[5] = float("nan")
    nan = ops.embedding_backward(bad, idx, v)
    assert torch.isnan(nan[idx[5]]).all() and int(torch.isnan(nan).any(1).sum()) == 1


def test_embedding_offsets_past_32_bits():
    v, d = 2100000, 1030
    table = torch.zeros(v, d, dtype=torch.bfloat16, device="cuda")
    table[-2:] = 3.0
    idx = torch.tensor([0, v - 1, v - 2, -1, v, 2 ** 40], device="cuda")
    assert ops.embedding(table, idx, 2.0)[:, 0].tolist() == [0.0, 6.0, 6.0, 0.0, 0.0, 0.0]
    del table
    g = ops.embedding_backward(torch.ones(6, d, dtype=torch.bfloat16, device="cuda"), idx, v)
    assert float(g[-1].float().sum()) == d and float(g[-2].float().sum()) == d and float(g[0].float().sum()) == d and float(g[1:-2].float().abs().max()) == 0.0


# ---- together ------------------------------------------------------------------------------------------------------------------
class Net(torch.nn.Module):
    """Per-view codes beside the inputs of a small residual network: what the two operators are for."""

    def __init__(self):
        super().__init__()
        self.code = layers.Embedding(20, 16, scale=0.25)
        self.l0, self.l1, self.l2 = layers.Linear(39 + 16, 128, activation="softplus", beta=1.0), layers.Linear(128, 128, activation="silu"), layers.Linear(128, 3, activation="sigmoid")

    def forward(self, x, view):
        h = self.l0(torch.cat([x, self.code(view)], dim=-1))
        return self.l2(self.l1(h, residual=h))


def net64(net, x, view):
    p = {k: v.detach().double().requires_grad_(True) for k, v in net.named_parameters()}
    h = F.softplus(F.linear(torch.cat([x.double(), 0.25 * p["code.weight"][view]], dim=-1), p["l0.weight"], p["l0.bias"]))
    h = F.silu(F.linear(h, p["l1.weight"], p["l1.bias"])) + h
    return torch.sigmoid(F.linear(h, p["l2.weight"], p["l2.bias"])), p


def test_a_network_of_layers_trains_like_its_definition():
    torch.manual_seed(0)
    net = Net().cuda()
    x, view = torch.randn(1536, 39, device="cuda"), torch.randint(0, 20, (1536,), device="cuda")
    out = net(x, view)
    want, p = net64(net, x, view)
    seed = torch.randn(1536, 3, device="cuda")
    out.backward(seed)
    want.backward(seed.double())
    # three layers of float32 sums of at most 1 536 terms against their float64 values, relative to a tensor's largest entry
    assert float((out.double() - want).abs().max()) < 1e-6
    for k, v in net.named_parameters():
        g = p[k].grad
        assert float((v.grad.double() - g).abs().max()) <= 1536 * U32 * float(g.abs().max()), k
    first = {k: v.grad.clone() for k, v in net.named_parameters()}
    net.zero_grad()
    net(x, view).backward(seed)
    assert all(torch.equal(first[k], v.grad) for k, v in net.named_parameters())       # the same bits


def test_second_derivatives_and_mixed_types_are_refused():
    x = torch.randn(8, 4, device="cuda", requires_grad=True)
    w = torch.randn(4, 4, device="cuda")
    (g,) = torch.autograd.grad(layers.linear(x, w, activation="silu").sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    for bad in (lambda: ops.linear(x, w.half()), lambda: ops.linear(x.double(), w.double()), lambda: ops.linear(x, w, activation="tanh"),
                lambda: ops.linear(x, w[:, :3]), lambda: ops.linear(x, w, torch.zeros(3, device="cuda")), lambda: ops.linear(x, w.cpu()),
                lambda: ops.linear(x, w, None, torch.zeros(1, 4, device="cuda")), lambda: ops.linear(x, w, activation="softplus", beta=0.0),
                lambda: ops.linear_backward(x, x, w, None, "silu"), lambda: ops.linear_backward(x[:4], x, w, None),
                lambda: ops.embedding(w, torch.zeros(3, device="cuda")), lambda: ops.embedding(w, torch.zeros(3, dtype=torch.int64)),
                lambda: ops.embedding_backward(x.detach(), torch.zeros(3, dtype=torch.int64, device="cuda"), 5),
                lambda: ops.embedding_backward(x.detach(), torch.zeros(8, dtype=torch.int64, device="cuda"), 0)):
        with pytest.raises(ValueError):
            bad()


def test_layers_on_a_side_stream_and_in_graphs():
    """The operators on another stream, and two captured graphs replayed in turn with eager calls between: every replay equals the
    eager result bit for bit (each capture holds its own workspaces)."""
    m, k, n, v = 3000, 96, 80, 50
    x, w, b, r, yb = operands(m, k, n, torch.float32, "silu", 12, True, True)
    idx = indices(m, v, "uneven", 5)
    table = torch.randn(v, n, generator=gen(6), device="cuda")

    def step(x_, t_):
        rows = ops.embedding(t_, idx, 0.5)
        y, d = ops.linear_train_forward(x_, w, b, rows, "silu")
        return [y, ops.embedding_backward(yb, idx, v, 0.5), *ops.linear_backward(yb, x_, w, d, "silu")]

    eager = step(x, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x, table)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(eager, other))
    sx, st = x.clone(), table.clone()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs = step(sx, st)
        graphs.append((gr, outs))
    for trial in range(3):
        sx.copy_(x * (trial + 1))
        st.copy_(table - trial)
        want = step(sx, st)
        for gr, outs in graphs:
            gr.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(want, outs)), trial


def test_a_captured_backward_pass():
    """Forward and backward through autograd inside a capture, replayed, against the eager gradients."""
    torch.manual_seed(1)
    net = Net().cuda()
    x, view, seed = torch.randn(512, 39, device="cuda"), torch.randint(0, 20, (512,), device="cuda"), torch.randn(512, 3, device="cuda")
    params = list(net.parameters())
    eager = torch.autograd.grad(net(x, view), params, seed)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(net(x, view), params, seed)
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        grads = torch.autograd.grad(net(x, view), params, seed)
    for _ in range(3):
        for t in grads:
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, grads))


def test_a_capture_beside_a_live_eager_graph_is_refused():
    """Parameters whose eager graph still lives would accumulate their gradients on the eager stream from inside a capture: refused with an
    exception; once the graph is gone the same capture works."""
    torch.manual_seed(2)
    net = Net().cuda()
    x, view, seed = torch.randn(64, 39, device="cuda"), torch.randint(0, 20, (64,), device="cuda"), torch.randn(64, 3, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = torch.autograd.grad(net(x, view), list(net.parameters()), seed)      # warm-up, its graph ends here
    torch.cuda.current_stream().wait_stream(side)
    alive = net(x, view)
    with pytest.raises(RuntimeError, match="outside this capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            net(x, view)
    torch.cuda.synchronize()
    del alive
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = net(x, view)
        y.backward(seed)
    del y
    grads = [p.grad for p in net.parameters()]
    for _ in range(3):
        for t in grads:
            t.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, grads))


@pytest.mark.parametrize("dtype", DT[1:], ids=IDS[1:])
@pytest.mark.parametrize("act", ["softplus", "sigmoid", "silu", "gelu"])
def test_small_gradients_are_rounded_once(dtype, act):
    """Small 16-bit products take ybar act' in two parts (the type's bits twice: 2^-16 of bfloat16 at least), so what a gradient is off by is
    its own rounding, that of the kept act' (beside bfloat16: float16) and float32's."""
    m, k, n, beta = 200, 96, 130, 1.0
    x, w, b, _, yb = operands(m, k, n, dtype, act, 77)
    y, dact = ops.linear_train_forward(x, w, b, activation=act, beta=beta)
    xb, wb, _ = ops.linear_backward(yb, x, w, dact, activation=act)
    X, W, YB = x.double(), w.double(), yb.double()
    z = (X @ W.t() + b.double()).requires_grad_(True)
    d = torch.autograd.grad(act64(z, act, beta).sum(), z)[0]
    z = z.detach()
    ez = (k + 8) * U32 * (X.abs() @ W.abs().t() + b.double().abs())
    ed = CURVATURE[act] * ez + 16 * U32 * (1.0 + (z.abs() if act in ("silu", "gelu") else 0.0))
    kept = ut(torch.float16) * d.abs() + 2.0 ** -25 if dtype == torch.bfloat16 else 0.0
    zb = YB * d
    ezb = YB.abs() * (ed + kept) + 2.0 ** -16 * zb.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    for got, want, err in ((xb, zb @ W, ezb @ W.abs() + (2 * n + 8) * U32 * (zb.abs() @ W.abs())),
                           (wb, zb.t() @ X, ezb.t() @ X.abs() + (2 * m + 8) * U32 * (zb.abs().t() @ X.abs()))):
        bound = err + 1.01 * ut(dtype) * want.abs() + tiny(dtype)
        assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("ld", [3950000, 4200000])
def test_linear_offsets_past_32_bits(ld):
    """Rows so far apart that the last ones lie beyond 2^32 elements, on either side of the 2^22 up to which lanes keep 32-bit offsets."""
    m, k, n = 1100, 72, 40
    g = gen(5)
    store = torch.empty((m, ld), dtype=torch.float16, device="cuda")
    assert store.stride(0) * (m - 1) > 2 ** 32
    x = store[:, 5:5 + k]
    x.copy_(torch.randn(m, k, generator=g, device="cuda"))
    w = (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).half()
    check_linear(x, w, None, None, torch.randn(m, n, generator=g, device="cuda").half(), "silu", 1.0)


def test_calls_at_once_and_two_graphs_of_one_pool():
    """The same bits from three streams at once and from two graphs that share a memory pool, replayed between eager work."""
    g = gen(12)
    x, yb = torch.randn(4096, 300, generator=g, device="cuda").half(), torch.randn(4096, 500, generator=g, device="cuda").half()
    w = (torch.randn(500, 300, generator=g, device="cuda") / 17).half()
    index, rows = torch.randint(0, 700, (20000,), generator=g, device="cuda"), torch.randn(20000, 37, generator=g, device="cuda")
    _, dact = ops.linear_train_forward(x, w, activation="gelu")

    def work():
        return (*ops.linear_backward(yb, x, w, dact, activation="gelu", want_bias=True), ops.embedding_backward(rows, index, 700))

    want = work()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(4):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(work())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o in got for a, b in zip(o, want))
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    with torch.cuda.graph(graphs[0]):
        work()
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        last = work()
    for _ in range(4):
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(last, want))
        ops.linear(x, w)
        torch.cuda.synchronize()


@pytest.mark.parametrize("v,d,n", [(1, 1, 1), (255, 8, 513), (256, 8, 1024), (256, 9, 1025), (5, 1 << 20, 3), (300, 3, 2049), (300, 100000, 40),
                                   (70000, 5, 65537), (2, 4, 0), (10, 7, 12), (60000, 20, 8193)])
def test_embedding_gradient_at_its_limits(v, d, n):
    """Either side of each rule (255 rows, 1 024 tokens, rows of 16 bytes, 64 tiles), against sums in float64: a row's sum of t terms is off
    by at most t u32 sum |rows| and one rounding."""
    for dtype in (torch.float32, torch.bfloat16):
        g = gen(v + d + n)
        rows, index = torch.randn(n, d, generator=g, device="cuda").to(dtype), torch.randint(-1, v + 1, (n,), generator=g, device="cuda")
        got = ops.embedding_backward(rows, index, v)
        ok = (index >= 0) & (index < v)
        want, size, terms = (torch.zeros(v, d, dtype=torch.float64, device="cuda") for _ in range(3))
        want.index_add_(0, index[ok], rows.double()[ok])
        size.index_add_(0, index[ok], rows.double()[ok].abs())
        terms.index_add_(0, index[ok], torch.ones_like(rows, dtype=torch.float64)[ok])
        assert bool(((got.double() - want).abs() <= (terms + 1) * U32 * size + 1.01 * ut(dtype) * want.abs() + tiny(dtype)).all())
