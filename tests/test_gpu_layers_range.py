"""The layer operators away from values of size one: saturated activations, small and large gradients, infinities, subnormal numbers.

u32 = 2^-24.  Arguments are one product with 1, so they are exact; act' is then off by at most 24 u32 of its value: 2 for the exponential,
6 for the complementary error function, 1 for every other step of at most ten, and (softplus) 4 for log or division by beta - never by an
absolute amount.  ybar act' as an operand of a 16-bit product: two bfloat16 parts leave out at most 2^-16 of it (half a step of a rest of
2^-8) and, where x and the weight are in parts too (float16), the rests' product 2^-16.  Float32 sums of R terms add (R + 8) u32 of the sum of magnitudes, twice
that in two parts; an output is rounded once (float16: half a subnormal step, 2^-25, at least)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from nrhints_amd import layers, ops  # noqa: E402

U32 = 2.0 ** -24
DT = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
LEFT_OUT = {torch.float32: 0.0, torch.float16: 2.0 ** -15, torch.bfloat16: 2.0 ** -16}
LOWEST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def slope(z, act, beta):
    """act'(z) in float64 without the cancellation of 1 + erf or 1 - sigmoid in the tails."""
    s = lambda t: torch.where(t > 0, 1 / (1 + torch.exp(-t.abs())), torch.exp(-t.abs()) / (1 + torch.exp(-t.abs())))
    if act == "sigmoid":
        return s(z) * s(-z)
    if act == "softplus":
        return s(beta * z)
    if act == "silu":
        return s(z) * (1 + z * s(-z))
    return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def value(z, act, beta):
    if act == "sigmoid":
        return torch.where(z > 0, 1 / (1 + torch.exp(-z.abs())), torch.exp(-z.abs()) / (1 + torch.exp(-z.abs())))
    if act == "softplus":
        return z.clamp(min=0) + torch.log1p(torch.exp(-(beta * z).abs())) / beta
    return z * (value(z, "sigmoid", 1.0) if act == "silu" else 0.5 * torch.special.erfc(-z / math.sqrt(2)))


def within(name, got, want, bound):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    # (a sum past the type's largest number, 65 504 of float16, is rounded to infinity: 16 384 rows of ybar act' x = -12 make -2e5)
    past = got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= torch.finfo(got.dtype).max)
    assert bool(((err <= bound) | past).all()), (name, float((err / bound).max()))


def check_gradients(xb, wb, bb, zb, x, w, dtype):
    """The three gradients against float64 ones of zb (float64, off by 24 u32 and what the type leaves out of it), purely relative."""
    X, W, (m, n), ut = x.double(), w.double(), zb.shape, torch.finfo(dtype).eps / 2
    size, rel = zb.abs(), 24 * U32 + LEFT_OUT[dtype]
    for name, got, want, sums, r in (("x", xb, zb @ W, size @ W.abs(), n), ("w", wb, zb.t() @ X, size.t() @ X.abs(), m)):
        within(name, got, want, (rel + (2 * r + 8) * U32) * sums + 1.01 * ut * want.abs() + LOWEST[dtype])
    if bb is not None:
        within("b", bb, zb.sum(0), (25 + m + 8) * U32 * size.sum(0) + 1.01 * ut * zb.sum(0).abs() + LOWEST[dtype])


def column_of_arguments(m, n, lo, hi, dtype, seed, k=24):
    """x [m, k], w [n, k] with z = x w^T = a number of the type in lo .. hi for every row: column 0 holds it beside a weight of 1, the next
    third meets zero weights (their weight gradients are sums over rows), the others are zero beside random weights."""
    g = gen(seed)
    z = (lo + (hi - lo) * torch.rand(m, generator=g, device="cuda")).to(dtype)
    x, w = torch.zeros(m, k, dtype=dtype, device="cuda"), torch.zeros(n, k, dtype=dtype, device="cuda")
    x[:, 0], w[:, 0] = z, 1.0
    x[:, 1:k // 3] = torch.rand(m, k // 3 - 1, generator=g, device="cuda").to(dtype) + 0.5
    w[:, k // 3:] = torch.rand(n, k - k // 3, generator=g, device="cuda").to(dtype) + 0.5
    return z, x, w


TAILS = [("sigmoid", 1.0, -20.0, -10.0), ("softplus", 1.0, -20.0, -10.0), ("softplus", 100.0, -0.8, -0.1), ("silu", 1.0, -20.0, -10.0), ("gelu", 1.0, -11.0, -5.0)]


@pytest.mark.parametrize("act,beta,lo,hi", TAILS + [("gelu", 1.0, -5.0, 8.0), ("softplus", 100.0, -0.1, 0.5)])
def test_float32_values_in_the_tails(act, beta, lo, hi):
    """y to 24 u32 of its own value (not of the argument's), on one row and on tiles."""
    for m in (4, 3000):
        z, x, w = column_of_arguments(m, 40, lo, hi, torch.float32, 8)
        y, dact = ops.linear_train_forward(x, w, None, None, act, beta)
        z = z.double()[:, None].expand(m, 40)
        within("y", y, value(z, act, beta), 24 * U32 * value(z, act, beta).abs())
        if hi < 0:
            within("act'", dact, slope(z, act, beta), 24 * U32 * slope(z, act, beta).abs())


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("act,beta,lo,hi", TAILS, ids=[f"{t[0]}{t[1]:g}" for t in TAILS])
@pytest.mark.parametrize("m,k,n", [(6, 24, 16), (300, 24, 130), (3, 12, 5), (4096, 24, 2048), (16384, 512, 512)])
def test_gradients_where_an_activation_is_saturated(m, k, n, act, beta, lo, hi, dtype):
    """Every argument in the tail: act' is far below 2^-24 there, and the gradients of a loss whose ybar makes up for it (1 / y of a
    logarithm, say) are ordinary numbers, right to their own last bits."""
    z, x, w = column_of_arguments(m, n, lo, hi, dtype, 3, k)
    y, dact = ops.linear_train_forward(x, w, None, None, act, beta)
    d = slope(z.double(), act, beta)[:, None].expand(m, n)
    big = (1.0 / d.abs()).clamp(max=3e4 if dtype == torch.float16 else 1e30)
    yb = (big * (0.5 + torch.rand(m, n, generator=gen(4), device="cuda"))).to(dtype)
    xb, wb, bb = ops.linear_backward(yb, x, w, dact, act)
    check_gradients(xb, wb, bb, yb.double() * d, x, w, dtype)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(200, 70, 130), (16384, 512, 512), (30, 9, 5)])
def test_infinities_in_gradients_have_the_sign_of_their_product(m, k, n, dtype):
    """One infinity in x, in the weight or in ybar: every entry it meets is that infinity with the sign of the other factor - which no sum of
    parts may turn into NaN -, the others are as without it."""
    g = gen(k)
    x, w = torch.randn(m, k, generator=g, device="cuda").to(dtype), torch.randn(n, k, generator=g, device="cuda").to(dtype)
    yb = torch.randn(m, n, generator=g, device="cuda").to(dtype)
    dact = 0.25 + torch.rand(m, n, generator=g, device="cuda")
    dact = (dact * 4).round() / 4                          # quarters: some products are exact in one part, some are not
    yb = torch.where(yb == 0, torch.ones_like(yb), yb)
    clean = ops.linear_backward(yb, x, w, dact, "silu")
    zb = yb.double() * dact.double()
    for what, at in (("x", (m // 2, k - 1)), ("w", (n // 3, k // 2)), ("yb", (m - 1, n // 2))):
        t = {"x": x, "w": w, "yb": yb}
        t[what] = t[what].clone()
        t[what][at] = -math.inf
        xb, wb, bb = ops.linear_backward(t["yb"], t["x"], t["w"], dact, "silu")
        inf = lambda s: -math.inf * s.double().sign()
        if what == "x":
            want = ((xb, clean[0], None, None), (wb, clean[1], (slice(None), at[1]), inf(zb[at[0]])), (bb, clean[2], None, None))
        elif what == "w":
            want = ((xb, clean[0], (slice(None), at[1]), inf(zb[:, at[0]])), (wb, clean[1], None, None), (bb, clean[2], None, None))
        else:
            want = ((xb, clean[0], at[0], inf(w[at[1]])), (wb, clean[1], at[1], inf(x[at[0]])), (bb, clean[2], at[1], torch.tensor(-math.inf, device="cuda")))
        for got, base, where, expect in want:
            got, base = got.double().clone(), base.double().clone()
            if where is not None:
                meets = expect != 0                        # (an infinity times zero is NaN)
                assert torch.equal(torch.where(expect.isnan(), 0.0, got[where]), torch.where(expect.isnan(), 0.0, expect.double())), what
                got[where], base[where] = 0.0, 0.0
            # the tile that met an infinity is summed in float32 instead of in parts: both are within the type's step of the exact sum
            assert float((got - base).abs().max()) <= 2 * torch.finfo(dtype).eps * float(base.abs().max()) + (m + n) * 8 * U32 * 8, what


@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("m,k,n", [(20000, 63, 129), (16384, 512, 512), (700, 40, 30)])
def test_float16_gradients_below_its_own_range(m, k, n, act):
    """ybar of 2^-12 times act' of 1e-2 to 1e-5: single products are below float16's smallest number, their sums are not."""
    g = gen(m)
    z = (-5.0 - 5.0 * torch.rand(m, generator=g, device="cuda")).half()
    x, w = torch.rand(m, k, generator=g, device="cuda").half() + 0.5, torch.rand(n, k, generator=g, device="cuda").half() + 0.5
    dact = slope(z.double(), act, 1.0)[:, None].expand(m, n).float().contiguous()
    yb = (2.0 ** -12 * (0.5 + torch.rand(m, n, generator=g, device="cuda"))).half()
    xb, wb, bb = ops.linear_backward(yb, x, w, dact, act)
    assert float(wb.abs().min()) > 0.0
    check_gradients(xb, wb, bb, yb.double() * dact.double(), x, w, torch.float16)


@pytest.mark.parametrize("m,k,n", [(16384, 512, 512), (700, 40, 30)])
def test_float16_gradients_past_its_own_range(m, k, n):
    """ybar near float16's largest number times an act' above one: the product does not fit the type, the gradients do."""
    g = gen(m)
    x, w = 2.0 ** -9 * torch.randn(m, k, generator=g, device="cuda").half(), 2.0 ** -9 * torch.randn(n, k, generator=g, device="cuda").half()
    dact = 1.05 + 0.07 * torch.rand(m, n, generator=g, device="cuda")
    yb = torch.where(torch.rand(m, n, generator=g, device="cuda") < 0.5, -65000.0, 65000.0).half()
    xb, wb, bb = ops.linear_backward(yb, x, w, dact, "gelu")
    zb = yb.double() * dact.double()
    # (16 384 terms of 7e4 2^-9 add up to 17 500 rms: a few of the weight's 262 144 sums, beyond 3.7 rms, are past the type and infinite)
    assert float(zb.abs().min()) > 65504.0 and torch.isfinite(xb).all() and float(wb.isinf().float().mean()) < 1e-3
    check_gradients(xb, wb, None, zb, x, w, torch.float16)


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "softplus"])
def test_gradients_have_one_precision_in_every_batch(act, dtype):
    """16 384 rows at once, the first 200 of them by themselves: both are off by the float32 sums, two parts' rest and their own rounding, the
    large tiles as the small ones."""
    g = gen(9)
    m, k, n = 16384, 512, 768
    x, w = torch.randn(m, k, generator=g, device="cuda").to(dtype), (torch.randn(n, k, generator=g, device="cuda") / 22).to(dtype)
    yb = torch.randn(m, n, generator=g, device="cuda").to(dtype)
    _, dact = ops.linear_train_forward(x, w, None, None, act, 2.0)
    for rows in (m, 200):
        xb, wb, _ = ops.linear_backward(yb[:rows], x[:rows], w, dact[:rows], act)
        zb, X, W = yb[:rows].double() * dact[:rows].double(), x[:rows].double(), w.double()
        rel, ut = LEFT_OUT[dtype], torch.finfo(dtype).eps / 2
        for name, got, want, size, r in (("x", xb, zb @ W, zb.abs() @ W.abs(), n), ("w", wb, zb.t() @ X, zb.abs().t() @ X.abs(), rows)):
            within(name, got, want, (rel + (2 * r + 8) * U32) * size + 1.01 * ut * want.abs() + LOWEST[dtype])
            # ... and the rms error is that of rounding exact values to the type, up to a twentieth
            own = (got.double() - want).norm() / want.norm()
            alone = (want.to(dtype).double() - want).norm() / want.norm()
            assert dtype == torch.float32 or float(own) <= 1.05 * float(alone), (name, rows, float(own), float(alone))


@pytest.mark.parametrize("dtype", DT, ids=IDS)
@pytest.mark.parametrize("m", [3, 200])
def test_relu_passes_gradients_of_arguments_that_round_to_zero(m, dtype):
    """z = 2^-26 is positive, y = relu(z) is 0 in float16: the gradient passes all the same, with a residual and without."""
    x, w = torch.full((m, 16), 2.0 ** -15, dtype=dtype, device="cuda"), torch.full((24, 16), 2.0 ** -15, dtype=dtype, device="cuda")
    w[12:] = -w[12:]
    yb = torch.randn(m, 24, generator=gen(2), device="cuda").to(dtype)
    zero = torch.zeros(m, 24, dtype=dtype, device="cuda")
    plain, beside = (ops.linear_train_forward(x, w, None, r, "relu") for r in (None, zero))
    if dtype == torch.float16:
        assert not plain[0].any()
    on = torch.where(torch.arange(24, device="cuda") < 12, yb, torch.zeros_like(yb))
    for _, mask in (plain, beside):
        xb, wb, bb = ops.linear_backward(yb, x, w, mask, "relu")
        check_gradients(xb, wb, bb, on.double(), x, w, dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]
    grads = torch.autograd.grad(layers.linear(*leaves, activation="relu"), leaves, yb)
    check_gradients(*grads, None, on.double(), x, w, dtype)


def test_many_rows_past_32_bits():
    """2^31 elements and more behind one operand with many rows: the last of 600 000 rows of 4 100 elements, bit for bit what the same rows
    give by themselves in a launch of as many tiles, and within the bound of a bfloat16 product."""
    m, ld, k, n = 600000, 4100, 96, 40
    big = torch.zeros(m, ld, dtype=torch.bfloat16, device="cuda")
    assert big.numel() > 2 ** 31
    g = gen(1)
    x = big[:, 2000:2000 + k]
    x.copy_(torch.randn(m, k, generator=g, device="cuda"))
    w = torch.randn(n, k, generator=g, device="cuda").bfloat16()
    y = ops.linear(x, w)
    assert torch.equal(y, ops.linear(x.contiguous(), w))
    want, size = x[-300:].double() @ w.double().t(), x[-300:].double().abs() @ w.double().abs().t()
    within("y", y[-300:], want, (k + 8) * U32 * size + 1.01 * 2.0 ** -8 * want.abs())
    yb = torch.randn(m, n, generator=g, device="cuda").bfloat16()
    _, wb, _ = ops.linear_backward(yb, x, w, None)
    want, size = yb.double().t() @ x.double(), yb.double().abs().t() @ x.double().abs()
    within("w", wb, want, (m + 8) * U32 * size + 1.01 * 2.0 ** -8 * want.abs())


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -112, 2.0 ** -120, 2.0 ** -126])
def test_float32_products_of_very_small_numbers(scale):
    """The three bfloat16 parts of a float32 number end at 2^-133, bfloat16's smallest: what they leave out of x is at most 2^-134, below
    2^-25 of it down to 2^-109, and each product misses at most that times |w|."""
    g = gen(6)
    m, k, n = 300, 200, 140
    x, w = torch.randn(m, k, generator=g, device="cuda") * scale, torch.randn(n, k, generator=g, device="cuda")
    X, W = x.double(), w.double()
    size = X.abs() @ W.abs().t()
    bound = (k + 8) * U32 * size + 2.0 ** -134 * W.abs().sum(1) + k * 2.0 ** -149
    within("y", ops.linear(x, w), X @ W.t(), bound)
