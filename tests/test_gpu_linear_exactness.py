"""What the float linear operator's results hold at the ends of their range, against the formula in 64 bits: the
three-part split of f32 products, infinities in them, the activations' tails. Each tolerance is relative to the
output and derived beside its test."""
import math

import pytest

import spatialdb_b200 as slx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
TYPES = {"f32": (slx.DTYPE_F32, torch.float32), "f16": (slx.DTYPE_F16, torch.float16), "bf16": (slx.DTYPE_BF16, torch.bfloat16)}
ACTS = {"silu": slx.ACT_SILU, "gelu_tanh": slx.ACT_GELU_TANH, "gelu_erf": slx.ACT_GELU_ERF}


@pytest.fixture(scope="module")
def ctx():
    return slx.Context(0)


def linear(ctx, x, w, dtype, act=0, gate=None):
    """act(x . w^T), or with gate weights act(x . gate^T) * (x . w^T)."""
    code, dt = TYPES[dtype]
    size = w.numel() * w.element_size()
    torch.cuda.synchronize()
    op = slx.Linear(code, w.data_ptr(), size, code, *w.shape, act=act, d_gate=gate.data_ptr() if gate is not None else 0,
                    gate_bytes=size if gate is not None else 0, ctx=ctx)
    y = torch.full((x.shape[0], w.shape[0]), 7.0, dtype=dt, device="cuda")
    op.apply_device(x.data_ptr(), x.shape[0], y.data_ptr(), ldx=x.stride(0), stream=slx.STREAM_LEGACY)
    ctx.status(slx.STREAM_LEGACY)
    return y


# ---- f32 products from three bf16 parts ----------------------------------------------------------------


@pytest.mark.parametrize("value", [1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -8 - 2.0 ** -23, 1 + 2.0 ** -8 + 2.0 ** -16, 1.9999999,
                                   1 + 2.0 ** -9 + 2.0 ** -17])
@pytest.mark.parametrize("M", [40, 600])
@pytest.mark.parametrize("K", [1, 16, 32, 256, 768, 4096])
def test_f32_products_of_one_sign(ctx, M, K, value):
    """Operands of one sign, where what the split leaves out and what the tensor core cuts off only add up. Parts
    rounded to nearest are at most 2^-8 and 2^-16 of the value, so x2 w3 + x3 w2 + x3 w3, left out, is at
    most (2 + 2^-8) 2^-24 of a product. An addition takes 16 products into an accumulator, which is promoted every 256
    values of K; it aligns them to the largest term, keeps 25 bits of each and 24 of the sum. Products of 8-bit parts of
    like size keep all their 16 bits beside a sum of up to 256 of them, so each addition of x1 w1 after the first (which
    adds to nothing) cuts off less than 2^-23 of the sum. The corrections, at most 2^-6.9 of it, lose up to 16 x 2^-25 + 2^-23
    of themselves in each of five times as many additions: 0.21 x 2^-23 of the sum for 16 values. Two roundings to promote
    the first 256 values, one more for each further 256."""
    x = torch.full((M, K), value, device="cuda")
    w = torch.full((130, K), value, device="cuda")
    x[1::2] *= -0.75  # whole rows: every sum keeps one sign
    w[1::3] *= 1.25
    y = linear(ctx, x, w, "f32").double()
    want = x.double() @ w.double().T
    steps = min(-(-K // 16), 16) - 1
    tol = (2 + 2.0 ** -8 + 2 * (steps + 0.21 * (steps + 1)) + 2 + K / 256) * 2.0 ** -24
    worst = float(((y - want).abs() / want.abs()).max())
    assert worst <= tol, f"{worst * 2 ** 24} of {tol * 2 ** 24} in units of 2^-24"


@pytest.mark.parametrize("M", [20, 300])
def test_f32_parts_near_the_largest_value(ctx, M):
    """A value whose leading part would round to infinity keeps a finite one."""
    top = torch.finfo(torch.float32).max
    x = torch.tensor([top, -top, top * (1 - 2.0 ** -9), 3.3961775e38], device="cuda").repeat(M // 4)[:, None].contiguous()
    w = torch.tensor([1.0, 0.5, -0.25, 2.0 ** -100, 1 - 2.0 ** -24], device="cuda")[:, None].contiguous()
    y = linear(ctx, x, w, "f32").double()
    want = x.double() @ w.double().T
    assert bool(y.isfinite().all())
    assert float(((y - want).abs() / want.abs()).max()) <= 2.0 ** -21  # cut at the top of the range: 2^-7, 2^-15 parts


# ---- infinities ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("K,exact16", [(200, True), (200, False), (700, True)])
@pytest.mark.parametrize("M", [1, 3, 6, 12, 40, 300, 2000])
def test_f32_infinities(ctx, M, K, exact16, gated):
    """Infinities and NaN in x and w end where fp32 arithmetic takes them, whichever kernel a call's sizes pick: an
    infinity of the product's sign, NaN against a zero or an infinity of the other sign. Weights that are exact in
    bf16 have zeros for their second and third parts."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(M + K)
    x = torch.randn(M, K, generator=gen, device="cuda")
    w = torch.randn(150, K, generator=gen, device="cuda") / math.sqrt(K)
    g = torch.rand(150, K, generator=gen, device="cuda") if gated else None
    if exact16:
        x, w = x.bfloat16().float(), w.bfloat16().float()
    inf, nan = float("inf"), float("nan")
    x[M // 2, K // 2] = inf
    x[M // 3, 5] = -inf
    w[4, K // 2] = 0.0
    w[9, 6] = inf
    w[11, 5] = -inf
    w[20, 1] = nan
    if M > 3:
        x[M - 1, 2], x[M - 1, K - 1] = inf, inf
        x[0, 3] = nan
    y = linear(ctx, x, w, "f32", act=slx.ACT_RELU if gated else 0, gate=g)

    def product(w):
        p, kinds = x.double()[:, None, :] * w.double()[None], (inf, -inf)
        up, down = ((p == k).any(-1) for k in kinds)
        s = torch.where(p.isfinite(), p, 0.0).sum(-1)
        s = torch.where(up, inf, torch.where(down, -inf, s))
        return torch.where(p.isnan().any(-1) | (up & down), nan, s)

    want = product(w)
    if gated:
        v = product(g)
        want = torch.where(v < 0, 0.0, v) * want  # a NaN stays one
    odd = ~want.isfinite()
    assert int(odd.sum()) >= 150
    assert torch.equal(y.isnan(), want.isnan())
    inf_at = want.isinf()
    assert torch.equal(y[inf_at].double(), want[inf_at])
    assert bool(y[~odd].isfinite().all())


# ---- activations ---------------------------------------------------------------------------------------


def act64(v, act):
    """Each activation as v times its factor, the factor formed without cancellation."""
    if act == "silu":
        return v * torch.special.expit(v)
    if act == "gelu_tanh":
        return v * torch.special.expit(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [1, 12, 40, 700])
def test_activation_tails(ctx, dtype, act, M):
    """act(v) for v given exactly (K = 1, x = 1), held to a tolerance relative to the output, so that the negative
    tails, where it is small, count as much as the rest. With u = 2^-24:

    The exponential of s (s = v, or GELU-tanh's 2 sqrt(2 / pi) (v + 0.044715 v^3)): CUDA's expf is good to 2 units of its
    last place (4 u), __expf, which 16-bit outputs may take, to 2 + 1.173 |s| units, 2 u each; s itself is off by two
    rounded constants and four roundings, 5 u at most, which the exponential makes 5 u |s|. Sum, quotient (its fast form: two
    units), product: 6 u.

    GELU-erf's tail is v e^(-v^2 / 2) t P(t) with t = 1 / (1 + a z). The exponent is off by one rounding, v^2 / 2 u of the
    exponential, itself 4 u or (2 + 1.173 v^2 / 2) 2 u. t is off by 3.5 u (z 1.5, sum and quotient; a hardware reciprocal
    1 more), of which t P(t) makes at most 3.8 times as much (its logarithm's slope in log t, erfc's 2 / sqrt(pi) over
    a = 0.3 at z = 0, falling to 1). Horner's steps: the terms' sizes add up to 2.5 P(t) at most, three roundings each: 7.5 u. P
    itself: u / 2 in f32, 2^-17.5 = 91 u for 16-bit outputs. Products 3 u. Together (28.3 + v^2 / 2) u and
    (91 + 32 + 1.7 v^2) u. Above zero v (1 - tail) is better than that.

    Then half a step of the type, and below its normal range half its smallest step (f32: |v| times it, and whole: the
    exponential itself lies there)."""
    code, dt = TYPES[dtype]
    v = torch.cat([torch.linspace(-14, 14, 2801), torch.linspace(-104, -13, 911), torch.linspace(14, 100, 44),
                   torch.tensor([0.0, -0.0, 1e-30, -1e-30, 6e4, -6e4, 2.0 ** -14, -(2.0 ** -14)])]).to(dt).cuda()
    if dtype != "f16":
        v = torch.cat([v, torch.tensor([3e38, -3e38, 1e19, -1e19, 2e13, -2e13], device="cuda").to(dt)])
    y = linear(ctx, torch.ones(M, 1, dtype=dt, device="cuda"), v[:, None].contiguous(), dtype, act=ACTS[act])
    assert torch.equal(y, y[:1].expand_as(y))
    a = v.double()
    want, u = act64(a, act), 2.0 ** -24
    s = (a if act == "silu" else 2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)).abs().clamp_max(105)
    if act == "gelu_erf":
        sq = a.square().clamp_max(220)
        rel = (28.3 + sq / 2 if dtype == "f32" else 91 + 32 + 1.7 * sq) * u
    else:
        rel = ((5 * s if act == "gelu_tanh" else 0) + (4 if dtype == "f32" else 2 * (2 + 1.173 * s)) + 6) * u
    least = {"f32": 2.0 ** -149 * (a.abs().clamp_max(105) + 1), "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[dtype]
    tol = rel * want.abs()
    tol = tol + torch.finfo(dt).eps / 2 * (want.abs() + tol) * (dtype != "f32") + least
    d = (y[0].double() - want).abs()
    at = int((d / tol).argmax())
    assert bool((d <= tol).all()), f"act({float(a[at])}) = {float(y[0, at])}, {float(want[at])} wanted: {float(d[at] / tol[at])} of the tolerance"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [2, 40])
def test_activations_of_what_is_not_finite(ctx, dtype, act, M):
    """+infinity is kept, a NaN stays one, and -infinity is the formula's -infinity times zero."""
    code, dt = TYPES[dtype]
    w = torch.tensor([float("inf"), -float("inf"), float("nan"), 1.0], device="cuda").to(dt)[:, None].contiguous()
    y = linear(ctx, torch.ones(M, 1, dtype=dt, device="cuda"), w, dtype, act=ACTS[act])
    assert bool((y[:, 0] == float("inf")).all()) and bool(y[:, 1:3].isnan().all()) and bool(y[:, 3].isfinite().all())
