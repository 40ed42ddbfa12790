"""The float linear operator (Linear: slx_linear_prepare / slx_linear_device) against its formula in 64 bits.

Tolerances, per output, from the arithmetic. With S = sum_k |x_k w_k| (+ |b|), a sum of K terms formed in
fp32 in any order is off by at most (K + 2) 2^-24 S where additions round, twice that where the tensor
core truncates: e_v = (K + 16) 2^-23 S. An activation's slope is at most 1.13 and its evaluation in fp32 is
good to 16 roundings of |v|: e_a = 1.13 e_v + 2^-20 |v|. A gated product adds |g| e_u + |u| e_g + e_g e_u and
three roundings; the residual's sum one; the last rounding is half a step of the type,
eps / 2 |y| (f16: or half its smallest step below its normal range).
F32 on the tensor cores adds at most 16 partial products to an accumulator before it is promoted to
rounded sums, so relative to the result's 2-norm random data stay below 16 x 2^-23.
"""
import ctypes
import math

import numpy as np
import pytest

import spatialdb_b200 as slx
from spatialdb_b200 import _lib, synth

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
TYPES = {"f32": (slx.DTYPE_F32, torch.float32), "f16": (slx.DTYPE_F16, torch.float16), "bf16": (slx.DTYPE_BF16, torch.bfloat16)}
ACTS = {"none": slx.ACT_NONE, "relu": slx.ACT_RELU, "silu": slx.ACT_SILU, "gelu_tanh": slx.ACT_GELU_TANH,
        "gelu_erf": slx.ACT_GELU_ERF}


@pytest.fixture(scope="module")
def ctx():
    return slx.Context(0)


def act64(v, act):
    if act == "relu":
        return v.clamp_min(0)
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))
    if act == "gelu_erf":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    return v


def want(x, w, dt, act="none", b=None, g=None, gb=None, r=None):
    """(y, tolerance) in float64."""
    K = x.shape[1]
    x, w = x.double(), w.double()

    def product(w, b):
        v, s = x @ w.T, x.abs() @ w.abs().T
        if b is not None:
            v, s = v + b.double(), s + b.double().abs()
        return v, (K + 16) * 2.0 ** -23 * s

    u, eu = product(w, b)
    if g is None:
        y, e = act64(u, act), 1.13 * eu + 2.0 ** -20 * u.abs() if act != "none" else eu
    else:
        v, ev = product(g.double(), gb)
        a, ea = act64(v, act), 1.13 * ev + 2.0 ** -20 * v.abs()
        y, e = a * u, a.abs() * eu + u.abs() * ea + ea * eu + 3 * 2.0 ** -24 * (a * u).abs()
    if r is not None:
        y = y + r.double()
        e = e + 2.0 ** -24 * (y.abs() + e)
    e = e + torch.finfo(dt).eps / 2 * (y.abs() + e)
    return y, e + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -126)


def rows(gen, m, n, dt, pad=0, scale=1.0):
    t = (scale * torch.randn(m, n + pad, generator=gen, device="cuda")).to(dt)
    return t[:, :n]


class Case:
    def __init__(self, ctx, dtype, M, K, N, act="none", gated=False, bias=False, residual=False, pad=0, seed=0):
        self.code, self.dt = TYPES[dtype]
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed * 1000003 + M * 131 + K * 17 + N)
        self.M, self.K, self.N, self.act = M, K, N, act
        s = 1 / math.sqrt(K)
        self.x = rows(gen, M, K, self.dt, pad)
        self.w = rows(gen, N, K, self.dt, 0, s)
        self.g = rows(gen, N, K, self.dt, 0, s) if gated else None
        self.b = torch.randn(N, generator=gen, device="cuda") if bias else None
        self.gb = torch.randn(N, generator=gen, device="cuda") if bias and gated else None
        self.r = rows(gen, M, N, self.dt, pad) if residual else None
        self.y = torch.full((M, N + pad), 7.0, dtype=self.dt, device="cuda")
        at = lambda t: t.data_ptr() if t is not None else 0  # noqa: E731
        size = N * K * self.w.element_size()
        torch.cuda.synchronize()
        self.op = slx.Linear(self.code, at(self.w), size, self.code, N, K, d_bias=at(self.b), act=ACTS[act], d_gate=at(self.g),
                             gate_bytes=size if gated else 0, d_gate_bias=at(self.gb), ctx=ctx)
        torch.cuda.synchronize()

    def run(self, y=None, stream=slx.STREAM_LEGACY):
        y = self.y if y is None else y
        self.op.apply_device(self.x.data_ptr(), self.M, y.data_ptr(), ldx=self.x.stride(0), ldo=y.stride(0),
                             d_residual=self.r.data_ptr() if self.r is not None else 0,
                             ldr=self.r.stride(0) if self.r is not None else 0, stream=stream)
        return y[:, : self.N]

    def want(self):
        return want(self.x, self.w, self.dt, self.act, self.b, self.g, self.gb, self.r)

    def check(self, got=None):
        got = self.run() if got is None else got
        y, e = self.want()
        self.op.ctx.status(slx.STREAM_LEGACY)
        d = (got.double() - y).abs()
        assert bool((d <= e).all()), f"worst {float((d / e).max())} of the tolerance at {int((d / e).argmax())}"
        return got


# every tile width of the tensor-core kernel, clusters of 1..8, K blocks of 1 and more, N across tiles
SIZES = [(1, 1, 1), (1, 7, 5), (1, 768, 768), (2, 64, 16), (3, 65, 17), (4, 200, 129), (5, 1000, 40), (8, 256, 300), (9, 96, 128),
         (15, 1001, 33), (16, 512, 1000), (17, 31, 128), (17, 32, 1), (24, 2048, 130), (32, 64, 640), (33, 640, 256),
         (40, 1001, 1111), (64, 1024, 128), (65, 33, 257), (100, 300, 300), (128, 4096, 136), (129, 257, 127), (200, 512, 200),
         (257, 96, 3000), (300, 768, 768), (20, 1, 5), (200, 3, 300), (3000, 2, 700)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N", SIZES)
def test_product_and_epilogue(ctx, dtype, M, K, N):
    Case(ctx, dtype, M, K, N).check()
    Case(ctx, dtype, M, K, N, act="gelu_erf", bias=True, residual=True, pad=3).check()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N", [(1, 96, 40), (3, 257, 130), (8, 512, 64), (12, 64, 129), (20, 2048, 128), (32, 40, 65),
                                   (48, 640, 256), (64, 1000, 30), (65, 65, 257), (130, 512, 384), (300, 300, 1000)])
def test_gated(ctx, dtype, M, K, N):
    Case(ctx, dtype, M, K, N, act="silu", gated=True).check()
    Case(ctx, dtype, M, K, N, act="gelu_tanh", gated=True, bias=True, residual=True, pad=8).check()


@pytest.mark.parametrize("dtype,M,K,N,pad", [("bf16", 120, 1024, 9900, 0), ("f16", 128, 2048, 11008, 0), ("bf16", 77, 1111, 10001, 1),
                                             ("f16", 513, 640, 2050, 1), ("bf16", 600, 768, 2048, 0), ("bf16", 130, 512, 9600, 0),
                                             ("f16", 300, 200, 70, 0), ("f32", 512, 1024, 2050, 0), ("f32", 700, 333, 1300, 1)])
def test_gated_pairs(ctx, dtype, M, K, N, pad):
    """Gated products on pairs of CTAs: half of each array's rows a CTA, and whole blocks of both for one activation tile."""
    Case(ctx, dtype, M, K, N, act="silu", gated=True, bias=True, residual=True, pad=pad).check()
    Case(ctx, dtype, M, K, N, act="gelu_tanh", gated=True, pad=pad, seed=1).check()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("M", [2, 70])
def test_activations(ctx, dtype, act, M):
    c = Case(ctx, dtype, M, 128, 96, act=act, bias=True)
    c.x *= 4  # the activations' tails
    c.check()


@pytest.mark.parametrize("dtype,M,K,N", [("bf16", 2500, 512, 2304), ("f16", 1111, 768, 3000), ("f32", 1500, 512, 1500),
                                         ("bf16", 512, 2048, 6000), ("f32", 2000, 300, 1500), ("f16", 5001, 100, 1111),
                                         ("bf16", 300, 64, 10001), ("f32", 4099, 33, 1027)])
def test_persistent_tiles(ctx, dtype, M, K, N):
    """More tiles than SMs: every CTA, or pair of CTAs, walks several, the accumulators in turn."""
    Case(ctx, dtype, M, K, N, act="silu", bias=True, residual=True, pad=8).check()
    Case(ctx, dtype, M, K, N, act="silu", gated=True).check()


@pytest.mark.parametrize("dtype,M,K,N,gated,pad", [("f32", 20, 2048, 19000, False, 0), ("f32", 30, 1111, 19000, True, 1),
                                                   ("f32", 60, 1500, 19000, False, 0), ("f16", 31, 3001, 19000, False, 3),
                                                   ("bf16", 64, 2500, 19000, True, 1), ("bf16", 100, 4096, 18000, False, 0),
                                                   ("f32", 7, 2100, 4100, False, 0), ("f32", 5, 2100, 2500, True, 2),
                                                   ("f32", 13, 300, 1111, False, 0), ("f32", 16, 513, 40, True, 1),
                                                   ("bf16", 2100, 301, 200, False, 3), ("f16", 1500, 1111, 1300, True, 1)])
def test_long_sums_of_one_tile(ctx, dtype, M, K, N, gated, pad):
    """So many weight tiles that none is split over K: one CTA goes through every K block, its stages many
    times over, and in f32 through many promotions, with its rows loaded by TMA and by the epilogue's warps."""
    Case(ctx, dtype, M, K, N, act="silu" if gated else "none", gated=gated, pad=pad).check()


@pytest.mark.parametrize("M,K,N", [(64, 768, 512), (300, 2048, 640), (1000, 4096, 768), (20, 4096, 256), (4, 4096, 512)])
def test_f32_is_as_exact_as_fp32(ctx, M, K, N):
    c = Case(ctx, "f32", M, K, N)
    got = c.check().double()
    y, _ = c.want()
    assert float((got - y).norm() / y.norm()) <= 16 * 2.0 ** -23


@pytest.mark.parametrize("M", [3, 50, 200])
def test_f32_range(ctx, M):
    """Large and small magnitudes keep fp32's relative precision; values near the ends of the range neither
    overflow nor lose their leading part."""
    c = Case(ctx, "f32", M, 256, 100)
    c.x *= 2.0 ** torch.randint(-40, 40, (M, 1), device="cuda").float()
    c.check()
    c.x.fill_(0)
    c.x[:, 5] = 3.0e38
    w = torch.zeros_like(c.w)
    w[:, 5] = 0.5
    op = slx.Linear(c.code, w.data_ptr(), w.numel() * 4, c.code, c.N, c.K, ctx=ctx)
    op.apply_device(c.x.data_ptr(), M, c.y.data_ptr(), ldx=c.x.stride(0), ldo=c.y.stride(0), stream=slx.STREAM_LEGACY)
    torch.cuda.synchronize()
    np.testing.assert_allclose(c.y[:, : c.N].double().cpu().numpy(), 1.5e38, rtol=2.0 ** -22)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [1, 6, 40, 300])
def test_rows_stay_apart(ctx, dtype, M):
    """A NaN or an infinity in one row of x reaches that row's outputs alone, and the elements between the
    rows of y keep what they held."""
    c = Case(ctx, dtype, M, 200, 150, pad=6, residual=True)
    clean = c.run().clone()
    bad = M // 2
    c.x[bad, 3] = float("nan")
    got = c.run().clone()
    keep = torch.arange(M, device="cuda") != bad
    assert torch.equal(got[keep], clean[keep])
    assert bool(got[bad].isnan().all())
    c.x[bad, 3] = float("inf")
    got = c.run()
    assert torch.equal(got[keep], clean[keep])
    assert not bool(got[bad].isfinite().any())
    assert bool((c.y[:, c.N:] == 7).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [2, 30, 140])
def test_output_over_the_residual(ctx, dtype, M):
    c = Case(ctx, dtype, M, 300, 260, act="silu", bias=True, residual=True)
    first = c.run().clone()
    c.run(y=c.r)
    torch.cuda.synchronize()
    assert torch.equal(c.r, first)


@pytest.mark.parametrize("dtype,M,K,N", [("bf16", 8, 1024, 512), ("f32", 4, 2048, 96), ("f16", 33, 4096, 200), ("f32", 40, 2048, 200),
                                         ("bf16", 700, 512, 1024)])
def test_same_result_every_time(ctx, dtype, M, K, N):
    c = Case(ctx, dtype, M, K, N, bias=True)
    first = c.run().clone()
    for _ in range(5):
        assert torch.equal(c.run(), first)


@pytest.mark.parametrize("wdtype", [synth.Q8_0, synth.Q4_0, synth.F16, synth.BF16, synth.F32])
@pytest.mark.parametrize("M", [1, 50])
def test_gguf_weights_under_f32(ctx, oracle, wdtype, M):
    rng = np.random.default_rng(wdtype + M)
    N, K = 70, 160
    if wdtype == synth.Q8_0:
        raw = synth.random_q8_0(rng, N * K)
    elif wdtype == synth.Q4_0:
        raw = synth.random_q4_0(rng, N * K)
    else:
        v = (rng.standard_normal(N * K) * 0.1).astype(np.float32)
        raw = v if wdtype == synth.F32 else v.astype(np.float16) if wdtype == synth.F16 else (v.view(np.uint32) >> 16).astype(np.uint16)
    raw = np.frombuffer(np.ascontiguousarray(raw).tobytes(), np.uint8).copy()
    w = torch.from_numpy(oracle.dequantize(wdtype, raw, N * K).reshape(N, K).copy()).cuda()
    d_raw = torch.from_numpy(raw).cuda()
    x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda()
    y = torch.empty(M, N, device="cuda")
    torch.cuda.synchronize()
    op = slx.Linear(slx.DTYPE_F32, d_raw.data_ptr(), raw.size, wdtype, N, K, ctx=ctx)
    del d_raw
    op.apply_device(x.data_ptr(), M, y.data_ptr(), stream=slx.STREAM_LEGACY)
    ref, tol = want(x, w, torch.float32)
    assert bool(((y.double() - ref).abs() <= tol).all())


def test_streams_and_graphs(ctx):
    """Calls on two streams at once, and two captured graphs whose calls need scratch (f32, and rows TMA
    cannot address), replayed together with an eager call between them: nothing is shared."""
    cases = [Case(ctx, "f32", 3000, 512, 1000, bias=True), Case(ctx, "f32", 200, 384, 300, residual=True),
             Case(ctx, "bf16", 3000, 257, 600, pad=3), Case(ctx, "f16", 4, 512, 300, bias=True)]
    firsts = [c.run().clone() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        for c, s in zip(cases, streams):
            c.run(stream=s.cuda_stream)
    torch.cuda.synchronize()
    for c, f in zip(cases, firsts):
        assert torch.equal(c.y[:, : c.N], f)
    graphs = []
    for c, s in zip(cases, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.run(stream=s.cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for c in cases:
            c.y.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        cases[0].run(y=torch.empty_like(cases[0].y))
        torch.cuda.synchronize()
        for c, f in zip(cases, firsts):
            assert torch.equal(c.y[:, : c.N], f)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [1, 7, 24, 200, 3000])
def test_calls_that_feed_each_other(ctx, dtype, M):
    """y = A x, x = B y + x over and over without a pause: each call reads what the one before it wrote and
    writes what that one read. The same as with a synchronisation after every call."""
    a, b = Case(ctx, dtype, M, 384, 384, act="gelu_tanh", seed=1), Case(ctx, dtype, M, 384, 384, bias=True, seed=2)
    start = (a.x * 0.1).to(a.dt)

    def chain(pause):
        x, y = start.clone(), torch.empty_like(start)
        torch.cuda.synchronize()
        for _ in range(25):
            a.op.apply_device(x.data_ptr(), M, y.data_ptr(), stream=s.cuda_stream)
            if pause:
                torch.cuda.synchronize()
            b.op.apply_device(y.data_ptr(), M, x.data_ptr(), stream=s.cuda_stream)
            if pause:
                torch.cuda.synchronize()
            with torch.cuda.stream(s):
                x.mul_(0.4)
        torch.cuda.synchronize()
        return x, y

    s = torch.cuda.Stream()
    ref = chain(True)
    assert bool(ref[0].isfinite().all())
    for _ in range(3):
        got = chain(False)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_first_call_inside_a_capture():
    """A context whose first calls are captured: nothing they need is made inside the capture."""
    own = slx.Context(0)
    cases = [Case(own, "f32", 2500, 320, 900), Case(own, "f16", 1700, 333, 800, pad=1), Case(own, "bf16", 50, 96, 70)]
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        for c in cases:
            c.run(stream=s.cuda_stream)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        for c in cases:
            c.check(got=c.y[:, : c.N])
            c.y.fill_(7)
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("M", [1, 12, 40])
def test_infinite_weights(ctx, dtype, M):
    """An infinite weight makes its own output infinite where x is not zero, whatever the padding around it."""
    c = Case(ctx, dtype, M, 70, 20)
    c.x.abs_().add_(0.5)
    w = c.w.clone()
    w[7, 3] = float("inf")
    torch.cuda.synchronize()
    op = slx.Linear(c.code, w.data_ptr(), w.numel() * 2, c.code, 20, 70, ctx=ctx)
    op.apply_device(c.x.data_ptr(), M, c.y.data_ptr(), ldx=c.x.stride(0), stream=slx.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert bool((c.y[:, 7] == float("inf")).all()) and bool(c.y[:, torch.arange(20) != 7].isfinite().all())


def test_wait_that_gives_up_is_reported():
    """The tensor-core kernel's bounded waits: with its MMA warp idle and a short limit the call ends,
    the status is reported once, and the context computes the next call."""
    own = slx.Context(0)
    # one tile a cluster (rows by TMA, by the epilogue's warps) and pairs, gated with both arrays' rows in a tile and wide
    for dtype, M, K, N, gated in (("bf16", 40, 512, 128, False), ("f32", 40, 512, 256, False), ("f32", 3000, 512, 2000, False),
                                  ("bf16", 2000, 512, 3000, False), ("f16", 513, 512, 4096, True), ("f32", 513, 512, 4096, True),
                                  ("bf16", 128, 1024, 11008, True)):
        c = Case(own, dtype, M, K, N, act="silu" if gated else "none", gated=gated)
        own.set_option(slx.OPT_WAIT_LIMIT_CYCLES, 2_000_000)
        own.set_option(slx.OPT_TEST_STALL_MMA, 1)
        c.run()
        with pytest.raises(slx.SlxError) as e:
            own.status(slx.STREAM_LEGACY)
        assert e.value.status == slx.SLX_ETIMEOUT
        own.status(slx.STREAM_LEGACY)
        own.set_option(slx.OPT_TEST_STALL_MMA, 0)
        own.set_option(slx.OPT_WAIT_LIMIT_CYCLES, 0)
        c.check()


def test_wait_limit_counts_from_the_kernels_ahead():
    """A call queued behind one that runs several times as long as the wait limit: its own waits start when that
    one has ended. The long call is one weight tile whose sums (promoted every 256 values) wait briefly each."""
    own = slx.Context(0)
    long, short = Case(own, "f32", 17, 1 << 19, 128), Case(own, "f32", 40, 512, 256)
    own.set_option(slx.OPT_WAIT_LIMIT_CYCLES, 400_000)
    for _ in range(3):
        long.run()
        short.run()
    own.status(slx.STREAM_LEGACY)
    short.check()


def test_empty_and_profile(ctx):
    c = Case(ctx, "bf16", 20, 64, 64)
    c.op.apply_device(0, 0, 0)
    n = ctypes.c_int64(0)
    ctx.check(ctx._lib.slx_launch_count(ctx._h, ctypes.byref(n)))
    before = n.value
    c.check()
    ctx.check(ctx._lib.slx_launch_count(ctx._h, ctypes.byref(n)))
    assert n.value == before + 1


def test_refusals(ctx):
    w = torch.zeros(64 * 64, device="cuda")
    b = torch.zeros(64, device="cuda")
    p = w.data_ptr()

    def refused(status, *a, **k):
        with pytest.raises(slx.SlxError) as e:
            slx.Linear(*a, ctx=ctx, **k)
        assert e.value.status == status

    f32, f16 = slx.DTYPE_F32, slx.DTYPE_F16
    refused(slx.SLX_EINVAL, f32, 0, 64 * 64 * 4, f32, 64, 64)
    refused(slx.SLX_EINVAL, f32, p, 64 * 64 * 4, f32, 0, 64)
    refused(slx.SLX_EINVAL, f32, p, 64 * 64 * 4, f32, 64, -1)
    refused(slx.SLX_EINVAL, f32, p, 64 * 64 * 4, f32, 64, 64, act=9)
    refused(slx.SLX_EINVAL, f32, p, 64 * 64 * 4, f32, 64, 64, d_gate_bias=b.data_ptr())
    refused(slx.SLX_EINVAL, f32, p + 2, 63 * 64 * 4, f32, 63, 64)
    refused(slx.SLX_EINVAL, f32, p, 64 * 64 * 4, f32, 64, 64, d_bias=b.data_ptr() + 1)
    refused(slx.SLX_EEOF, f32, p, 64 * 64 * 4 - 1, f32, 64, 64)
    refused(slx.SLX_EUNSUPPORTED, slx.DTYPE_Q30, p, 64 * 64 * 4, f32, 64, 64)
    refused(slx.SLX_EUNSUPPORTED, f16, p, 64 * 64 * 4, f32, 64, 64)
    refused(slx.SLX_EUNSUPPORTED, f32, p, 64 * 64 * 4, 99, 64, 64)
    c = Case(ctx, "f16", 20, 64, 64)
    x, y = c.x.data_ptr(), c.y.data_ptr()
    for a, k in (((x, -1, y), {}), ((0, 20, y), {}), ((x, 20, 0), {}), ((x, 20, y), {"ldx": 63}), ((x, 20, y), {"ldo": 63}),
                 ((x, 20, y), {"d_residual": y, "ldr": 63}), ((x + 1, 19, y), {}), ((x, 20, y + 1), {}), ((x, 1 << 31, y), {})):
        with pytest.raises(slx.SlxError) as e:
            c.op.apply_device(*a, **k)
        assert e.value.status == slx.SLX_EINVAL
    c.check()


def test_failed_allocation_is_reported_once(ctx):
    """Weights no device holds: the allocation's failure ends that call alone. (The buffer is not read.)"""
    w = torch.zeros(64, dtype=torch.float16, device="cuda")
    n = 1 << 21
    for dtype, size in ((slx.DTYPE_F32, 2), (slx.DTYPE_F16, 2)):
        with pytest.raises(slx.SlxError) as e:
            slx.Linear(dtype, w.data_ptr(), n * n * size, slx.DTYPE_F16, n, n, ctx=ctx)
        assert e.value.status == slx.SLX_EOOM
        Case(ctx, "f32", 20, 64, 64).check()


def test_handle_outlives_its_context():
    own = slx.Context(0)
    c = Case(own, "bf16", 20, 64, 64)
    lib, h = own._lib, c.op._h
    lib.slx_destroy(own._h)
    own._h = None
    c.op._h = None
    assert lib.slx_linear_device(h, slx._LINEAR_ARGS(c.x.data_ptr(), 64, 20, 0, 64, c.y.data_ptr(), 64, slx.STREAM_LEGACY)) == 0
    torch.cuda.synchronize()
    y, e = c.want()
    assert bool(((c.y.double() - y).abs() <= e).all())
    assert lib.slx_linear_free(h) == 0
