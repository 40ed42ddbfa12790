"""The fused query/key norm and rotation (RopeTable, QkNormRope): the float form against its formula in 64
bits, the Q30 form bit for bit against the oracle's RmsNormPerHead and ApplyRoPE, and the operators of a
block run together.

Tolerances of the float form, from the arithmetic: the sum of hd squares in fp32 is off by at most
hd 2^-24 of itself (half of that in its root), the division, root, products, table entries and the
rotation's two terms by a dozen roundings, so a rotated value is off by at most
(hd / 2 + 12) 2^-24 (|u_p| + |u_{p+h}|) before the last rounding, half a step of the type.
"""
import math

import numpy as np
import pytest

import spatialdb_b200 as slx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
TYPES = {"f32": (slx.DTYPE_F32, torch.float32), "f16": (slx.DTYPE_F16, torch.float16), "bf16": (slx.DTYPE_BF16, torch.bfloat16)}
ONE = float(1 << 30)


@pytest.fixture(scope="module")
def ctx():
    return slx.Context(0)


def heads64(x, hd, rot, base, pos, w, eps, dt):
    """(y, tolerance) in float64 for rows x [M][heads * hd]."""
    v = x.double().reshape(x.shape[0], -1, hd)
    if w is not None:
        v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    h = rot // 2
    theta = torch.tensor([base ** (-2.0 * i / rot) for i in range(h)], dtype=torch.float64, device="cuda")
    a = (pos.double()[:, None] * theta)[:, None, :]
    p, q = v[..., :h], v[..., h:rot]
    y = torch.cat([p * a.cos() - q * a.sin(), p * a.sin() + q * a.cos(), v[..., rot:]], -1)
    s = p.abs() + q.abs()
    e = (hd / 2 + 12) * 2.0 ** -24 * torch.cat([s, s, v[..., rot:].abs()], -1)
    e = e + torch.finfo(dt).eps / 2 * (y.abs() + e) + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -126)
    return y.reshape(x.shape), e.reshape(x.shape)


class Case:
    def __init__(self, ctx, dtype, M, H, KV, hd, rot=None, rows=64, base=10000.0, norm=(True, True), pad=0, fused=False,
                 pos=None, T=0, eps=1e-6, seed=0):
        self.code, self.dt = TYPES[dtype]
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed + M * 31 + hd)
        self.M, self.H, self.KV, self.hd, self.rot, self.base, self.eps, self.T = M, H, KV, hd, rot or hd, base, eps, T
        nq, nk = H * hd, KV * hd
        if fused:
            x = torch.randn(M, nq + 2 * nk + pad, generator=gen, device="cuda").to(self.dt)
            self.q, self.k = x[:, :nq], x[:, nq:nq + nk]
        else:
            self.q = torch.randn(M, nq + pad, generator=gen, device="cuda").to(self.dt)[:, :nq]
            self.k = torch.randn(M, nk + pad, generator=gen, device="cuda").to(self.dt)[:, :nk]
        self.w = [1 + 0.3 * torch.randn(hd, generator=gen, device="cuda") if n else None for n in norm]
        self.pos = pos
        self.at = pos.clamp_min(0).long() if pos is not None else torch.arange(M, device="cuda") % (T or M)
        torch.cuda.synchronize()
        self.table = slx.RopeTable(rows, self.rot, base, ctx=ctx)
        self.op = slx.QkNormRope(self.table, self.code, H, KV, hd, *[w.data_ptr() if w is not None else 0 for w in self.w], eps=eps)
        self.qo = torch.full((M, nq + pad), 7.0, dtype=self.dt, device="cuda")
        self.ko = torch.full((M, nk + pad), 7.0, dtype=self.dt, device="cuda")
        torch.cuda.synchronize()

    def run(self, qo=None, ko=None, stream=slx.STREAM_LEGACY):
        qo, ko = self.qo if qo is None else qo, self.ko if ko is None else ko
        self.op.apply_device(self.q.data_ptr(), self.k.data_ptr(), self.M, qo.data_ptr(), ko.data_ptr(), T=self.T,
                             d_pos=0 if self.pos is None else self.pos.data_ptr(), ldq=self.q.stride(0), ldk=self.k.stride(0),
                             ldqo=qo.stride(0), ldko=ko.stride(0), stream=stream)
        return qo[:, : self.H * self.hd], ko[:, : self.KV * self.hd]

    def want(self):
        return [heads64(x, self.hd, self.rot, self.base, self.at, w, self.eps, self.dt) for x, w in zip((self.q, self.k), self.w)]

    def check(self, got=None):
        got = got or self.run()
        self.op.ctx.status(slx.STREAM_LEGACY)
        for g, (y, e) in zip(got, self.want()):
            d = (g.double() - y).abs()
            assert bool((d <= e).all()), f"worst {float((d / e).max())} of the tolerance"


LAYOUTS = [(1, 8, 1, 256, None), (1, 1, 1, 2, None), (2, 3, 1, 16, None), (3, 12, 12, 64, None), (5, 4, 2, 6, None), (7, 2, 2, 80, 32),
           (9, 20, 4, 96, 64), (10, 5, 1, 128, 2), (11, 3, 3, 130, 100), (13, 2, 1, 512, None), (4, 2, 1, 1000, 998),
           (17, 32, 8, 128, None), (64, 6, 2, 32, 16), (33, 2, 2, 48, 24), (6, 1, 1, 2048, 64)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,H,KV,hd,rot", LAYOUTS)
def test_float_layouts(ctx, dtype, M, H, KV, hd, rot):
    Case(ctx, dtype, M, H, KV, hd, rot).check()
    Case(ctx, dtype, M, H, KV, hd, rot, norm=(True, False), fused=True, pad=3).check()
    Case(ctx, dtype, M, H, KV, hd, rot, norm=(False, True), fused=True, T=3).check()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("H,KV", [(4, 0), (0, 3)])
def test_one_side_only(ctx, dtype, H, KV):
    Case(ctx, dtype, 9, H, KV, 64, T=4).check()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_many_rows(ctx, dtype):
    """Enough rows that a group of lanes walks several heads."""
    Case(ctx, dtype, 5000, 16, 4, 64, rows=1250, T=1250).check()
    Case(ctx, dtype, 4001, 7, 1, 96, rot=32, rows=4001, fused=True).check()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_far_positions(ctx, dtype):
    pos = torch.tensor([0, 1, 99999, 131071, 65536, 131070], dtype=torch.int32, device="cuda")
    Case(ctx, dtype, 6, 2, 1, 128, rows=131072, base=500000.0, pos=pos).check()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("hd,pad", [(64, 0), (66, 5)])
def test_in_place(ctx, dtype, hd, pad):
    c = Case(ctx, dtype, 21, 4, 2, hd, fused=True, pad=pad)
    ref = [t.clone() for t in c.run()]
    want = c.want()
    got = c.run(qo=c.q, ko=c.k)
    torch.cuda.synchronize()
    for g, r, (y, e) in zip(got, ref, want):
        assert torch.equal(g, r)
        assert bool(((g.double() - y).abs() <= e).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("hd", [64, 70])
def test_rows_left_alone(ctx, dtype, hd):
    """Padding rows (position -1) and the elements between rows keep what they held; a position outside
    the table does too, and is reported once."""
    pos = torch.tensor([3, -1, 0, 63, -1, 5, 5], dtype=torch.int32, device="cuda")
    c = Case(ctx, dtype, 7, 2, 1, hd, pos=pos, pad=4)
    q, k = c.run()
    ctx.status(slx.STREAM_LEGACY)
    for g, (y, e), o in zip((q, k), c.want(), (c.qo, c.ko)):
        live = pos >= 0
        assert bool(((g.double() - y).abs() <= e)[live].all())
        assert bool((g[~live] == 7).all()) and bool((o[:, g.shape[1]:] == 7).all())
    for bad in (64, -2, 2 ** 31 - 1, -2 ** 31):
        c.qo.fill_(7)
        pos[2] = bad
        c.run()
        with pytest.raises(slx.IndexOutOfRangeError):
            ctx.status(slx.STREAM_LEGACY)
        ctx.status(slx.STREAM_LEGACY)
        assert bool((c.qo[2] == 7).all()) and bool((c.qo[0, : 2 * hd] != 7).all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_zero_heads_and_nan_rows(ctx, dtype):
    c = Case(ctx, dtype, 6, 3, 2, 64)
    c.q[1] = 0
    c.check()  # 0 / sqrt(eps)
    clean = c.run()[0].clone()
    c.q[4, 64:128] = float("nan")
    got = c.run()[0]
    assert bool(got[4, 64:128].isnan().all())
    got[4, 64:128] = clean[4, 64:128]
    assert torch.equal(got, clean)


def q30_rows(rng, m, n, mag):
    return rng.integers(-mag, mag, (m, n), dtype=np.int64)


def q30_want(oracle, x, heads, hd, w, pos, rows, base):
    """RmsNormPerHead, then ApplyRoPE at the given positions."""
    M = x.shape[0]
    y = x.copy()
    if w is not None:
        y = oracle.rmsnorm_per_head(y, M, heads, hd, w).reshape(M, heads * hd)
    out = np.empty_like(y)
    for m in range(M):  # ApplyRoPE rotates row t of a sequence at position t
        seq = np.zeros((pos[m] + 1, heads * hd), np.int64)
        seq[-1] = y[m]
        out[m] = oracle.apply_rope(seq, pos[m] + 1, heads * hd, heads, rows, hd, base).reshape(pos[m] + 1, -1)[-1]
    return out


@pytest.mark.parametrize("M,H,KV,hd", [(1, 8, 1, 256), (5, 2, 2, 2), (7, 4, 2, 32), (9, 3, 1, 66), (6, 2, 1, 130), (5, 1, 1, 512),
                                       (3, 2, 1, 600), (12, 12, 12, 64)])
@pytest.mark.parametrize("mag", [4, 1 << 31, 1 << 36, (1 << 62) - 1])
def test_q30_matches_oracle(ctx, oracle, M, H, KV, hd, mag):
    rng = np.random.default_rng(M * 7 + hd + mag % 1009)
    rows, base = 40, 10000.0
    q, k = q30_rows(rng, M, H * hd, mag), q30_rows(rng, M, KV * hd, mag)
    q[0, :hd] = 0  # a row the norm leaves as it is
    wq, wk = q30_rows(rng, 1, hd, 1 << 31)[0], q30_rows(rng, 1, hd, 1 << 31)[0]
    pos = rng.integers(0, rows, M).astype(np.int32)
    table = slx.RopeTable(rows, hd, base, q30=True, ctx=ctx)
    dq, dk, dwq, dwk, dp = (torch.from_numpy(a.copy()).cuda() for a in (q, k, wq, wk, pos))
    torch.cuda.synchronize()
    for norm in ((True, True), (False, True)):
        op = slx.QkNormRope(table, slx.DTYPE_Q30, H, KV, hd, dwq.data_ptr() if norm[0] else 0, dwk.data_ptr() if norm[1] else 0)
        qo, ko = torch.empty_like(dq), torch.empty_like(dk)
        op.apply_device(dq.data_ptr(), dk.data_ptr(), M, qo.data_ptr(), ko.data_ptr(), d_pos=dp.data_ptr(), stream=slx.STREAM_LEGACY)
        ctx.status(slx.STREAM_LEGACY)
        np.testing.assert_array_equal(qo.cpu().numpy(), q30_want(oracle, q, H, hd, wq if norm[0] else None, pos, rows, base))
        np.testing.assert_array_equal(ko.cpu().numpy(), q30_want(oracle, k, KV, hd, wk if norm[1] else None, pos, rows, base))
    op.apply_device(dq.data_ptr(), dk.data_ptr(), M, dq.data_ptr(), dk.data_ptr(), d_pos=dp.data_ptr(), stream=slx.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(dq, qo) and torch.equal(dk, ko)  # in place


def test_streams_and_graph(ctx):
    cs = [Case(ctx, "bf16", 300, 8, 2, 128, T=100, rows=100, seed=i) for i in range(2)]
    firsts = [[t.clone() for t in c.run()] for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    for c, s in zip(cs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.run(stream=s.cuda_stream)
        c.graph = g
        c.qo.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                c.graph.replay()
    torch.cuda.synchronize()
    for c, f in zip(cs, firsts):
        assert torch.equal(c.qo, f[0]) and torch.equal(c.ko, f[1])


def test_refusals(ctx):
    def refused(status, fn, *a, **k):
        with pytest.raises(slx.SlxError) as e:
            fn(*a, **k)
        assert e.value.status == status

    for a in ((0, 64), (10, 0), (10, 63), (10, 64, 0.0), (10, 64, float("inf")), (10, 64, -1.0),
              (2 ** 31 - 1, 65536)):
        refused(slx.SLX_EINVAL, slx.RopeTable, *a, ctx=ctx)
    t, ti = slx.RopeTable(32, 64, ctx=ctx), slx.RopeTable(32, 64, q30=True, ctx=ctx)
    w = torch.ones(64, device="cuda")
    refused(slx.SLX_EUNSUPPORTED, slx.QkNormRope, t, 8, 2, 1, 64)
    for a, k in (((t, slx.DTYPE_Q30, 2, 1, 64), {}), ((ti, slx.DTYPE_F32, 2, 1, 64), {}), ((t, slx.DTYPE_F32, 0, 0, 64), {}),
                 ((t, slx.DTYPE_F32, -1, 1, 64), {}), ((t, slx.DTYPE_F32, 2, 1, 62), {}), ((ti, slx.DTYPE_Q30, 2, 1, 128), {}),
                 ((ti, slx.DTYPE_Q30, 2, 1, 64), {"eps": 1e-6}), ((t, slx.DTYPE_F32, 2, 1, 64), {"eps": -1.0}),
                 ((t, slx.DTYPE_F32, 2, 1, 64), {"d_wq": w.data_ptr() + 2})):
        refused(slx.SLX_EINVAL, slx.QkNormRope, *a, **k)
    c = Case(ctx, "bf16", 8, 2, 1, 64, rows=32)
    q, k, o, p = c.q.data_ptr(), c.k.data_ptr(), c.qo.data_ptr(), c.ko.data_ptr()
    ap = c.op.apply_device
    for a, kw in (((q, k, -1, o, p), {}), ((0, k, 8, o, p), {}), ((q, k, 8, o, 0), {}), ((q, k, 8, o, p), {"ldq": 127}),
                  ((q, k, 8, o, p), {"ldko": 63}), ((q + 1, k, 7, o, p), {}), ((q, k, 8, o, p), {"T": -3}),
                  ((q, k, 8, o, p), {"d_pos": q + 2}), ((q, k, 1 << 40, o, p), {"T": 1})):
        refused(slx.SLX_EINVAL, ap, *a, **kw)
    big = Case(ctx, "bf16", 40, 2, 1, 64, rows=64)
    big.op.close()
    refused(slx.SLX_ERANGE, c.op.apply_device, big.q.data_ptr(), big.k.data_ptr(), 40, big.qo.data_ptr(), big.ko.data_ptr())
    c.op.apply_device(0, 0, 0, 0, 0)
    c.check()


def test_table_and_context_freed_first():
    own = slx.Context(0)
    c = Case(own, "f32", 5, 2, 1, 64)
    c.table.close()
    lib, h = own._lib, c.op._h
    lib.slx_destroy(own._h)
    own._h = c.op._h = None
    a = (c.q.data_ptr(), 128, c.k.data_ptr(), 64, 5, 5, 0, c.qo.data_ptr(), 128, c.ko.data_ptr(), 64, slx.STREAM_LEGACY)
    assert lib.slx_qk_norm_rope_device(h, slx._QK_ARGS(*a)) == 0
    torch.cuda.synchronize()
    (y, e), _ = c.want()
    assert bool(((c.qo.double() - y).abs() <= e).all())
    assert lib.slx_qk_norm_free(h) == 0


@pytest.mark.parametrize("dtype,M,T", [("bf16", 70, 35), ("f32", 70, 35), ("f16", 4, 4), ("f32", 1, 1)])
def test_block_of_operators(ctx, dtype, M, T):
    """A transformer block's products, norms and rotation in a row, on one stream, against the block in 64
    bits: fused QKV with a bias, norms and rotation in place, attention (torch, 64 bits, rounded), output
    projection onto the residual, gated FFN and its down projection onto the residual.

    The block's roundings to the type happen at six places, each of at most eps / 2 of a value, and the
    maps between them have gains of a few units here; 64 eps of the output's largest value covers them."""
    code, dt = TYPES[dtype]
    H, KV, hd, d, F = 4, 2, 64, 192, 320
    gen = torch.Generator(device="cuda")
    gen.manual_seed(M)
    rnd = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=gen, device="cuda")).to(dt)  # noqa: E731
    n = (H + 2 * KV) * hd
    x = rnd(M, d)
    wqkv, wo = rnd(n, d, scale=d ** -0.5), rnd(d, H * hd, scale=(H * hd) ** -0.5)
    wg, wu, wd = rnd(F, d, scale=d ** -0.5), rnd(F, d, scale=d ** -0.5), rnd(d, F, scale=F ** -0.5)
    b = torch.randn(n, generator=gen, device="cuda") * 0.1
    nq, nk = (1 + 0.2 * torch.randn(hd, generator=gen, device="cuda") for _ in range(2))
    size = x.element_size()
    torch.cuda.synchronize()

    def linear(w, **k):
        return slx.Linear(code, w.data_ptr(), w.numel() * size, code, w.shape[0], w.shape[1], ctx=ctx, **k)

    ops = [linear(wqkv, d_bias=b.data_ptr()), linear(wo),
           linear(wu, d_gate=wg.data_ptr(), gate_bytes=wg.numel() * size, act=slx.ACT_SILU), linear(wd)]
    qk = slx.QkNormRope(slx.RopeTable(T, hd, ctx=ctx), code, H, KV, hd, nq.data_ptr(), nk.data_ptr(), eps=1e-6)

    def attention(q, k, v):
        q, k, v = (t.double().reshape(M // T, T, -1, hd).transpose(1, 2) for t in (q, k, v))
        k, v = (t.repeat_interleave(H // KV, 1) for t in (k, v))
        return (torch.softmax(q @ k.transpose(2, 3) / math.sqrt(hd), -1) @ v).transpose(1, 2).reshape(M, H * hd)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        s = stream.cuda_stream
        qkv, h, u, y = torch.empty(M, n, dtype=dt, device="cuda"), *(torch.empty(M, w, dtype=dt, device="cuda") for w in (d, F, d))
        ops[0].apply_device(x.data_ptr(), M, qkv.data_ptr(), stream=s)
        q, k, v = qkv[:, : H * hd], qkv[:, H * hd: (H + KV) * hd], qkv[:, (H + KV) * hd:]
        qk.apply_device(q.data_ptr(), k.data_ptr(), M, q.data_ptr(), k.data_ptr(), T=T, ldq=n, ldk=n, ldqo=n, ldko=n, stream=s)
        att = attention(q, k, v).to(dt)
        ops[1].apply_device(att.data_ptr(), M, h.data_ptr(), d_residual=x.data_ptr(), stream=s)
        ops[2].apply_device(h.data_ptr(), M, u.data_ptr(), stream=s)
        ops[3].apply_device(u.data_ptr(), M, y.data_ptr(), d_residual=h.data_ptr(), stream=s)
    ctx.status(stream.cuda_stream)
    X = x.double()
    ref = X @ wqkv.double().T + b.double()
    at = torch.arange(M, device="cuda") % T
    rq, _ = heads64(ref[:, : H * hd], hd, hd, 10000.0, at, nq, 1e-6, torch.float64)
    rk, _ = heads64(ref[:, H * hd: (H + KV) * hd], hd, hd, 10000.0, at, nk, 1e-6, torch.float64)
    r1 = attention(rq, rk, ref[:, (H + KV) * hd:]) @ wo.double().T + X
    g = r1 @ wg.double().T
    r2 = (g * torch.sigmoid(g) * (r1 @ wu.double().T)) @ wd.double().T + r1
    assert float((y.double() - r2).abs().max()) <= 64 * torch.finfo(dt).eps * float(r2.abs().max())
