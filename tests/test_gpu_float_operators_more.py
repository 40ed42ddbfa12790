"""Float operators beyond the sizes of their first tests: GGUF weights under f32 on every path, gated, and the Q30
norm and rotation of heads wider than a warp's registers."""
import numpy as np
import pytest

import spatialdb_b200 as slx
from spatialdb_b200 import synth
from test_gpu_linear import want
from test_gpu_qk_norm_rope import q30_rows, q30_want

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def ctx():
    return slx.Context(0)


def raw_weights(rng, dtype, n):
    if dtype == synth.Q8_0:
        raw = synth.random_q8_0(rng, n)
    elif dtype == synth.Q4_0:
        raw = synth.random_q4_0(rng, n)
    else:
        v = (rng.standard_normal(n) * 0.1).astype(np.float32)
        raw = v.astype(np.float16) if dtype == synth.F16 else (v.view(np.uint32) >> 16).astype(np.uint16)
    return np.frombuffer(np.ascontiguousarray(raw).tobytes(), np.uint8).copy()


@pytest.mark.parametrize("wdtype", [synth.Q8_0, synth.Q4_0, synth.F16, synth.BF16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [1, 4, 7, 16, 130, 2000])
def test_gguf_weights(ctx, oracle, wdtype, gated, M):
    rng = np.random.default_rng(wdtype * 100 + M)
    N, K = 330, 288
    raws = [raw_weights(rng, wdtype, N * K) for _ in range(1 + gated)]
    mats = [torch.from_numpy(oracle.dequantize(wdtype, r, N * K).reshape(N, K).copy()).cuda() for r in raws]
    bufs = [torch.from_numpy(r).cuda() for r in raws]
    x = torch.from_numpy(rng.standard_normal((M, K)).astype(np.float32)).cuda()
    y = torch.empty(M, N, device="cuda")
    torch.cuda.synchronize()
    op = slx.Linear(slx.DTYPE_F32, bufs[0].data_ptr(), raws[0].size, wdtype, N, K, act=slx.ACT_SILU,
                    d_gate=bufs[1].data_ptr() if gated else 0, gate_bytes=raws[1].size if gated else 0, ctx=ctx)
    del bufs
    op.apply_device(x.data_ptr(), M, y.data_ptr(), stream=slx.STREAM_LEGACY)
    ctx.status(slx.STREAM_LEGACY)
    ref, tol = want(x, mats[0], torch.float32, "silu", g=mats[1] if gated else None)
    assert bool(((y.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("hd", [514, 768, 1024, 2050])
@pytest.mark.parametrize("mag", [4, 1 << 31, 1 << 36, (1 << 62) - 1])
def test_q30_wide_heads(ctx, oracle, hd, mag):
    rng = np.random.default_rng(hd + mag % 1009)
    M, H, KV, rows, base = 4, 2, 1, 20, 10000.0
    q, k = q30_rows(rng, M, H * hd, mag), q30_rows(rng, M, KV * hd, mag)
    q[0, :hd] = 0  # a row the norm leaves as it is
    w = q30_rows(rng, 1, hd, 1 << 31)[0]
    pos = rng.integers(0, rows, M).astype(np.int32)
    dq, dk, dw, dp = (torch.from_numpy(a.copy()).cuda() for a in (q, k, w, pos))
    torch.cuda.synchronize()
    op = slx.QkNormRope(slx.RopeTable(rows, hd, base, q30=True, ctx=ctx), slx.DTYPE_Q30, H, KV, hd, dw.data_ptr(), 0)
    op.apply_device(dq.data_ptr(), dk.data_ptr(), M, dq.data_ptr(), dk.data_ptr(), d_pos=dp.data_ptr(), stream=slx.STREAM_LEGACY)
    ctx.status(slx.STREAM_LEGACY)
    np.testing.assert_array_equal(dq.cpu().numpy(), q30_want(oracle, q, H, hd, w, pos, rows, base))
    np.testing.assert_array_equal(dk.cpu().numpy(), q30_want(oracle, k, KV, hd, None, pos, rows, base))
