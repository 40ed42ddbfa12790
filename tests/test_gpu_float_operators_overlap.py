"""Calls of the float operators whose rows share memory: outputs over inputs that other blocks still read are refused,
rows that only lie between one another are computed."""
import pytest

import spatialdb_b200 as slx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
F16 = torch.float16


@pytest.fixture(scope="module")
def ctx():
    return slx.Context(0)


def refused(fn, *a, **k):
    with pytest.raises(slx.SlxError) as e:
        fn(*a, **k)
    assert e.value.status == slx.SLX_EINVAL


@pytest.mark.parametrize("M", [1, 5, 40])
def test_linear(ctx, M):
    w = (torch.randn(64, 64, device="cuda") / 8).to(F16)
    x = torch.randn(M, 64, device="cuda").to(F16)
    torch.cuda.synchronize()
    op = slx.Linear(slx.DTYPE_F16, w.data_ptr(), w.numel() * 2, slx.DTYPE_F16, 64, 64, ctx=ctx)
    y = torch.empty_like(x)
    op.apply_device(x.data_ptr(), M, y.data_ptr(), d_residual=x.data_ptr(), stream=slx.STREAM_LEGACY)
    kept = x.clone()
    p = x.data_ptr()
    refused(op.apply_device, p, M, p)  # y over x
    refused(op.apply_device, p, M, p, d_residual=p)  # x is the residual too
    refused(op.apply_device, p, M, p + 2 * 63)
    refused(op.apply_device, p, M, y.data_ptr(), d_residual=y.data_ptr() + 2)
    if M > 1:
        refused(op.apply_device, p, M - 1, y.data_ptr(), d_residual=y.data_ptr(), ldr=128)
        refused(op.apply_device, p, M, p + 2 * 64 * (M - 1))  # the last row alone
    torch.cuda.synchronize()
    assert torch.equal(x, kept)
    buf = torch.full((M, 200), 7.0, dtype=F16, device="cuda")  # x and y side by side in the same rows
    buf[:, :64] = x
    op.apply_device(buf.data_ptr(), M, buf.data_ptr() + 2 * 128, ldx=200, ldo=200, d_residual=buf.data_ptr(), ldr=200,
                    stream=slx.STREAM_LEGACY)
    torch.cuda.synchronize()
    assert torch.equal(buf[:, 128:192], y) and torch.equal(buf[:, :64], x)
    assert bool((buf[:, 64:128] == 7).all()) and bool((buf[:, 192:] == 7).all())


def test_qk_norm_rope(ctx):
    H, KV, hd, M = 4, 2, 64, 6
    op = slx.QkNormRope(slx.RopeTable(8, hd, ctx=ctx), slx.DTYPE_F16, H, KV, hd)
    n = (H + 2 * KV) * hd
    x = torch.randn(M, n, device="cuda").to(F16)
    kept, p, k = x.clone(), x.data_ptr(), x.data_ptr() + 2 * H * hd
    o = torch.empty(M, n, dtype=F16, device="cuda")
    go, ok = (lambda qo, ko, **s: op.apply_device(p, k, M, qo, ko, ldq=n, ldk=n, stream=slx.STREAM_LEGACY, **s)), dict(ldqo=n, ldko=n)
    q_o, k_o = o.data_ptr(), o.data_ptr() + 2 * H * hd
    refused(go, p, k_o, ldko=n)  # over q with another stride
    refused(go, p + 16, k_o, **ok)
    refused(go, k, k_o, **ok)  # q's output over k
    refused(go, q_o, p, **ok)  # k's output over q
    refused(go, q_o, q_o + 16, **ok)  # the outputs over each other
    torch.cuda.synchronize()
    assert torch.equal(x, kept)
    go(q_o, k_o, **ok)
    go(p, k, **ok)  # in place
    torch.cuda.synchronize()
    m = (H + KV) * hd
    assert torch.equal(x[:, :m], o[:, :m]) and torch.equal(x[:, m:], kept[:, m:])


def test_one_row_has_no_stride(ctx):
    """A single row in place, whatever the strides say."""
    w = (torch.randn(64, 64, device="cuda") / 8).to(F16)
    x, r = torch.randn(1, 64, device="cuda").to(F16), torch.randn(1, 64, device="cuda").to(F16)
    y = torch.empty_like(x)
    q, k = torch.randn(1, 256, device="cuda").to(F16), torch.randn(1, 128, device="cuda").to(F16)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    torch.cuda.synchronize()
    op = slx.Linear(slx.DTYPE_F16, w.data_ptr(), w.numel() * 2, slx.DTYPE_F16, 64, 64, ctx=ctx)
    op.apply_device(x.data_ptr(), 1, y.data_ptr(), d_residual=r.data_ptr(), stream=slx.STREAM_LEGACY)
    op.apply_device(x.data_ptr(), 1, r.data_ptr(), ldo=100, d_residual=r.data_ptr(), stream=slx.STREAM_LEGACY)
    qk = slx.QkNormRope(slx.RopeTable(8, 64, ctx=ctx), slx.DTYPE_F16, 4, 2, 64)
    for a, b, s in ((qo, ko, {}), (q, k, dict(ldq=512, ldk=512))):
        qk.apply_device(q.data_ptr(), k.data_ptr(), 1, a.data_ptr(), b.data_ptr(), stream=slx.STREAM_LEGACY, **s)
    torch.cuda.synchronize()
    assert torch.equal(r, y) and torch.equal(q, qo) and torch.equal(k, ko)
