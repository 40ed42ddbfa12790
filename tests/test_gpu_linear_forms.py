"""Every form of the linear operator's tensor-core kernel by name (SLX_OPT_TEST_LINEAR_FORM), not only those that the
estimate picks for the other tests' sizes: each tile width and cluster size, pairs, wide pairs, rows that TMA reads and
rows that it cannot, gated and not, each type; what ran is the form asked for, or the call is refused."""
import pytest

import spatialdb_b200 as slx
from test_gpu_linear import Case

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
ONE, PAIR, WIDE = 0, 1, 2


def forms(dtype, gated):
    f32 = dtype == "f32"
    for nt in (32, 64) if f32 and gated else (32, 64, 128):
        for log2 in range(4):
            yield ONE, nt, log2
    for nt in (32, 64, 128) if f32 else (64, 128, 256):
        yield PAIR, nt, 0
    if gated and not f32:
        yield WIDE, 128, 0


ALL = [(d, g, *f) for d in ("f32", "f16", "bf16") for g in (False, True) for f in forms(d, g)]


@pytest.fixture(scope="module")
def ctx():
    return slx.Context(0)


@pytest.fixture
def form(ctx):
    def set_form(mode, nt, log2):
        ctx.set_option(slx.OPT_TEST_LINEAR_FORM, nt + 1024 * mode + 4096 * log2)
    yield set_form
    ctx.set_option(slx.OPT_TEST_LINEAR_FORM, 0)


@pytest.mark.parametrize("dtype,gated,mode,nt,log2", ALL)
def test_every_form(ctx, form, dtype, gated, mode, nt, log2):
    form(mode, nt, log2)
    for M, K, N, pad in ((1, 1100, 129, 0), (70, 1100, 300, 0), (129, 1101, 257, 1), (300, 2048, 128, 8), (37, 1032, 1024, 4)):
        Case(ctx, dtype, M, K, N, act="silu", gated=gated, bias=True, residual=True, pad=pad).check()
    Case(ctx, dtype, 200, 1030, 130, act="gelu_tanh" if gated else "none", gated=gated, pad=3).check()


@pytest.mark.parametrize("dtype,gated,mode,nt,log2", [f for f in ALL if f[4] in (0, 3)])
def test_every_form_over_many_tiles(ctx, form, dtype, gated, mode, nt, log2):
    """Several tiles a CTA, or a grid past what is resident; the same result on every call."""
    form(mode, nt, log2)
    for pad in (0, 5) if dtype != "f32" or not gated or mode else (0,):
        c = Case(ctx, dtype, 2600, 1032, 2600, act="silu", gated=gated, residual=True, pad=pad)
        first = c.check().clone()
        for _ in range(3):
            assert torch.equal(c.run(), first)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("K", [1, 31, 64, 65])
def test_every_form_of_short_sums(ctx, form, dtype, gated, K):
    for mode, nt, log2 in forms(dtype, gated):
        if log2:
            continue
        form(mode, nt, log2)
        Case(ctx, dtype, 140, K, 140, act="silu", gated=gated, bias=True).check()


def test_refused_forms(ctx, form):
    def refused(dtype, gated, K, *f):
        form(*f)
        c = Case(ctx, dtype, 20, K, 64, gated=gated)
        with pytest.raises(slx.SlxError) as e:
            c.run()
        assert e.value.status == slx.SLX_EUNSUPPORTED

    for dtype, gated, f in (("f32", False, (PAIR, 256, 0)), ("f32", True, (ONE, 128, 0)), ("f16", False, (PAIR, 32, 0)), ("f16", False, (ONE, 256, 0)),
                            ("f16", False, (WIDE, 128, 0)), ("f32", True, (WIDE, 128, 0)), ("f16", True, (WIDE, 64, 0)), ("f16", True, (PAIR, 64, 1)),
                            ("bf16", False, (ONE, 48, 0)), ("bf16", False, (3, 64, 0))):
        refused(dtype, gated, 640, *f)
    refused("f16", False, 64, ONE, 32, 1)  # one block of K for two CTAs
    for value in (-1, 1 << 14):
        with pytest.raises(slx.SlxError) as e:
            ctx.set_option(slx.OPT_TEST_LINEAR_FORM, value)
        assert e.value.status == slx.SLX_EINVAL
