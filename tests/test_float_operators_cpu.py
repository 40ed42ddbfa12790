"""Host-side checks of the float operators: the packed call arguments against the header's structures, refusals
that need no device, and CPU models of the exactness claims their kernels rest on (the three-way bf16 split,
the 64-bit forms of the Q30 norm and rotation)."""
import ctypes
import math
import os
import re
import struct
from fractions import Fraction

import numpy as np
import pytest

import spatialdb_b200 as slx
from spatialdb_b200 import _lib, build

M64 = (1 << 64) - 1


def signed(v):
    v &= M64
    return v - (1 << 64) if v >> 63 else v


def fields(name):
    src = open(os.path.join(build.INCLUDE, "slx.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    out = []
    for decl in body.split(";"):
        decl = " ".join(decl.split())
        if decl:
            kind = "Q" if "*" in decl else "q"
            out += [kind] * (decl.count(",") + 1)
    return "".join(out)


@pytest.mark.parametrize("name,pack", [("slx_linear_args", slx._LINEAR_ARGS), ("slx_qk_args", slx._QK_ARGS)])
def test_packed_arguments_match_the_header(name, pack):
    fmt = fields(name)
    values = [7 + i if f == "Q" else -1 - i for i, f in enumerate(fmt)]
    assert pack(*values) == struct.pack("=" + fmt, *values)


def test_null_handles_are_refused_without_a_device():
    lib = _lib.lib()
    out = ctypes.c_void_p(1)
    assert lib.slx_linear_device(None, slx._LINEAR_ARGS(0, 0, 0, 0, 0, 0, 0, 0)) == slx.SLX_EINVAL
    assert lib.slx_qk_norm_rope_device(None, slx._QK_ARGS(*[0] * 12)) == slx.SLX_EINVAL
    for fn in (lib.slx_linear_free, lib.slx_rope_free, lib.slx_qk_norm_free):
        assert fn(None) == slx.SLX_EINVAL
    assert lib.slx_linear_prepare(None, 0, 1, 4, 0, 1, 1, None, 0, None, 0, None, ctypes.byref(out)) == slx.SLX_EINVAL
    assert lib.slx_rope_create(None, 4, 4, 10000.0, 0, ctypes.byref(out)) == slx.SLX_EINVAL
    assert lib.slx_qk_norm_prepare(None, 0, 1, 1, 4, None, None, 0.0, ctypes.byref(out)) == slx.SLX_EINVAL
    assert lib.slx_linear_info(None, (ctypes.c_int64 * 6)(), 6) == slx.SLX_EINVAL


def cut(v):
    """The leading eight significant bits of an fp32 value, the rest cut off."""
    return (v.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)


def test_three_bf16_parts_sum_to_the_value():
    rng = np.random.default_rng(1)
    v = np.concatenate([rng.standard_normal(20000), 10.0 ** rng.uniform(-25, 38, 20000) * rng.choice([-1, 1], 20000),
                        [0.0, -0.0, 3.4028234e38, -3.4028234e38, 1.0, 1 + 2 ** -23, 2 ** -100]]).astype(np.float32)
    a = cut(v)
    r = v - a
    b = cut(r)
    c = cut(r - b)
    assert (a.astype(np.float64) + b + c == v).all()
    assert np.isfinite(a).all() and (np.abs(b) <= np.abs(v) * 2.0 ** -7).all() and (np.abs(c) <= np.abs(v) * 2.0 ** -15).all()


def mean_square(ss, n):
    """The kernel's quotient: a double estimate, the wrapping remainder, one more estimate, then single steps."""
    rn = 1.0 / n
    sd = float(ss >> 64) * 18446744073709551616.0 + float(ss & M64)
    ms = int(sd * rn)
    rem = signed(ss - ms * n)
    assert rem == ss - ms * n  # the true remainder fits: wrapping arithmetic is exact
    ms += math.floor(float(rem) * rn)
    left, steps = signed(ss - ms * n), 0
    while left < 0:
        ms, left, steps = ms - 1, left + n, steps + 1
    while left >= n:
        ms, left, steps = ms + 1, left - n, steps + 1
    assert steps <= 2
    return ms


def test_q30_mean_square_quotient():
    rng = np.random.default_rng(2)
    for n in (2, 6, 62, 64, 66, 96, 128, 250, 256, 512):
        top = n << 62
        for ss in [n, n + 1, top - 1, top - n, top // 2, top // 3] + [int(rng.integers(1, 1 << 62)) * n // int(rng.integers(1, 1 << 20))
                                                                       for _ in range(400)]:
            if n <= ss < top:
                assert mean_square(ss, n) == ss // n
        for ms in rng.integers(1, 1 << 62, 200):  # remainders around zero
            for d in (-1, 0, 1):
                ss = int(ms) * n + d
                if n <= ss < top:
                    assert mean_square(ss, n) == ss // n


def test_q30_quotients_from_one_range_check():
    """floor(P rd) with P = ux uw rounded and rd = 1 / root rounded is exact unless its fraction lies within
    (q + 1) 2^-50 of an integer, where the wrapping remainder decides: quotients built around integers."""
    rng = np.random.default_rng(3)
    near, draws = 0, []
    for _ in range(4000):
        n = int(rng.choice([2, 64, 256, 512]))
        root = int(rng.integers(1, 1 << 31))
        ux = int(rng.integers(0, min(1 << 32, 2 * int(math.sqrt(n)) * root + 1)))
        uw = int(rng.integers(0, 1 << 43))
        if rng.random() < 0.5 and ux:  # a quotient within ux / root of an integer
            uw = min((int(rng.integers(1, 1 << 40)) * root + int(rng.integers(-1, 2))) // ux, (1 << 43) - 1)
            uw = max(uw, 0)
        draws.append((root, ux, uw))
    for _ in range(2000):  # ux uw = -1, 0 or 1 modulo root: on an integer and one step of the numerator beside it
        root = int(rng.integers(2, 1 << 31))
        ux = int(rng.integers(1, min(1 << 32, 2 * root)))
        e = int(rng.integers(-1, 2))
        if math.gcd(ux, root) != 1:
            continue
        uw = pow(ux, -1, root) * e % root
        uw += root * int(rng.integers(0, ((1 << 43) - 1 - uw) // root + 1))
        if ux * uw // root < 1 << 49:
            draws.append((root, ux, uw))
    for root, ux, uw in draws:
        assert ux * uw // root < 1 << 49
        P, rd = float(ux) * float(uw), 1.0 / float(root)
        exact = Fraction(P) * Fraction(rd)
        q = math.floor(exact)
        frac = float(exact - q)
        tol = (q + 1) * 2.0 ** -50
        if frac < tol or frac > 1.0 - tol:
            near += 1
            r = signed(ux * uw - q * root)
            assert abs(r) < 1 << 62
            while r < 0:
                q, r = q - 1, r + root
            while r >= root:
                q, r = q + 1, r - root
        assert q == ux * uw // root
    assert near > 100


def test_q30_rotation_in_64_bits():
    """|a|, |b| < 6e9 and a Q30 cosine and sine: the sums fit 64 bits whatever the angle."""
    lim = 6_000_000_000 - 1
    for t in np.linspace(0, 2 * math.pi, 2001):
        c, s = int(math.cos(t) * 2 ** 30), int(math.sin(t) * 2 ** 30)
        assert c * c + s * s <= 1 << 60
        for a in (lim, -lim):
            for b in (lim, -lim):
                for v in (a * c - b * s, a * s + b * c):
                    assert signed(v) == v


def test_q30_lane_sums_in_three_limbs():
    """A lane's 16 squares stay below 2^68, and 32 limbs of 27 bits below 2^32."""
    top = 16 * ((1 << 32) - 1) ** 2
    assert top < 1 << 68 and 32 * ((1 << 27) - 1) < 1 << 32 and 32 * (top >> 54) < 1 << 32
    rng = np.random.default_rng(4)
    sums = [int(rng.integers(0, 1 << 62)) * int(rng.integers(0, 64)) % top for _ in range(32)]
    mask = (1 << 27) - 1
    limbs = [sum((s >> k) & mask for s in sums) if k < 54 else sum(s >> 54 for s in sums) for k in (0, 27, 54)]
    assert limbs[0] + (limbs[1] << 27) + (limbs[2] << 54) == sum(sums)
