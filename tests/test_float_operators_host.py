"""Host-side checks of the float operators' sources and helpers that need no device."""
import itertools
import math
import os
import re
import subprocess

import numpy as np

from spatialdb_b200 import build


def source(name):
    text = open(os.path.join(build.CSRC, name)).read()
    return re.sub(r"//[^\n]*", "", text)


def test_dependents_start_after_the_tensor_memory_is_taken():
    """A kernel that may run beside this one must find its tensor memory taken: every CTA of the product allocates,
    meets at a barrier, and only then lets dependents start."""
    body = source("k_linear_tc.cu")
    body = body[body.index("k_linear_tc(const __grid_constant__"):]
    alloc = [m.start() for m in re.finditer(r"tcgen05\.alloc\.", body)]
    release = [m.start() for m in re.finditer(r"grid_release\(\)", body)]
    assert len(alloc) == 2 and len(release) == 1
    barrier = body.index("__syncthreads()", max(alloc))
    assert max(alloc) < barrier < release[0] < body.index("grid_wait()")


def nearest(v):
    """fp32 values rounded to the nearest bf16 (ties to even), finite where cutting off would be."""
    u = v.view(np.uint32)
    up = ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) & np.uint32(0xFFFF0000)).view(np.float32)
    return np.where(np.isfinite(up), up, (u & np.uint32(0xFFFF0000)).view(np.float32))


def test_rounded_bf16_parts_sum_to_the_value():
    """x = x1 + x2 + x3 exactly, with remainders of 2^-8 and 2^-17 (twice that where x1 is cut off at the range's top),
    the product of two such sums short of six of its nine terms by 2^-23.9, and no bias to one side."""
    rng = np.random.default_rng(6)
    near = (1 + rng.integers(0, 1 << 23, 20000) * 2.0 ** -23) * 2.0 ** rng.integers(-90, 120, 20000)
    ties = (1 + (2 * rng.integers(0, 128, 2000) + 1) * 2.0 ** -8 + rng.integers(-2, 3, 2000) * 2.0 ** -23) * 2.0 ** rng.integers(-90, 120, 2000)
    v = np.concatenate([near, ties, -near, [0.0, -0.0, 1.0, 1 + 2 ** -23, 2 - 2 ** -23]]).astype(np.float32)
    top = np.array([3.4028234e38, -3.4028234e38, 3.3961775e38, 3.39e38, 3.395e38], np.float32)
    for values, first in ((v, 2.0 ** -8), (top, 2.0 ** -7)):
        a = nearest(values)
        r = values - a
        b = nearest(r)
        c = nearest(r - b)
        assert (a.astype(np.float64) + b + c == values).all() and np.isfinite(a).all()
        size = np.abs(values.astype(np.float64))
        assert (np.abs(b) <= first * size).all() and (np.abs(c) <= first * 2.0 ** -9 * size).all()
    x, w = rng.permutation(np.abs(near)).astype(np.float32), np.abs(near).astype(np.float32)

    def parts(v):
        a = nearest(v)
        b = nearest(v - a)
        return [t.astype(np.float64) for t in (a, b, v - a - b)]

    (_, x2, x3), (_, w2, w3) = parts(x), parts(w)
    left = (x2 * w3 + x3 * w2 + x3 * w3) / (x.astype(np.float64) * w)
    assert np.abs(left).max() <= 2.0 ** -23.9
    assert abs(left.mean()) <= 6 * left.std() / math.sqrt(left.size)


def test_erfc_polynomials():
    """erfc(z) = e^(-z^2) t P(t), t = 1 / (1 + a z), with the kernels' constants: the relative errors their comment states,
    over the z whose results the output's type can hold."""
    text = source("slx_linear_dev.cuh")
    a32, a16 = (float(np.float32(x)) for x in re.search(r"A = F \? ([0-9.]+)f : ([0-9.]+)f", text).groups())
    for name, a, top, bound in (("c32", a32, 10.2, 2.7e-8), ("c16", a16, 9.6, 2.0 ** -17.5)):
        c = [float(np.float32(x.strip(" f"))) for x in re.search(name + r"\[\d+\] = \{(.*?)\}", text).group(1).split(",")]
        worst = 0.0
        for z in np.linspace(0.0, top, 20001):
            t = 1.0 / (1.0 + a * z)
            p = t * sum(v * t ** i for i, v in enumerate(c))
            worst = max(worst, abs(p * math.exp(-z * z) / math.erfc(z) - 1.0))
        assert worst <= bound, (name, worst)


def test_overlap_of_strided_rows(tmp_path):
    """rows_overlap against the bytes themselves, over every small arrangement of two arrays of rows."""
    main = tmp_path / "rows.cpp"
    main.write_text('''
#include <cstdio>
#include "slx_rows.h"
int main() {
    long long p[8];
    while (std::scanf("%lld %lld %lld %lld %lld %lld %lld %lld", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6, p + 7) == 8)
        std::printf("%d", (int)slx::rows_overlap((void*)p[0], p[1], p[2], (void*)p[3], p[4], p[5], p[6], (int)p[7]));
}
''')
    exe = str(tmp_path / "rows")
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", build.CSRC, str(main), "-o", exe], check=True)
    calls, want = [], []
    for lda, ldb, M, e in itertools.product((3, 5), (3, 4, 5, 9), (1, 2, 3), (1, 2)):
        for wa, wb, d in itertools.product((1, 2, 3), (1, 3), range(-20, 21)):
            a, b = 4096, 4096 + d * e
            at = [{p + m * ld * e + i for m in range(M) for i in range(w * e)} for p, ld, w in ((a, lda, wa), (b, ldb, wb))]
            calls.append((a, lda, wa, b, ldb, wb, M, e))
            want.append(bool(at[0] & at[1]))
    big = 1 << 40  # strides past 32 bits, and nothing to read
    calls += [(64, big, 8, 64 + big * 4, big, 8, 100, 4), (64, big, 8, 80, big, 8, 1 << 20, 4), (64, big, 8, 96, big, 8, 1 << 20, 4), (0, 8, 8, 0, 8, 8, 4, 4)]
    want += [True, True, False, False]
    out = subprocess.run([exe], input="\n".join(" ".join(map(str, c)) for c in calls), capture_output=True, text=True, check=True).stdout
    assert [c == "1" for c in out] == want


def test_freeing_the_last_object_leaves_the_current_device(tmp_path):
    """ctx_release, as it stands, against stand-ins of the CUDA runtime: whichever device was current still is."""
    text = source("slx_model.cu")
    body = text[text.index("void slx::ctx_release"):]
    body = body[:body.index("\n}\n") + 3]
    header = source("slx_ctx.h")
    guard = header[header.index("struct OnDevice {"):]
    guard = guard[:guard.index("};") + 2]
    main = tmp_path / "release.cpp"
    main.write_text("""
#include <atomic>
#include <cstdio>
#include <vector>
typedef int cudaError_t; enum { cudaSuccess = 0 };
int current = 0, freed_on = -1;
int cudaGetDevice(int* d) { *d = current; return 0; }
int cudaSetDevice(int d) { current = d; return 0; }
template <class T> int cudaFree(T) { freed_on = current; return 0; }
template <class T> int cudaEventDestroy(T) { return 0; }
template <class T> int cudaStreamSynchronize(T) { return 0; }
template <class T> int cudaStreamDestroy(T) { return 0; }
template <class T> int cudaMemPoolDestroy(T) { return 0; }
template <class T> void gemm_workspace_free(T) {}
typedef int cudaEvent_t;
struct Record { int a, b; };
struct slx_ctx { std::atomic<int> refs{1}; int device = 3, stream = 1, d_flag = 1, kws = 0, pool = 1;
                 std::vector<Record> records; std::vector<int> event_pool; };
namespace slx { void ctx_release(slx_ctx*); %s }
using namespace slx;
%s
int main() {
    current = 1;
    slx::ctx_release(new slx_ctx());
    std::printf("%%d %%d", current, freed_on);
}
""" % (guard, body))
    exe = str(tmp_path / "release")
    subprocess.run(["g++", "-std=c++17", str(main), "-o", exe], check=True)
    assert subprocess.run([exe], capture_output=True, text=True, check=True).stdout == "1 3"
