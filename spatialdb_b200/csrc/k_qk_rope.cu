// k_qk_rope.cu -- RmsNorm of every query and key head and the rotary positions in one pass.
//
// Float: for a head row x of hd values, s = 1 / sqrt(sum x^2 / hd + eps), u_j = x_j s w_j; the pair
// (u_p, u_{p+h}), p < h, becomes (u_p c - u_{p+h} s', u_p s' + u_{p+h} c) with (c, s') the table's entry of the
// row's position; values past 2 h keep u. All in fp32 from the loaded values to the one rounding at
// the store; the root and its reciprocal are one rsqrtf, good to two units of 2^-23 for each head. Q30: RmsNormRow, then
// ApplyRoPE, on int64 values.
//
// Both are bound by memory at many rows (every value is read and written once, the table's row once
// per token) and by latency at one token. A pair's two values belong to one lane, so the rotation
// needs no exchange, the reduction is the only traffic between lanes, and in-place calls are safe.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "slx_attr.h"
#include "slx_device.cuh"
#include "slx_kernels.h"
#include "slx_qk_rope.h"

namespace slx {
namespace {

constexpr int QT = 256;  // threads per block
constexpr int QV = 128;  // of k_qk_vec

SLX_DEV float to_f(float v) { return v; }
SLX_DEV float to_f(__half v) { return __half2float(v); }
SLX_DEV float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
SLX_DEV T from_f(float v);
template <>
SLX_DEV float from_f<float>(float v) { return v; }
template <>
SLX_DEV __half from_f<__half>(float v) { return __float2half_rn(v); }
template <>
SLX_DEV __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two fp32 values in a 64-bit register: the packed FMA and multiply do both in one instruction.
typedef unsigned long long f32x2;
SLX_DEV f32x2 pack2(float lo, float hi) {
    f32x2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
SLX_DEV void unpack2(f32x2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
SLX_DEV f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
SLX_DEV f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}

// 16 bytes of a row as pairs of fp32 values, and back with one rounding.
template <class T>
struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    uint4 raw;
};
SLX_DEV void widen(const Vec16<float>& v, f32x2 (&o)[2]) {
    o[0] = pack2(__uint_as_float(v.raw.x), __uint_as_float(v.raw.y));
    o[1] = pack2(__uint_as_float(v.raw.z), __uint_as_float(v.raw.w));
}
SLX_DEV f32x2 widen2(uint32_t w, __nv_bfloat16) { return pack2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
SLX_DEV f32x2 widen2(uint32_t w, __half) {
    const float2 f = __half22float2(*(const __half2*)&w);
    return pack2(f.x, f.y);
}
template <class T>
SLX_DEV void widen(const Vec16<T>& v, f32x2 (&o)[4]) {
    o[0] = widen2(v.raw.x, T());
    o[1] = widen2(v.raw.y, T());
    o[2] = widen2(v.raw.z, T());
    o[3] = widen2(v.raw.w, T());
}
SLX_DEV uint32_t narrow2(f32x2 v, __nv_bfloat16) {
    float lo, hi;
    unpack2(v, lo, hi);
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *(const uint32_t*)&h;
}
SLX_DEV uint32_t narrow2(f32x2 v, __half) {
    float lo, hi;
    unpack2(v, lo, hi);
    const __half2 h = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&h;
}
SLX_DEV uint4 narrow(const f32x2 (&v)[2], float) {
    float f[4];
    unpack2(v[0], f[0], f[1]);
    unpack2(v[1], f[2], f[3]);
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <class T>
SLX_DEV uint4 narrow(const f32x2 (&v)[4], T t) {
    return make_uint4(narrow2(v[0], t), narrow2(v[1], t), narrow2(v[2], t), narrow2(v[3], t));
}

// a / b and a % b for a below `most`, in 32 bits where they suffice (a 64-bit division costs ten times as much).
SLX_DEV void divide(int64_t a, int b, int64_t most, int64_t& quo, int& rem) {
    if (most < (1ll << 32)) {
        const uint32_t q = (uint32_t)a / (uint32_t)b;
        quo = q;
        rem = (int)((uint32_t)a - q * (uint32_t)b);
    } else {
        quo = a / b;
        rem = (int)(a - quo * b);
    }
}

// Row m's position, or -1 when the row is to be left alone (a negative entry, or one outside the
// table, which raises KERR_RANGE unless it is exactly -1).
SLX_DEV int position(const QkRope& p, int64_t m) {
    if (!p.pos) return p.M < (1ll << 31) && p.T < (1ll << 31) ? (int)((uint32_t)m % (uint32_t)p.T) : (int)(m % p.T);
    const int t = p.pos[m];
    if (t >= 0 && t < p.table_rows) return t;
    if (t != -1) atomicOr(p.err, KERR_RANGE);
    return -1;
}

// 16-byte chunks. Lane j of a head's group of G lanes owns chunk j and its partner chunk j + h for
// j < h = half / N, and past those the two unrotated chunks 2h + 2(j - h) and the next one. A warp takes one
// row's query heads or key heads, 32 / G at a time in up to STEPS steps: the row's table entries are read once.
// Every step's values are asked for before the position is known, so that a warp has up to STEPS KB in flight
// while it waits for the position and then for the table (with one step in flight at a time 24 warps an SM
// kept 24 KB in flight, where the memory's rate times its latency is about 44).
struct Slabs {
    int q, k;  // warps to a row's query and key heads
};
template <class T, int G, int STEPS>
__global__ void __launch_bounds__(QV) k_qk_vec(QkRope p, Slabs sl) {
    constexpr int N = Vec16<T>::N;
    const int lane = threadIdx.x & 31, j = lane & (G - 1), grp = lane / G;
    const unsigned gmask = (G == 32 ? 0xffffffffu : (1u << (G & 31)) - 1u) << (grp * G & 31);
    int64_t m;
    int slab;
    divide((int64_t)blockIdx.x * (QV / 32) + (threadIdx.x >> 5), sl.q + sl.k, p.M * (sl.q + sl.k) + QV, m, slab);
    grid_release();
    grid_wait();
    if (m >= p.M) return;
    const bool isq = slab < sl.q;
    const QkSide& s = isq ? p.q : p.k;
    constexpr int PER = 32 / G;
    const int head = (isq ? slab : slab - sl.q) * STEPS * PER + grp;
    const int h = p.half / N, chunks = p.hd / N;
    const bool pair = j < h;
    const int ca = pair ? j : 2 * j, cb = pair ? j + h : 2 * j + 1;  // 2h + 2(j - h) = 2j
    const bool has_a = ca < chunks, has_b = cb < chunks;
    const T* x = (const T*)s.in + m * s.ld_in + (int64_t)head * p.hd;
    T* y = (T*)s.out + m * s.ld_out + (int64_t)head * p.hd;
    Vec16<T> va[STEPS], vb[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; i++) {
        const bool live = head + i * PER < s.nh;
        const T* from = x + (int64_t)i * PER * p.hd;
        va[i].raw = live && has_a ? *(const uint4*)(from + ca * N) : make_uint4(0, 0, 0, 0);
        vb[i].raw = live && has_b ? *(const uint4*)(from + cb * N) : make_uint4(0, 0, 0, 0);
    }
    const int pos = position(p, m);
    if (pos < 0) return;
    constexpr int P = N / 2;
    f32x2 cs[P], sn[P], ns[P];  // cosines, sines and the sines' negatives
    if (pair) {
        const float4* t = (const float4*)(p.table + (int64_t)pos * p.half + (int64_t)j * N);
#pragma unroll
        for (int e = 0; e < P; e++) {
            const float4 v = t[e];
            cs[e] = pack2(v.x, v.z);
            sn[e] = pack2(v.y, v.w);
            ns[e] = pack2(-v.y, -v.w);
        }
    }
    const float inv_n = 1.0f / (float)p.hd;
    const float* w = (const float*)s.w;
#pragma unroll
    for (int i = 0; i < STEPS; i++, y += PER * p.hd) {
        if (head + i * PER >= s.nh) break;
        f32x2 a[P], b[P];
        widen(va[i], a);
        widen(vb[i], b);
        if (w) {
            f32x2 sq = 0;  // 0.0, 0.0
#pragma unroll
            for (int e = 0; e < P; e++) sq = fma2(a[e], a[e], fma2(b[e], b[e], sq));
            float lo, hi;
            unpack2(sq, lo, hi);
            float ss = lo + hi;
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(gmask, ss, o);
            const float r1 = rsqrtf(fmaf(ss, inv_n, p.eps));
            const f32x2 r = pack2(r1, r1);
#pragma unroll
            for (int e = 0; e < P; e += 2) {
                if (has_a) {
                    const float4 v = *(const float4*)(w + ca * N + 2 * e);
                    a[e] = mul2(a[e], mul2(r, pack2(v.x, v.y)));
                    a[e + 1] = mul2(a[e + 1], mul2(r, pack2(v.z, v.w)));
                }
                if (has_b) {
                    const float4 v = *(const float4*)(w + cb * N + 2 * e);
                    b[e] = mul2(b[e], mul2(r, pack2(v.x, v.y)));
                    b[e + 1] = mul2(b[e + 1], mul2(r, pack2(v.z, v.w)));
                }
            }
        }
        if (pair) {
#pragma unroll
            for (int e = 0; e < P; e++) {
                const f32x2 t = fma2(a[e], cs[e], mul2(b[e], ns[e]));
                b[e] = fma2(a[e], sn[e], mul2(b[e], cs[e]));
                a[e] = t;
            }
        }
        if (has_a) *(uint4*)(y + ca * N) = narrow(a, T());
        if (has_b) *(uint4*)(y + cb * N) = narrow(b, T());
    }
}

// Any even head size, rotation width, stride and alignment: one warp per head row, single values. The
// row is read a second time (from cache) after its norm is known.
template <class T>
__global__ void __launch_bounds__(QT) k_qk_any(QkRope p) {
    const int lane = threadIdx.x & 31, nheads = p.q.nh + p.k.nh;
    int64_t m;
    int head;
    divide((int64_t)blockIdx.x * (QT / 32) + (threadIdx.x >> 5), nheads, p.M * nheads + QT, m, head);
    grid_release();
    grid_wait();
    if (m >= p.M) return;
    const int pos = position(p, m);
    if (pos < 0) return;
    const bool isq = head < p.q.nh;
    const QkSide& s = isq ? p.q : p.k;
    const int hh = isq ? head : head - p.q.nh;
    const T* x = (const T*)s.in + m * s.ld_in + (int64_t)hh * p.hd;
    T* y = (T*)s.out + m * s.ld_out + (int64_t)hh * p.hd;
    const float* w = (const float*)s.w;
    float r = 1.0f;
    if (w) {
        float ss = 0.0f;
        for (int i = lane; i < p.hd; i += 32) {
            const float v = to_f(x[i]);
            ss = fmaf(v, v, ss);
        }
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        r = rsqrtf(fmaf(ss, 1.0f / (float)p.hd, p.eps));
    }
    const float2* t = p.table + (int64_t)pos * p.half;
    for (int i = lane; i < p.half; i += 32) {
        float a = to_f(x[i]), b = to_f(x[i + p.half]);
        if (w) {
            a = a * r * w[i];
            b = b * r * w[i + p.half];
        }
        const float2 c = t[i];
        y[i] = from_f<T>(fmaf(a, c.x, -(b * c.y)));
        y[i + p.half] = from_f<T>(fmaf(a, c.y, b * c.x));
    }
    for (int i = 2 * p.half + lane; i < p.hd; i += 32) {
        const float a = to_f(x[i]);
        y[i] = from_f<T>(w ? a * r * w[i] : a);
    }
}

template <class T, int G, int STEPS>
int launch_steps(const QkRope& p, cudaStream_t st) {
    const int heads = 32 / G * STEPS;  // of a warp
    const Slabs sl{(p.q.nh + heads - 1) / heads, (p.k.nh + heads - 1) / heads};
    const int64_t units = p.M * (sl.q + sl.k);
    launch_early(k_qk_vec<T, G, STEPS>, (unsigned)((units + QV / 32 - 1) / (QV / 32)), QV, 0, st, 1, p, sl);
    return 1;
}
// One step to a warp while that leaves SMs without work (the least latency), then two and four (f16 3001 x (20 + 4) x
// 96, in us with 1, 2, 3, 4 steps: 12.3, 10.3, 12.3, 14.4; bf16 8192 x (32 + 8) x 128: 44.6, 36.9, 39.7, 36.9).
template <class T, int G>
int launch_vec(const QkRope& p, cudaStream_t st) {
    const int per = 32 / G;
    const int64_t steps = p.M * ((p.q.nh + per - 1) / per + (p.k.nh + per - 1) / per), warps = (int64_t)device_sm_count() * 20;
    if (steps < 2 * warps) return launch_steps<T, G, 1>(p, st);
    if (steps < 12 * warps) return launch_steps<T, G, 2>(p, st);
    return launch_steps<T, G, 4>(p, st);
}

template <class T>
int launch_float(const QkRope& p, cudaStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    auto aligned = [](const QkSide& s) {
        return s.nh == 0 || (((uintptr_t)s.in | (uintptr_t)s.out) % 16 == 0 && s.ld_in % N == 0 && s.ld_out % N == 0);
    };
    const int h = p.half / N, rest = (p.hd - 2 * p.half) / N, lanes = h + (rest + 1) / 2;
    if (p.half % N == 0 && p.hd % N == 0 && lanes <= 32 && aligned(p.q) && aligned(p.k)) {
        if (lanes <= 2) return launch_vec<T, 2>(p, st);
        if (lanes <= 4) return launch_vec<T, 4>(p, st);
        if (lanes <= 8) return launch_vec<T, 8>(p, st);
        if (lanes <= 16) return launch_vec<T, 16>(p, st);
        return launch_vec<T, 32>(p, st);
    }
    const int64_t units = p.M * (p.q.nh + p.k.nh);
    launch_early(k_qk_any<T>, (unsigned)((units + QT / 32 - 1) / (QT / 32)), QT, 0, st, 1, p);
    return 1;
}

// ---- Q30 -------------------------------------------------------------------------------------------

// RmsNormRow's root for a head's wrapping sum of squares, and its reciprocal; skip: the row is left as it is
// (ms <= 0). A mean square below 2^62 (values below 2 in Q30) takes 64-bit arithmetic: its quotient from a double
// estimate (off by at most 2^10), corrected by the exact remainder, and its root corrected by squaring. rn = 1 / n.
SLX_DEV int64_t q30_root(u128 ss, int n, double rn, bool& skip, double& rd) {
    skip = (i128)ss < (i128)n;
    rd = 1.0;
    if (skip) return 1;
    if ((ss >> 62) < (u128)(uint32_t)n) {
        const double sd = fma((double)(uint32_t)(ss >> 64), 18446744073709551616.0, (double)(uint64_t)ss);
        uint64_t ms = (uint64_t)(sd * rn);
        const int64_t rem = (int64_t)((uint64_t)ss - ms * (uint64_t)n);  // exact: the true value is small
        ms += (uint64_t)(int64_t)floor((double)rem * rn);
        int64_t left = (int64_t)((uint64_t)ss - ms * (uint64_t)n);
        while (left < 0) { ms--; left += n; }
        while (left >= n) { ms++; left -= n; }
        uint64_t r = (uint64_t)sqrt((double)ms);
        while (r * r > ms) r--;
        while ((r + 1) * (r + 1) <= ms) r++;
        rd = 1.0 / (double)r;
        return (int64_t)r;
    }
    int64_t r = isqrt_u128(udiv128_u32(ss, (uint32_t)n, ~0ULL / (uint32_t)n));
    if (r == 0) r = 1;
    rd = 1.0 / (double)r;
    return r;
}

// floor((a c - b s) / 2^30) and floor((a s + b c) / 2^30). With c, s a Q30 cosine and sine (c^2 + s^2 <= 2^60) and
// |a|, |b| < 6e9 the sums stay below sqrt(a^2 + b^2) 2^30 < 2^63: wrapping 64-bit arithmetic is exact.
SLX_DEV void q30_rotate(int64_t a, int64_t b, int64_t c, int64_t s, int64_t& ya, int64_t& yb) {
    constexpr int64_t lim = 6000000000ll;
    if (a > -lim && a < lim && b > -lim && b < lim) {
        const int64_t c32 = (int32_t)c, s32 = (int32_t)s;
        ya = wsub(wmul(a, c32), wmul(b, s32)) >> 30;
        yb = wadd(wmul(a, s32), wmul(b, c32)) >> 30;
        return;
    }
    ya = lo64(sar128((i128)((u128)((i128)a * c) - (u128)((i128)b * s)), 30));
    yb = lo64(sar128((i128)((u128)((i128)a * s) + (u128)((i128)b * c)), 30));
}

// trunc(x w / root) for a value of a row whose |x| are all below 2^32 and whose root is `root`: muldiv_trunc with
// one range check. sum x^2 < n (root + 1)^2, so |x| < 2 sqrt(n) root and the quotient is below 2 sqrt(n) |w|: for
// |w| < 2^43 and n <= 512 below 2^49, muldiv_trunc's own bound for its estimate.
SLX_DEV int64_t q30_scale(int64_t x, int64_t w, int64_t root, double rd) {
    const bool minus = (x ^ w) < 0;
    const uint64_t uw = w < 0 ? 0 - (uint64_t)w : (uint64_t)w;
    const uint32_t ux = (uint32_t)(x < 0 ? -x : x);
    if (uw >= (1ull << 43)) return muldiv_trunc(x, w, d_i64(w), root, rd);
    const double P = d_u32(ux) * d_i64((int64_t)uw);
    const double y = rd_floor(P, rd);
    int64_t q = rd_i64(y);
    const double fl = y - RD_BASE, frac = __fma_rn(P, rd, -fl), tol = __fma_rn(fl, 0x1p-50, 0x1p-50);
    if (frac < tol || frac > 1.0 - tol) {
        int64_t r = (int64_t)(ux * uw - (uint64_t)q * (uint64_t)root);
        while (r < 0) { q--; r += root; }
        while (r >= root) { q++; r -= root; }
    }
    return minus ? -q : q;
}

// One warp per head row, lane l owning the pairs l, l + 32, ... (PL of them, held in registers). Bound by the
// latency of a warp's chain (sum, root, exact quotients, rotation) at 32 warps an SM: four blocks (64 registers) of
// 513 rows' 4617 warps run at once, 9.1 us; three (70 registers) take two waves, 12.2.
template <int PL>
__global__ void __launch_bounds__(QT, PL <= 4 ? 4 : 2) k_qk_q30(QkRope p) {
    const int lane = threadIdx.x & 31, nheads = p.q.nh + p.k.nh;
    int64_t m;
    int head;
    divide((int64_t)blockIdx.x * (QT / 32) + (threadIdx.x >> 5), nheads, p.M * nheads + QT, m, head);
    grid_release();
    grid_wait();
    if (m >= p.M) return;
    const int pos = position(p, m);
    if (pos < 0) return;
    const bool isq = head < p.q.nh;
    const QkSide& s = isq ? p.q : p.k;
    const int hh = isq ? head : head - p.q.nh;
    const int64_t* x = (const int64_t*)s.in + m * s.ld_in + (int64_t)hh * p.hd;
    int64_t* y = (int64_t*)s.out + m * s.ld_out + (int64_t)hh * p.hd;
    const int64_t* w = (const int64_t*)s.w;
    const int64_t *cs = p.cs + (int64_t)pos * p.half, *sn = p.sn + (int64_t)pos * p.half;
    int64_t a[PL], b[PL];
#pragma unroll
    for (int e = 0; e < PL; e++) {
        const int i = lane + 32 * e;
        a[e] = i < p.half ? x[i] : 0;
        b[e] = i < p.half ? x[i + p.half] : 0;
    }
    bool skip = true, narrow = true;  // narrow: every |x| of the head below 2^32, a square is one 32-bit product
    int64_t root = 1;
    double rd = 1.0;
    if (w) {
        u128 ss = 0;
#pragma unroll
        for (int e = 0; e < PL; e++) {
            const uint64_t ua = a[e] < 0 ? 0 - (uint64_t)a[e] : (uint64_t)a[e], ub = b[e] < 0 ? 0 - (uint64_t)b[e] : (uint64_t)b[e];
            narrow = narrow && ((ua | ub) >> 32) == 0;
            ss += (u128)((uint64_t)(uint32_t)ua * (uint32_t)ua);
            ss += (u128)((uint64_t)(uint32_t)ub * (uint32_t)ub);
        }
        narrow = __all_sync(0xffffffffu, narrow);
        if (narrow) {  // below 2^68 in a lane: three limbs of 27 bits, each summed over the lanes in one instruction
            constexpr uint32_t MASK = (1u << 27) - 1;
            const uint32_t l0 = __reduce_add_sync(0xffffffffu, (uint32_t)ss & MASK);
            const uint32_t l1 = __reduce_add_sync(0xffffffffu, (uint32_t)(ss >> 27) & MASK);
            const uint32_t l2 = __reduce_add_sync(0xffffffffu, (uint32_t)(ss >> 54));
            ss = (u128)l0 + ((u128)l1 << 27) + ((u128)l2 << 54);
        } else {
            ss = 0;
#pragma unroll
            for (int e = 0; e < PL; e++) ss += (u128)((i128)a[e] * a[e]) + (u128)((i128)b[e] * b[e]);
            ss = warp_sum_u128(ss);
        }
        root = q30_root(ss, p.hd, p.inv_hd, skip, rd);
    }
#pragma unroll
    for (int e = 0; e < PL; e++) {
        const int i = lane + 32 * e;
        if (i >= p.half) continue;
        int64_t u = a[e], v = b[e];
        if (!skip) {
            const int64_t wu = w[i], wv = w[i + p.half];
            if (narrow) {
                u = q30_scale(u, wu, root, rd);
                v = q30_scale(v, wv, root, rd);
            } else {
                u = muldiv_trunc(u, wu, d_i64(wu), root, rd);
                v = muldiv_trunc(v, wv, d_i64(wv), root, rd);
            }
        }
        q30_rotate(u, v, cs[i], sn[i], y[i], y[i + p.half]);
    }
}

// Heads wider than the registers of k_qk_q30 hold: the row is read again after its norm is known.
__global__ void __launch_bounds__(QT) k_qk_q30_wide(QkRope p) {
    const int lane = threadIdx.x & 31, nheads = p.q.nh + p.k.nh;
    int64_t m;
    int head;
    divide((int64_t)blockIdx.x * (QT / 32) + (threadIdx.x >> 5), nheads, p.M * nheads + QT, m, head);
    grid_release();
    grid_wait();
    if (m >= p.M) return;
    const int pos = position(p, m);
    if (pos < 0) return;
    const bool isq = head < p.q.nh;
    const QkSide& s = isq ? p.q : p.k;
    const int hh = isq ? head : head - p.q.nh;
    const int64_t* x = (const int64_t*)s.in + m * s.ld_in + (int64_t)hh * p.hd;
    int64_t* y = (int64_t*)s.out + m * s.ld_out + (int64_t)hh * p.hd;
    const int64_t* w = (const int64_t*)s.w;
    bool skip = true;
    int64_t root = 1;
    double rd = 1.0;
    if (w) {
        u128 ss = 0;
        for (int i = lane; i < p.hd; i += 32) ss += (u128)((i128)x[i] * x[i]);
        root = q30_root(warp_sum_u128(ss), p.hd, p.inv_hd, skip, rd);
    }
    for (int i = lane; i < p.half; i += 32) {
        int64_t u = x[i], v = x[i + p.half];
        if (!skip) {
            u = muldiv_trunc(u, w[i], d_i64(w[i]), root, rd);
            v = muldiv_trunc(v, w[i + p.half], d_i64(w[i + p.half]), root, rd);
        }
        q30_rotate(u, v, p.cs[(int64_t)pos * p.half + i], p.sn[(int64_t)pos * p.half + i], y[i], y[i + p.half]);
    }
}
}  // namespace

int qk_norm_rope(int dtype, const QkRope& p, cudaStream_t st) {
    if (p.M <= 0 || p.q.nh + p.k.nh <= 0) return 0;
    if (dtype == DT_F16) return launch_float<__half>(p, st);
    if (dtype == DT_BF16) return launch_float<__nv_bfloat16>(p, st);
    return launch_float<float>(p, st);
}

int qk_norm_rope_q30(const QkRope& given, cudaStream_t st) {
    QkRope p = given;
    if (p.M <= 0 || p.q.nh + p.k.nh <= 0) return 0;
    p.inv_hd = 1.0 / (double)p.hd;
    const int64_t units = p.M * (p.q.nh + p.k.nh);
    const unsigned grid = (unsigned)((units + QT / 32 - 1) / (QT / 32));
    if (p.half <= 32) launch_early(k_qk_q30<1>, grid, QT, 0, st, 1, p);
    else if (p.half <= 64) launch_early(k_qk_q30<2>, grid, QT, 0, st, 1, p);
    else if (p.half <= 128) launch_early(k_qk_q30<4>, grid, QT, 0, st, 1, p);
    else if (p.half <= 256) launch_early(k_qk_q30<8>, grid, QT, 0, st, 1, p);
    else launch_early(k_qk_q30_wide, grid, QT, 0, st, 1, p);
    return 1;
}

}  // namespace slx
