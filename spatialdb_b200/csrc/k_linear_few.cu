// k_linear_few.cu -- the linear operator for few rows (decoded tokens): the weights are read once and
// nothing else matters, so the kernels are built around the weight stream.
//
// 16-bit, up to 16 rows: one block per 16 weight rows, its eight warps taking 64-wide K blocks in turn, two
// at a time (everything they need is asked for before any of it is used; four at a time take the registers
// of half the blocks: 18.3 against 16.5 us, short runs of the first figure below). In the tiled layout 16 rows of a K block are 2 KB in a
// row; a lane loads 16-byte chunks t and t + 4 of rows g and g + 8 (g = lane / 4, t = lane % 4). A chunk's
// eight values feed two m16n8k16 products whose K order is permuted alike on both sides (a sum does not
// care), so weights go from memory to the matrix instruction without shared memory or shuffles; x comes from
// cache in the same order. The tensor pipe is idle most of the time: what counts is the bytes in flight.
// The matrix instructions cut off what they add to a sum; a warp adds an eighth of K, and the eight sums are joined by
// fp32 additions (K 8192, f16, operands of one sign: low by 6e-6; the output's half step is 2.4e-4).
// In a loop of calls bf16 1 x 4096 x 11008 takes 17.7 us, 5100 GB/s; f16 8 x 4096 x 4096 8.5 us, 3960; bf16 1 x 2048 x
// 16384 gated 22.1 us, 6070.
// f32, up to 16 rows: one block per 8 weight rows (4 + 4 when gated), four consecutive K values a lane,
// fp32 FMAs. 1 x 4096 x 11008: 29.4 us, 6130 GB/s.
// Both join the warps' partial sums in shared memory in a fixed order and apply the epilogue there.
#include <algorithm>
#include <cstdint>

#include <cuda_runtime.h>

#include "slx_attr.h"
#include "slx_device.cuh"
#include "slx_linear.h"
#include "slx_linear_dev.cuh"

namespace slx {
namespace lin {
namespace {

constexpr int WARPS = 8, FT = WARPS * 32;

struct FewParams {
    const uint8_t *w, *g;  // tiles (16-bit) or rows (f32)
    const float *bias, *gbias;
    const void *x, *r;
    void* y;
    int64_t ldx, ldr, ldo, k4;
    int M, N, K, nkb, act, parts;
};

template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                        uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                 uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight values of x row m from column k, zeros past K (and a zero row for m >= M).
template <class T, bool VEC>
__device__ __forceinline__ uint4 load_x8(const FewParams& p, int m, int k) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (m >= p.M || k >= p.K) return v;
    const T* x = (const T*)p.x + (int64_t)m * p.ldx + k;
    if (VEC && k + 8 <= p.K) return *(const uint4*)x;
    alignas(16) T e[8];
    *(uint4*)e = v;
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (k + i < p.K) e[i] = x[i];
    return *(const uint4*)e;
}

template <class T>
__device__ __forceinline__ void finish(const FewParams& p, int m, int n, float acc, float gacc, bool gated) {
    float v = acc + (p.bias ? p.bias[n] : 0.0f);
    float a[1] = {gated ? gacc + (p.gbias ? p.gbias[n] : 0.0f) : v};
    activate_all<T>(a, p.act);
    v = gated ? v * a[0] : a[0];
    if (p.r) v += to_f(((const T*)p.r)[(int64_t)m * p.ldr + n]);
    ((T*)p.y)[(int64_t)m * p.ldo + n] = from_f<T>(v);
}

// MT: tiles of 8 activation rows. VEC: x rows start on 16-byte boundaries.
template <class T, int MT, bool GATED, bool VEC>
__global__ void __launch_bounds__(FT) k_few16(FewParams p) {
    constexpr int S = GATED ? 2 : 1, U = GATED ? 1 : 2;  // K blocks a warp has in flight
    __shared__ float red[WARPS][S][MT][8][16];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int grp = blockIdx.x, n0 = grp * 16;
    const int64_t base = ((int64_t)(grp >> 3) * p.nkb * TR + (grp & 7) * 16) * 128;
    const uint8_t* src[2] = {p.w + base, GATED ? p.g + base : nullptr};
    const int off = g * 128 + ((t ^ g) << 4);  // chunk t of row g; chunk t + 4 lies at off ^ 64, row g + 8 1 KB on
    float acc[S][MT][4];
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[s][i][j] = 0.0f;
    grid_wait();
    for (int kb0 = warp; kb0 < p.nkb; kb0 += WARPS * U) {
        // everything the U blocks need is asked for before any of it is used
        uint4 w[U][S][4];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int s = 0; s < S; s++) {
                const int kb = kb0 + u * WARPS;
                const bool live = kb < p.nkb;
                const uint8_t* q = src[s] + (int64_t)kb * TR * 128;
                const uint4 none = make_uint4(0, 0, 0, 0);
                w[u][s][0] = live ? __ldg((const uint4*)(q + off)) : none;
                w[u][s][1] = live ? __ldg((const uint4*)(q + off + 1024)) : none;
                w[u][s][2] = live ? __ldg((const uint4*)(q + (off ^ 64))) : none;
                w[u][s][3] = live ? __ldg((const uint4*)(q + (off ^ 64) + 1024)) : none;
            }
        uint4 x[U][MT][2];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int kb = kb0 + u * WARPS;
                    x[u][i][c] = load_x8<T, VEC>(p, kb < p.nkb ? g + 8 * i : p.M, kb * 64 + c * 32 + t * 8);
                }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int s = 0; s < S; s++) {
                        const uint4 lo = w[u][s][2 * c], hi = w[u][s][2 * c + 1], v = x[u][i][c];
                        mma16816<T>(acc[s][i], lo.x, hi.x, lo.y, hi.y, v.x, v.y);
                        mma16816<T>(acc[s][i], lo.z, hi.z, lo.w, hi.w, v.z, v.w);
                    }
    }
    grid_release();  // not earlier: the next kernel's blocks would share the memory's rate with this one's
#pragma unroll
    for (int s = 0; s < S; s++)
#pragma unroll
        for (int i = 0; i < MT; i++) {
            red[warp][s][i][2 * t][g] = acc[s][i][0];
            red[warp][s][i][2 * t + 1][g] = acc[s][i][1];
            red[warp][s][i][2 * t][g + 8] = acc[s][i][2];
            red[warp][s][i][2 * t + 1][g + 8] = acc[s][i][3];
        }
    __syncthreads();
    for (int o = threadIdx.x; o < 128 * MT; o += FT) {
        const int row = o & 15, col = (o >> 4) & 7, i = o >> 7, m = col + 8 * i, n = n0 + row;
        if (m >= p.M || n >= p.N) continue;
        float v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int q = 0; q < WARPS; q++) v[s] += red[q][s][i][col][row];
        finish<T>(p, m, n, v[0], v[1], GATED);
    }
}

template <bool VEC>
__device__ __forceinline__ float4 load_x4(const FewParams& p, int m, int64_t k) {
    const float* x = (const float*)p.x + (int64_t)m * p.ldx + k;
    if (VEC && k + 4 <= p.K) return *(const float4*)x;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (k < p.K) v.x = x[0];
    if (k + 1 < p.K) v.y = x[1];
    if (k + 2 < p.K) v.z = x[2];
    if (k + 3 < p.K) v.w = x[3];
    return v;
}

// MB: activation rows of a block (1, 2, 4, 8). More rows than that are shared by p.parts neighbouring blocks,
// which read the same weights at about the same time (from L2, but for the first).
template <int MB, bool GATED, bool VEC>
__global__ void __launch_bounds__(FT, MB >= 4 ? 2 : 3) k_few32(FewParams p) {
    constexpr int S = GATED ? 2 : 1, R = 8 / S, NV = 8 * MB;  // weight rows a block, sums a lane
    __shared__ float red[WARPS][NV];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = (int)(blockIdx.x / p.parts) * R, m0 = (int)(blockIdx.x % p.parts) * MB, rows = min(p.M - m0, MB);
    const float* row[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int n = min(n0 + i % R, p.N - 1);  // rows past N repeat the last one and are not stored
        row[i] = (const float*)(i < R ? p.w : p.g) + (int64_t)n * p.k4;
    }
    float acc[NV];
#pragma unroll
    for (int i = 0; i < NV; i++) acc[i] = 0.0f;
    grid_release();
    float4 w[8];
    auto weights = [&](int64_t k) {
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = __ldg((const float4*)(row[i] + k));
    };
    const int64_t k0 = (int64_t)threadIdx.x * 4;
    if (k0 < p.k4) weights(k0);  // the handle's own memory: no kernel in the stream writes it
    grid_wait();
    for (int64_t k = k0; k < p.k4; k += FT * 4) {
        if (k != k0) weights(k);
#pragma unroll
        for (int m = 0; m < MB; m++) {
            if (m >= rows) break;
            const float4 x = load_x4<VEC>(p, m0 + m, k);
#pragma unroll
            for (int i = 0; i < 8; i++)
                acc[i * MB + m] = fmaf(w[i].x, x.x, fmaf(w[i].y, x.y, fmaf(w[i].z, x.z, fmaf(w[i].w, x.w, acc[i * MB + m]))));
        }
    }
    // sums over the lanes, halving the values each lane carries while there are any to halve
    int have = NV, first = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        if (have > 1) {
            const bool up = lane & o;
            have /= 2;
#pragma unroll
            for (int i = 0; i < NV / 2; i++) {
                if (i >= have) break;
                const float send = up ? acc[i] : acc[i + have];
                const float keep = up ? acc[i + have] : acc[i];
                acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
            }
            first += up ? have : 0;
        } else {
            acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
        }
    }
#pragma unroll
    for (int i = 0; i < (NV > 32 ? NV / 32 : 1); i++) red[warp][first + i] = acc[i];
    __syncthreads();
    for (int o = threadIdx.x; o < R * MB; o += FT) {
        const int i = o / MB, m = o % MB, n = n0 + i;
        if (m >= rows || n >= p.N) continue;
        float v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int q = 0; q < WARPS; q++) v[s] += red[q][(i + s * R) * MB + m];
        finish<float>(p, m0 + m, n, v[0], v[1], GATED);
    }
}

template <class T, bool GATED, bool VEC>
void launch16(const FewParams& p, cudaStream_t st) {
    const unsigned grid = (unsigned)((p.N + 15) / 16);
    if (p.M <= 8) launch_early(k_few16<T, 1, GATED, VEC>, grid, FT, 0, st, 1, p);
    else launch_early(k_few16<T, 2, GATED, VEC>, grid, FT, 0, st, 1, p);
}
template <bool GATED, bool VEC>
void launch32(FewParams p, cudaStream_t st) {
    // Up to eight rows to a block, four where eight would leave SMs without work (8 x 768 x 768: 4.0 and 3.2 us;
    // 5 x 768 x 2304: 4.0 and 5.2).
    const int64_t groups = GATED ? (p.N + 3) / 4 : (p.N + 7) / 8;
    const int most = 2 * groups * ((p.M + 7) / 8) < 3 * device_sm_count() ? 4 : 8;
    p.parts = (p.M + most - 1) / most;
    const int mb = (p.M + p.parts - 1) / p.parts;
    const unsigned grid = (unsigned)(groups * p.parts);
    if (p.M <= 1) launch_early(k_few32<1, GATED, VEC>, grid, FT, 0, st, 1, p);
    else if (p.M <= 2) launch_early(k_few32<2, GATED, VEC>, grid, FT, 0, st, 1, p);
    else if (mb <= 4) launch_early(k_few32<4, GATED, VEC>, grid, FT, 0, st, 1, p);
    else launch_early(k_few32<8, GATED, VEC>, grid, FT, 0, st, 1, p);
}
}  // namespace

// f32 past 4 rows: the sums leave few registers for loads, and the tensor-core form, which reads six bytes a
// weight instead of four, catches up (us here and there: 8 x 768 x 2304 4.2, 9.1; 8 x 4096 x 4096 30.8, 24.2;
// 16 x 768 x 2304 7.8, 9.1; 10 x 8096 x 32 9.6, 24.8; 11 x 1632 x 10016 38.2, 36.2; 16 x 4096 x 4096 46.7, 24.2).
bool few_supported(const Plan& p, int64_t M) {
    if (p.dtype != DT_F32 || M <= 4) return M <= 16;
    const int64_t weights = (int64_t)p.N * p.K * (p.gated ? 2 : 1);
    return M <= 16 && weights <= (M <= 8 ? 8 << 20 : 4 << 20);
}

int few(const Plan& pl, const Call& c, cudaStream_t st) {
    FewParams p;
    const bool f32 = pl.dtype == DT_F32;
    p.w = f32 ? (const uint8_t*)pl.rows : pl.tiles;
    p.g = f32 ? (const uint8_t*)pl.grows : pl.gtiles;
    p.bias = pl.bias; p.gbias = pl.gbias;
    p.x = c.x; p.r = c.r; p.y = c.y;
    p.ldx = c.ldx; p.ldr = c.ldr; p.ldo = c.ldo; p.k4 = pl.k4();
    p.M = (int)c.M; p.N = pl.N; p.K = pl.K; p.nkb = pl.nkb(); p.act = pl.act; p.parts = 1;
    const bool vec = (uintptr_t)c.x % 16 == 0 && (c.M == 1 || c.ldx % (f32 ? 4 : 8) == 0);
#define SLX_PICK(fn, ...)                                                         \
    do {                                                                          \
        if (pl.gated) vec ? fn<__VA_ARGS__ true, true>(p, st) : fn<__VA_ARGS__ true, false>(p, st);  \
        else vec ? fn<__VA_ARGS__ false, true>(p, st) : fn<__VA_ARGS__ false, false>(p, st);         \
    } while (0)
#define SLX_COMMA ,
    if (f32) SLX_PICK(launch32, );
    else if (pl.dtype == DT_F16) SLX_PICK(launch16, __half SLX_COMMA);
    else SLX_PICK(launch16, __nv_bfloat16 SLX_COMMA);
#undef SLX_PICK
#undef SLX_COMMA
    return 1;
}

}  // namespace lin
}  // namespace slx
