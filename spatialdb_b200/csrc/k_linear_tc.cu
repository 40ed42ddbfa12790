// k_linear_tc.cu -- the linear operator on the 5th-generation tensor cores (tcgen05.mma kind::f16, fp32
// accumulators in TMEM).
//
// A tile is 128 weight rows (the MMA's M: one TMEM lane each) x NT activation rows (its N). Weights are
// laid out once in the swizzled blocks that the MMA reads, so a K block of a tile is one contiguous
// untiled bulk copy; activations come through a TMA tensor map on the caller's rows (a packed copy when
// their base or stride is not a multiple of 16 bytes). Warp 0 loads, warp 1 issues the MMAs, eight
// warps run the epilogue: bias, activation, gate, residual and the one rounding, out of TMEM.
//
// f32 (PLANES = 3): each value is the exact sum of three bf16 parts (8 significant bits each, by
// truncation), x = x1 + x2 + x3. x1 w1 goes to one accumulator, the corrections x1 w2 + x2 w1 + x2 w2 +
// x1 w3 + x3 w1 (at most 2^-8 of it) to another; what is left out is below 2^-23 |x| |w|. The tensor core
// truncates when it adds to an accumulator, which biases long sums, so every 256 values of K both
// accumulators are added to fp32 registers (rounded to nearest) and started anew.
//
// SPLIT: fewer tiles than SMs; a cluster of S CTAs shares a tile, each with a range of the K blocks. The
// partial sums meet in shared memory: CTA c adds columns c NT / S... of all S partials, in rank order, over
// distributed shared memory, and finishes them. One launch, no workspace, the same result every time.
// Otherwise the kernel is persistent: one CTA per SM walks the tiles, the epilogue of one under the
// MMAs of the next (two accumulators). Every mbarrier wait is bounded.
#include <cuda.h>

#include <algorithm>
#include <cstring>

#include "slx_attr.h"
#include "slx_device.cuh"
#include "slx_gemm.h"
#include "slx_linear.h"
#include "slx_linear_dev.cuh"
#include "tc_ptx.cuh"

namespace slx {
namespace lin {
namespace {

using namespace tc;

constexpr int EPI = 8;                      // epilogue warps: two per TMEM lane quarter
constexpr int LT = 32 * (2 + EPI);          // threads
constexpr int SMEM_MAX = 227 * 1024;
constexpr int CHUNK = 8;                    // f32: K blocks (of 32) between promotions to registers

struct TcParams {
    const uint8_t *w, *g;
    const float *bias, *gbias;
    const void* r;
    void* y;
    int64_t ldr, ldo;
    int M, N, nkb, act, f16;
    int tiles_n, tiles, split;
    int* err;
    long long wait_limit;
    int stall_mma;
};

template <int NT, int PLANES, bool GATED>
struct Shape {
    static constexpr int S = GATED ? 2 : 1;
    static constexpr int ROWB = PLANES == 3 ? 64 : 128;        // bytes of K per operand row and block
    static constexpr int WB = PLANES * TR * ROWB;              // one weight array's block
    static constexpr int XB = PLANES * NT * ROWB;
    static constexpr int STAGE = S * WB + XB;
    static constexpr int ACC = S * (PLANES == 3 ? 2 : 1);      // accumulators of NT columns
    static constexpr int COLS = 2 * ACC * NT;                  // two buffers
    static constexpr int STAGES = (SMEM_MAX - 1024 - 512) / STAGE > 8 ? 8 : (SMEM_MAX - 1024 - 512) / STAGE;
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + 1024 + 512;
    static_assert(COLS <= 512 && STAGES >= 2, "tile does not fit");
    static_assert((size_t)S * NT * TR * 4 <= (size_t)STAGES * STAGE, "split partials reuse the stages");
};

__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_ld(uint32_t addr, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// Instruction descriptor, kind::f16: D f32, A and B both f16 (0) or both bf16 (1), K-major, M = 128, N = n.
__device__ __forceinline__ uint32_t idesc_f16(int n, int bf16) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

template <class T>
__device__ __forceinline__ void store_one(const TcParams& p, int64_t m, int n, float v, float gv, float b, float gb, bool gated,
                                          float res) {
    v += b;
    if (gated) v *= activate(gv + gb, p.act);
    else v = activate(v, p.act);
    ((T*)p.y)[m * p.ldo + n] = from_f<T>(v + res);
}

template <class T, int NT, int PLANES, bool GATED, bool SPLIT>
__global__ void __launch_bounds__(LT, 1) k_linear_tc(const __grid_constant__ CUtensorMap tmx, TcParams p) {
    using Sh = Shape<NT, PLANES, GATED>;
    constexpr int S = Sh::S, ST = Sh::STAGES, ROWB = Sh::ROWB;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = (uint64_t*)(smem + (size_t)ST * Sh::STAGE);
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + ST);
    const uint32_t tfull0 = smem_u32(bars + 2 * ST), tfree0 = smem_u32(bars + 2 * ST + 2);
    const uint32_t drain = smem_u32(bars + 2 * ST + 4);
    uint32_t* tmem_slot = (uint32_t*)(bars + 2 * ST + 5);
    __shared__ int s_fail;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long limit = p.wait_limit;
    if (threadIdx.x == 0) {
        s_fail = 0;
        for (int i = 0; i < ST; i++) {
            mbar_init(full0 + 8 * i, 1);
            mbar_init(empty0 + 8 * i, 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(tfull0 + 8 * b, 1);
            mbar_init(tfree0 + 8 * b, EPI);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    constexpr int ALLOC = Sh::COLS <= 32 ? 32 : Sh::COLS <= 64 ? 64 : Sh::COLS <= 128 ? 128 : Sh::COLS <= 256 ? 256 : 512;
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(ALLOC));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot, sbase = smem_u32(smem);

    // This CTA's tiles and K blocks.
    const int rank = SPLIT ? (int)cluster_rank() : 0;
    const int tile0 = SPLIT ? (int)blockIdx.x / p.split : (int)blockIdx.x;
    const int tstep = SPLIT ? p.tiles : (int)gridDim.x;
    const int kb0 = SPLIT ? (int)((int64_t)p.nkb * rank / p.split) : 0;
    const int kb1 = SPLIT ? (int)((int64_t)p.nkb * (rank + 1) / p.split) : p.nkb;
    constexpr int CH = PLANES == 3 ? CHUNK : 1 << 30;

    if (warp == 0) {
        if (lane == 0) {  // producer, running ahead across tiles
            int done = 0, s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = tile0; ok && t < p.tiles; t += tstep) {
                const int nt = t % p.tiles_n, m0 = (t / p.tiles_n) * NT;
                const int64_t blk0 = (int64_t)nt * p.nkb;
                for (int kb = kb0; kb < kb1; kb++, done++) {
                    if (!mbar_wait(empty0 + 8 * s, ph ^ 1u, limit) || *(volatile int*)&s_fail) {
                        s_fail = 1;
                        ok = false;
                        break;
                    }
                    const uint32_t dst = sbase + s * Sh::STAGE, bar = full0 + 8 * s;
                    mbar_expect_tx(bar, Sh::STAGE);
                    bulk_load(dst, p.w + (blk0 + kb) * Sh::WB, Sh::WB, bar);
                    if (GATED) bulk_load(dst + Sh::WB, p.g + (blk0 + kb) * Sh::WB, Sh::WB, bar);
                    tma_load_3d(dst + S * Sh::WB, &tmx, kb * (ROWB / 2), m0, 0, bar);
                    if (++s == ST) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok)  // let copies still in flight land before the CTA exits (they always complete)
                for (int j = done - ST < 0 ? 0 : done - ST; j < done; j++)
                    mbar_wait(full0 + 8 * (j % ST), (uint32_t)(j / ST) & 1u);
        }
    } else if (warp == 1) {
        if (lane == 0) {  // MMA issuer
            const uint32_t idesc = idesc_f16(NT, !p.f16);
            int use = 0, s = 0;
            uint32_t ph = 0;
            bool ok = true, issued = false;
            for (int t = tile0; ok && t < p.tiles; t += tstep) {
                for (int c0 = kb0; ok && c0 < kb1; c0 += CH, use++) {
                    const int c1 = kb1 - c0 < CH ? kb1 : c0 + CH, b = use & 1;
                    if (!mbar_wait(tfree0 + 8 * b, ((uint32_t)(use >> 1) & 1u) ^ 1u, limit)) { ok = false; break; }
                    fence_after();
                    const uint32_t d = tmem + b * Sh::ACC * NT;
                    for (int kb = c0; kb < c1; kb++) {
                        if (p.stall_mma || !mbar_wait(full0 + 8 * s, ph, limit)) { ok = false; break; }
                        fence_after();
                        const uint32_t w = sbase + s * Sh::STAGE, x = w + S * Sh::WB;
#pragma unroll
                        for (int kk = 0; kk < ROWB / 32; kk++) {
                            const uint32_t first = kb == c0 && kk == 0 ? 0u : 1u;
#pragma unroll
                            for (int v = 0; v < S; v++) {
                                if (PLANES == 1) {
                                    umma_f16(d + v * NT, sw128_desc(w + v * Sh::WB + kk * 32), sw128_desc(x + kk * 32), idesc, first);
                                } else {
                                    const uint32_t wb = w + v * Sh::WB + kk * 32, xb = x + kk * 32;
                                    const uint64_t w1 = sw64_desc(wb), w2 = sw64_desc(wb + TR * ROWB), w3 = sw64_desc(wb + 2 * TR * ROWB);
                                    const uint64_t x1 = sw64_desc(xb), x2 = sw64_desc(xb + NT * ROWB), x3 = sw64_desc(xb + 2 * NT * ROWB);
                                    const uint32_t da = d + 2 * v * NT, db = da + NT;
                                    umma_f16(da, w1, x1, idesc, first);
                                    umma_f16(db, w1, x2, idesc, first);
                                    umma_f16(db, w2, x1, idesc, 1u);
                                    umma_f16(db, w2, x2, idesc, 1u);
                                    umma_f16(db, w1, x3, idesc, 1u);
                                    umma_f16(db, w3, x1, idesc, 1u);
                                }
                            }
                        }
                        umma_commit(empty0 + 8 * s);
                        issued = true;
                        if (++s == ST) { s = 0; ph ^= 1u; }
                    }
                    if (!ok) break;
                    umma_commit(tfull0 + 8 * b);
                }
            }
            if (!ok) {
                s_fail = 1;
                if (issued) {  // MMAs still in flight write TMEM: let them retire before it is freed
                    umma_commit(drain);
                    mbar_wait(drain, 0u);
                }
            }
        }
    } else {  // epilogue: thread = weight row (TMEM lane), half of the tile's activation rows
        const int q4 = warp & 3, part = (warp - 2) >> 2;
        constexpr int HC = NT / 2;  // columns of a thread
        const uint32_t lane_base = (uint32_t)(32 * q4) << 16;
        int use = 0;
        for (int t = tile0; t < p.tiles; t += tstep) {
            const int nt = t % p.tiles_n;
            const int64_t m0 = (int64_t)(t / p.tiles_n) * NT + part * HC;
            const int n = nt * TR + 32 * q4 + lane;
            const bool in = n < p.N;
            const float b = in && p.bias ? p.bias[n] : 0.0f, gb = GATED && in && p.gbias ? p.gbias[n] : 0.0f;
            float acc[PLANES == 3 ? S : 1][PLANES == 3 ? HC : 1];  // f32: the promoted sums
            bool ok = true;
            int chunks = 0;
            for (int c0 = kb0; c0 < kb1; c0 += CH, use++, chunks++) {
                const int buf = use & 1;
                if (!__all_sync(0xffffffffu, mbar_wait(tfull0 + 8 * buf, (uint32_t)(use >> 1) & 1u, limit))) {
                    s_fail = 1;
                    ok = false;
                    break;
                }
                fence_after();
                if (PLANES == 3) {
#pragma unroll
                    for (int v = 0; v < S; v++)
#pragma unroll
                        for (int c = 0; c < HC; c += 16) {
                            uint32_t a[16], k[16];
                            const uint32_t at = tmem + lane_base + (buf * Sh::ACC + 2 * v) * NT + part * HC + c;
                            tmem_ld16(at, a);
                            tmem_ld16(at + NT, k);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int j = 0; j < 16; j++) {
                                const float sum = __uint_as_float(a[j]) + __uint_as_float(k[j]);
                                acc[v][c + j] = chunks ? acc[v][c + j] + sum : sum;
                            }
                        }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tfree0 + 8 * buf);
                }
            }
            if (!ok) break;
            const int buf = (use - 1) & 1;
            if (!SPLIT) {
#pragma unroll
                for (int c = 0; c < HC; c += 16) {
                    float res[16], v[16], g[16];
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        res[j] = p.r && in && m0 + c + j < p.M ? to_f(((const T*)p.r)[(m0 + c + j) * p.ldr + n]) : 0.0f;
                    if (PLANES == 1) {
                        uint32_t a[16], k[16];
                        const uint32_t at = tmem + lane_base + buf * Sh::ACC * NT + part * HC + c;
                        tmem_ld16(at, a);
                        if (GATED) tmem_ld16(at + NT, k);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            v[j] = __uint_as_float(a[j]);
                            g[j] = GATED ? __uint_as_float(k[j]) : 0.0f;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            v[j] = acc[0][c + j];
                            g[j] = GATED ? acc[S - 1][c + j] : 0.0f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (in && m0 + c + j < p.M) store_one<T>(p, m0 + c + j, n, v[j], g[j], b, gb, GATED, res[j]);
                }
                if (PLANES == 1) {
                    fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tfree0 + 8 * buf);
                }
            } else {  // this CTA's partial sums, [v][column][weight row], over the stages (all consumed)
                float* part_sums = (float*)smem;
#pragma unroll
                for (int v = 0; v < S; v++)
#pragma unroll
                    for (int c = 0; c < HC; c += 16) {
                        float* dst = part_sums + ((int64_t)v * NT + part * HC + c) * TR + 32 * q4 + lane;
                        if (PLANES == 1) {
                            uint32_t a[16];
                            tmem_ld16(tmem + lane_base + (buf * Sh::ACC + v) * NT + part * HC + c, a);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int j = 0; j < 16; j++) dst[j * TR] = __uint_as_float(a[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 16; j++) dst[j * TR] = acc[v][c + j];
                        }
                    }
            }
        }
    }
    fence_before();
    __syncthreads();
    if (SPLIT) {
        cluster_sync();  // every CTA's partial sums are in its shared memory (or it failed and said so)
        if (!s_fail && warp >= 2) {
            const int i = (int)threadIdx.x - 64, row = i & (TR - 1), sub = i >> 7;
            const int n = (tile0 % p.tiles_n) * TR + row, cols = NT / p.split;
            const int64_t m0 = (int64_t)(tile0 / p.tiles_n) * NT;
            const float b = n < p.N && p.bias ? p.bias[n] : 0.0f, gb = GATED && n < p.N && p.gbias ? p.gbias[n] : 0.0f;
            for (int c = rank * cols + sub; c < (rank + 1) * cols; c += EPI * 32 / TR) {
                const int64_t m = m0 + c;
                if (m >= p.M || n >= p.N) continue;
                float v = 0.0f, g = 0.0f;
                for (int q = 0; q < p.split; q++) {
                    v += peer_ld(sbase + (uint32_t)(c * TR + row) * 4, q);
                    if (GATED) g += peer_ld(sbase + (uint32_t)((NT + c) * TR + row) * 4, q);
                }
                const float res = p.r ? to_f(((const T*)p.r)[m * p.ldr + n]) : 0.0f;
                store_one<T>(p, m, n, v, g, b, gb, GATED, res);
            }
        }
        cluster_sync();  // no CTA leaves while another reads its partial sums
    }
    if (s_fail && threadIdx.x == 0 && p.err) atomicOr(p.err, KERR_TIMEOUT);
    if (warp == 1) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(ALLOC));
    }
}

// ---- layouts ----------------------------------------------------------------------------------------

__device__ __forceinline__ uint16_t bf16_cut(float v) { return (uint16_t)(__float_as_uint(v) >> 16); }

// The three bf16 parts of an fp32 value, each the leading eight significant bits of what is left
// (truncated, so no part overflows): their sum is the value exactly. A value that is not finite keeps
// itself in the first part (a NaN stays one) and zeros in the others.
__device__ __forceinline__ void split3(float v, uint16_t (&o)[3]) {
    o[0] = bf16_cut(v);
    o[1] = o[2] = 0;
    if (!isfinite(v)) {
        if (isnan(v)) o[0] |= 0x40;
        return;
    }
    const float r1 = v - __uint_as_float((uint32_t)o[0] << 16);
    o[1] = bf16_cut(r1);
    o[2] = bf16_cut(r1 - __uint_as_float((uint32_t)o[1] << 16));
}

// One thread per 16-byte chunk of the tiles.
__global__ void k_tiles16(const uint16_t* __restrict__ w, int N, int K, int nkb, int64_t chunks, uint4* __restrict__ out) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * blockDim.x) {
        const int c = (int)(i & 7), row = (int)(i >> 3) & (TR - 1);
        const int64_t blk = i >> 10;  // tile * nkb + kb
        const int64_t n = blk / nkb * TR + row;
        const int k = (int)(blk % nkb) * 64 + c * 8;
        uint16_t e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = n < N && k + j < K ? w[n * K + k + j] : (uint16_t)0;
        out[(i & ~(int64_t)7) | (c ^ (row & 7))] = *(const uint4*)e;
    }
}

// f32: a thread forms one 16-byte chunk (eight values) of each of the three planes of a block.
__global__ void k_tiles32(const float* __restrict__ w, int N, int K, int nkb, int64_t chunks, uint8_t* __restrict__ out) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * blockDim.x) {
        const int c = (int)(i & 3), row = (int)(i >> 2) & (TR - 1);
        const int64_t blk = i >> 9;
        const int64_t n = blk / nkb * TR + row;
        const int k = (int)(blk % nkb) * 32 + c * 8;
        uint16_t e[3][8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint16_t o[3];
            split3(n < N && k + j < K ? w[n * K + k + j] : 0.0f, o);
#pragma unroll
            for (int q = 0; q < 3; q++) e[q][j] = o[q];
        }
#pragma unroll
        for (int q = 0; q < 3; q++)
            *(uint4*)(out + blk * (3 * TR * 64) + q * (TR * 64) + row * 64 + ((c ^ ((row >> 1) & 3)) << 4)) = *(const uint4*)e[q];
    }
}

__global__ void k_rows4(const float* __restrict__ w, int64_t N, int K, int64_t k4, float* __restrict__ out) {
    const int64_t total = N * k4;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x)
        out[i] = i % k4 < K ? w[i / k4 * K + i % k4] : 0.0f;
}

// The activations' three planes [3][M][kp], kp a multiple of 32, zeros past K.
__global__ void k_split_x(const float* __restrict__ x, int64_t ldx, int64_t M, int K, int kp, uint16_t* __restrict__ out) {
    const int64_t total = M * (kp / 8);
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t m = i / (kp / 8);
        const int k = (int)(i % (kp / 8)) * 8;
        const float* src = x + m * ldx + k;
        float f[8];
        if (k + 8 <= K && ((uintptr_t)src & 15) == 0) {
            *(float4*)f = *(const float4*)src;
            *(float4*)(f + 4) = *(const float4*)(src + 4);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = k + j < K ? src[j] : 0.0f;
        }
        uint16_t e[3][8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            uint16_t o[3];
            split3(f[j], o);
#pragma unroll
            for (int q = 0; q < 3; q++) e[q][j] = o[q];
        }
#pragma unroll
        for (int q = 0; q < 3; q++) *(uint4*)(out + (q * M + m) * kp + k) = *(const uint4*)e[q];
    }
}

// 16-bit rows whose base or stride TMA cannot address, packed to rows of kp (a multiple of 8).
__global__ void k_pack_x(const uint16_t* __restrict__ x, int64_t ldx, int64_t M, int K, int kp, uint16_t* __restrict__ out) {
    const int64_t total = M * (kp / 8);
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t m = i / (kp / 8);
        const int k = (int)(i % (kp / 8)) * 8;
        uint16_t e[8];
#pragma unroll
        for (int j = 0; j < 8; j++) e[j] = k + j < K ? x[m * ldx + k + j] : (uint16_t)0;
        *(uint4*)(out + m * kp + k) = *(const uint4*)e;
    }
}

unsigned grid_for(int64_t items) { return (unsigned)std::min<int64_t>((items + 255) / 256, (int64_t)device_sm_count() * 16); }

int kp_of(const Plan& p) { return p.planes() == 3 ? p.nkb() * 32 : (p.K + 7) / 8 * 8; }

bool tma_rows(const Plan& p, const Call& c) {  // the caller's 16-bit rows as they are
    return p.planes() == 1 && (uintptr_t)c.x % 16 == 0 && c.ldx % 8 == 0;
}

template <class T, int NT, int PLANES, bool GATED, bool SPLIT>
bool launch(const CUtensorMap& tm, const TcParams& p, int grid, cudaStream_t st) {
    using Sh = Shape<NT, PLANES, GATED>;
    auto* fn = k_linear_tc<T, NT, PLANES, GATED, SPLIT>;
    if (ensure_smem((const void*)fn, Sh::SMEM) != cudaSuccess) return false;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(LT);
    cfg.dynamicSmemBytes = Sh::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    if (SPLIT) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)p.split;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, fn, tm, p) == cudaSuccess;
}

template <class T, int NT, int PLANES, bool GATED>
bool run(const Plan& pl, const Call& c, const void* x, int64_t ldx, cudaStream_t st) {
    CUtensorMap tm;
    const int kp = kp_of(pl);
    if (!tc::encode_rows_planes(&tm, x, PLANES == 1 && x == c.x ? pl.K : kp, c.M, ldx, PLANES, pl.bk(), NT)) return false;
    TcParams p;
    p.w = pl.tiles; p.g = pl.gtiles; p.bias = pl.bias; p.gbias = pl.gbias;
    p.r = c.r; p.y = c.y; p.ldr = c.ldr; p.ldo = c.ldo;
    p.M = (int)c.M; p.N = pl.N; p.nkb = pl.nkb(); p.act = pl.act; p.f16 = pl.dtype == DT_F16;
    p.tiles_n = pl.tiles_n();
    p.tiles = p.tiles_n * (int)((c.M + NT - 1) / NT);
    p.err = c.err;
    p.wait_limit = c.wait_limit > 0 ? c.wait_limit : tc::kWaitCycles;
    p.stall_mma = c.stall_mma;
    const int sms = device_sm_count();
    p.split = 1;
    while (p.split < 8 && p.tiles * p.split * 2 <= sms && p.nkb >= p.split * 4) p.split *= 2;
    if (p.split > 1) return launch<T, NT, PLANES, GATED, true>(tm, p, p.tiles * p.split, st);
    return launch<T, NT, PLANES, GATED, false>(tm, p, std::min(p.tiles, sms), st);
}

template <class T, int PLANES>
bool pick_tile(const Plan& pl, const Call& c, const void* x, int64_t ldx, cudaStream_t st) {
    if (pl.gated) {
        if (c.M <= 32) return run<T, 32, PLANES, true>(pl, c, x, ldx, st);
        if (PLANES == 3 || c.M <= 64) return run<T, 64, PLANES, true>(pl, c, x, ldx, st);
        return run<T, PLANES == 3 ? 64 : 128, PLANES, true>(pl, c, x, ldx, st);
    }
    if (c.M <= 32) return run<T, 32, PLANES, false>(pl, c, x, ldx, st);
    if (c.M <= 64) return run<T, 64, PLANES, false>(pl, c, x, ldx, st);
    const int64_t wide = (c.M + 255) / 256 * pl.tiles_n();
    if (PLANES == 3 || c.M <= 128 || wide < device_sm_count()) return run<T, 128, PLANES, false>(pl, c, x, ldx, st);
    return run<T, PLANES == 3 ? 128 : 256, PLANES, false>(pl, c, x, ldx, st);
}
}  // namespace

void layout(const Plan& p, const void* w, uint8_t* tiles, float* rows, cudaStream_t st) {
    const int64_t chunks = (int64_t)p.tiles_n() * p.nkb() * TR * (p.bk() / 8);
    if (p.planes() == 1) {
        k_tiles16<<<grid_for(chunks), 256, 0, st>>>((const uint16_t*)w, p.N, p.K, p.nkb(), chunks, (uint4*)tiles);
        return;
    }
    k_tiles32<<<grid_for(chunks), 256, 0, st>>>((const float*)w, p.N, p.K, p.nkb(), chunks, tiles);
    k_rows4<<<grid_for(p.N * p.k4()), 256, 0, st>>>((const float*)w, p.N, p.K, p.k4(), rows);
}

size_t tc_workspace(const Plan& p, const Call& c) {
    if (tma_rows(p, c)) return 0;
    return (size_t)p.planes() * c.M * kp_of(p) * 2;
}

int tc(const Plan& p, const Call& c, void* ws, cudaStream_t st) {
    const void* x = c.x;
    int64_t ldx = c.ldx;
    int n = 0;
    if (!tma_rows(p, c)) {
        const int kp = kp_of(p);
        const unsigned grid = grid_for(c.M * (kp / 8));
        if (p.planes() == 3) k_split_x<<<grid, 256, 0, st>>>((const float*)c.x, c.ldx, c.M, p.K, kp, (uint16_t*)ws);
        else k_pack_x<<<grid, 256, 0, st>>>((const uint16_t*)c.x, c.ldx, c.M, p.K, kp, (uint16_t*)ws);
        x = ws;
        ldx = kp;
        n++;
    }
    bool ok;
    if (p.dtype == DT_F32) ok = pick_tile<float, 3>(p, c, x, ldx, st);
    else if (p.dtype == DT_F16) ok = pick_tile<__half, 1>(p, c, x, ldx, st);
    else ok = pick_tile<__nv_bfloat16, 1>(p, c, x, ldx, st);
    return ok ? n + 1 : -1;
}

}  // namespace lin
}  // namespace slx
