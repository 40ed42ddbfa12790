// k_linear_tc.cu -- the linear operator on the 5th-generation tensor cores (tcgen05.mma kind::f16, fp32
// accumulators in TMEM).
//
// A tile is 128 weight rows a CTA (one TMEM lane each) x NT activation rows (the MMA's N). Weights are
// laid out once in the swizzled blocks that the MMA reads, so a K block of a tile is one contiguous
// copy; activations come through a TMA tensor map on the caller's rows (a packed copy when their base
// or stride is not a multiple of 16 bytes). Warp 0 loads, warp 1 issues the MMAs, eight warps run the
// epilogue: 16 columns at a time go from TMEM through shared memory, so that bias, activation, gate,
// residual and the one rounding run on eight consecutive outputs of a row with 16-byte accesses.
//
// f32 (PLANES = 3): each value is the exact sum of three bf16 parts (8 significant bits each, by
// truncation), x = x1 + x2 + x3. x1 w1 goes to one accumulator, the corrections x1 w2 + x2 w1 + x2 w2 +
// x1 w3 + x3 w1 (at most 2^-8 of it) to another; what is left out is below 2^-23 |x| |w|. The tensor core
// truncates when it adds to an accumulator, which biases long sums, so every 256 values of K both
// accumulators are added to fp32 registers (rounded to nearest) and started anew.
//
// Three forms, by the number of tiles:
//   SPLIT   fewer tiles than SMs: a cluster of up to 8 CTAs shares a tile, each with a range of the K
//           blocks. CTA c of S adds columns c NT / S... of all partial sums, in rank order, over
//           distributed shared memory, and finishes them. One launch, no workspace, the same result every time.
//   SINGLE  persistent, one CTA per SM, the epilogue of a tile under the MMAs of the next (two accumulators).
//   PAIR    persistent, two CTAs (cta_group::2) on 256 weight rows: each loads its own 128 weight rows and
//           half of the activation rows, which halves the activation bytes per MMA.
// Every mbarrier wait is bounded.
#include <cuda.h>

#include <algorithm>
#include <atomic>
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

enum Mode { SINGLE = 0, SPLIT = 1, PAIR = 2 };

constexpr int EPI = 8;                      // epilogue warps: two per TMEM lane quarter
constexpr int LT = 32 * (2 + EPI);          // threads
constexpr int SMEM_MAX = 227 * 1024;
constexpr int CHUNK = 8;                    // f32: K blocks (of 32) between promotions to registers
constexpr int SLAB = 16;                    // columns the epilogue moves through shared memory at a time
constexpr int GROUP_M = 8;                  // activation tiles walked together (their rows stay in L2)

struct TcParams {
    const uint8_t *w, *g;
    const float *bias, *gbias;
    const void* r;
    void* y;
    int64_t ldr, ldo;
    int M, N, nkb, act, f16, vec;
    int tiles_n, tiles_m, tiles, split;
    int* err;
    long long wait_limit;
    int stall_mma;
};

template <int NT, int PLANES, bool GATED, int MODE>
struct Shape {
    static constexpr int S = GATED ? 2 : 1;
    static constexpr int ROWB = PLANES == 3 ? 64 : 128;        // bytes of K per operand row and block
    static constexpr int WB = PLANES * TR * ROWB;              // one weight array's block
    static constexpr int XR = MODE == PAIR ? NT / 2 : NT;      // activation rows this CTA loads
    static constexpr int STAGE = S * WB + PLANES * XR * ROWB;
    static constexpr int ACC = S * (PLANES == 3 ? 2 : 1);      // accumulators of NT columns
    static constexpr int COLS = 2 * ACC * NT;                  // two buffers
    static constexpr int OUT = 2 * S * SLAB * TR * 4;          // epilogue staging, both groups of four warps
    static constexpr int FIT = (SMEM_MAX - 1024 - 512 - OUT) / STAGE;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + OUT + 1024 + 512;
    static_assert(COLS <= 512 && STAGES >= 2, "tile does not fit");
    static_assert((size_t)S * NT * TR * 4 <= (size_t)STAGES * STAGE || MODE != SPLIT, "split partials reuse the stages");
};

template <int CG>
__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if (CG == 1)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc));
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

// Completion of the MMAs issued so far: one arrival at `bar`, in a pair at the same place of both CTAs.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
    if (CG == 1)
        umma_commit(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                     "h"((uint16_t)3)
                     : "memory");
}

// Tiled loads of a pair: into this CTA's shared memory, counted on a barrier of the leading CTA.
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            dst),
        "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
        : "memory");
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
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ float4 peer_ld4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ void peer_arrive(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

// Instruction descriptor, kind::f16: D f32, A and B both f16 (0) or both bf16 (1), K-major, N = n.
__device__ __forceinline__ uint32_t idesc_f16(int m, int n, int bf16) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Eight consecutive outputs n.. of row m from their sums (and gate sums): the epilogue proper.
template <class T>
struct Eight {
    float r[8];  // residual
    bool vec, any;

    __device__ __forceinline__ void load(const TcParams& p, int64_t m, int n) {
        any = m < p.M && n < p.N;
        vec = any && p.vec && n + 8 <= p.N;
#pragma unroll
        for (int j = 0; j < 8; j++) r[j] = 0.0f;
        if (!p.r || !any) return;
        const T* src = (const T*)p.r + m * p.ldr + n;
        if (vec) {
            uint4 raw[sizeof(T) / 2];
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) raw[i] = ((const uint4*)src)[i];
#pragma unroll
            for (int j = 0; j < 8; j++) r[j] = to_f(((const T*)raw)[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (n + j < p.N) r[j] = to_f(src[j]);
        }
    }

    __device__ __forceinline__ void store(const TcParams& p, int64_t m, int n, float (&v)[8], float (&g)[8], bool gated) {
        if (!any) return;
        const bool full = n + 8 <= p.N;
        if (p.bias) add8(v, p.bias, n, p.N, full);
        if (gated && p.gbias) add8(g, p.gbias, n, p.N, full);
        float(&a)[8] = gated ? g : v;
        switch (p.act) {
            case ACT_RELU: each<ACT_RELU>(a); break;
            case ACT_SILU: each<ACT_SILU>(a); break;
            case ACT_GELU_TANH: each<ACT_GELU_TANH>(a); break;
            case ACT_GELU_ERF: each<ACT_GELU_ERF>(a); break;
            default: break;
        }
        T o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = from_f<T>((gated ? g[j] * v[j] : v[j]) + r[j]);
        T* dst = (T*)p.y + m * p.ldo + n;
        if (vec) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++) ((uint4*)dst)[i] = ((const uint4*)o)[i];
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (n + j < p.N) dst[j] = o[j];
        }
    }

    static __device__ __forceinline__ void add8(float (&v)[8], const float* b, int n, int N, bool full) {
        if (full) {  // n is a multiple of 8 and the vector is 16-byte aligned
            const float4 x = *(const float4*)(b + n), y = *(const float4*)(b + n + 4);
            v[0] += x.x; v[1] += x.y; v[2] += x.z; v[3] += x.w;
            v[4] += y.x; v[5] += y.y; v[6] += y.z; v[7] += y.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (n + j < N) v[j] += b[n + j];
        }
    }
    template <int ACT>
    static __device__ __forceinline__ void each(float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = activate(v[j], ACT);
    }
};

// Tile t as (activation tile, weight tile): weight tiles slowest inside groups of GROUP_M activation tiles, so
// that the CTAs at work share both operands in L2.
__device__ __forceinline__ void tile_at(const TcParams& p, int tiles_n, int t, int& tm, int& tn) {
    const int group = t / (GROUP_M * tiles_n), first = group * GROUP_M;
    const int width = p.tiles_m - first < GROUP_M ? p.tiles_m - first : GROUP_M;
    const int i = t - group * GROUP_M * tiles_n;
    tm = first + i % width;
    tn = i / width;
}

template <class T, int NT, int PLANES, bool GATED, int MODE>
__global__ void __launch_bounds__(LT, 1)
k_linear_tc(const __grid_constant__ CUtensorMap tmx, const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmg,
            const __grid_constant__ TcParams p) {
    using Sh = Shape<NT, PLANES, GATED, MODE>;
    constexpr int S = Sh::S, ST = Sh::STAGES, ROWB = Sh::ROWB, CG = MODE == PAIR ? 2 : 1;
    extern __shared__ uint8_t smem_raw[];
    // The pair's MMA reads both CTAs' operands at the same offsets: the dynamic area starts at the same
    // address in every CTA of a launch, so its rounded-up base does too.
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* out_stage = (float*)(smem + (size_t)ST * Sh::STAGE);
    uint64_t* bars = (uint64_t*)(smem + (size_t)ST * Sh::STAGE + Sh::OUT);
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
            mbar_init(tfree0 + 8 * b, EPI * CG);
        }
        mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    constexpr int ALLOC = Sh::COLS <= 32 ? 32 : Sh::COLS <= 64 ? 64 : Sh::COLS <= 128 ? 128 : Sh::COLS <= 256 ? 256 : 512;
    if (warp == 1) {
        if (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(ALLOC));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(ALLOC));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        }
    }
    fence_before();
    __syncthreads();
    if (MODE == PAIR) cluster_sync();  // both CTAs' barriers exist before either is signalled
    fence_after();
    const uint32_t tmem = *tmem_slot, sbase = smem_u32(smem);

    // This CTA's tiles and K blocks.
    const int rank = MODE == SINGLE ? 0 : (int)cluster_rank();
    const int tiles_n = MODE == PAIR ? (p.tiles_n + 1) / 2 : p.tiles_n;
    const int tile0 = MODE == SPLIT ? (int)blockIdx.x / p.split : (int)blockIdx.x / CG;
    const int tstep = MODE == SPLIT ? p.tiles : (int)gridDim.x / CG;
    const int kb0 = MODE == SPLIT ? (int)((int64_t)p.nkb * rank / p.split) : 0;
    const int kb1 = MODE == SPLIT ? (int)((int64_t)p.nkb * (rank + 1) / p.split) : p.nkb;
    constexpr int CH = PLANES == 3 ? CHUNK : 1 << 30;

    if (warp == 0) {
        if (lane == 0) {  // producer, running ahead across tiles
            int done = 0, s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = tile0; ok && t < p.tiles; t += tstep) {
                int tm, tn;
                tile_at(p, tiles_n, t, tm, tn);
                const int m0 = tm * NT + (MODE == PAIR ? rank * Sh::XR : 0);
                const int64_t blk0 = (int64_t)(MODE == PAIR ? 2 * tn + rank : tn) * p.nkb;
                for (int kb = kb0; kb < kb1; kb++, done++) {
                    if (!mbar_wait(empty0 + 8 * s, ph ^ 1u, limit) || *(volatile int*)&s_fail) {
                        s_fail = 1;
                        ok = false;
                        break;
                    }
                    const uint32_t dst = sbase + s * Sh::STAGE, bar = full0 + 8 * s;
                    if (MODE == PAIR) {
                        const uint32_t lead = peer_addr(bar, 0);
                        if (rank == 0) mbar_expect_tx(bar, 2 * Sh::STAGE);
                        const int line = (int)((blk0 + kb) * (Sh::WB / 128));
                        pair_load_2d(dst, &tmw, 0, line, lead);
                        if (GATED) pair_load_2d(dst + Sh::WB, &tmg, 0, line, lead);
                        pair_load_3d(dst + S * Sh::WB, &tmx, kb * (ROWB / 2), m0, 0, lead);
                    } else {
                        mbar_expect_tx(bar, Sh::STAGE);
                        bulk_load(dst, p.w + (blk0 + kb) * Sh::WB, Sh::WB, bar);
                        if (GATED) bulk_load(dst + Sh::WB, p.g + (blk0 + kb) * Sh::WB, Sh::WB, bar);
                        tma_load_3d(dst + S * Sh::WB, &tmx, kb * (ROWB / 2), m0, 0, bar);
                    }
                    if (++s == ST) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok) {  // let copies still in flight land before the CTA exits (they always complete)
                if (MODE != PAIR) {
                    for (int j = done - ST < 0 ? 0 : done - ST; j < done; j++)
                        mbar_wait(full0 + 8 * (j % ST), (uint32_t)(j / ST) & 1u);
                } else {  // counted on the leader's barriers, whose phases may stay open: a millisecond instead
                    const long long t0 = clock64();
                    while (clock64() - t0 < 2000000) __nanosleep(1000);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && (MODE != PAIR || rank == 0)) {  // MMA issuer
            const uint32_t idesc = idesc_f16(128 * CG, NT, !p.f16);
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
                                    umma_f16<CG>(d + v * NT, sw128_desc(w + v * Sh::WB + kk * 32), sw128_desc(x + kk * 32), idesc, first);
                                } else {
                                    const uint32_t wb = w + v * Sh::WB + kk * 32, xb = x + kk * 32;
                                    constexpr int WP = TR * ROWB, XP = Sh::XR * ROWB;
                                    const uint64_t w1 = sw64_desc(wb), w2 = sw64_desc(wb + WP), w3 = sw64_desc(wb + 2 * WP);
                                    const uint64_t x1 = sw64_desc(xb), x2 = sw64_desc(xb + XP), x3 = sw64_desc(xb + 2 * XP);
                                    const uint32_t da = d + 2 * v * NT, db = da + NT;
                                    umma_f16<CG>(da, w1, x1, idesc, first);
                                    umma_f16<CG>(db, w1, x2, idesc, first);
                                    umma_f16<CG>(db, w2, x1, idesc, 1u);
                                    umma_f16<CG>(db, w2, x2, idesc, 1u);
                                    umma_f16<CG>(db, w1, x3, idesc, 1u);
                                    umma_f16<CG>(db, w3, x1, idesc, 1u);
                                }
                            }
                        }
                        commit<CG>(empty0 + 8 * s);
                        issued = true;
                        if (++s == ST) { s = 0; ph ^= 1u; }
                    }
                    if (!ok) break;
                    commit<CG>(tfull0 + 8 * b);
                }
            }
            if (!ok) {
                s_fail = 1;
                if (issued) {  // MMAs still in flight write TMEM: let them retire before it is freed
                    commit<CG>(drain);
                    mbar_wait(drain, 0u);
                }
            }
        }
    } else {  // epilogue: two groups of four warps, each half of the tile's columns; thread = weight row (TMEM lane)
        const int q4 = warp & 3, part = (warp - 2) >> 2, row = 32 * q4 + lane;
        constexpr int HC = NT / 2;  // columns of a group
        const uint32_t tbase = tmem + ((uint32_t)(32 * q4) << 16) + part * HC;
        const uint32_t free0 = MODE == PAIR ? peer_addr(tfree0, 0) : tfree0;
        float* st = out_stage + part * S * SLAB * TR;
        int use = 0;
        auto release = [&](int buf) {  // this warp has read the buffer
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (MODE == PAIR) peer_arrive(free0 + 8 * buf);
                else mbar_arrive(tfree0 + 8 * buf);
            }
        };
        for (int t = tile0; t < p.tiles; t += tstep) {
            int tm, tn;
            tile_at(p, tiles_n, t, tm, tn);
            const int64_t m0 = (int64_t)tm * NT + part * HC;
            const int n0 = (MODE == PAIR ? 2 * tn + rank : tn) * TR;
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
                            const uint32_t at = tbase + (buf * Sh::ACC + 2 * v) * NT + c;
                            tmem_ld16(at, a);
                            tmem_ld16(at + NT, k);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int j = 0; j < 16; j++) {
                                const float sum = __uint_as_float(a[j]) + __uint_as_float(k[j]);
                                acc[v][c + j] = chunks ? acc[v][c + j] + sum : sum;
                            }
                        }
                    release(buf);
                }
            }
            // A warp that gave up still takes the barriers of its group, so that none waits for it.
            const int buf = (use - 1) & 1;
            if (MODE == SPLIT) {  // this CTA's partial sums, [v][column][weight row], over the stages (all consumed)
                float* sums = (float*)smem;
                if (ok) {
#pragma unroll
                    for (int v = 0; v < S; v++)
#pragma unroll
                        for (int c = 0; c < HC; c += 16) {
                            float* dst = sums + ((int64_t)v * NT + part * HC + c) * TR + row;
                            uint32_t a[16];
                            if (PLANES == 1) {
                                tmem_ld16(tbase + (buf * Sh::ACC + v) * NT + c, a);
                                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                            }
#pragma unroll
                            for (int j = 0; j < 16; j++) dst[j * TR] = PLANES == 1 ? __uint_as_float(a[j]) : acc[v][PLANES == 1 ? 0 : c + j];
                        }
                }
            } else {
                const int tid = (int)threadIdx.x - 64 - 128 * part;
                auto slab = [&](int c) {
                    Eight<T> e[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) e[i].load(p, m0 + c + 8 * i + (tid >> 4), n0 + (tid & 15) * 8);
#pragma unroll
                    for (int v = 0; v < S; v++) {
                        uint32_t a[16];
                        if (PLANES == 1) {
                            tmem_ld16(tbase + (buf * Sh::ACC + v) * NT + c, a);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                        }
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            st[(v * SLAB + j) * TR + row] = PLANES == 1 ? __uint_as_float(a[j]) : acc[v][PLANES == 1 ? 0 : c + j];
                    }
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
#pragma unroll 1
                    for (int i = 0; i < 2; i++) {
                        const float* src = st + (8 * i + (tid >> 4)) * TR + (tid & 15) * 8;
                        // the two 16-byte halves in an order that keeps eight lanes on different banks
                        const int h = (tid >> 2) & 1;
                        float v[8], g[8];
                        const float4 a = *(const float4*)(src + 4 * h), b = *(const float4*)(src + 4 * (h ^ 1));
                        *(float4*)v = h ? b : a;
                        *(float4*)(v + 4) = h ? a : b;
                        if (GATED) {
                            const float4 ga = *(const float4*)(src + SLAB * TR + 4 * h), gb = *(const float4*)(src + SLAB * TR + 4 * (h ^ 1));
                            *(float4*)g = h ? gb : ga;
                            *(float4*)(g + 4) = h ? ga : gb;
                        }
                        if (i == 0) e[0].store(p, m0 + c + (tid >> 4), n0 + (tid & 15) * 8, v, g, GATED);
                        else e[1].store(p, m0 + c + 8 + (tid >> 4), n0 + (tid & 15) * 8, v, g, GATED);
                    }
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                };
                // whole group or nothing: a warp whose wait ran out takes the others with it
                int alive;
                asm volatile("{\n .reg .pred q, r;\n setp.ne.b32 q, %1, 0;\n bar.red.and.pred r, %2, 128, q;\n selp.b32 %0, 1, 0, r;\n}\n"
                             : "=r"(alive)
                             : "r"((int)ok), "r"(1 + part)
                             : "memory");
                if (!alive) break;
                if (PLANES == 1) {
#pragma unroll 1
                    for (int c = 0; c < HC; c += SLAB) slab(c);
                    release(buf);
                } else {
#pragma unroll
                    for (int c = 0; c < HC; c += SLAB) slab(c);
                }
            }
            if (!ok) break;
        }
    }
    fence_before();
    __syncthreads();
    if (MODE == SPLIT) {
        cluster_sync();  // every CTA's partial sums are in its shared memory (or it failed and said so)
        if (!s_fail && warp >= 2) {
            const int cols = NT / p.split;
            int tm, tn;
            tile_at(p, tiles_n, tile0, tm, tn);
            for (int i = (int)threadIdx.x - 64; i < cols * (TR / 8); i += EPI * 32) {
                const int c = rank * cols + (i >> 4), n = tn * TR + (i & 15) * 8;
                const int64_t m = (int64_t)tm * NT + c;
                Eight<T> e;
                e.load(p, m, n);
                if (!e.any) continue;
                float v[8], g[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = g[j] = 0.0f;
                const uint32_t at = sbase + (uint32_t)(c * TR + (i & 15) * 8) * 4;
                for (int q = 0; q < p.split; q++) {
                    const uint32_t from = peer_addr(at, q);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float4 a = peer_ld4(from + 16 * h);
                        v[4 * h] += a.x; v[4 * h + 1] += a.y; v[4 * h + 2] += a.z; v[4 * h + 3] += a.w;
                        if (GATED) {
                            const float4 b = peer_ld4(from + NT * TR * 4 + 16 * h);
                            g[4 * h] += b.x; g[4 * h + 1] += b.y; g[4 * h + 2] += b.z; g[4 * h + 3] += b.w;
                        }
                    }
                }
                e.store(p, m, n, v, g, GATED);
            }
        }
    }
    if (MODE != SINGLE) cluster_sync();  // no CTA leaves while another reads its memory or signals its barriers
    if (s_fail && threadIdx.x == 0 && p.err) atomicOr(p.err, KERR_TIMEOUT);
    if (warp == 1) {
        fence_after();
        if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(ALLOC));
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(ALLOC));
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

// Clusters of `size` CTAs that can be resident at once (a GPC with an odd number of SMs leaves one out).
int resident_clusters(const void* fn, size_t smem, int size) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(device_sm_count() / size * size));
    cfg.blockDim = dim3(LT);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)size;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n;
}

struct Operands {
    const void* x;
    int64_t ldx;
    int width;  // 16-bit values of a row that hold data
};

template <class T, int NT, int PLANES, bool GATED, int MODE>
bool launch(const Plan& pl, const Call& c, const Operands& op, int split, cudaStream_t st) {
    using Sh = Shape<NT, PLANES, GATED, MODE>;
    auto* fn = k_linear_tc<T, NT, PLANES, GATED, MODE>;
    if (ensure_smem((const void*)fn, Sh::SMEM) != cudaSuccess) return false;
    CUtensorMap tmx, tmw, tmg;
    if (!tc::encode_rows_planes(&tmx, op.x, op.width, c.M, op.ldx, PLANES, pl.bk(), Sh::XR)) return false;
    if (MODE == PAIR) {  // the weights' blocks as lines of 128 bytes, swizzled already
        const int64_t lines = pl.tile_bytes() / 128;
        if (!tc::encode_rows_u16(&tmw, pl.tiles, 64, lines, 64, Sh::WB / 128)) return false;
        if (GATED && !tc::encode_rows_u16(&tmg, pl.gtiles, 64, lines, 64, Sh::WB / 128)) return false;
    } else {
        tmw = tmx;
    }
    if (!GATED || MODE != PAIR) tmg = tmw;
    TcParams p;
    p.w = pl.tiles; p.g = pl.gtiles; p.bias = pl.bias; p.gbias = pl.gbias;
    p.r = c.r; p.y = c.y; p.ldr = c.ldr; p.ldo = c.ldo;
    p.M = (int)c.M; p.N = pl.N; p.nkb = pl.nkb(); p.act = pl.act; p.f16 = pl.dtype == DT_F16;
    constexpr int PER = 16 / (int)sizeof(T);
    p.vec = (uintptr_t)c.y % 16 == 0 && c.ldo % PER == 0 && (!c.r || ((uintptr_t)c.r % 16 == 0 && c.ldr % PER == 0));
    p.tiles_n = pl.tiles_n();
    p.tiles_m = (int)((c.M + NT - 1) / NT);
    p.tiles = p.tiles_m * (MODE == PAIR ? (p.tiles_n + 1) / 2 : p.tiles_n);
    p.split = split;
    p.err = c.err;
    p.wait_limit = c.wait_limit > 0 ? c.wait_limit : tc::kWaitCycles;
    p.stall_mma = c.stall_mma;
    int clusters = 0;
    if (MODE == PAIR) {
        static std::atomic<int> cached{0};  // the same on every device this library is built for
        clusters = cached.load();
        if (!clusters) {
            clusters = std::max(1, resident_clusters((const void*)fn, Sh::SMEM, 2));
            cached.store(clusters);
        }
    }
    const int size = MODE == PAIR ? 2 : MODE == SPLIT ? split : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(MODE == SPLIT ? p.tiles * split
                                  : MODE == PAIR ? 2 * std::min(p.tiles, clusters) : std::min(p.tiles, device_sm_count())));
    cfg.blockDim = dim3(LT);
    cfg.dynamicSmemBytes = Sh::SMEM;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    if (MODE != SINGLE) {
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = (unsigned)size;
        at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&cfg, fn, tmx, tmw, tmg, p) == cudaSuccess;
}

// One tile width: split over K when the tiles leave half of the SMs idle, one CTA per SM otherwise.
template <class T, int NT, int PLANES, bool GATED>
bool run(const Plan& pl, const Call& c, const Operands& op, cudaStream_t st) {
    const int64_t tiles = (c.M + NT - 1) / NT * pl.tiles_n();
    int split = 1;
    while (split < 8 && tiles * split * 2 <= device_sm_count() && pl.nkb() >= split * 4) split *= 2;
    if (split > 1) return launch<T, NT, PLANES, GATED, SPLIT>(pl, c, op, split, st);
    return launch<T, NT, PLANES, GATED, SINGLE>(pl, c, op, 1, st);
}

template <class T, int PLANES>
bool pick_tile(const Plan& pl, const Call& c, const Operands& op, cudaStream_t st) {
    constexpr int WIDE = PLANES == 3 ? 128 : 256;  // widest tile whose accumulators fit in TMEM, ungated
    auto pairs = [&](int nt) { return (c.M + nt - 1) / nt * ((pl.tiles_n() + 1) / 2); };
    const int enough = device_sm_count() / 2;  // a tile for every pair of CTAs
    if (pl.gated) {
        if (pairs(WIDE / 2) >= enough && c.M > WIDE / 2) return launch<T, WIDE / 2, PLANES, true, PAIR>(pl, c, op, 1, st);
        if (c.M <= 32) return run<T, 32, PLANES, true>(pl, c, op, st);
        if (PLANES == 3 || c.M <= 64) return run<T, 64, PLANES, true>(pl, c, op, st);
        return run<T, WIDE / 2, PLANES, true>(pl, c, op, st);
    }
    if (pairs(WIDE) >= enough && c.M > WIDE / 2) return launch<T, WIDE, PLANES, false, PAIR>(pl, c, op, 1, st);
    if (c.M <= 32) return run<T, 32, PLANES, false>(pl, c, op, st);
    if (c.M <= 64) return run<T, 64, PLANES, false>(pl, c, op, st);
    return run<T, 128, PLANES, false>(pl, c, op, st);
}
}  // namespace

void layout(const Plan& p, const void* w, uint8_t* tiles, float* rows, cudaStream_t st) {
    const int64_t chunks = p.tile_bytes() / (16 * p.planes());
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
    const Operands op{x, ldx, x == c.x ? p.K : kp_of(p)};
    bool ok;
    if (p.dtype == DT_F32) ok = pick_tile<float, 3>(p, c, op, st);
    else if (p.dtype == DT_F16) ok = pick_tile<__half, 1>(p, c, op, st);
    else ok = pick_tile<__nv_bfloat16, 1>(p, c, op, st);
    return ok ? n + 1 : -1;
}

}  // namespace lin
}  // namespace slx
