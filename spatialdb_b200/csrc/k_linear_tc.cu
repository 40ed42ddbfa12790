// k_linear_tc.cu -- the linear operator on the 5th-generation tensor cores (tcgen05.mma kind::f16, fp32
// accumulators in TMEM).
//
// A tile is 128 weight rows a CTA (one TMEM lane each) x NT activation rows (the MMA's N). Weights are
// laid out once in the swizzled blocks that the MMA reads, so a K block of a tile is one contiguous
// copy; activations come through a TMA tensor map on the caller's rows (a packed copy when their base
// or stride is not a multiple of 16 bytes). Warp 0 loads, warp 1 issues the MMAs, 16 warps run the
// epilogue: 16 columns at a time go from TMEM through shared memory, so that bias, activation, gate,
// residual and the one rounding run on runs of a row's outputs with vector accesses.
//
// f32 (PLANES = 3): each value is the exact sum of three bf16 parts, each rounded to nearest, x = x1 + x2 + x3 with
// |x2| <= 2^-8 |x| and |x3| <= 2^-17 |x|. x1 w1 goes to one accumulator, the corrections x1 w2 + x2 w1 + x2 w2 +
// x1 w3 + x3 w1 (at most 2^-6.9 of it) to another; x2 w3 + x3 w2 + x3 w3, left out, is at most 2^-23.9 |x| |w| and of
// either sign. (Parts cut off instead of rounded leave out up to 2^-21 |x| |w|, all of the product's sign: 7.8 x 2^-24 of
// 1.0078^2.) The tensor core truncates what it adds, which biases long sums, so every 256 values
// of K both accumulators are added to fp32 registers (rounded to nearest) and started anew. x1 w1 may pass the sum it
// stands for by 2^-7 of it: a sum within 2^-7 of the largest finite value may end infinite. An infinity or NaN is all
// in its first part, so x1 w1 alone is what fp32 makes of it, and the corrections, where it meets the zeros of exact
// bf16 values, are left out of a sum that is not finite.
//
// 16 bits: the sums stay in the truncating accumulator over all of K. An addition aligns 16 products and the sum to the
// largest of them, keeps 25 bits of each and 24 of the result (measured): operands of one sign come out low by about
// K x 6e-9, 1.2e-5 at K = 2048 and 5e-5 at 8192 (a sixth of that with random signs), where half a step of an f16 output
// is 2.4e-4 to 4.9e-4 and of a bf16 output eight times that. Against 64 bits the outputs' error stays that of their
// rounding (bf16 512 x 2048 x 16384 gated: 1.66e-3, as with sums in fp32 FMAs, against which 0.2 % of the outputs round
// the other way). Promoting the sums as in f32 would take 64 registers a thread with 256 columns a tile; of 96 the
// epilogue uses all.
//
// Three forms, the cheapest by an estimate of its cycles (choose):
//   ONE   one tile at a time. A cluster of S = 1, 2, 4 or 8 CTAs shares the tile, each with a range of the K
//         blocks, so that few tiles still occupy the SMs. CTA c of S finishes columns c NT / S...: the others
//         store their partial sums of them into its shared memory, and it adds them in rank order. One
//         launch, no workspace, the same result every time. The epilogue's warps have nothing to do before the
//         sums are there: f32 rows, and 16-bit rows TMA cannot address, are loaded, split and swizzled by
//         them (MANUAL), without a pass of its own.
//   PAIR  persistent, two CTAs (cta_group::2) on 256 weight rows: each loads its own 128 weight rows and half
//         of the activation rows, which halves the activation bytes per MMA; the epilogue of a tile runs
//         under the MMAs of the next (two accumulators). With a gate a CTA's 128 rows are 64 of the weights and the
//         same 64 of the gate's, in one accumulator of all 256 columns: they meet in the epilogue's shared memory.
//   WIDE  (16 bits, gated) pairs with 128 rows of each array a CTA, an accumulator each, on 128 activation rows: for
//         products of one such tile whose PAIR tiles just miss a wave.
// What bounds PAIR is shared memory as much as the tensor pipe: a K block of a 256-column tile takes 512 cycles
// of MMA and, at 128 bytes a cycle, 250 each for the operands' reads and the TMA's writes plus 170 for the
// epilogue's staging (K 768): 543 cycles a block measured without a concurrent epilogue, 713 with one. Gated, 810
// (K 2048); with 128 columns of each array in accumulators of their own, the form before, 950.
// Leaving out the loads of either operand changes the times by 2 to 8 %.
// Measured in loops of calls, inputs larger than L2, the large products at the power cap (sustained cuBLAS bf16 is 1391.3
// TFLOP/s): bf16 8192^3 838 us, 1312 TFLOP/s; 4096 x 4096 x 11008 with bias, GELU and residual 312 us, 1184; 512 x 2048 x
// 16384 gated 71 us, 970; 8192 x 768 x 2304 32.7 us, 887; f32 8192 x 768 x 2304 165 us, 176 (1057 of bf16 products), 512
// x 2048 x 8192 gated 200 us, 172 (one array's rows a tile, the form before, took 1.6 times as long); f16 129 x 1001 x
// 1111 7.9 us. In short runs, above the sustained clock: 703, 276, 59, 27.3, 147 and 169 us. Tensor pipe active (ncu): 79 %
// at bf16 2048 x 4096 x 8192, 66 % gated, 52 % at 8192 x 768 x 2304, 67 % in f32.
// Every mbarrier wait is bounded.
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <type_traits>

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

enum Mode { ONE = 0, PAIR = 1, WIDE = 2 };

constexpr int EPI = 16;                     // epilogue warps: four groups of one warp per TMEM lane quarter
constexpr int GROUPS = EPI / 4;
constexpr int LT = 32 * (2 + EPI);          // threads
constexpr int SMEM_MAX = 227 * 1024;
constexpr int CHUNK = 8;                    // f32: K blocks (of 32) between promotions to registers
constexpr int GROUP_M = 8;                  // activation tiles walked together (their rows stay in L2)

struct TcParams {
    const uint8_t *w, *g;
    const float *bias, *gbias;
    const void* r;
    void* y;
    int64_t ldr, ldo;
    const void* x;   // MANUAL: the caller's rows
    int64_t ldx;
    int M, N, K, nkb, act, f16, vec;
    int tiles_n, tiles_m, tiles, log2_split;
    int* err;
    long long wait_limit;
    int stall_mma;
};

template <int NT, int PLANES, bool GATED, int MODE>
struct Shape {
    static constexpr bool DUO = MODE != ONE, MIX = GATED && MODE == PAIR;  // a CTA's 128 rows are 64 of the weights and 64 of the gate's
    static constexpr int S = GATED && !MIX ? 2 : 1;
    static constexpr int ROWB = PLANES == 3 ? 64 : 128;        // bytes of K per operand row and block
    static constexpr int WB = PLANES * TR * ROWB;              // one weight array's block
    static constexpr int XR = DUO ? NT / 2 : NT;      // activation rows this CTA loads
    static constexpr int STAGE = S * WB + PLANES * XR * ROWB;
    static constexpr int ACC = S * (PLANES == 3 ? 2 : 1);      // accumulators of NT columns
    static constexpr int COLS = 2 * ACC * NT;                  // two buffers
    static constexpr int HC = NT / GROUPS;                     // columns of an epilogue group
    static constexpr int SLAB = HC < 16 || PLANES == 3 || S == 2 ? 8 : 16;  // columns it moves through shared memory at a time
    // the epilogue's shared memory: the groups' staging, or in ONE the partial sums this CTA finishes
    static constexpr int OUT = MODE == ONE ? S * NT * TR * 4 : GROUPS * S * SLAB * TR * 4;
    static constexpr int FIT = (SMEM_MAX - 1024 - 512 - OUT) / STAGE;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int GROUPS_X = XR * (ROWB / 16) / 32;     // MANUAL: groups of 32 chunks of eight values a block
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + OUT + 1024 + 512;
    static_assert(COLS <= 512 && STAGES >= 2, "tile does not fit");
    static_assert(2 * SMEM > SMEM_MAX, "two CTAs on an SM would share its tensor memory");
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
// All 32 lanes of every warp of the cluster arrive, and wait before they arrive again.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
    cluster_arrive();
    cluster_wait();
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
    return a;
}
__device__ __forceinline__ void peer_st(uint32_t addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
__device__ __forceinline__ void peer_arrive(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}

// Instruction descriptor, kind::f16: D f32, A and B both f16 (0) or both bf16 (1), K-major, N = n.
__device__ __forceinline__ uint32_t idesc_f16(int m, int n, int bf16) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// A thread's share of a tile's outputs: of rows m of y, the values of four weight rows n.. and with H = 2 of four
// more from n + 64 (a warp's reads of the staged sums then fall on different banks, and its stores are runs of
// 128 bytes or more). FAST: the tile lies inside y and rows take vectors of four values.
template <class T, bool GATED, int H>
struct Columns {
    static constexpr int V = 4 * H;
    float b[V], gb[V];
    int n;

    __device__ __forceinline__ void begin(const TcParams& p, int first) {
        n = first;
        fill(b, p.bias, p.N);
        if (GATED) fill(gb, p.gbias, p.N);
    }
    __device__ __forceinline__ int at(int j) const { return n + (j & 3) + (j >> 2) * 64; }
    __device__ __forceinline__ void fill(float (&v)[V], const float* from, int N) const {
#pragma unroll
        for (int j = 0; j < V; j++) v[j] = from && at(j) < N ? from[at(j)] : 0.0f;
    }

    struct __align__(4 * sizeof(T)) Four {
        T v[4];
    };
    struct __align__(8) Residual {
        Four f[H];
    };
    template <bool FAST>
    __device__ __forceinline__ void load(const TcParams& p, int64_t m, Residual& r) const {
        if (!p.r) return;
        const T* src = (const T*)p.r + m * p.ldr;
        if (FAST) {
#pragma unroll
            for (int h = 0; h < H; h++) copy(&r.f[h], src + n + 64 * h);
        } else if (m < p.M) {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (at(j) < p.N) r.f[j >> 2].v[j & 3] = src[at(j)];
        }
    }
    // Items' sums (and gate sums) to outputs, R rows of m apart `step`.
    template <bool FAST, int R>
    __device__ __forceinline__ void store(const TcParams& p, int64_t m, int step, float (&v)[V * R], float (&g)[V * R],
                                          const Residual (&r)[R]) const {
#pragma unroll
        for (int j = 0; j < V * R; j++) {
            v[j] += b[j % V];
            if (GATED) g[j] += gb[j % V];
        }
        if (GATED) {
            activate_all<T>(g, p.act);
#pragma unroll
            for (int j = 0; j < V * R; j++) v[j] *= g[j];
        } else {
            activate_all<T>(v, p.act);
        }
        if (p.r) {
#pragma unroll
            for (int j = 0; j < V * R; j++) v[j] += to_f(r[j / V].f[j % V >> 2].v[j & 3]);
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int64_t row = m + i * step;
            T* dst = (T*)p.y + row * p.ldo;
            Four o[H];
#pragma unroll
            for (int j = 0; j < V; j++) o[j >> 2].v[j & 3] = from_f<T>(v[V * i + j]);
            if (FAST) {
#pragma unroll
                for (int h = 0; h < H; h++) copy(dst + n + 64 * h, &o[h]);
            } else if (row < p.M) {
#pragma unroll
                for (int j = 0; j < V; j++)
                    if (at(j) < p.N) dst[at(j)] = o[j >> 2].v[j & 3];
            }
        }
    }
    static __device__ __forceinline__ void copy(void* dst, const void* src) {  // four values
        if (sizeof(T) == 4) *(uint4*)dst = *(const uint4*)src;
        else *(uint2*)dst = *(const uint2*)src;
    }
};

// C consecutive accumulator columns of this thread's lane.
template <int C>
__device__ __forceinline__ void tmem_cols(uint32_t at, float (&v)[C]) {
    static_assert(C == 8 || C == 16, "columns");
    uint32_t a[C];
    if constexpr (C == 16) tmem_ld16(at, a);
    else tmem_ld8(at, a);
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int j = 0; j < C; j++) v[j] = __uint_as_float(a[j]);
}

// Tile t as (activation tile, weight tile): weight tiles slowest inside groups of GROUP_M activation tiles, so
// that the CTAs at work share both operands in L2.
__device__ __forceinline__ void tile_at(const TcParams& p, int tiles_n, int t, int& tm, int& tn) {
    const int group = t / (GROUP_M * tiles_n), first = group * GROUP_M;
    const int width = p.tiles_m - first < GROUP_M ? p.tiles_m - first : GROUP_M;
    const int i = t - group * GROUP_M * tiles_n;
    tm = first + i % width;
    tn = i / width;
}

// The three bf16 parts of eight fp32 values, each what is left rounded to nearest: x1 takes 8 of the 24 significant
// bits, what it leaves is a multiple of x's last place and at most 2^-8 of x, what x2 leaves of that at most 2^-17,
// which fits x3: the sum is the value exactly, and the parts' signs favour no side. A finite value whose x1 would
// round to infinity has its x1 cut off instead. Of a value that is not finite the first part keeps it (a NaN stays
// one) and the others are zero.
__device__ __forceinline__ void split3(const float (&f)[8], uint4 (&part)[3]) {
    float r[8], q[8];
    uint32_t w[3][4];
    auto high = [](float v) { return __float_as_uint(v) & 0xFFFF0000u; };
    auto pair = [](float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *(const uint32_t*)&h;
    };
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int a = 2 * j, b = a + 1;
        w[0][j] = pair(f[a], f[b]);
        r[a] = f[a] - __uint_as_float(w[0][j] << 16);
        r[b] = f[b] - __uint_as_float(high(__uint_as_float(w[0][j])));
        w[1][j] = pair(r[a], r[b]);
        q[a] = r[a] - __uint_as_float(w[1][j] << 16);
        q[b] = r[b] - __uint_as_float(high(__uint_as_float(w[1][j])));
        w[2][j] = pair(q[a], q[b]);
    }
    const float sum = ((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7]));
    if (!isfinite(sum)) {  // some value, or its first part, is not finite (finite remainders cannot reach the largest value)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (isfinite(r[j])) continue;
            const float x1 = __uint_as_float(high(f[j])), x2 = f[j] - x1;
            const bool cut = isfinite(f[j]);
            const float c2 = __bfloat162float(__float2bfloat16_rn(x2));
            const uint32_t p[3] = {high(f[j]) | (isnan(f[j]) ? 0x00400000u : 0u), cut ? high(c2) : 0u, cut ? high(x2 - c2) : 0u};
#pragma unroll
            for (int i = 0; i < 3; i++) w[i][j / 2] = j & 1 ? (w[i][j / 2] & 0x0000FFFFu) | p[i] : (w[i][j / 2] & 0xFFFF0000u) | p[i] >> 16;
        }
    }
#pragma unroll
    for (int i = 0; i < 3; i++) part[i] = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
}

// Shared-memory matrix descriptors, K-major: the operand's start goes into the low word (in 16-byte units),
// the rest is constant: rows of 128 bytes in groups of 1 KB with the 128-byte swizzle, or of 64 bytes in groups of
// 512 with the 64-byte one.
template <int ROWB>
__device__ __forceinline__ uint64_t operand(uint32_t start) {
    constexpr uint32_t HI = (uint32_t)(8 * ROWB >> 4) | 1u << 14 | (ROWB == 128 ? 2u : 4u) << 29;  // group stride, version, swizzle
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(start), "n"(HI));
    return d;
}

// Eight values of a row from column k (a multiple of 8), zeros past K. Where they do not start on a 16-byte
// boundary, the two aligned vectors around them, shifted together, while both lie inside the row (7 values
// before, 8 behind); single values at the row's ends.
__device__ __forceinline__ uint4 row8(const uint16_t* row, int k, int K) {
    const uint16_t* src = row + k;
    const uint32_t off = (uint32_t)(uintptr_t)src & 15;
    if (off == 0 && k + 8 <= K) return *(const uint4*)src;
    if (k >= 8 && k + 16 <= K) {
        const uint4* at = (const uint4*)((uintptr_t)src & ~(uintptr_t)15);
        const uint4 lo = at[0], hi = at[1];
        uint32_t w[7] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z};
        const uint32_t last = hi.w;
        // by two words, by one, by half of one
        const bool two = off & 8, one = off & 4;
        uint32_t t[6], u[5];
#pragma unroll
        for (int j = 0; j < 6; j++) t[j] = two ? (j + 2 < 7 ? w[j + 2] : last) : w[j];
#pragma unroll
        for (int j = 0; j < 5; j++) u[j] = one ? t[j + 1] : t[j];
        const uint32_t bits = (off & 2) * 8;
        return make_uint4(__funnelshift_r(u[0], u[1], bits), __funnelshift_r(u[1], u[2], bits), __funnelshift_r(u[2], u[3], bits),
                          __funnelshift_r(u[3], u[4], bits));
    }
    alignas(16) uint16_t e[8];
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = k + j < K ? src[j] : (uint16_t)0;
    return *(const uint4*)e;
}
__device__ __forceinline__ void row8(const float* row, int k, int K, float (&f)[8]) {
    const float* src = row + k;
    if (k + 8 <= K && ((uintptr_t)src & 15) == 0) {
        *(float4*)f = *(const float4*)src;
        *(float4*)(f + 4) = *(const float4*)(src + 4);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = k + j < K ? src[j] : 0.0f;
    }
}

// Eight values of one chunk of x, on their way from the caller's rows to a stage.
template <int PLANES>
struct Chunk {
    uint4 v;
    __device__ __forceinline__ void load(const TcParams& p, int64_t m, int k) {
        v = m < p.M ? row8((const uint16_t*)p.x + m * p.ldx, k, p.K) : make_uint4(0, 0, 0, 0);
    }
    // Chunk c of row r of a stage's activation area: 128-byte rows, chunks XORed with r % 8.
    __device__ __forceinline__ void store(uint32_t area, int rows, int r, int c) const {
        const uint32_t at = area + r * 128 + ((c ^ (r & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
    }
};
template <>
struct Chunk<3> {
    alignas(16) float f[8];
    __device__ __forceinline__ void load(const TcParams& p, int64_t m, int k) {
        if (m < p.M) {
            row8((const float*)p.x + m * p.ldx, k, p.K, f);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) f[j] = 0.0f;
        }
    }
    // The three parts' planes of 64-byte rows, chunks XORed with (r / 2) % 4.
    __device__ __forceinline__ void store(uint32_t area, int rows, int r, int c) const {
        uint4 w[3];
        split3(f, w);
#pragma unroll
        for (int q = 0; q < 3; q++) {
            const uint32_t at = area + q * rows * 64 + r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[q].x), "r"(w[q].y), "r"(w[q].z), "r"(w[q].w) : "memory");
        }
    }
};

// MANUAL: the epilogue's warps fill the stages' activation areas. A warp takes every LW-th group of 32
// chunks (a group lies in one K block), the next group's values in flight while it stores this one's; a
// stage's full barrier counts its groups. LW is such that a warp has a group in at least every ST-th block:
// when it waits for block n's stage it then knows block n - 2 ST consumed (it has waited for a later one), so
// the parity it waits for cannot be an older phase's.
template <class Sh, int PLANES>
struct RowLoader {
    static constexpr int PER = Sh::ROWB / 16, ST = Sh::STAGES;  // chunks of a row in a block
    static constexpr int LW = Sh::GROUPS_X * ST < EPI ? Sh::GROUPS_X * ST : EPI;
    static_assert(Sh::GROUPS_X >= EPI || LW % Sh::GROUPS_X == 0, "a warp's groups lie LW / GROUPS_X blocks apart");
    const TcParams& p;
    int m0, kb0, lane, next;  // next: the warp's next group, counted from block kb0
    uint32_t sbase, full0, empty0;

    __device__ RowLoader(const TcParams& params, int m, int kb, int warp, int ln, uint32_t base, uint32_t full, uint32_t empty)
        : p(params), m0(m), kb0(kb), lane(ln), next(warp < LW ? warp : 1 << 30), sbase(base), full0(full), empty0(empty) {}

    __device__ __forceinline__ void fetch(Chunk<PLANES>& c, int g, int groups) const {
        const int i = (g % Sh::GROUPS_X) * 32 + lane;
        if (g < groups) c.load(p, m0 + i / PER, (kb0 + g / Sh::GROUPS_X) * (Sh::ROWB / 2) + i % PER * 8);
    }
    __device__ __forceinline__ bool put(const Chunk<PLANES>& c, int g, long long limit) const {
        const int i = (g % Sh::GROUPS_X) * 32 + lane, n = g / Sh::GROUPS_X, s = n % ST;
        if (!__all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, ((uint32_t)(n / ST) & 1u) ^ 1u, limit))) return false;
        c.store(sbase + s * Sh::STAGE + Sh::S * Sh::WB, Sh::XR, i / PER, i % PER);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(full0 + 8 * s);
        return true;
    }
    // Fills this warp's groups of the first `blocks` K blocks that it has not filled yet.
    __device__ bool fill(int blocks, long long limit) {
        const int groups = blocks * Sh::GROUPS_X;
        Chunk<PLANES> buf[2];
        fetch(buf[0], next, groups);
        while (next < groups) {
            fetch(buf[1], next + LW, groups);
            if (!put(buf[0], next, limit)) return false;
            next += LW;
            if (next >= groups) break;
            fetch(buf[0], next + LW, groups);
            if (!put(buf[1], next, limit)) return false;
            next += LW;
        }
        return true;
    }
};

template <class T, int NT, int PLANES, bool GATED, int MODE, bool MANUAL>
__global__ void __launch_bounds__(LT, 1)
k_linear_tc(const __grid_constant__ CUtensorMap tmx, const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmg,
            const __grid_constant__ TcParams p) {
    using Sh = Shape<NT, PLANES, GATED, MODE>;
    constexpr int S = Sh::S, ST = Sh::STAGES, ROWB = Sh::ROWB, CG = Sh::DUO ? 2 : 1;
    constexpr bool DUO = Sh::DUO, MIX = Sh::MIX;
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
            mbar_init(full0 + 8 * i, MANUAL ? 1 + Sh::GROUPS_X : 1);
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
    // Not before this CTA holds its tensor memory: a kernel let in earlier, of another library perhaps, could take the
    // columns first and hold them while it waits for this kernel, which would then wait for them without a limit.
    grid_release();
    if (DUO) cluster_sync();   // both CTAs' barriers exist before either is signalled
    if (MODE == ONE) cluster_arrive();  // waited for before the first store to another CTA
    bool met = false;
    fence_after();
    const uint32_t tmem = *tmem_slot, sbase = smem_u32(smem);

    // This CTA's tiles and K blocks.
    const int rank = (int)cluster_rank(), split = 1 << p.log2_split;
    const int tiles_n = DUO && !MIX ? (p.tiles_n + 1) / 2 : p.tiles_n;
    const int tile0 = MODE == ONE ? (int)blockIdx.x >> p.log2_split : (int)blockIdx.x / CG;
    const int tstep = MODE == ONE ? p.tiles : (int)gridDim.x / CG;
    const int kb0 = MODE == ONE ? (int)(((int64_t)p.nkb * rank) >> p.log2_split) : 0;
    const int kb1 = MODE == ONE ? (int)(((int64_t)p.nkb * (rank + 1)) >> p.log2_split) : p.nkb;
    constexpr int CH = PLANES == 3 ? CHUNK : 1 << 28;

    if (warp == 0) {
        if (lane == 0) {  // producer, running ahead across tiles
            auto load_w = [&](int kb, int stage, int64_t blk0) {
                const uint32_t dst = sbase + stage * Sh::STAGE, bar = full0 + 8 * stage;
                if (DUO) {
                    const uint32_t lead = peer_addr(bar, 0);
                    if (rank == 0) mbar_expect_tx(bar, 2 * Sh::STAGE);
                    const int line = (int)((blk0 + kb) * (Sh::WB / 128));
                    if (MIX) {  // of every part's block this CTA's half of the weights' rows, then of the gate's
                        constexpr int HALF = TR * ROWB / 2;
#pragma unroll
                        for (int q = 0; q < PLANES; q++) {
                            pair_load_2d(dst + 2 * q * HALF, &tmw, 0, line + (2 * q + rank) * (HALF / 128), lead);
                            pair_load_2d(dst + 2 * q * HALF + HALF, &tmg, 0, line + (2 * q + rank) * (HALF / 128), lead);
                        }
                    } else {
                        pair_load_2d(dst, &tmw, 0, line, lead);
                        if (GATED) pair_load_2d(dst + Sh::WB, &tmg, 0, line, lead);
                    }
                } else {
                    mbar_expect_tx(bar, MANUAL ? S * Sh::WB : Sh::STAGE);
                    bulk_load(dst, p.w + (blk0 + kb) * Sh::WB, Sh::WB, bar);
                    if (GATED) bulk_load(dst + Sh::WB, p.g + (blk0 + kb) * Sh::WB, Sh::WB, bar);
                }
            };
            int done = 0, s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = tile0; ok && t < p.tiles; t += tstep) {
                int tm, tn;
                tile_at(p, tiles_n, t, tm, tn);
                const int m0 = tm * NT + (DUO ? rank * Sh::XR : 0);
                const int64_t blk0 = (int64_t)(DUO && !MIX ? 2 * tn + rank : tn) * p.nkb;
                // Weights are the handle's own memory, which no kernel in the stream writes: the first stages' are
                // asked for before the kernels ahead of this one are waited for, the activations after it.
                const int ahead = MODE == ONE ? (kb1 - kb0 < ST ? kb1 - kb0 : ST) : 0;
                for (int i = 0; i < ahead; i++) load_w(kb0 + i, i, blk0);
                if (done == 0) grid_wait();
                for (int kb = kb0; kb < kb1; kb++, done++) {
                    const bool asked = done < ahead;
                    if (!asked && (!mbar_wait(empty0 + 8 * s, ph ^ 1u, limit) || *(volatile int*)&s_fail)) {
                        s_fail = 1;
                        ok = false;
                        break;
                    }
                    if (!asked) load_w(kb, s, blk0);
                    const uint32_t dst = sbase + s * Sh::STAGE + S * Sh::WB, bar = full0 + 8 * s;
                    if (DUO) pair_load_3d(dst, &tmx, kb * (ROWB / 2), m0, 0, peer_addr(bar, 0));
                    else if (!MANUAL) tma_load_3d(dst, &tmx, kb * (ROWB / 2), m0, 0, bar);
                    if (++s == ST) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok) {  // let copies still in flight land before the CTA exits (they always complete)
                if (!DUO && !MANUAL) {
                    for (int j = done - ST < 0 ? 0 : done - ST; j < done; j++)
                        mbar_wait(full0 + 8 * (j % ST), (uint32_t)(j / ST) & 1u);
                } else {  // their barriers also count the other CTA's copies, or rows that may not come: a millisecond
                    const long long t0 = clock64();
                    while (clock64() - t0 < 2000000) __nanosleep(1000);
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0 && (!DUO || rank == 0)) {  // MMA issuer
            const uint32_t idesc = idesc_f16(128 * CG, NT, !p.f16);
            grid_wait();  // the bounded waits below are for this kernel's copies, not for the kernels ahead
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
                        // operand starts in 16-byte units (the leading byte offset's 1 is ignored for these layouts)
                        const uint32_t w0 = ((sbase + s * Sh::STAGE) >> 4) | 1u << 16, x0 = w0 + (S * Sh::WB >> 4);
#pragma unroll
                        for (int kk = 0; kk < ROWB / 32; kk++) {
                            const uint32_t first = kb == c0 && kk == 0 ? 0u : 1u;
#pragma unroll
                            for (int v = 0; v < S; v++) {
                                const uint32_t w = w0 + (v * Sh::WB >> 4) + 2 * kk, x = x0 + 2 * kk;
                                if (PLANES == 1) {
                                    umma_f16<CG>(d + v * NT, operand<ROWB>(w), operand<ROWB>(x), idesc, first);
                                } else {
                                    constexpr uint32_t WP = TR * ROWB >> 4, XP = Sh::XR * ROWB >> 4;
                                    const uint64_t w1 = operand<ROWB>(w), w2 = operand<ROWB>(w + WP), w3 = operand<ROWB>(w + 2 * WP);
                                    const uint64_t x1 = operand<ROWB>(x), x2 = operand<ROWB>(x + XP), x3 = operand<ROWB>(x + 2 * XP);
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
    } else {  // epilogue: groups of four warps, each a quarter of the tile's columns; thread = weight row (TMEM lane)
        const int q4 = warp & 3, part = (warp - 2) >> 2, row = 32 * q4 + lane;
        constexpr int HC = Sh::HC, SLAB = Sh::SLAB;
        const uint32_t tbase = tmem + ((uint32_t)(32 * q4) << 16) + part * HC;
        const uint32_t free0 = DUO ? peer_addr(tfree0, 0) : tfree0;
        float* st = out_stage + part * S * SLAB * TR;
        const int tid = (int)threadIdx.x - 64 - 128 * part, col = tid >> 4;
        const float* src = st + col * TR + (tid & 15) * 4;
        constexpr int OH = MIX ? 1 : 2;  // runs of four outputs a thread has in a row of y
        grid_wait();  // x, the residual and y belong to the kernels ahead until they have ended
        int use = 0;
        auto release = [&](int buf) {  // this warp has read the buffer
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (DUO) peer_arrive(free0 + 8 * buf);
                else mbar_arrive(tfree0 + 8 * buf);
            }
        };
        for (int t = tile0; t < p.tiles; t += tstep) {
            int tm, tn;
            tile_at(p, tiles_n, t, tm, tn);
            const int64_t m0 = (int64_t)tm * NT + part * HC;
            const int n0 = MIX ? tn * TR + rank * (TR / 2) : (DUO ? 2 * tn + rank : tn) * TR;
            Columns<T, GATED, OH> out;
            out.begin(p, n0 + (tid & 15) * 4);
            // The rows of two accumulator chunks ahead of the one being read: the MMAs of chunk i wait for the
            // sums of chunk i - 2 to be read, so rows past chunk i + 1 must not be waited for before that.
            RowLoader<Sh, PLANES> rows(p, tm * NT, kb0, warp - 2, lane, sbase, full0, empty0);
            if (MANUAL && !rows.fill(kb1 - kb0 < 2 * CH ? kb1 - kb0 : 2 * CH, limit)) s_fail = 1;  // the wait below runs out too
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
                        for (int c = 0; c < HC; c += SLAB) {
                            float a[SLAB], k[SLAB];
                            const uint32_t at = tbase + (buf * Sh::ACC + 2 * v) * NT + c;
                            tmem_cols<SLAB>(at, a);
                            tmem_cols<SLAB>(at + NT, k);
                            float all = a[0];
#pragma unroll
                            for (int j = 1; j < SLAB; j++) all += a[j];
                            if (!isfinite(all)) {  // some sum may not be finite: it keeps clear of the corrections
#pragma unroll
                                for (int j = 0; j < SLAB; j++) k[j] = isfinite(a[j]) ? k[j] : 0.0f;
                            }
#pragma unroll
                            for (int j = 0; j < SLAB; j++) acc[v][c + j] = chunks ? acc[v][c + j] + (a[j] + k[j]) : a[j] + k[j];
                        }
                    release(buf);
                    if (MANUAL && !rows.fill(kb1 - c0 < 3 * CH ? kb1 - kb0 : c0 - kb0 + 3 * CH, limit)) s_fail = 1;
                }
            }
            const int buf = (use - 1) & 1;
            if (MODE == ONE) {  // partial sums to the CTAs that finish the columns: [v][column of the part][source][weight row]
                cluster_wait();  // every CTA of the cluster is running
                met = true;
                if (!ok) break;
                const int sh = __popc(NT - 1) - p.log2_split, cols = 1 << sh;
                const uint32_t base = smem_u32(out_stage) + (uint32_t)(rank * TR + row) * 4;
#pragma unroll
                for (int v = 0; v < S; v++)
#pragma unroll
                    for (int c = 0; c < HC; c += SLAB) {
                        float a[SLAB];
                        if (PLANES == 1) tmem_cols<SLAB>(tbase + (buf * Sh::ACC + v) * NT + c, a);
                        const int k0 = part * HC + c;
                        if (tm * NT + k0 >= p.M) break;  // columns past the last row of x
#pragma unroll
                        for (int j = 0; j < SLAB; j++) {
                            const int k = k0 + j;
                            const uint32_t at = base + (((v << sh) + (k & (cols - 1))) << p.log2_split) * (TR * 4);
                            peer_st(peer_addr(at, k >> sh), PLANES == 1 ? a[j] : acc[v][PLANES == 1 ? 0 : c + j]);
                        }
                    }
            } else {
                // whole group or nothing: a warp whose wait ran out takes the others with it, so that none is
                // left at a barrier
                int alive;
                asm volatile("{\n .reg .pred q, r;\n setp.ne.b32 q, %1, 0;\n bar.red.and.pred r, %2, 128, q;\n selp.b32 %0, 1, 0, r;\n}\n"
                             : "=r"(alive)
                             : "r"((int)ok), "r"(1 + part)
                             : "memory");
                if (!alive) break;
                auto slab = [&](int c, auto fast) {
                    constexpr bool FAST = decltype(fast)::value;
                    constexpr int R = SLAB / 8;
                    typename Columns<T, GATED, OH>::Residual res[R];
#pragma unroll
                    for (int i = 0; i < R; i++) out.template load<FAST>(p, m0 + c + 8 * i + col, res[i]);
#pragma unroll
                    for (int v = 0; v < S; v++) {
                        float a[SLAB];
                        if (PLANES == 1) tmem_cols<SLAB>(tbase + (buf * Sh::ACC + v) * NT + c, a);
#pragma unroll
                        for (int j = 0; j < SLAB; j++)
                            st[(v * SLAB + j) * TR + row] = PLANES == 1 ? a[j] : acc[v][PLANES == 1 ? 0 : c + j];
                    }
                    if (PLANES == 1 && c + SLAB == HC) release(buf);
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                    alignas(16) float v[4 * OH * R], g[4 * OH * R];
#pragma unroll
                    for (int i = 0; i < 2 * R; i++) {
                        float* to = MIX && (i & 1) ? g + 4 * (i >> 1) : v + 4 * (MIX ? i >> 1 : i);
                        *(float4*)to = *(const float4*)(src + (i >> 1) * 8 * TR + (i & 1) * 64);
                        if (S == 2) *(float4*)(g + 4 * i) = *(const float4*)(src + (SLAB + (i >> 1) * 8) * TR + (i & 1) * 64);
                    }
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + part) : "memory");
                    out.template store<FAST, R>(p, m0 + c + col, 8, v, g, res);
                };
                if (p.vec && n0 + 64 * OH <= p.N && m0 + HC <= p.M) {
                    if (PLANES == 1) {
#pragma unroll 1
                        for (int c = 0; c < HC; c += SLAB) slab(c, std::true_type{});
                    } else {
#pragma unroll
                        for (int c = 0; c < HC; c += SLAB) slab(c, std::true_type{});
                    }
                } else if (PLANES == 1) {
#pragma unroll 1
                    for (int c = 0; c < HC; c += SLAB) slab(c, std::false_type{});
                } else {
#pragma unroll
                    for (int c = 0; c < HC; c += SLAB) slab(c, std::false_type{});
                }
            }
        }
    }
    fence_before();
    __syncwarp();
    if (MODE == ONE && !met) cluster_wait();
    Columns<T, GATED, 2> last;
    typename Columns<T, GATED, 2>::Residual res[1];
    const int chunk = (int)threadIdx.x & 15, first = ((int)threadIdx.x - 64) >> 4;
    int tm = 0, tn = 0;
    int64_t mr = 0;
    bool fast = false;
    if (MODE == ONE && warp >= 2) {  // what the finish needs besides the sums, asked for before they are there
        tile_at(p, tiles_n, tile0, tm, tn);
        last.begin(p, tn * TR + chunk * 4);
        fast = p.vec && (tn + 1) * TR <= p.N;
        mr = (int64_t)tm * NT + rank * (NT >> p.log2_split);
        if (fast && mr + first < p.M) last.template load<true>(p, mr + first, res[0]);
    }
    __syncthreads();
    cluster_sync();  // ONE: all partial sums have arrived; PAIR: no CTA leaves while the other signals it
    if (MODE == ONE && !s_fail && warp >= 2) {
        const int cols = NT >> p.log2_split;
        for (int i = first; i < cols; i += EPI * 2) {
            const int64_t m = mr + i;
            if (m >= p.M) break;
            if (!fast) last.template load<false>(p, m, res[0]);
            else if (i != first) last.template load<true>(p, m, res[0]);
            float v[8], g[8];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = g[j] = 0.0f;
            const float* src = out_stage + (int64_t)i * split * TR + chunk * 4;
#pragma unroll 4
            for (int q = 0; q < split; q++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const float4 a = *(const float4*)(src + q * TR + 64 * h);
                    v[4 * h] += a.x; v[4 * h + 1] += a.y; v[4 * h + 2] += a.z; v[4 * h + 3] += a.w;
                    if (GATED) {
                        const float4 b = *(const float4*)(src + (cols * split + q) * TR + 64 * h);
                        g[4 * h] += b.x; g[4 * h + 1] += b.y; g[4 * h + 2] += b.z; g[4 * h + 3] += b.w;
                    }
                }
            }
            if (fast) last.template store<true, 1>(p, m, 0, v, g, res);
            else last.template store<false, 1>(p, m, 0, v, g, res);
        }
    }
    if (s_fail && threadIdx.x == 0 && p.err) atomicOr(p.err, KERR_TIMEOUT);
    if (warp == 1) {
        fence_after();
        if (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(ALLOC));
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(ALLOC));
    }
}

// ---- layouts ----------------------------------------------------------------------------------------

// One thread per 16-byte chunk of the tiles.
__global__ void k_tiles16(const uint16_t* __restrict__ w, int N, int K, int nkb, int64_t chunks, uint4* __restrict__ out) {
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < chunks; i += (int64_t)gridDim.x * blockDim.x) {
        const int c = (int)(i & 7), row = (int)(i >> 3) & (TR - 1);
        const int64_t blk = i >> 10;  // tile * nkb + kb
        const int64_t n = blk / nkb * TR + row;
        const int k = (int)(blk % nkb) * 64 + c * 8;
        alignas(16) uint16_t e[8];
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
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = n < N && k + j < K ? w[n * K + k + j] : 0.0f;
        uint4 part[3];
        split3(f, part);
#pragma unroll
        for (int q = 0; q < 3; q++)
            *(uint4*)(out + blk * (3 * TR * 64) + q * (TR * 64) + row * 64 + ((c ^ ((row >> 1) & 3)) << 4)) = part[q];
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
        alignas(16) float f[8];
        row8(x + m * ldx, k, K, f);
        uint4 part[3];
        split3(f, part);
#pragma unroll
        for (int q = 0; q < 3; q++) *(uint4*)(out + (q * M + m) * kp + k) = part[q];
    }
}

// 16-bit rows whose base or stride TMA cannot address, packed to rows of kp (a multiple of 8).
__global__ void k_pack_x(const uint16_t* __restrict__ x, int64_t ldx, int64_t M, int K, int kp, uint16_t* __restrict__ out) {
    const int64_t total = M * (kp / 8);
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t m = i / (kp / 8);
        const int k = (int)(i % (kp / 8)) * 8;
        *(uint4*)(out + m * kp + k) = row8(x + m * ldx, k, K);
    }
}

// Clusters of `size` CTAs of a kernel that can be resident at once (a GPC whose SMs are not a multiple of the
// size leaves some out). Asked once per kernel and size: the library is built for one GPU.
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
    if (cudaOccupancyMaxActiveClusters(&n, fn, &cfg) != cudaSuccess) cudaGetLastError();
    return std::max(n, 1);
}

struct Operands {
    const void* x;
    int64_t ldx;
    int width;  // 16-bit values of a row that hold data
};

template <class T, int NT, int PLANES, bool GATED, int MODE, bool MANUAL>
bool launch(const Plan& pl, const Call& c, const Operands& op, int log2_split, cudaStream_t st) {
    using Sh = Shape<NT, PLANES, GATED, MODE>;
    auto* fn = k_linear_tc<T, NT, PLANES, GATED, MODE, MANUAL>;
    if (ensure_smem((const void*)fn, Sh::SMEM) != cudaSuccess) return false;
    CUtensorMap tmx, tmw, tmg;
    if (MANUAL) {
        std::memset(&tmx, 0, sizeof tmx);
    } else if (!tc::encode_rows_planes(&tmx, op.x, op.width, c.M, op.ldx, PLANES, pl.bk(), Sh::XR)) {
        return false;
    }
    if (Sh::DUO) {  // the weights' blocks as lines of 128 bytes, swizzled already
        const int64_t lines = pl.tile_bytes() / 128;
        const int box = Sh::MIX ? TR * Sh::ROWB / 2 / 128 : Sh::WB / 128;
        if (!tc::encode_rows_u16(&tmw, pl.tiles, 64, lines, 64, box)) return false;
        if (GATED && !tc::encode_rows_u16(&tmg, pl.gtiles, 64, lines, 64, box)) return false;
    } else {
        tmw = tmx;
    }
    if (!GATED || !Sh::DUO) tmg = tmw;
    TcParams p;
    p.w = pl.tiles; p.g = pl.gtiles; p.bias = pl.bias; p.gbias = pl.gbias;
    p.r = c.r; p.y = c.y; p.ldr = c.ldr; p.ldo = c.ldo;
    p.x = c.x; p.ldx = c.ldx;
    p.M = (int)c.M; p.N = pl.N; p.K = pl.K; p.nkb = pl.nkb(); p.act = pl.act; p.f16 = pl.dtype == DT_F16;
    auto fours = [](const void* at, int64_t ld) { return (uintptr_t)at % (4 * sizeof(T)) == 0 && ld % 4 == 0; };
    p.vec = fours(c.y, c.ldo) && (!c.r || fours(c.r, c.ldr));
    p.tiles_n = pl.tiles_n();
    p.tiles_m = (int)((c.M + NT - 1) / NT);
    p.tiles = p.tiles_m * (Sh::DUO && !Sh::MIX ? (p.tiles_n + 1) / 2 : p.tiles_n);
    p.log2_split = log2_split;
    p.err = c.err;
    p.wait_limit = c.wait_limit > 0 ? c.wait_limit : tc::kWaitCycles;
    p.stall_mma = c.stall_mma;
    int grid = p.tiles << log2_split;
    if (Sh::DUO) {
        static std::atomic<int> clusters{0};
        int n = clusters.load();
        if (!n) clusters.store(n = resident_clusters((const void*)fn, Sh::SMEM, 2));
        grid = 2 * std::min(p.tiles, n);
    }
    const int size = Sh::DUO ? 2 : 1 << log2_split;
    return launch_early(fn, dim3((unsigned)grid), dim3(LT), Sh::SMEM, st, size, tmx, tmw, tmg, p) == cudaSuccess;
}

bool tma_rows(const Plan& p, const Call& c) {  // the caller's 16-bit rows as they are
    return p.planes() == 1 && (uintptr_t)c.x % 16 == 0 && c.ldx % 8 == 0;
}

template <class T, int PLANES, bool GATED, bool MANUAL>
bool run_one(const Plan& pl, const Call& c, const Operands& op, const Choice& ch, cudaStream_t st) {
    if (ch.nt == 32) return launch<T, 32, PLANES, GATED, ONE, MANUAL>(pl, c, op, ch.log2_split, st);
    if (ch.nt == 64) return launch<T, 64, PLANES, GATED, ONE, MANUAL>(pl, c, op, ch.log2_split, st);
    return launch<T, PLANES == 3 && GATED ? 64 : 128, PLANES, GATED, ONE, MANUAL>(pl, c, op, ch.log2_split, st);
}
template <class T, int PLANES, bool GATED>
bool run_pair(const Plan& pl, const Call& c, const Operands& op, const Choice& ch, cudaStream_t st) {
    constexpr int W = PLANES == 3 ? 128 : 256;
    if (ch.nt == W) return launch<T, W, PLANES, GATED, PAIR, false>(pl, c, op, 0, st);
    if (ch.nt == W / 2) return launch<T, W / 2, PLANES, GATED, PAIR, false>(pl, c, op, 0, st);
    return launch<T, W / 4, PLANES, GATED, PAIR, false>(pl, c, op, 0, st);
}
template <class T, int PLANES, bool GATED>
bool run(const Plan& pl, const Call& c, const Operands& op, const Choice& ch, cudaStream_t st) {
    if (ch.mode == PAIR) return run_pair<T, PLANES, GATED>(pl, c, op, ch, st);
    if constexpr (GATED && PLANES == 1)
        if (ch.mode == WIDE) return launch<T, 128, PLANES, GATED, WIDE, false>(pl, c, op, 0, st);
    if constexpr (PLANES == 3) return run_one<T, PLANES, GATED, true>(pl, c, op, ch, st);
    else return tma_rows(pl, c) ? run_one<T, PLANES, GATED, false>(pl, c, op, ch, st) : run_one<T, PLANES, GATED, true>(pl, c, op, ch, st);
}
template <class T, int PLANES>
bool run(const Plan& pl, const Call& c, const Operands& op, const Choice& ch, cudaStream_t st) {
    return pl.gated ? run<T, PLANES, true>(pl, c, op, ch, st) : run<T, PLANES, false>(pl, c, op, ch, st);
}

unsigned grid_for(int64_t items) { return (unsigned)std::min<int64_t>((items + 255) / 256, (int64_t)device_sm_count() * 16); }
int kp_of(const Plan& p) { return p.planes() == 3 ? p.nkb() * 32 : (p.K + 7) / 8 * 8; }
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

// The form and tile of a call, by an estimate of its SM cycles. Fixed parts and rates as measured
// (clock64 stamps in the kernel, and every form and tile of 60 shapes timed): about 3000 cycles from launch to the
// first MMA, a K block the larger of its MMAs (64 cycles each up to N = 128, N / 2 above) and its bytes at 56 a
// cycle, 1500 cycles for the exchange in a cluster and 64 bytes a cycle stored in it, four outputs a cycle in the
// epilogue. Clusters of 8 and 4 fit 15 and 33 times, pairs on all SMs. Gated 16-bit blocks wait for their bytes:
// 3300 cycles of latency over the stages in ONE, 420 cycles and their bytes at 100 a cycle in PAIR, 1000 in WIDE.
// 128 x 4096 x 11008, 86 tiles of 128 rows on 74 pairs: WIDE 41 us, PAIR 49, ONE 57; 512 x 2048 x 16384: PAIR 60,
// WIDE 68, ONE 120.
Choice choose(const Plan& p, const Call& c) {
    const int64_t M = c.M;
    const bool pass = !tma_rows(p, c);  // pairs need the rows split or packed, ONE loads them itself
    const int S = p.gated ? 2 : 1, planes = p.planes(), rowb = planes == 3 ? 64 : 128;
    const int steps = planes == 3 ? 12 : 4, sms = device_sm_count();
    const int widest = planes == 3 ? 128 / S : 256 / S, pair_widest = planes == 3 ? 128 : 256;  // accumulators in TMEM
    // Cycles of a K block whose weights come from memory (3300 bytes a cycle), read by `ctas` CTAs at a time; those of
    // up to GROUP_M activation tiles share three quarters of them.
    auto dram = [](double ctas, double bytes, double tiles_m) {
        return ctas * bytes / 3300.0 / (0.25 + 0.75 * std::min<double>(tiles_m, GROUP_M));
    };
    Choice best;
    for (int nt = 32; nt <= 256; nt *= 2) {
        const double tiles_m = (double)((M + nt - 1) / nt), mma = std::max(64, nt / 2);
        const double rows = std::min<double>(nt, (double)M), out = rows * TR * S / 4.0;
        if (nt <= std::min(widest, 128)) {
            for (int l = 0; l < 4; l++) {
                const int split = 1 << l;
                if (l && p.nkb() < 2 * split) break;
                const int fit = split == 8 ? 15 : split == 4 ? 33 : sms / split;
                const double tiles = tiles_m * p.tiles_n();
                const double waves = std::ceil(tiles / fit);
                double block = std::max(S * steps * mma, (S * planes * TR * rowb + planes * nt * rowb) / 56.0);
                if (p.gated && planes == 1) {
                    const int stage = (2 * TR + nt) * rowb, stages = std::min(8, (SMEM_MAX - 1536 - 2 * nt * TR * 4) / stage);
                    block = std::max({block, 3300.0 / stages, dram(std::min<double>(tiles * split, sms), 2 * TR * rowb, tiles_m)});
                }
                if (pass) block = std::max(block, planes == 3 ? 1100.0 + 6.0 * nt : 200.0 + 22.0 * nt);
                const double t = waves * (3000 + std::ceil((double)p.nkb() / split) * block + out / split +
                                          (l ? 1500 + S * rows * TR * 4 / 64.0 : rows * TR * S * 4 / 256.0));
                if (!best.nt || t < best.cycles) best = Choice{nt, ONE, l, t};
            }
        }
        for (const int mode : {PAIR, WIDE}) {
            if (mode == PAIR ? nt > pair_widest || nt * 4 < pair_widest : !p.gated || planes == 3 || nt != 128) continue;
            const bool mix = p.gated && mode == PAIR;
            const double tiles = tiles_m * (mix ? p.tiles_n() : (p.tiles_n() + 1) / 2), sums = rows * TR * (mode == WIDE ? 2 : 1) / 4.0;
            const double loads = planes * rowb * (TR + nt / 2);
            double block = mode == WIDE ? 1000.0 : mix && planes == 1 ? 420.0 + loads / 100.0 : std::max(steps * mma * 1.15, loads / 56.0);
            if (mix && planes == 1) block = std::max(block, dram(std::min<double>(2 * tiles, sms), TR * rowb, tiles_m));
            const double work = p.nkb() * block;
            double t = 4500 + std::ceil(tiles / (sms / 2)) * std::max(work, sums) + std::min(work, sums);
            if (pass) t += 3500 + (double)M * p.K * (planes == 3 ? 10 : 4) / 3000.0;
            if (t < best.cycles) best = Choice{nt, mode, 0, t};
        }
    }
    return best;
}

bool has_form(const Plan& p, const Choice& ch) {
    const int planes = p.planes(), widest = (planes == 3 ? 128 : 256) / (p.gated ? 2 : 1), pair_widest = planes == 3 ? 128 : 256;
    const bool width = ch.nt == 32 || ch.nt == 64 || ch.nt == 128 || ch.nt == 256;
    if (ch.mode == ONE) return width && ch.nt <= std::min(widest, 128) && (!ch.log2_split || p.nkb() >= 2 << ch.log2_split);
    if (ch.log2_split) return false;
    return ch.mode == PAIR ? width && ch.nt <= pair_widest && ch.nt * 4 >= pair_widest : ch.mode == WIDE && p.gated && planes == 1 && ch.nt == 128;
}

size_t tc_workspace(const Plan& p, const Call& c, const Choice& ch) {
    if (tma_rows(p, c) || ch.mode == ONE) return 0;
    return (size_t)p.planes() * c.M * kp_of(p) * 2;
}

int tc(const Plan& p, const Call& c, const Choice& ch, void* ws, cudaStream_t st) {
    const bool direct = tma_rows(p, c);
    Operands op{c.x, c.ldx, p.K};
    int n = 0;
    if (!direct && ch.mode != ONE) {
        const int kp = kp_of(p);
        const unsigned grid = grid_for(c.M * (kp / 8));
        if (p.planes() == 3) k_split_x<<<grid, 256, 0, st>>>((const float*)c.x, c.ldx, c.M, p.K, kp, (uint16_t*)ws);
        else k_pack_x<<<grid, 256, 0, st>>>((const uint16_t*)c.x, c.ldx, c.M, p.K, kp, (uint16_t*)ws);
        op = Operands{ws, kp, kp};
        n++;
    }
    bool ok;
    if (p.dtype == DT_F32) ok = run<float, 3>(p, c, op, ch, st);
    else if (p.dtype == DT_F16) ok = run<__half, 1>(p, c, op, ch, st);
    else ok = run<__nv_bfloat16, 1>(p, c, op, ch, st);
    return ok ? n + 1 : -1;
}

}  // namespace lin
}  // namespace slx
