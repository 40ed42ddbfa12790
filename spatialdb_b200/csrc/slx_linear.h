// slx_linear.h -- float matrix product with bias, activation, gate and residual in its epilogue.
//   y[m][n] = act(sum_k x[m][k] w[n][k] + b[n]) + r[m][n]
//   gated:    act(x . g^T + gb) * (x . w^T + b) + r
// Weights are laid out once (linear_prepare); calls stream them.
#pragma once
#include <cstdint>
#include <string>

#include <cuda_runtime.h>

#include "slx_gemm.h"

namespace slx {
namespace lin {

constexpr int TR = 128;  // weight rows per tile (the MMA's M, one TMEM lane each)

// One operator's weights in device memory, owned by the handle.
//   f16 / bf16: tiles [N / 128][K / 64] of 128 rows x 128 bytes, 16-byte chunks XORed with row % 8 (the
//               128-byte swizzle the tensor core reads), rows and columns past N and K zero;
//   f32:        rows [N][k4] as given (k4 = K rounded up to 4) for the products of few rows, and for the
//               tensor core tiles [N / 128][K / 32][3] of 128 rows x 64 bytes: the three bf16 parts of
//               each value, 64-byte swizzle.
struct Plan {
    int dtype = 0;  // DT_F32, DT_F16 or DT_BF16: activations, residual and output
    int N = 0, K = 0, act = 0;
    bool gated = false;
    uint8_t *tiles = nullptr, *gtiles = nullptr;
    float *rows = nullptr, *grows = nullptr;
    float *bias = nullptr, *gbias = nullptr;
    size_t bytes = 0;
    int planes() const { return dtype == 0 ? 3 : 1; }
    int bk() const { return dtype == 0 ? 32 : 64; }                  // K values per block
    int nkb() const { return (K + bk() - 1) / bk(); }
    int64_t block_bytes() const { return (int64_t)planes() * TR * bk() * 2; }
    int tiles_n() const { return (N + TR - 1) / TR; }
    int64_t tile_bytes() const { return (int64_t)(tiles_n() + 1) / 2 * 2 * nkb() * block_bytes(); }  // a pair of tiles at a time
    int64_t k4() const { return (K + 3) / 4 * 4; }
};

struct Call {
    const void* x = nullptr;
    int64_t ldx = 0;
    const void* r = nullptr;
    int64_t ldr = 0;
    void* y = nullptr;
    int64_t ldo = 0;
    int64_t M = 0;
    int* err = nullptr;
    long long wait_limit = 0;
    int stall_mma = 0;
};

// Lays out N x K weights given as f32 (dtype f32) or as 16-bit values of the plan's type.
void layout(const Plan& p, const void* w, uint8_t* tiles, float* rows, cudaStream_t st);

// Products of few rows on the CUDA cores' load path (k_linear_few.cu); false when M is past its range.
bool few_supported(const Plan& p, int64_t M);
int few(const Plan& p, const Call& c, cudaStream_t st);

// The tensor-core product (k_linear_tc.cu): its form and tile for a call, the scratch that form needs (0: none),
// laid out by the call, and the call itself, which returns the kernels queued, -1 when a tensor map could not
// be encoded or a launch failed.
struct Choice {
    int nt = 0, mode = 0, log2_split = 0;
    double cycles = 0;
};
Choice choose(const Plan& p, const Call& c);
bool has_form(const Plan& p, const Choice& ch);  // whether the kernel is built for it and the sums can be split so
size_t tc_workspace(const Plan& p, const Call& c, const Choice& ch);
int tc(const Plan& p, const Call& c, const Choice& ch, void* ws, cudaStream_t st);

}  // namespace lin
}  // namespace slx
