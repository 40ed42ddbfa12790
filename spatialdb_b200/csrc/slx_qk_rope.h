// slx_qk_rope.h -- norms of queries and keys for each head and the position rotation in one pass
// (k_qk_rope.cu): float rows (f32, f16, bf16) and the Q30 integers of the causal path.
#pragma once
#include <cstdint>
#include <vector>

#include <cuda_runtime.h>

namespace slx {

// IntegerRoPECache (Math/IntegerAttention.cs:14-32): Q30 cos / sin tables [rows][hd / 2] on the host.
void rope_table(int rows, int hd, float base, std::vector<int64_t>& cs, std::vector<int64_t>& sn);

// One tensor's rows: row m at in + m * ld_in holds nh heads of hd; w (nullable: no norm) has hd values.
struct QkSide {
    const void* in = nullptr;
    void* out = nullptr;
    int64_t ld_in = 0, ld_out = 0;
    int nh = 0;
    const void* w = nullptr;
};

struct QkRope {
    QkSide q, k;
    int hd = 0, half = 0;          // head size, pairs rotated (2 * half <= hd)
    int64_t M = 0, T = 0;          // rows; without pos, row m stands at position m % T
    const int32_t* pos = nullptr;  // positions (-1: the row is left as it is)
    int table_rows = 0;
    const float2* table = nullptr;                       // float: (cos, sin) [table_rows][half]
    const int64_t *cs = nullptr, *sn = nullptr;          // Q30: [table_rows][half]
    float eps = 0.0f;
    double inv_hd = 0.0;           // 1 / hd, set by the Q30 launcher
    int* err = nullptr;            // context error word: KERR_RANGE for a position outside the table
};

// u = x / sqrt(mean(x^2) + eps) * w for each head (u = x without a weight), then each pair
// (u_p, u_{p + half}) rotated by its position's angle; values past 2 * half keep u. dtype: DT_F32, DT_F16
// or DT_BF16, weights float. out may be in (same pointer and row stride). Returns the kernels queued.
int qk_norm_rope(int dtype, const QkRope& p, cudaStream_t st);

// RmsNormRow of every head (IntegerLayerNorm.cs:71-93), then ApplyRoPE (IntegerAttention.cs:35-58) with
// half = hd / 2, int64 Q30 rows and weights: the same integers as rmsnorm_rows followed by rope_rows.
int qk_norm_rope_q30(const QkRope& p, cudaStream_t st);

}  // namespace slx
