// slx_operators.cu -- C ABI of the float linear operator and of the fused query/key norm and rotation.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <memory>
#include <new>
#include <vector>

#include <cuda_runtime.h>

#include "gguf.hpp"
#include "slx.h"
#include "slx_ctx.h"
#include "slx_kernels.h"
#include "slx_linear.h"
#include "slx_qk_rope.h"
#include "slx_rows.h"

using namespace slx;

static_assert(SLX_DTYPE_F32 == GG_F32 && SLX_DTYPE_F16 == GG_F16 && SLX_DTYPE_BF16 == GG_BF16, "GGUF dtype ids");

namespace {

bool is_float(int dtype) { return dtype == SLX_DTYPE_F32 || dtype == SLX_DTYPE_F16 || dtype == SLX_DTYPE_BF16; }
int width_of(int dtype) { return dtype == SLX_DTYPE_F32 ? 4 : dtype == SLX_DTYPE_Q30 ? 8 : 2; }

// The pool of the calls' stream-ordered scratch, made with the first operator (a call may be in a capture).
// Every call has its own allocation, so calls on several streams and captured graphs (whose allocations belong
// to the graph) never share one. The pool keeps what is freed.
int ensure_pool(slx_ctx* ctx) {
    if (ctx->pool) return SLX_OK;
    cudaMemPoolProps props = {};
    props.allocType = cudaMemAllocationTypePinned;
    props.location.type = cudaMemLocationTypeDevice;
    props.location.id = ctx->device;
    CK(cudaMemPoolCreate(&ctx->pool, &props));
    uint64_t keep = ~0ull;
    CK(cudaMemPoolSetAttribute(ctx->pool, cudaMemPoolAttrReleaseThreshold, &keep));
    return SLX_OK;
}

}  // namespace

struct slx_linear {
    slx_ctx* ctx = nullptr;
    lin::Plan plan;
    ~slx_linear() {
        for (void* p : {(void*)plan.tiles, (void*)plan.gtiles, (void*)plan.rows, (void*)plan.grows, (void*)plan.bias,
                        (void*)plan.gbias})
            cudaFree(p);
    }
};

struct slx_rope {
    slx_ctx* ctx = nullptr;
    std::atomic<int> refs{1};  // slx_rope_free's reference plus one per slx_qk_norm
    int rows = 0, rot = 0, q30 = 0;
    float2* table = nullptr;
    int64_t *cs = nullptr, *sn = nullptr;
    ~slx_rope() {
        cudaFree(table);
        cudaFree(cs);
        cudaFree(sn);
    }
};

struct slx_qk_norm {
    slx_ctx* ctx = nullptr;
    slx_rope* rope = nullptr;
    int dtype = 0, heads = 0, kv_heads = 0, hd = 0;
    float eps = 0.0f;
    void *wq = nullptr, *wk = nullptr;
    ~slx_qk_norm() {
        cudaFree(wq);
        cudaFree(wk);
    }
};

namespace {

void rope_release(slx_rope* r) {
    if (r->refs.fetch_sub(1) != 1) return;
    slx_ctx* ctx = r->ctx;
    delete r;
    ctx_release(ctx);
}

// One weight array laid out for the operator: any decodable GGUF type through f32 for f32 activations, the
// activations' own type otherwise.
int linear_weights(slx_ctx* ctx, lin::Plan& p, const uint8_t* d_w, int64_t w_bytes, int w_dtype, uint8_t** tiles,
                   float** rows) {
    const int64_t n = (int64_t)p.N * p.K;
    const int64_t need = gguf_decode_bytes((uint32_t)w_dtype, n);
    if (need < 0) return set_err(ctx, SLX_EUNSUPPORTED, "Dequantization of dtype %d is not yet implemented", w_dtype);
    if (p.dtype != SLX_DTYPE_F32 && w_dtype != p.dtype)
        return set_err(ctx, SLX_EUNSUPPORTED, "weights of dtype %d with activations of dtype %d", w_dtype, p.dtype);
    if (w_bytes < need)
        return set_err(ctx, SLX_EEOF, "weight buffer too small: expected %lld bytes, got %lld", (long long)need, (long long)w_bytes);
    const int align = w_dtype == GG_F32 ? 4 : w_dtype == GG_MXFP4 ? 1 : 2;
    if ((uintptr_t)d_w % align) return set_err(ctx, SLX_EINVAL, "weights not aligned to %d bytes", align);
    const void* src = d_w;
    float* wide = nullptr;
    if (p.dtype == SLX_DTYPE_F32 && w_dtype != GG_F32) {
        int* flag = nullptr;
        int bad = 0;
        CK(cudaMalloc(&wide, sizeof(float) * n + 16));
        flag = (int*)(wide + n);
        cudaMemsetAsync(flag, 0, sizeof(int), ctx->stream);
        dequant_f32(w_dtype, d_w, n, wide, flag, ctx->stream);
        cudaMemcpyAsync(&bad, flag, sizeof(int), cudaMemcpyDeviceToHost, ctx->stream);
        const cudaError_t e = cudaStreamSynchronize(ctx->stream);
        if (e != cudaSuccess || bad) {
            cudaFree(wide);
            if (bad) return set_err(ctx, SLX_ERANGE, "MXFP4 nibble 15 (index outside the 15-entry table)");
            return set_err(ctx, SLX_ECUDA, "%s", cudaGetErrorString(e));
        }
        src = wide;
    }
    const size_t tb = (size_t)p.tile_bytes(), rb = p.dtype == SLX_DTYPE_F32 ? sizeof(float) * p.N * p.k4() : 0;
    cudaError_t e = cudaMalloc(tiles, tb);
    if (e == cudaSuccess && rb) e = cudaMalloc(rows, rb);
    if (e == cudaSuccess) {
        lin::layout(p, src, *tiles, rb ? *rows : nullptr, ctx->stream);
        e = cudaGetLastError();
        const cudaError_t s = cudaStreamSynchronize(ctx->stream);
        if (e == cudaSuccess) e = s;
    }
    cudaFree(wide);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_err(ctx, e == cudaErrorMemoryAllocation ? SLX_EOOM : SLX_ECUDA, "%s", cudaGetErrorString(e));
    }
    p.bytes += tb + rb;
    return SLX_OK;
}

int copy_vector(slx_ctx* ctx, const void* d_v, size_t bytes, void** out) {
    if (!d_v) return SLX_OK;
    CK(cudaMalloc(out, bytes));
    CK(cudaMemcpyAsync(*out, d_v, bytes, cudaMemcpyDeviceToDevice, ctx->stream));
    CK(cudaStreamSynchronize(ctx->stream));
    return SLX_OK;
}

}  // namespace

extern "C" {

// ---- linear ------------------------------------------------------------------------------------------

slx_status slx_linear_prepare(slx_ctx* ctx, int dtype, const uint8_t* d_w, int64_t w_bytes, int w_dtype, int N, int K,
                              const float* d_bias, int act, const uint8_t* d_gate, int64_t gate_bytes,
                              const float* d_gate_bias, slx_linear** out) {
    if (!ctx || !out) return set_err(ctx, SLX_EINVAL, "null argument");
    *out = nullptr;
    if (!d_w || N <= 0 || K <= 0 || w_bytes < 0 || gate_bytes < 0) return set_err(ctx, SLX_EINVAL, "bad arguments");
    if (!is_float(dtype)) return set_err(ctx, SLX_EUNSUPPORTED, "activations of dtype %d", dtype);
    if (act < SLX_ACT_NONE || act > SLX_ACT_GELU_ERF) return set_err(ctx, SLX_EINVAL, "unknown activation %d", act);
    if (!d_gate && d_gate_bias) return set_err(ctx, SLX_EINVAL, "a gate bias without gate weights");
    if (N > (1 << 30) || K > (1 << 30)) return set_err(ctx, SLX_EINVAL, "weights of %d x %d", N, K);
    if (((uintptr_t)d_bias | (uintptr_t)d_gate_bias) % 4) return set_err(ctx, SLX_EINVAL, "bias not aligned to 4 bytes");
    OnDevice on(ctx->device);
    CK(on.err);
    if (int rc = ensure_pool(ctx)) return rc;
    std::unique_ptr<slx_linear> h(new (std::nothrow) slx_linear());
    if (!h) return set_err(ctx, SLX_EOOM, "host memory");
    h->ctx = ctx;
    lin::Plan& p = h->plan;
    p.dtype = dtype; p.N = N; p.K = K; p.act = act; p.gated = d_gate != nullptr;
    int st = linear_weights(ctx, p, d_w, w_bytes, w_dtype, &p.tiles, &p.rows);
    if (!st && d_gate) st = linear_weights(ctx, p, d_gate, gate_bytes, w_dtype, &p.gtiles, &p.grows);
    if (!st) st = copy_vector(ctx, d_bias, sizeof(float) * N, (void**)&p.bias);
    if (!st) st = copy_vector(ctx, d_gate_bias, sizeof(float) * N, (void**)&p.gbias);
    if (st) return st;
    ctx->refs.fetch_add(1);
    *out = h.release();
    return SLX_OK;
}

slx_status slx_linear_free(slx_linear* l) {
    if (!l) return SLX_EINVAL;
    slx_ctx* ctx = l->ctx;
    {
        OnDevice on(ctx->device);
        delete l;  // cudaFree waits for the work that still reads the weights
    }
    ctx_release(ctx);
    return SLX_OK;
}

slx_status slx_linear_info(slx_linear* l, int64_t* info, int n) {
    if (!l || !info) return SLX_EINVAL;
    const lin::Plan& p = l->plan;
    const int64_t v[6] = {p.dtype, p.N, p.K, p.act, p.gated, (int64_t)p.bytes};
    for (int i = 0; i < n && i < 6; i++) info[i] = v[i];
    return SLX_OK;
}

slx_status slx_linear_device(slx_linear* l, const slx_linear_args* a) {
    if (!l) return SLX_EINVAL;
    slx_ctx* ctx = l->ctx;
    if (!a) return set_err(ctx, SLX_EINVAL, "null argument");
    const lin::Plan& p = l->plan;
    const int64_t M = a->M;
    if (M < 0) return set_err(ctx, SLX_EINVAL, "M %lld < 0", (long long)M);
    if (M == 0) return SLX_OK;
    const int e = width_of(p.dtype);
    if (!a->x || !a->y) return set_err(ctx, SLX_EINVAL, "null argument");
    if (a->ldx < p.K || a->ldy < p.N || (a->residual && a->ldr < p.N))
        return set_err(ctx, SLX_EINVAL, "row stride below the row's width (K %d, N %d)", p.K, p.N);
    if (((uintptr_t)a->x | (uintptr_t)a->y | (uintptr_t)a->residual) % e)
        return set_err(ctx, SLX_EINVAL, "rows not aligned to %d bytes", e);
    if (M > (1 << 30) || (M + 31) / 32 * p.tiles_n() > (1ll << 27) || a->ldx > (1ll << 36))
        return set_err(ctx, SLX_EINVAL, "M %lld with N %d, row stride %lld", (long long)M, p.N, (long long)a->ldx);
    if (rows_overlap(a->x, a->ldx, p.K, a->y, a->ldy, p.N, M, e)) return set_err(ctx, SLX_EINVAL, "y overlaps x");
    if ((a->residual != a->y || (M > 1 && a->ldr != a->ldy)) && rows_overlap(a->residual, a->ldr, p.N, a->y, a->ldy, p.N, M, e))
        return set_err(ctx, SLX_EINVAL, "y overlaps the residual without being it");
    OnDevice on(ctx->device);
    CK(on.err);
    cudaStream_t st = pick(ctx, a->stream);
    lin::Call c;
    c.x = a->x; c.ldx = a->ldx; c.r = a->residual; c.ldr = a->ldr; c.y = a->y; c.ldo = a->ldy; c.M = M;
    c.err = ctx->d_flag;
    c.wait_limit = ctx->wait.limit_cycles;
    c.stall_mma = ctx->wait.stall_mma;
    const double macs = (double)M * p.N * p.K * (p.gated ? 2 : 1);
    const double bytes = (double)e * (M * p.K + (double)p.N * p.K * (p.gated ? 2 : 1) + M * p.N * (a->residual ? 2 : 1));
    if (!ctx->linear_form && lin::few_supported(p, M)) {
        run_k(ctx, KC_GEMV, macs, bytes, st, [&] { return lin::few(p, c, st); });
        CK(cudaGetLastError());
        return SLX_OK;
    }
    lin::Choice ch;
    if (const int form = ctx->linear_form) {
        ch.nt = form % 1024; ch.mode = form / 1024 % 4; ch.log2_split = form / 4096;
        if (!lin::has_form(p, ch))
            return set_err(ctx, SLX_EUNSUPPORTED, "linear form %d (width %d, mode %d, split %d)", form, ch.nt, ch.mode, 1 << ch.log2_split);
    } else {
        ch = lin::choose(p, c);
    }
    void* ws = nullptr;
    if (const size_t need = lin::tc_workspace(p, c, ch)) {
        CK(cudaMallocFromPoolAsync(&ws, need, ctx->pool, st));
    }
    int n = 0;
    run_k(ctx, KC_GEMM, macs, bytes, st, [&] { return (n = lin::tc(p, c, ch, ws, st)) < 0 ? 0 : n; });
    const cudaError_t launched = cudaGetLastError();
    if (ws) CK(cudaFreeAsync(ws, st));
    if (launched != cudaSuccess || n < 0)
        return set_err(ctx, SLX_ECUDA, "linear launch: %s", cudaGetErrorString(launched));
    return SLX_OK;
}

// ---- query / key norm and rotation -------------------------------------------------------------------

slx_status slx_rope_create(slx_ctx* ctx, int rows, int rot_dim, float base, int q30, slx_rope** out) {
    if (!ctx || !out) return set_err(ctx, SLX_EINVAL, "null argument");
    *out = nullptr;
    if (rows <= 0 || rot_dim <= 0 || rot_dim % 2 || rot_dim > 65536 || !(base > 0.0f) || !std::isfinite(base))
        return set_err(ctx, SLX_EINVAL, "bad rotation table: %d rows, width %d, base %g", rows, rot_dim, (double)base);
    if ((int64_t)rows * (rot_dim / 2) > (1 << 28))
        return set_err(ctx, SLX_EINVAL, "rotation table of %d rows x %d: more than 2^28 entries", rows, rot_dim / 2);
    OnDevice on(ctx->device);
    CK(on.err);
    std::unique_ptr<slx_rope> r;
    try {
        r.reset(new slx_rope());
        r->ctx = ctx;
        r->rows = rows; r->rot = rot_dim; r->q30 = q30 ? 1 : 0;
        const int half = rot_dim / 2;
        const size_t n = (size_t)rows * half;
        if (q30) {
            std::vector<int64_t> cs, sn;
            rope_table(rows, rot_dim, base, cs, sn);
            CK(cudaMalloc(&r->cs, n * 8));
            CK(cudaMalloc(&r->sn, n * 8));
            CK(cudaMemcpyAsync(r->cs, cs.data(), n * 8, cudaMemcpyHostToDevice, ctx->stream));
            CK(cudaMemcpyAsync(r->sn, sn.data(), n * 8, cudaMemcpyHostToDevice, ctx->stream));
            CK(cudaStreamSynchronize(ctx->stream));
        } else {
            // Angles in double, each entry rounded to fp32 once: far positions keep their angle.
            std::vector<double> theta((size_t)half);
            for (int i = 0; i < half; i++) theta[i] = std::pow((double)base, -2.0 * i / rot_dim);
            std::vector<float2> t(n);
            for (int m = 0; m < rows; m++)
                for (int i = 0; i < half; i++) {
                    const double a = m * theta[i];
                    t[(size_t)m * half + i] = make_float2((float)std::cos(a), (float)std::sin(a));
                }
            CK(cudaMalloc(&r->table, n * sizeof(float2)));
            CK(cudaMemcpyAsync(r->table, t.data(), n * sizeof(float2), cudaMemcpyHostToDevice, ctx->stream));
            CK(cudaStreamSynchronize(ctx->stream));
        }
    } catch (const std::bad_alloc&) {
        return set_err(ctx, SLX_EOOM, "host memory for a rotation table of %d rows", rows);
    }
    ctx->refs.fetch_add(1);
    *out = r.release();
    return SLX_OK;
}

slx_status slx_rope_free(slx_rope* r) {
    if (!r) return SLX_EINVAL;
    OnDevice on(r->ctx->device);
    rope_release(r);
    return SLX_OK;
}

slx_status slx_qk_norm_prepare(slx_rope* r, int dtype, int heads, int kv_heads, int head_dim, const void* d_wq,
                               const void* d_wk, float eps, slx_qk_norm** out) {
    if (!r) return SLX_EINVAL;
    slx_ctx* ctx = r->ctx;
    if (!out) return set_err(ctx, SLX_EINVAL, "null argument");
    *out = nullptr;
    const bool q30 = dtype == SLX_DTYPE_Q30;
    if (!q30 && !is_float(dtype)) return set_err(ctx, SLX_EUNSUPPORTED, "heads of dtype %d", dtype);
    if (q30 != (r->q30 != 0)) return set_err(ctx, SLX_EINVAL, "a %s rotation table for dtype %d", r->q30 ? "Q30" : "float", dtype);
    if (heads < 0 || kv_heads < 0 || heads + (int64_t)kv_heads <= 0 || heads + (int64_t)kv_heads > 65536 || head_dim <= 0 ||
        head_dim > 65536 || r->rot > head_dim)
        return set_err(ctx, SLX_EINVAL, "bad heads: %d + %d of %d, %d rotated", heads, kv_heads, head_dim, r->rot);
    if (q30 && (r->rot != head_dim || eps != 0.0f))
        return set_err(ctx, SLX_EINVAL, "the Q30 form rotates whole heads and has no eps");
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return set_err(ctx, SLX_EINVAL, "eps %g", (double)eps);
    const int e = q30 ? 8 : 4;
    if (((uintptr_t)d_wq | (uintptr_t)d_wk) % e) return set_err(ctx, SLX_EINVAL, "norm weights not aligned to %d bytes", e);
    OnDevice on(ctx->device);
    CK(on.err);
    std::unique_ptr<slx_qk_norm> h(new (std::nothrow) slx_qk_norm());
    if (!h) return set_err(ctx, SLX_EOOM, "host memory");
    h->ctx = ctx;
    h->dtype = dtype; h->heads = heads; h->kv_heads = kv_heads; h->hd = head_dim; h->eps = eps;
    if (int st = copy_vector(ctx, d_wq, (size_t)e * head_dim, &h->wq)) return st;
    if (int st = copy_vector(ctx, d_wk, (size_t)e * head_dim, &h->wk)) return st;
    h->rope = r;
    r->refs.fetch_add(1);
    ctx->refs.fetch_add(1);
    *out = h.release();
    return SLX_OK;
}

slx_status slx_qk_norm_free(slx_qk_norm* h) {
    if (!h) return SLX_EINVAL;
    slx_ctx* ctx = h->ctx;
    {
        OnDevice on(ctx->device);
        slx_rope* r = h->rope;
        delete h;
        rope_release(r);
    }
    ctx_release(ctx);
    return SLX_OK;
}

slx_status slx_qk_norm_rope_device(slx_qk_norm* h, const slx_qk_args* a) {
    if (!h) return SLX_EINVAL;
    slx_ctx* ctx = h->ctx;
    if (!a) return set_err(ctx, SLX_EINVAL, "null argument");
    const slx_rope* r = h->rope;
    const int64_t M = a->M, T = a->T;
    if (M < 0) return set_err(ctx, SLX_EINVAL, "M %lld < 0", (long long)M);
    if (M == 0) return SLX_OK;
    const int e = width_of(h->dtype);
    const int64_t nq = (int64_t)h->heads * h->hd, nk = (int64_t)h->kv_heads * h->hd;
    if ((nq && (!a->q || !a->qo)) || (nk && (!a->k || !a->ko))) return set_err(ctx, SLX_EINVAL, "null argument");
    if ((nq && (a->ldq < nq || a->ldqo < nq)) || (nk && (a->ldk < nk || a->ldko < nk)))
        return set_err(ctx, SLX_EINVAL, "row stride below the row's width (q %lld, k %lld)", (long long)nq, (long long)nk);
    if (((nq ? (uintptr_t)a->q | (uintptr_t)a->qo : 0) | (nk ? (uintptr_t)a->k | (uintptr_t)a->ko : 0)) % e)
        return set_err(ctx, SLX_EINVAL, "rows not aligned to %d bytes", e);
    if ((uintptr_t)a->pos % 4) return set_err(ctx, SLX_EINVAL, "positions not aligned to 4 bytes");
    if (!a->pos && T <= 0) return set_err(ctx, SLX_EINVAL, "sequence length %lld", (long long)T);
    if (!a->pos && std::min(T, M) > r->rows)
        return set_err(ctx, SLX_ERANGE, "sequence length %lld exceeds the RoPE table (%d rows)", (long long)T, r->rows);
    if (M > (1ll << 32) / (h->heads + h->kv_heads))
        return set_err(ctx, SLX_EINVAL, "M %lld rows of %d heads", (long long)M, h->heads + h->kv_heads);
    auto meet = [&](const void* x, int64_t ldx, int64_t wx, const void* y, int64_t ldy, int64_t wy) {
        return wx && wy && rows_overlap(x, ldx, wx, y, ldy, wy, M, e);
    };
    if (((a->qo != a->q || (M > 1 && a->ldqo != a->ldq)) && meet(a->q, a->ldq, nq, a->qo, a->ldqo, nq)) ||
        ((a->ko != a->k || (M > 1 && a->ldko != a->ldk)) && meet(a->k, a->ldk, nk, a->ko, a->ldko, nk)) ||
        meet(a->q, a->ldq, nq, a->ko, a->ldko, nk) || meet(a->k, a->ldk, nk, a->qo, a->ldqo, nq) ||
        meet(a->qo, a->ldqo, nq, a->ko, a->ldko, nk))
        return set_err(ctx, SLX_EINVAL, "an output overlaps the inputs, or the other output, without being its input");
    OnDevice on(ctx->device);
    CK(on.err);
    cudaStream_t st = pick(ctx, a->stream);
    QkRope p;
    p.q.in = a->q; p.q.out = a->qo; p.q.ld_in = a->ldq; p.q.ld_out = a->ldqo; p.q.nh = h->heads; p.q.w = h->wq;
    p.k.in = a->k; p.k.out = a->ko; p.k.ld_in = a->ldk; p.k.ld_out = a->ldko; p.k.nh = h->kv_heads; p.k.w = h->wk;
    p.hd = h->hd; p.half = r->rot / 2; p.M = M; p.T = T; p.pos = a->pos;
    p.table_rows = r->rows; p.table = r->table; p.cs = r->cs; p.sn = r->sn;
    p.eps = h->eps; p.err = ctx->d_flag;
    run_k(ctx, KC_ROPE, 0, 2.0 * e * M * (nq + nk), st,
          [&] { return h->dtype == SLX_DTYPE_Q30 ? qk_norm_rope_q30(p, st) : qk_norm_rope(h->dtype, p, st); });
    CK(cudaGetLastError());
    return SLX_OK;
}

}  // extern "C"
