// slx_ctx.h -- the context behind the C ABI's slx_ctx handle and the helpers its entry points share.
#pragma once
#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <string>
#include <vector>

#include <cuda_runtime.h>

#include "slx.h"
#include "slx_gemm.h"

// Kernel classes reported by slx_profile_end.
enum KClass { KC_GEMM, KC_ATTENTION, KC_NORM, KC_ROPE, KC_FFN_GATE, KC_EMBED, KC_POOL, KC_ADD, KC_ARGMAX, KC_GEMV,
              KC_SPLIT, KC_FALLBACK, KC_SEARCH, KC_VOCAB, KC_COUNT };

struct ProfRecord {
    int cls;
    int launches;
    cudaEvent_t a, b;
    double macs, bytes, tc_macs;
};

struct slx_ctx {
    int device = 0;
    cudaStream_t stream = nullptr;
    std::string err;
    int* d_flag = nullptr;
    int64_t launches = 0;            // kernels queued by the library on this context
    bool prof = false;
    std::vector<ProfRecord> records;
    slx::GemmWorkspace kws;          // scratch of the kernel-level matmul entry points
    slx::WaitOptions wait;           // bounded-wait settings of the tensor-core GEMMs (slx_ctx_set_option)
    int linear_form = 0;             // SLX_OPT_TEST_LINEAR_FORM
    std::atomic<int> refs{1};        // slx_destroy's reference plus one per live object created on it
    cudaMemPool_t pool = nullptr;    // stream-ordered scratch of the float operators, made at first use
    std::vector<cudaEvent_t> event_pool;
    cudaEvent_t event() {
        if (!event_pool.empty()) { cudaEvent_t e = event_pool.back(); event_pool.pop_back(); return e; }
        cudaEvent_t e = nullptr;
        cudaEventCreate(&e);
        return e;
    }
};

// Runs one launcher (which returns how many kernels it queued), counting launches and, when
// profiling, bracketing it with events on the launch stream.
template <class F>
static inline void run_k(slx_ctx* c, int cls, double macs, double bytes, cudaStream_t st, F&& f, double tc_macs = 0) {
    if (!c->prof) {
        c->launches += f();
        return;
    }
    ProfRecord r{cls, 0, c->event(), c->event(), macs, bytes, tc_macs};
    cudaEventRecord(r.a, st);
    r.launches = f();
    cudaEventRecord(r.b, st);
    c->launches += r.launches;
    c->records.push_back(r);
}

namespace slx {

inline int set_err(slx_ctx* c, int code, const char* fmt, ...) {
    if (!c) return code;
    char buf[1024];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    c->err = buf;
    return code;
}

#define CK(call)                                                                                 \
    do {                                                                                         \
        cudaError_t e_ = (call);                                                                 \
        if (e_ != cudaSuccess) {                                                                 \
            cudaGetLastError(); /* reported here: not once more by the next call's check */      \
            return set_err(ctx, e_ == cudaErrorMemoryAllocation ? SLX_EOOM : SLX_ECUDA, "%s: %s", \
                           #call, cudaGetErrorString(e_));                                      \
        }                                                                                        \
    } while (0)

// Makes a device current for one scope and puts the caller's back.
struct OnDevice {
    int prev = -1;
    cudaError_t err;
    explicit OnDevice(int dev) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != dev) err = cudaSetDevice(dev);
        else prev = -1;
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

inline cudaStream_t pick(slx_ctx* ctx, void* s) { return s ? (cudaStream_t)s : ctx->stream; }

// Drops one reference; the last one frees the context. The current device stays what it is.
void ctx_release(slx_ctx* ctx);

}  // namespace slx
