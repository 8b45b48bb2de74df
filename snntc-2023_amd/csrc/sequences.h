// The operators over sequences of tokens and choices (embed.hip, gated.hip, choice.hip): element types, what their kernels share and
// their launches.
#pragma once

#include "snntc_common.h"

namespace snntc {

// Element types of tables, gates and times (SNNTC_F32 / SNNTC_BF16 / SNNTC_F16).  Arithmetic is fp32, in 64 bits where a
// file says so; a result is rounded to its type once, to nearest even, when it is stored.
inline size_t type_bytes(int type) { return type == SNNTC_F32 ? 4 : 2; }
template <typename F>
int with_type(int type, F&& f) {
    switch (type) {
        case SNNTC_F32: return f(float{});
        case SNNTC_BF16: return f(__bf16{});
        default: return f(_Float16{});
    }
}

// One dimension of a launch holds less than 2^32 threads; more workgroups than that go on in the second one.  A kernel that is launched so
// counts by workgroup() and leaves out what lies behind its last one (there may be up to kGridRow - 1 too many).
constexpr int64_t kGridRow = 1 << 20;
inline dim3 wide_grid(int64_t blocks, int threads) {
    if (blocks * threads < (1ll << 32)) return dim3((unsigned)blocks);
    return dim3((unsigned)kGridRow, (unsigned)((blocks + kGridRow - 1) / kGridRow));
}
__device__ __forceinline__ int64_t workgroup() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }

// Calls that touch more than the caches hold (256 MB, the memory's own included) store their results past them: otherwise what the next
// kernel reads waits for the write-back of what this one has left.  Smaller calls leave their results where the next kernel finds them.
constexpr int64_t kStreamBytes = 256ll << 20;

// exp(v) by the hardware's base-2 exponential: v log2(e) is rounded once, and what the rounding and log2(e)'s own have lost is put back to
// first order, so the result is off by the hardware's step and half of one (one half-step of t is worth |t| half-steps of 2^t otherwise).
// The library's function is off by one step; this is about half of its instructions.  Below 2^-126 the result is 0.
__device__ __forceinline__ float exp_close(float v) {
    const float t = v * 1.44269502f;                                     // float(log2 e)
    const float lost = fmaf(v, 1.44269502f, -t) + v * 1.92596299e-8f;    // log2 e - float(log2 e)
    const float near = __builtin_amdgcn_exp2f(t);
    return fabsf(t) < 128.0f ? fmaf(near, lost * 0.693147181f, near) : near;           // (else 0, infinity or NaN)
}

int launch_embed_forward(const void* tokens, int token_bytes, const void* table, int type, float* z, int64_t N, int64_t V, int64_t D,
                         float scale, bool encode, hipStream_t stream);
size_t embed_backward_workspace(int64_t N, int64_t V, int64_t D);
int launch_embed_backward(const float* grad, const void* tokens, int token_bytes, const void* table, int type, void* dtable, int64_t N,
                          int64_t V, int64_t D, float scale, bool encode, void* ws, hipStream_t stream);

size_t gated_scan_workspace(int64_t B, int64_t T, int64_t D);
int launch_gated_scan_forward(const float* x, const void* gate, int type, const float* state, const int64_t* lengths, float* y,
                              float* final_state, int64_t B, int64_t T, int64_t D, void* ws, hipStream_t stream);
int launch_gated_scan_backward(const float* dy, const float* dfinal, const float* x, const void* gate, int type, const float* y,
                               const float* state, const int64_t* lengths, float* dx, void* dgate, float* dstate, int64_t B, int64_t T,
                               int64_t D, void* ws, hipStream_t stream);
int launch_gated_step(const float* x, const void* gate, int type, const float* state, float* out, int64_t n, hipStream_t stream);

// The policy loss as the kernels take it; ref_logp, weight: may be NULL.
struct PolicyArgs {
    const float* old_logp;
    const float* advantage;
    const float* ref_logp;
    const float* weight;
    float low, high;                       // ends of the clipped ratio
    float kl, mean;                        // mean: weight of a row where weight is NULL
};
struct PreferenceArgs {
    const float* ref_logp;
    const float* weight;
    float beta, smoothing;
};
size_t choice_workspace(int64_t rows, int64_t J);
size_t preference_workspace(int64_t rows, int64_t J);
int launch_time_logp(const void* times, int type, const int64_t* tokens, const float* weight, float* logp, float* stats, int64_t rows,
                     int64_t J, void* ws, hipStream_t stream);
int launch_time_logp_backward(const void* times, int type, const int64_t* tokens, const float* stats, const float* coef,
                              const float* upstream, void* dtimes, int64_t rows, int64_t J, hipStream_t stream);
int launch_policy_loss(const void* times, int type, const int64_t* actions, const PolicyArgs& a, float* row_loss, float* logp, float* stats,
                       float* coef, void* dtimes, int64_t rows, int64_t J, void* ws, hipStream_t stream);
int launch_preference_loss(const void* times, int type, const int64_t* tokens, const PreferenceArgs& a, float* pair_loss,
                           float* seq_logp, float* stats, float* coef, void* dtimes, int64_t P, int64_t T, int64_t J, void* ws,
                           hipStream_t stream);
int launch_loss_total(const float* loss, const float* weight, float* total, int64_t n, hipStream_t stream);

}  // namespace snntc
