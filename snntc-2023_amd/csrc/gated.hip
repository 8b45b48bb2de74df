// Gated running mean along a sequence, per channel:
//     a_t = sigmoid(gate_t),   h_t = a_t h_{t-1} + (1 - a_t) x_t,   y_t = h_t
// and its gradient, with u the gradient that reaches h_t:
//     u_t = dy_t + a_{t+1} u_{t+1}  (the last step of a sequence: dy_t + dfinal)
//     dx_t = (1 - a_t) u_t,   dgate_t = u_t (h_{t-1} - x_t) a_t (1 - a_t),   dstate = a_1 u_1
// A step mixes two spike times, so what comes out lies between those that went in and is a spike time itself.
#include "snntc_common.h"

namespace snntc {
namespace {

// a = sigmoid(g) and 1 - a, each to its own precision: with e = exp(-g), a = 1 / (1 + e) and 1 - a = e a.  (Below -80, where 1 - a
// is 1 and a below 2e-35, e is held finite.  A NaN stays one.)
struct Gate { float a, rest; };
__device__ __forceinline__ Gate gate_of(float g) {
    const float e = expf(g < -80.0f ? 80.0f : -g);
    const float a = 1.0f / (1.0f + e);
    return Gate{a, e * a};
}

__device__ __forceinline__ int length_of(const int64_t* lengths, int64_t b, int64_t T) {
    if (!lengths) return (int)T;
    const int64_t n = lengths[b];
    return (int)(n < 0 ? 0 : n > T ? T : n);
}

template <typename G>
__global__ void __launch_bounds__(256)
gated_scan_forward_kernel(const float* __restrict__ x, const G* __restrict__ gate, const float* __restrict__ state,
                          const int64_t* __restrict__ lengths, float* __restrict__ y, float* __restrict__ final_state, int T, int D) {
    const int64_t b = blockIdx.y;
    const int d = blockIdx.x * 256 + threadIdx.x;
    if (d >= D) return;
    const int n = length_of(lengths, b, T);
    const size_t base = (size_t)b * T * D + d;
    float h = state ? state[b * D + d] : 0.0f;
    for (int t = 0; t < T; ++t) {
        const size_t e = base + (size_t)t * D;
        if (t < n) {
            const Gate g = gate_of((float)gate[e]);
            h = g.a * h + g.rest * x[e];
        }
        y[e] = t < n ? h : 0.0f;
    }
    if (final_state) final_state[b * D + d] = h;
}

template <typename G>
__global__ void __launch_bounds__(256)
gated_scan_backward_kernel(const float* __restrict__ dy, const float* __restrict__ dfinal, const float* __restrict__ x,
                           const G* __restrict__ gate, const float* __restrict__ y, const float* __restrict__ state,
                           const int64_t* __restrict__ lengths, float* __restrict__ dx, G* __restrict__ dgate, float* __restrict__ dstate,
                           int T, int D) {
    const int64_t b = blockIdx.y;
    const int d = blockIdx.x * 256 + threadIdx.x;
    if (d >= D) return;
    const int n = length_of(lengths, b, T);
    const size_t base = (size_t)b * T * D + d;
    float u = dfinal ? dfinal[b * D + d] : 0.0f;
    for (int t = T - 1; t >= 0; --t) {
        const size_t e = base + (size_t)t * D;
        if (t >= n) {
            if (dx) dx[e] = 0.0f;
            if (dgate) dgate[e] = (G)0.0f;
            continue;
        }
        const Gate g = gate_of((float)gate[e]);
        const float before = t > 0 ? y[e - D] : state ? state[b * D + d] : 0.0f;
        if (dy) u += dy[e];
        if (dx) dx[e] = g.rest * u;
        if (dgate) dgate[e] = (G)(u * (before - x[e]) * (g.a * g.rest));
        u *= g.a;
    }
    if (dstate) dstate[b * D + d] = u;
}

template <typename G>
__global__ void __launch_bounds__(256)
gated_step_kernel(const float* x, const G* gate, const float* state, float* out, long long n) {
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
    if (e >= n) return;
    const Gate g = gate_of((float)gate[e]);
    out[e] = g.a * (state ? state[e] : 0.0f) + g.rest * x[e];
}

}  // namespace

size_t gated_scan_workspace(int64_t, int64_t, int64_t) { return 0; }

int launch_gated_scan_forward(const float* x, const void* gate, int type, const float* state, const int64_t* lengths, float* y,
                              float* final_state, int64_t B, int64_t T, int64_t D, void*, hipStream_t stream) {
    if (B > 65535) return fail(SNNTC_ERR_TOO_LARGE, "gated scan: too many sequences");
    with_type(type, [&](auto g) {
        using G = decltype(g);
        KernelTimerScope timer_("gated_scan_forward", stream);
        hipLaunchKernelGGL(gated_scan_forward_kernel<G>, dim3((unsigned)((D + 255) / 256), (unsigned)B), dim3(256), 0, stream, x,
                           static_cast<const G*>(gate), state, lengths, y, final_state, (int)T, (int)D);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

int launch_gated_scan_backward(const float* dy, const float* dfinal, const float* x, const void* gate, int type, const float* y,
                               const float* state, const int64_t* lengths, float* dx, void* dgate, float* dstate, int64_t B, int64_t T,
                               int64_t D, void*, hipStream_t stream) {
    if (B > 65535) return fail(SNNTC_ERR_TOO_LARGE, "gated scan: too many sequences");
    with_type(type, [&](auto g) {
        using G = decltype(g);
        KernelTimerScope timer_("gated_scan_backward", stream);
        hipLaunchKernelGGL(gated_scan_backward_kernel<G>, dim3((unsigned)((D + 255) / 256), (unsigned)B), dim3(256), 0, stream, dy, dfinal,
                           x, static_cast<const G*>(gate), y, state, lengths, dx, static_cast<G*>(dgate), dstate, (int)T, (int)D);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

int launch_gated_step(const float* x, const void* gate, int type, const float* state, float* out, int64_t n, hipStream_t stream) {
    const int64_t blocks = (n + 255) / 256;
    if (blocks > 0x7fffffffLL) return fail(SNNTC_ERR_TOO_LARGE, "gated step: too many elements");
    with_type(type, [&](auto g) {
        using G = decltype(g);
        KernelTimerScope timer_("gated_step", stream);
        hipLaunchKernelGGL(gated_step_kernel<G>, dim3((unsigned)blocks), dim3(256), 0, stream, x, static_cast<const G*>(gate), state, out,
                           (long long)n);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

}  // namespace snntc
