// Losses over choices.  A row of spike times t[J] stands for the distribution softmax(-t): the earlier an output, the likelier.
// Of every row one output a was chosen;
//     logp = -t_a - log sum_j exp(-t_j),     d logp / d t_j = p_j - [j = a],   p = softmax(-t),
// and any loss that is a function of the rows' logp has the gradient c (p_j - [j = a]) in row times, c = d loss / d logp.
//   policy       loss = k (exp(d) - d - 1) - min(r A, clip(r) A),  r = exp(logp - old), d = ref - logp
//                c    = k (1 - exp(d)) - (r A where r A <= clip(r) A)
//   preference   S_q = sum_t w_qt logp_qt,  m = beta ((S - R)_preferred - (S - R)_rejected)
//                loss = -(1 - e) log sig(m) - e log sig(-m),  d loss / d m = e sig(m) - (1 - e) sig(-m)
// logsumexp is kept as the pair (maximum, log of the sum above it): neurons that never fire sit at MAX_SPIKE_TIME, and in a row of
// them the one number 10^5 + log J would have lost the logarithm's digits.
// A row of weight 0 is not read: its loss, logp and gradient are 0.
#include "snntc_common.h"

namespace snntc {
namespace {

constexpr int kThreads = 256;

// Running maximum m and sum s of exp(v - m); empty: m = -inf, s = 0.
struct Soft { float m, s; };
__device__ __forceinline__ Soft join(const Soft& a, const Soft& b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return Soft{m, a.s + b.s};                     // nothing yet (or a NaN sum to keep)
    return Soft{m, a.s * expf(a.m - m) + b.s * expf(b.m - m)};
}
__device__ __forceinline__ Soft wave_join(Soft v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v = join(v, Soft{__shfl_xor(v.m, d, kWave), __shfl_xor(v.s, d, kWave)});
    return v;
}

__device__ __forceinline__ float row_weight(const float* weight, int64_t r) { return weight ? weight[r] : 1.0f; }

// logp of the row's token; NaN for a token outside [0, J).
template <typename E>
__device__ __forceinline__ float token_logp(const E* t, long long token, int J, float2 soft) {
    return token >= 0 && token < J ? (-(float)t[token] - soft.x) - soft.y : NAN;
}

template <typename E>
__global__ void __launch_bounds__(kThreads)
time_logp_kernel(const E* __restrict__ times, const long long* __restrict__ tokens, const float* __restrict__ weight,
                 float* __restrict__ logp, float2* __restrict__ stats, int J) {
    __shared__ Soft part[kThreads / kWave];
    const int64_t r = blockIdx.x;
    if (row_weight(weight, r) == 0.0f) {
        if (threadIdx.x == 0) { logp[r] = 0.0f; if (stats) stats[r] = float2{0.0f, 0.0f}; }
        return;
    }
    const E* __restrict__ t = times + (size_t)r * J;
    float m = -INFINITY;
    for (int j = threadIdx.x; j < J; j += kThreads) m = fmaxf(m, -(float)t[j]);
    float s = 0.0f;
    for (int j = threadIdx.x; j < J; j += kThreads) s += expf(-(float)t[j] - (m == -INFINITY ? 0.0f : m));
    const Soft w = wave_join(Soft{m, s});
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = w;
    __syncthreads();
    if (threadIdx.x == 0) {
        Soft v = part[0];
        for (int i = 1; i < kThreads / kWave; ++i) v = join(v, part[i]);
        const float2 soft{v.m, logf(v.s)};
        logp[r] = token_logp(t, tokens[r], J, soft);
        if (stats) stats[r] = soft;
    }
}

template <typename E>
__global__ void __launch_bounds__(kThreads)
time_logp_backward_kernel(const E* __restrict__ times, const long long* __restrict__ tokens, const float2* __restrict__ stats,
                          const float* __restrict__ coef, const float* __restrict__ upstream, E* __restrict__ dtimes, int J) {
    const int64_t r = blockIdx.x;
    const float c = coef[r];
    const float up = upstream ? *upstream : 1.0f;
    E* __restrict__ g = dtimes + (size_t)r * J;
    if (c == 0.0f) {
        for (int j = threadIdx.x; j < J; j += kThreads) g[j] = (E)0.0f;
        return;
    }
    const E* __restrict__ t = times + (size_t)r * J;
    const long long token = tokens[r];
    const float2 soft = stats[r];
    const float cu = c * up;
    for (int j = threadIdx.x; j < J; j += kThreads) g[j] = (E)(cu * (expf((-(float)t[j] - soft.x) - soft.y) - (j == token ? 1.0f : 0.0f)));
}

__global__ void __launch_bounds__(kThreads)
policy_rows_kernel(const float* __restrict__ logp, PolicyArgs a, float* __restrict__ row_loss, float* __restrict__ coef, int64_t rows) {
    const int64_t r = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (r >= rows) return;
    const float w = a.weight ? a.weight[r] : a.mean;
    if (w == 0.0f) {
        row_loss[r] = 0.0f;
        coef[r] = 0.0f;
        return;
    }
    const float lp = logp[r], adv = a.advantage[r];
    const float ratio = expf(lp - a.old_logp[r]);
    const float plain = ratio * adv, clipped = fminf(fmaxf(ratio, a.low), a.high) * adv;
    float loss = -(plain <= clipped ? plain : clipped), c = plain <= clipped ? -plain : 0.0f;
    if (isnan(ratio) || isnan(plain)) loss = c = NAN;
    if (a.ref_logp && a.kl != 0.0f) {
        const float d = a.ref_logp[r] - lp, e = expm1f(d);
        loss += a.kl * (d == INFINITY ? d : e - d);                    // (inf - inf where the output can never be chosen)
        c -= a.kl * e;
    }
    row_loss[r] = loss;
    coef[r] = c * w;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
}

// log(1 + exp(v))
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))); }

// One wavefront per pair.
__global__ void __launch_bounds__(kWave)
preference_pairs_kernel(const float* __restrict__ logp, PreferenceArgs a, float* __restrict__ pair_loss, float* __restrict__ seq_logp,
                        float* __restrict__ coef, int64_t P, int T) {
    const int64_t p = blockIdx.x;
    float seq[2];
    for (int half = 0; half < 2; ++half) {
        const int64_t q = p + half * P;
        float s = 0.0f;
        for (int t = threadIdx.x; t < T; t += kWave) {
            const float w = row_weight(a.weight, q * T + t);
            if (w != 0.0f) s = fmaf(w, logp[q * T + t], s);
        }
        seq[half] = wave_sum(s);
        if (threadIdx.x == 0) seq_logp[q] = seq[half];
    }
    const float m = a.beta * ((seq[0] - a.ref_logp[p]) - (seq[1] - a.ref_logp[p + P]));
    if (threadIdx.x == 0) pair_loss[p] = (1.0f - a.smoothing) * softplus(-m) + a.smoothing * softplus(m);
    const float slope = a.beta / (float)P * (a.smoothing / (1.0f + expf(-m)) - (1.0f - a.smoothing) / (1.0f + expf(m)));
    for (int half = 0; half < 2; ++half) {
        const int64_t q = p + half * P;
        for (int t = threadIdx.x; t < T; t += kWave) coef[q * T + t] = row_weight(a.weight, q * T + t) * (half ? -slope : slope);
    }
}

// total = sum weight loss, or the mean where weight is NULL; one workgroup, so that the order of the sum is fixed.
__global__ void __launch_bounds__(1024)
loss_total_kernel(const float* __restrict__ loss, const float* __restrict__ weight, float* __restrict__ total, int64_t n) {
    __shared__ float part[1024 / kWave];
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        if (!weight) s += loss[i];
        else if (weight[i] != 0.0f) s = fmaf(weight[i], loss[i], s);
    }
    s = wave_sum(s);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0f;
        for (int i = 0; i < 1024 / kWave; ++i) s += part[i];
        *total = weight ? s : s / (float)n;
    }
}

}  // namespace

size_t choice_workspace(int64_t rows, int64_t) { return align_up((size_t)rows * sizeof(float)) * 4; }

int launch_time_logp(const void* times, int type, const int64_t* tokens, const float* weight, float* logp, float* stats, int64_t rows,
                     int64_t J, void*, hipStream_t stream) {
    with_type(type, [&](auto e) {
        using E = decltype(e);
        KernelTimerScope timer_("time_logp", stream);
        hipLaunchKernelGGL(time_logp_kernel<E>, dim3((unsigned)rows), dim3(kThreads), 0, stream, static_cast<const E*>(times),
                           reinterpret_cast<const long long*>(tokens), weight, logp, reinterpret_cast<float2*>(stats), (int)J);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

int launch_time_logp_backward(const void* times, int type, const int64_t* tokens, const float* stats, const float* coef,
                              const float* upstream, void* dtimes, int64_t rows, int64_t J, hipStream_t stream) {
    with_type(type, [&](auto e) {
        using E = decltype(e);
        KernelTimerScope timer_("time_logp_backward", stream);
        hipLaunchKernelGGL(time_logp_backward_kernel<E>, dim3((unsigned)rows), dim3(kThreads), 0, stream, static_cast<const E*>(times),
                           reinterpret_cast<const long long*>(tokens), reinterpret_cast<const float2*>(stats), coef, upstream, static_cast<E*>(dtimes), (int)J);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

namespace {
// Row arrays the caller does not want are kept in the workspace.
struct RowArrays {
    float *logp, *stats, *coef;
    RowArrays(float* logp_, float* stats_, float* coef_, int64_t rows, void* ws) : logp(logp_), stats(stats_), coef(coef_) {
        char* scratch = static_cast<char*>(ws);
        const size_t piece = align_up((size_t)rows * sizeof(float));
        if (!coef) coef = reinterpret_cast<float*>(scratch);
        if (!logp) logp = reinterpret_cast<float*>(scratch + piece);
        if (!stats) stats = reinterpret_cast<float*>(scratch + 2 * piece);
    }
};
}  // namespace

int launch_policy_loss(const void* times, int type, const int64_t* actions, const PolicyArgs& a, float* row_loss, float* logp, float* stats,
                       float* coef, void* dtimes, int64_t rows, int64_t J, void* ws, hipStream_t stream) {
    const RowArrays ra(logp, stats, coef, rows, ws);
    int rc = launch_time_logp(times, type, actions, a.weight, ra.logp, ra.stats, rows, J, ws, stream);
    if (rc) return rc;
    {
        KernelTimerScope timer_("policy_rows", stream);
        hipLaunchKernelGGL(policy_rows_kernel, dim3((unsigned)((rows + kThreads - 1) / kThreads)), dim3(kThreads), 0, stream, ra.logp, a,
                           row_loss, ra.coef, rows);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return dtimes ? launch_time_logp_backward(times, type, actions, ra.stats, ra.coef, nullptr, dtimes, rows, J, stream) : SNNTC_OK;
}

int launch_preference_loss(const void* times, int type, const int64_t* tokens, const PreferenceArgs& a, float* pair_loss,
                           float* seq_logp, float* stats, float* coef, void* dtimes, int64_t P, int64_t T, int64_t J, void* ws,
                           hipStream_t stream) {
    const int64_t rows = 2 * P * T;
    const RowArrays ra(nullptr, stats, coef, rows, ws);
    int rc = SNNTC_OK;
    if (rows > 0) rc = launch_time_logp(times, type, tokens, a.weight, ra.logp, ra.stats, rows, J, ws, stream);
    if (rc) return rc;
    {
        KernelTimerScope timer_("preference_pairs", stream);
        hipLaunchKernelGGL(preference_pairs_kernel, dim3((unsigned)P), dim3(kWave), 0, stream, ra.logp, a, pair_loss, seq_logp, ra.coef, P,
                           (int)T);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    if (!dtimes || rows == 0) return SNNTC_OK;
    return launch_time_logp_backward(times, type, tokens, ra.stats, ra.coef, nullptr, dtimes, rows, J, stream);
}

int launch_loss_total(const float* loss, const float* weight, float* total, int64_t n, hipStream_t stream) {
    {
        KernelTimerScope timer_("loss_total", stream);
        hipLaunchKernelGGL(loss_total_kernel, dim3(1), dim3(1024), 0, stream, loss, weight, total, n);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

}  // namespace snntc
