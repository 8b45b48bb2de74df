// Spike times of tokens, and the gradient of their table.
//     z[n,:] = scale E[tok_n,:]   or, encoded like an image's intensities, exp(1 - scale E[tok_n,:])
//     dE[v,:] = k_v sum over the n with tok_n = v of g[n,:],   k_v = scale, or -scale exp(1 - scale E[v,:])
// The gradient is a sum of rows by token.  Atomic adds would make its last digits depend on the order in which workgroups run;
// here the tokens are sorted first (by token, then by position), and the rows are added in that order.
#include "snntc_common.h"

namespace snntc {
namespace {

// ---- forward -------------------------------------------------------------------------------------

__device__ __forceinline__ float time_of(float e, float scale, bool encode) {
    return encode ? expf(1.0f - scale * e) : scale * e;
}

template <typename E, typename I>
__global__ void __launch_bounds__(256)
embed_forward_kernel(const I* __restrict__ tokens, const E* __restrict__ table, float* __restrict__ z, int V, int D, float scale,
                     bool encode) {
    const int64_t n = blockIdx.x;
    const long long tok = tokens[n];
    const bool known = tok >= 0 && tok < V;
    const E* __restrict__ row = table + (size_t)(known ? tok : 0) * D;
    for (int d = threadIdx.x; d < D; d += 256) z[(size_t)n * D + d] = known ? time_of((float)row[d], scale, encode) : NAN;
}

// ---- gradient ------------------------------------------------------------------------------------

// Place of every position in the order (token, position): the number of positions that come before it.  Positions whose token
// lies outside the table count as token V and end up last.
constexpr int kRankThreads = 256;
template <typename I>
__global__ void __launch_bounds__(kRankThreads)
token_rank_kernel(const I* __restrict__ tokens, int* __restrict__ sorted_token, int* __restrict__ sorted_pos, int N, int V) {
    const int n = blockIdx.x * kRankThreads + threadIdx.x;
    auto key = [&](int i) {
        const long long t = tokens[i];
        return t >= 0 && t < V ? (int)t : V;
    };
    __shared__ int tile[kRankThreads];
    const int own = n < N ? key(n) : 0;
    int rank = 0;
    for (int i0 = 0; i0 < N; i0 += kRankThreads) {
        __syncthreads();
        if (i0 + (int)threadIdx.x < N) tile[threadIdx.x] = key(i0 + threadIdx.x);
        __syncthreads();
        const int count = min(kRankThreads, N - i0);
        for (int i = 0; i < count; ++i) rank += tile[i] < own || (tile[i] == own && i0 + i < n);
    }
    if (n < N) {
        sorted_token[rank] = own;
        sorted_pos[rank] = n;
    }
}

// A wavefront owns 64 columns of one table row and adds up its rows of g in order.
template <typename E>
__global__ void __launch_bounds__(256)
embed_backward_kernel(const float* __restrict__ grad, const int* __restrict__ sorted_token, const int* __restrict__ sorted_pos,
                      const E* __restrict__ table, E* __restrict__ dtable, int N, int D, float scale, bool encode) {
    const int v = blockIdx.x;
    int lo = 0, hi = N;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (sorted_token[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    for (int d = threadIdx.x; d < D; d += 256) {
        float s = 0.0f;
        for (int i = lo; i < N && sorted_token[i] == v; ++i) s += grad[(size_t)sorted_pos[i] * D + d];
        const size_t e = (size_t)v * D + d;
        dtable[e] = (E)(encode ? -scale * expf(1.0f - scale * (float)table[e]) * s : scale * s);
    }
}

}  // namespace

int launch_embed_forward(const void* tokens, int token_bytes, const void* table, int type, float* z, int64_t N, int64_t V, int64_t D,
                         float scale, bool encode, hipStream_t stream) {
    with_type(type, [&](auto e) {
        using E = decltype(e);
        KernelTimerScope timer_("embed_forward", stream);
        if (token_bytes == 8)
            hipLaunchKernelGGL((embed_forward_kernel<E, int64_t>), dim3((unsigned)N), dim3(256), 0, stream,
                               static_cast<const int64_t*>(tokens), static_cast<const E*>(table), z, (int)V, (int)D, scale, encode);
        else
            hipLaunchKernelGGL((embed_forward_kernel<E, int32_t>), dim3((unsigned)N), dim3(256), 0, stream,
                               static_cast<const int32_t*>(tokens), static_cast<const E*>(table), z, (int)V, (int)D, scale, encode);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

size_t embed_backward_workspace(int64_t N, int64_t, int64_t) { return align_up((size_t)N * sizeof(int)) * 2; }

int launch_embed_backward(const float* grad, const void* tokens, int token_bytes, const void* table, int type, void* dtable, int64_t N,
                          int64_t V, int64_t D, float scale, bool encode, void* ws, hipStream_t stream) {
    int* sorted_token = static_cast<int*>(ws);
    int* sorted_pos = reinterpret_cast<int*>(static_cast<char*>(ws) + align_up((size_t)N * sizeof(int)));
    if (N > 0) {
        KernelTimerScope timer_("token_rank", stream);
        const dim3 grid((unsigned)((N + kRankThreads - 1) / kRankThreads));
        if (token_bytes == 8)
            hipLaunchKernelGGL(token_rank_kernel<int64_t>, grid, dim3(kRankThreads), 0, stream, static_cast<const int64_t*>(tokens),
                               sorted_token, sorted_pos, (int)N, (int)V);
        else
            hipLaunchKernelGGL(token_rank_kernel<int32_t>, grid, dim3(kRankThreads), 0, stream, static_cast<const int32_t*>(tokens),
                               sorted_token, sorted_pos, (int)N, (int)V);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    with_type(type, [&](auto e) {
        using E = decltype(e);
        KernelTimerScope timer_("embed_backward", stream);
        hipLaunchKernelGGL(embed_backward_kernel<E>, dim3((unsigned)V), dim3(256), 0, stream, grad, sorted_token, sorted_pos,
                           static_cast<const E*>(table), static_cast<E*>(dtable), (int)N, (int)D, scale, encode);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

}  // namespace snntc
