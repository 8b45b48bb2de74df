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
#include "sequences.h"

namespace snntc {
namespace {

// Running maximum m and sum s of exp(v - m); empty: m = -inf, s = 0.
struct Soft { float m, s; };
// exp by the hardware's base-2 exponential: the argument's product with log2(e) adds its own size in half steps to the result's
// error, of terms that shrink faster than that grows.  For the terms of sums, and for gradients that are rounded to 16 bits; an element of
// a float32 gradient is one exponential by itself (off by up to 32 half steps at times of 13 that way, by 5 with what the product loses).
__device__ __forceinline__ float exp_fast(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
__device__ __forceinline__ Soft join(const Soft& a, const Soft& b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return Soft{m, a.s + b.s};                     // nothing yet (or a NaN sum to keep)
    return Soft{m, a.s * exp_close(a.m - m) + b.s * exp_close(b.m - m)};
}
template <int WIDTH>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int d = WIDTH / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, kWave));
    return v;
}
template <int WIDTH>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = WIDTH / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
}

__device__ __forceinline__ float row_weight(const float* weight, int64_t r) { return weight ? weight[r] : 1.0f; }

struct RowLoss { float loss, coef; };
// The policy loss of a row, and its derivative by logp.  In float32: logp is one, half a step of which (2^-24 |logp|) goes into the ratio and
// the distance from the reference whatever is done with it, and what these operations add is no more.  expm1 keeps the digits of a small
// distance, of which the KL term is half the square.
__device__ __forceinline__ RowLoss policy_row(const PolicyArgs& a, int64_t r, float lp) {
    const float adv = a.advantage[r];
    const float ratio = expf(lp - a.old_logp[r]);
    const float plain = ratio * adv, clipped = fminf(fmaxf(ratio, a.low), a.high) * adv;
    RowLoss out{-(plain <= clipped ? plain : clipped), plain <= clipped ? -plain : 0.0f};
    if (isnan(ratio) || isnan(plain)) out.loss = out.coef = NAN;
    if (a.ref_logp && a.kl != 0.0f) {
        const float d = a.ref_logp[r] - lp, e = expm1f(d);
        out.loss += a.kl * (d == INFINITY ? d : e - d);                // (inf - inf where the output can never be chosen)
        out.coef -= a.kl * e;
    }
    return out;
}

// What a kernel over rows does with them.
enum Mode {
    LOGP,                                           // logp and statistics
    POLICY,                                         // the same, the row's loss and, if wanted, its gradient
    GRAD                                            // the gradient from statistics and coef
};
struct RowArgs {
    const long long* tokens;
    const float* weight;
    float* logp;
    float2* stats;
    float* coef;
    float* row_loss;
    const float* upstream;                          // GRAD: a factor, NULL: 1
    PolicyArgs policy;
    int64_t rows;
    int J;
};

// A row in pieces of VEC elements (16 bytes): those at 16-byte boundaries, `lead` elements before the first and `tail` behind the
// last one.  VEC = 1: every element a piece, for times and dtimes that lie differently to such boundaries.
template <typename E, int VEC>
struct alignas(VEC * sizeof(E)) Piece { E v[VEC]; };
// Keeps the compiler from carrying a piece's elements in float32 from one use to the next: sixteen 16-bit pieces a thread would take
// all registers that way, eight half of the wavefronts a SIMD can have.
template <typename P>
__device__ __forceinline__ void forget(P& p) {
    if constexpr (sizeof(P) == 16) {
        typedef unsigned Words __attribute__((ext_vector_type(4)));
        Words w = __builtin_bit_cast(Words, p);
        asm volatile("" : "+v"(w));
        p = __builtin_bit_cast(P, w);
    }
}
template <bool STREAM, typename P>
__device__ __forceinline__ void store_piece(P* to, const P& p) {
    if constexpr (STREAM) {
        typedef unsigned Words __attribute__((ext_vector_type(sizeof(P) / sizeof(unsigned))));
        __builtin_nontemporal_store(__builtin_bit_cast(Words, p), reinterpret_cast<Words*>(to));
    } else {
        *to = p;
    }
}
struct Cut { int lead, pieces, tail; };
template <typename E, int VEC>
__device__ __forceinline__ Cut cut_row(const E* t, int J) {
    if (VEC == 1) return Cut{0, J, 0};
    Cut c;
    c.lead = min(J, (int)((-(uintptr_t)t & (VEC * sizeof(E) - 1)) / sizeof(E)));
    c.pieces = (J - c.lead) / VEC;
    c.tail = J - c.lead - c.pieces * VEC;
    return c;
}
// The single element thread k < 2 * VEC takes apart from its pieces, -1: none.
template <int VEC>
__device__ __forceinline__ int odd_element(const Cut& c, int k) {
    if (VEC == 1) return -1;
    if (k < c.lead) return k;
    return k >= VEC && k < VEC + c.tail ? c.lead + c.pieces * VEC + k - VEC : -1;
}

// c p of an element, from the row's maximum and c over its sum.
template <typename E>
__device__ __forceinline__ float grad_of(E t, float top, float share) {
    const float v = -(float)t - top;
    return share * (sizeof(E) == sizeof(float) ? exp_close(v) : exp_fast(v));
}

// WIDTH threads own a row and hold all of it in registers, so that it is read once: R pieces each, at most WIDTH * R * VEC elements and
// the odd ones.  Up to 64 threads a row: several rows a workgroup.
// Bound by memory: 4096 rows of 32000 outputs in 16 bits, a part of them of weight 0, with their gradient 95 us, 5.0 TB/s.
template <typename E, int VEC, int WIDTH, int R, Mode MODE, bool STREAM>
__global__ void __launch_bounds__(WIDTH < 256 ? 256 : WIDTH)
choice_row_kernel(const E* __restrict__ times, E* __restrict__ dtimes, RowArgs a) {
    constexpr int kRows = WIDTH < 256 ? 256 / WIDTH : 1, kWaves = WIDTH <= kWave ? 1 : WIDTH / kWave;
    constexpr int kGroup = WIDTH < kWave ? WIDTH : kWave;
    __shared__ Soft part[kWaves];
    using P = Piece<E, VEC>;
    const int k = threadIdx.x % WIDTH;
    // the gradient pass begins with the rows that were read last: they may still be in a cache (16 x 512 rows of 32768 outputs, a part
    // of them of weight 0: 199 -> 176 us; 1 GB of times, or 30 MB: alike)
    const int64_t block = MODE == GRAD ? (int64_t)gridDim.x * gridDim.y - 1 - workgroup() : workgroup();
    const int64_t r = block * kRows + threadIdx.x / WIDTH;
    if (r >= a.rows) return;                                             // (whole rows; no barrier where rows share a workgroup)
    const E* __restrict__ t = times + (size_t)r * a.J;
    E* __restrict__ g = dtimes + (size_t)r * a.J;
    const Cut cut = cut_row<E, VEC>(t, a.J);
    const int odd = odd_element<VEC>(cut, k);
    const float w = MODE == GRAD ? a.coef[r] : MODE == POLICY && !a.weight ? a.policy.mean : row_weight(a.weight, r);
    if (w == 0.0f) {
        if (MODE != GRAD && k == 0) {
            if (a.logp) a.logp[r] = 0.0f;
            if (a.stats) a.stats[r] = float2{0.0f, 0.0f};
            if (MODE == POLICY) a.row_loss[r] = 0.0f;
            if (MODE == POLICY && a.coef) a.coef[r] = 0.0f;
        }
        if (MODE == LOGP || !dtimes) return;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i * WIDTH + k < cut.pieces) store_piece<STREAM>(reinterpret_cast<P*>(g + cut.lead) + i * WIDTH + k, P{});
        if (odd >= 0) g[odd] = (E)0.0f;
        return;
    }
    P held[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (i * WIDTH < cut.pieces) held[i] = reinterpret_cast<const P*>(t + cut.lead)[min(i * WIDTH + k, cut.pieces - 1)];
    const float single = odd >= 0 ? (float)t[odd] : INFINITY;            // (infinity adds nothing)
    const long long token = a.tokens[r];
    const bool known = token >= 0 && token < a.J;
    float2 soft;
    float c = w, share;
    if (MODE == GRAD) {
        soft = a.stats[r];
        if (a.upstream) c *= *a.upstream;
        share = c * exp_close(-soft.y);
    } else {
        const float chosen = known ? (float)t[token] : NAN;
        float m = -single;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i * WIDTH + k < cut.pieces)
#pragma unroll
                for (int v = 0; v < VEC; ++v) m = fmaxf(m, -(float)held[i].v[v]);
        m = group_max<kGroup>(m);
        const float base = m == -INFINITY ? 0.0f : m;
        float sum = odd >= 0 ? exp_fast(-single - base) : 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (R >= 8) forget(held[i]);
            if (i * WIDTH + k < cut.pieces)
#pragma unroll
                for (int v = 0; v < VEC; ++v) sum += exp_fast(-(float)held[i].v[v] - base);
        }
        Soft all{m, group_sum<kGroup>(sum)};
        if (kWaves > 1) {
            if (k % kWave == 0) part[k / kWave] = all;
            __syncthreads();
            all = part[0];
#pragma unroll
            for (int i = 1; i < kWaves; ++i) all = join(all, part[i]);
        }
        soft = float2{all.m, logf(all.s)};
        const float lp = (-chosen - soft.x) - soft.y;
        RowLoss loss{0.0f, 0.0f};
        if (MODE == POLICY) {
            loss = policy_row(a.policy, r, lp);
            c = loss.coef * w;
        }
        if (k == 0) {
            if (a.logp) a.logp[r] = lp;
            if (a.stats) a.stats[r] = soft;
            if (MODE == POLICY) a.row_loss[r] = loss.loss;
            if (MODE == POLICY && a.coef) a.coef[r] = c;
        }
        if (MODE == LOGP || !dtimes) return;
        share = c / all.s;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if (i * WIDTH + k >= cut.pieces) continue;
        if (R >= 8) forget(held[i]);
        const int j0 = cut.lead + (i * WIDTH + k) * VEC;
        float d[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) d[v] = grad_of<E>(held[i].v[v], soft.x, share);
        if (token >= j0 && token < j0 + VEC) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) d[v] -= token == j0 + v ? c : 0.0f;
        }
        P out;
#pragma unroll
        for (int v = 0; v < VEC; ++v) out.v[v] = (E)d[v];
        store_piece<STREAM>(reinterpret_cast<P*>(g + cut.lead) + i * WIDTH + k, out);
    }
    if (odd >= 0) g[odd] = (E)(grad_of<E>((E)single, soft.x, share) - (token == odd ? c : 0.0f));
}

// Rows longer than a workgroup holds: slices of slice_pieces() pieces, a workgroup each.  One pass leaves (maximum, sum) of every slice; what
// follows joins those of a row in order and reads the row again for its gradient.
constexpr int kSliceThreads = 256;
template <int VEC>
constexpr int slice_pieces() { return VEC == 1 ? 4096 : 1024; }          // 16 KiB of float32, 8 or 16 of 16-bit times

template <typename E, int VEC>
__global__ void __launch_bounds__(kSliceThreads)
choice_slice_kernel(const E* __restrict__ times, const float* __restrict__ weight, Soft* __restrict__ partial, int64_t rows, int J, int slices) {
    __shared__ Soft part[kSliceThreads / kWave];
    using P = Piece<E, VEC>;
    constexpr int kPieces = slice_pieces<VEC>(), kEach = kPieces / kSliceThreads, kBatch = 4;
    const int64_t block = workgroup(), r = block / slices;
    const int slice = block % slices, k = threadIdx.x;
    if (r >= rows || row_weight(weight, r) == 0.0f) return;
    const E* __restrict__ t = times + (size_t)r * J;
    const Cut cut = cut_row<E, VEC>(t, J);
    const int odd = slice == 0 ? odd_element<VEC>(cut, k) : -1;
    const P* __restrict__ pieces = reinterpret_cast<const P*>(t + cut.lead);
    Soft all{-INFINITY, 0.0f};
    if (odd >= 0) all = Soft{-(float)t[odd], 1.0f};
    if (odd >= 0 && !(fabsf(all.m) < INFINITY)) all.s = all.m == -INFINITY ? 0.0f : NAN;
#pragma unroll
    for (int i0 = 0; i0 < kEach; i0 += kBatch) {
        const int first = slice * kPieces + i0 * kSliceThreads;
        if (first >= cut.pieces) break;                                  // (uniform)
        P held[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) held[i] = pieces[min(first + i * kSliceThreads + k, cut.pieces - 1)];
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (first + i * kSliceThreads + k < cut.pieces)
#pragma unroll
                for (int v = 0; v < VEC; ++v) m = fmaxf(m, -(float)held[i].v[v]);
        const float base = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (first + i * kSliceThreads + k < cut.pieces)
#pragma unroll
                for (int v = 0; v < VEC; ++v) sum += exp_fast(-(float)held[i].v[v] - base);
        all = join(all, Soft{m, sum});
    }
    const float m = group_max<kWave>(all.m);
    all = Soft{m, group_sum<kWave>(m == -INFINITY ? all.s : all.s * exp_close(all.m - m))};
    if (k % kWave == 0) part[k / kWave] = all;
    __syncthreads();
    if (k != 0) return;
#pragma unroll
    for (int i = 1; i < kSliceThreads / kWave; ++i) all = join(all, part[i]);
    partial[r * slices + slice] = all;
}

// A wavefront joins the slices of row r: its statistics, log-probability, loss and derivative (0 for a row of weight 0).
struct Joined { float2 soft; float lp, loss, coef, sum; };
template <typename E, Mode MODE>
__device__ __forceinline__ Joined join_slices(const E* times, const Soft* partial, const RowArgs& a, int64_t r, int slices, int lane) {
    Joined out{float2{0.0f, 0.0f}, 0.0f, 0.0f, 0.0f, 1.0f};
    const float w = MODE == POLICY && !a.weight ? a.policy.mean : row_weight(a.weight, r);
    if (w == 0.0f) return out;
    const long long token = a.tokens[r];
    const float chosen = token >= 0 && token < a.J ? (float)times[(size_t)r * a.J + token] : NAN;
    Soft all{-INFINITY, 0.0f};
    for (int i = lane; i < slices; i += kWave) all = join(all, partial[r * slices + i]);
    const float m = group_max<kWave>(all.m);
    all = Soft{m, group_sum<kWave>(m == -INFINITY ? all.s : all.s * exp_close(all.m - m))};
    out.soft = float2{all.m, logf(all.s)};
    out.sum = all.s;
    out.lp = (-chosen - out.soft.x) - out.soft.y;
    if (MODE == POLICY) {
        const RowLoss loss = policy_row(a.policy, r, out.lp);
        out.loss = loss.loss;
        out.coef = loss.coef * w;
    }
    return out;
}
template <Mode MODE>
__device__ __forceinline__ void store_joined(const RowArgs& a, int64_t r, const Joined& j) {
    if (a.logp) a.logp[r] = j.lp;
    if (a.stats) a.stats[r] = j.soft;
    if (MODE == POLICY) a.row_loss[r] = j.loss;
    if (MODE == POLICY && a.coef) a.coef[r] = j.coef;
}

template <typename E, Mode MODE>
__global__ void __launch_bounds__(kWave)
choice_join_kernel(const E* __restrict__ times, const Soft* __restrict__ partial, RowArgs a, int slices) {
    const Joined j = join_slices<E, MODE>(times, partial, a, blockIdx.x, slices, threadIdx.x);
    if (threadIdx.x == 0) store_joined<MODE>(a, blockIdx.x, j);
}

// POLICY: every workgroup of a row joins its slices by itself, which is a load per lane, instead of waiting for a kernel that does.
template <typename E, int VEC, Mode MODE, bool STREAM>
__global__ void __launch_bounds__(kSliceThreads)
choice_slice_grad_kernel(const E* __restrict__ times, E* __restrict__ dtimes, const Soft* __restrict__ partial, RowArgs a, int slices) {
    using P = Piece<E, VEC>;
    constexpr int kPieces = slice_pieces<VEC>(), kEach = kPieces / kSliceThreads, kBatch = 4;
    const int64_t block = (int64_t)gridDim.x * gridDim.y - 1 - workgroup();            // (what was read last comes first)
    const int64_t r = block / slices;
    if (r >= a.rows) return;
    const int slice = block % slices, k = threadIdx.x;
    const E* __restrict__ t = times + (size_t)r * a.J;
    E* __restrict__ g = dtimes + (size_t)r * a.J;
    const Cut cut = cut_row<E, VEC>(t, a.J);
    const int odd = slice == 0 ? odd_element<VEC>(cut, k) : -1;
    float c, top, share;
    if (MODE == POLICY) {
        __shared__ float shared[3];
        if (k < kWave) {
            const Joined j = join_slices<E, MODE>(times, partial, a, r, slices, k);
            if (k == 0) {
                shared[0] = j.coef; shared[1] = j.soft.x; shared[2] = j.coef / j.sum;
                if (slice == 0) store_joined<MODE>(a, r, j);
            }
        }
        __syncthreads();
        c = shared[0]; top = shared[1]; share = shared[2];
    } else {
        c = a.coef[r];
    }
    const bool off = c == 0.0f;
    if (MODE == GRAD) {
        const float2 soft = a.stats[r];
        if (a.upstream) c *= *a.upstream;
        top = soft.x;
        share = c * exp_close(-soft.y);
    }
    const long long token = off ? -1 : a.tokens[r];
#pragma unroll
    for (int i0 = 0; i0 < kEach; i0 += kBatch) {
        const int first = slice * kPieces + i0 * kSliceThreads;
        if (first >= cut.pieces) break;                                  // (uniform)
        P held[kBatch];
        if (!off) {
#pragma unroll
            for (int i = 0; i < kBatch; ++i) held[i] = reinterpret_cast<const P*>(t + cut.lead)[min(first + i * kSliceThreads + k, cut.pieces - 1)];
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int piece = first + i * kSliceThreads + k, j0 = cut.lead + piece * VEC;
            if (piece >= cut.pieces) continue;
            P out{};
            if (!off) {
                float d[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) d[v] = grad_of<E>(held[i].v[v], top, share);
                if (token >= j0 && token < j0 + VEC) {
#pragma unroll
                    for (int v = 0; v < VEC; ++v) d[v] -= token == j0 + v ? c : 0.0f;
                }
#pragma unroll
                for (int v = 0; v < VEC; ++v) out.v[v] = (E)d[v];
            }
            store_piece<STREAM>(reinterpret_cast<P*>(g + cut.lead) + piece, out);
        }
    }
    if (odd >= 0) g[odd] = off ? (E)0.0f : (E)(grad_of<E>(t[odd], top, share) - (token == odd ? c : 0.0f));
}

__device__ __forceinline__ float wave_sum(float v) { return group_sum<kWave>(v); }
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
}

// log(1 + exp(v))
__device__ __forceinline__ double softplus(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }

// One workgroup per pair.  A sequence's log-probability is a sum of hundreds of terms, of which the reference's takes almost all away
// again: both are held in 64 bits (in 32 the margin of sequences of 512 rows was off by 1e-4 of itself).
constexpr int kPairThreads = 256;
__global__ void __launch_bounds__(kPairThreads)
preference_pairs_kernel(const float* __restrict__ logp, PreferenceArgs a, float* __restrict__ pair_loss, float* __restrict__ seq_logp,
                        float* __restrict__ coef, int64_t P, int T) {
    __shared__ double part[2][kPairThreads / kWave];
    __shared__ float shared_slope;
    const int64_t p = blockIdx.x;
    // (logp is 0 where the weight is, so both are requested together)
    double sum[2] = {0.0, 0.0};
    for (int t = threadIdx.x; t < T; t += kPairThreads)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t e = (p + half * P) * T + t;
            sum[half] = fma((double)row_weight(a.weight, e), (double)logp[e], sum[half]);
        }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const double s = wave_sum(sum[half]);
        if (threadIdx.x % kWave == 0) part[half][threadIdx.x / kWave] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        double seq[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            seq[half] = part[half][0];
#pragma unroll
            for (int i = 1; i < kPairThreads / kWave; ++i) seq[half] += part[half][i];
            seq_logp[p + half * P] = (float)seq[half];
        }
        const double e = a.smoothing, m = a.beta * ((seq[0] - a.ref_logp[p]) - (seq[1] - a.ref_logp[p + P]));
        // (a term of factor 0 is none: at an infinite margin, from a sequence that cannot occur, it would be 0 times infinity)
        const double towards = e < 1.0 ? (1.0 - e) * softplus(-m) : 0.0, against = e > 0.0 ? e * softplus(m) : 0.0;
        pair_loss[p] = isnan(m) ? NAN : (float)(towards + against);
        shared_slope = (float)(a.beta / (double)P * (e / (1.0 + exp(-m)) - (1.0 - e) / (1.0 + exp(m))));
    }
    __syncthreads();
    const float slope = shared_slope;
    for (int t = threadIdx.x; t < T; t += kPairThreads)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t e = (p + half * P) * T + t;
            const float w = row_weight(a.weight, e);
            coef[e] = w == 0.0f ? 0.0f : w * (half ? -slope : slope);    // (a slope may be NaN: a row of weight 0 has none)
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

namespace {

// Whether a workgroup holds a row of so many pieces, or it is sliced.  Held with its gradient / sliced, us, 16-bit times: 48000 outputs (6000
// pieces) 16 rows 11.0 / 12.6, 1024 rows 42 / 51; 96000 outputs (12000 pieces, a CU to a workgroup) 16 rows 16 / 9.5, 128 rows 19.4 / 16.8,
// 192 rows 21.1 / 21.4, 256 rows 22.6 / 25.8; float32 times, 48000 outputs (12000 pieces) 16 rows 12.3 / 10.4, 64 rows 13.7 / 11.0, 128 rows
// 15.4 / 15.1, 192 rows 17.9 / 20.0, 256 rows 19.9 / 24.0; 65536 outputs 128 rows 20.3 / 18.1, 192 rows 23.3 / 24.5; without the gradient 48000 outputs,
// 1024 rows 45 / 37.  Nothing has to be held for a gradient from statistics: there the slices' smaller workgroups serve from 1024 pieces on.
constexpr int kMostPieces = 16 * 1024;
template <int VEC, Mode MODE>
bool held(int pieces, int64_t rows, bool gradient) {
    if (MODE == GRAD) return pieces <= 1024;
    if (VEC == 1) return pieces <= kMostPieces;
    return pieces <= 8192 || (MODE == POLICY && gradient && rows >= 192 && pieces <= kMostPieces);
}

template <typename E, int VEC, Mode MODE, bool STREAM>
int launch_rows(const E* times, E* dtimes, const RowArgs& a, hipStream_t stream) {
    const int pieces = VEC == 1 ? a.J : a.J / VEC;
    auto launch = [&](auto kern, int width) -> int {
        const int64_t per = width < 256 ? 256 / width : 1, blocks = (a.rows + per - 1) / per;
        const int threads = width < 256 ? 256 : width;
        {
            KernelTimerScope timer_(MODE == LOGP ? "time_logp" : MODE == POLICY ? "policy_loss" : "time_logp_backward", stream);
            hipLaunchKernelGGL(kern, wide_grid(blocks, threads), dim3((unsigned)threads), 0, stream, times, dtimes, a);
        }
        SNNTC_HIP_CHECK(hipGetLastError());
        return SNNTC_OK;
    };
    if (pieces <= 16) return launch(choice_row_kernel<E, VEC, 16, 1, MODE, STREAM>, 16);
    if (pieces <= 64) return launch(choice_row_kernel<E, VEC, 64, 1, MODE, STREAM>, 64);
    if constexpr (VEC == 1) {
        if (pieces <= 1024) return launch(choice_row_kernel<E, 1, 64, 16, MODE, STREAM>, 64);
        if constexpr (MODE != GRAD) return launch(choice_row_kernel<E, 1, 1024, 16, MODE, STREAM>, 1024);
    } else {
        if (pieces <= 256) return launch(choice_row_kernel<E, VEC, 64, 4, MODE, STREAM>, 64);
        if (pieces <= 1024) return launch(choice_row_kernel<E, VEC, 256, 4, MODE, STREAM>, 256);
        if constexpr (MODE != GRAD) {
            if (pieces <= 2048) return launch(choice_row_kernel<E, VEC, 256, 8, MODE, STREAM>, 256);
            if (pieces <= 4096) return launch(choice_row_kernel<E, VEC, 512, 8, MODE, STREAM>, 512);
            if (pieces <= 8192) return launch(choice_row_kernel<E, VEC, 1024, 8, MODE, STREAM>, 1024);
            if constexpr (MODE == POLICY) return launch(choice_row_kernel<E, VEC, 1024, 16, MODE, STREAM>, 1024);
        }
    }
    return fail(SNNTC_ERR_UNSUPPORTED, "loss: a row of %d pieces", pieces);
}

template <typename E, int VEC, Mode MODE, bool STREAM>
int launch_slices(const E* times, E* dtimes, const RowArgs& a, Soft* partial, hipStream_t stream) {
    const int per = slice_pieces<VEC>(), pieces = a.J / VEC, slices = (pieces + per - 1) / per;
    const int64_t blocks = a.rows * slices;
    if constexpr (MODE != GRAD) {
        {
            KernelTimerScope timer_("choice_slice", stream);
            hipLaunchKernelGGL((choice_slice_kernel<E, VEC>), wide_grid(blocks, kSliceThreads), dim3(kSliceThreads), 0, stream, times, a.weight,
                               partial, a.rows, a.J, slices);
        }
        if (MODE == LOGP || !dtimes) {
            KernelTimerScope timer_("choice_join", stream);
            hipLaunchKernelGGL((choice_join_kernel<E, MODE>), dim3((unsigned)a.rows), dim3(kWave), 0, stream, times, partial, a, slices);
        }
    }
    if constexpr (MODE != LOGP) {
        if (dtimes) {
            KernelTimerScope timer_("choice_slice_grad", stream);
            hipLaunchKernelGGL((choice_slice_grad_kernel<E, VEC, MODE, STREAM>), wide_grid(blocks, kSliceThreads), dim3(kSliceThreads), 0, stream, times,
                               dtimes, partial, a, slices);
        }
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

// Everything a mode does with the rows.
template <Mode MODE>
int launch_choice(const void* times, int type, void* dtimes, const RowArgs& a, Soft* partial, hipStream_t stream) {
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        constexpr int VEC = 16 / sizeof(E);
        const E* t = static_cast<const E*>(times);
        E* g = static_cast<E*>(dtimes);
        // pieces of 16 bytes where times and dtimes lie alike to 16-byte boundaries (and to their own type's)
        const bool vec = ((uintptr_t)t % sizeof(E)) == 0 && (!g || (((uintptr_t)t ^ (uintptr_t)g) & 15) == 0);
        auto go = [&](auto width, auto past) -> int {
            constexpr int W = decltype(width)::value;
            constexpr bool STREAM = decltype(past)::value;
            return held<W, MODE>(a.J / W, a.rows, g) ? launch_rows<E, W, MODE, STREAM>(t, g, a, stream)
                                                     : launch_slices<E, W, MODE, STREAM>(t, g, a, partial, stream);
        };
        if (!vec) return go(std::integral_constant<int, 1>{}, std::false_type{});
        if constexpr (MODE != LOGP)
            // rows of 32000 outputs in 16 bits, times and gradient 300 MB 66 -> 52 us, 500 MB 105 -> 78, 1 GB 199 -> 189; up to 200 MB alike
            if (g && 2 * a.rows * a.J * (int64_t)sizeof(E) > kStreamBytes)
                return go(std::integral_constant<int, VEC>{}, std::true_type{});
        return go(std::integral_constant<int, VEC>{}, std::false_type{});
    });
}

// What the rows of a pair's sequences need between the kernels, where the caller does not want it: in the workspace, before the slices' sums.
struct RowArrays {
    float *logp, *stats, *coef;
    size_t bytes;
    RowArrays(float* stats_, float* coef_, int64_t rows, void* ws) : stats(stats_), coef(coef_) {
        char* scratch = static_cast<char*>(ws);
        const size_t piece = align_up((size_t)rows * sizeof(float));
        logp = reinterpret_cast<float*>(scratch);
        if (!coef) coef = reinterpret_cast<float*>(scratch + piece);
        if (!stats) stats = reinterpret_cast<float*>(scratch + 2 * piece);
        bytes = 4 * piece;
    }
};

RowArgs row_args(const int64_t* tokens, const float* weight, float* logp, float* stats, float* coef, int64_t rows, int64_t J) {
    RowArgs a{};
    a.tokens = reinterpret_cast<const long long*>(tokens);
    a.weight = weight;
    a.logp = logp; a.stats = reinterpret_cast<float2*>(stats); a.coef = coef;
    a.rows = rows; a.J = (int)J;
    return a;
}

}  // namespace

// The slices' sums; rows of at most kMostPieces outputs are held whatever their type and alignment.
size_t choice_workspace(int64_t rows, int64_t J) { return J > kMostPieces ? align_up((size_t)rows * (J / 4096 + 1) * sizeof(Soft)) : 0; }
size_t preference_workspace(int64_t rows, int64_t J) { return RowArrays(nullptr, nullptr, rows, nullptr).bytes + choice_workspace(rows, J); }

int launch_time_logp(const void* times, int type, const int64_t* tokens, const float* weight, float* logp, float* stats, int64_t rows,
                     int64_t J, void* ws, hipStream_t stream) {
    return launch_choice<LOGP>(times, type, nullptr, row_args(tokens, weight, logp, stats, nullptr, rows, J), static_cast<Soft*>(ws), stream);
}

int launch_time_logp_backward(const void* times, int type, const int64_t* tokens, const float* stats, const float* coef,
                              const float* upstream, void* dtimes, int64_t rows, int64_t J, hipStream_t stream) {
    RowArgs a = row_args(tokens, nullptr, nullptr, const_cast<float*>(stats), const_cast<float*>(coef), rows, J);
    a.upstream = upstream;
    return launch_choice<GRAD>(times, type, dtimes, a, nullptr, stream);
}

int launch_policy_loss(const void* times, int type, const int64_t* actions, const PolicyArgs& p, float* row_loss, float* logp, float* stats,
                       float* coef, void* dtimes, int64_t rows, int64_t J, void* ws, hipStream_t stream) {
    RowArgs a = row_args(actions, p.weight, logp, stats, coef, rows, J);
    a.row_loss = row_loss;
    a.policy = p;
    return launch_choice<POLICY>(times, type, dtimes, a, static_cast<Soft*>(ws), stream);
}

int launch_preference_loss(const void* times, int type, const int64_t* tokens, const PreferenceArgs& a, float* pair_loss,
                           float* seq_logp, float* stats, float* coef, void* dtimes, int64_t P, int64_t T, int64_t J, void* ws,
                           hipStream_t stream) {
    const int64_t rows = 2 * P * T;
    const RowArrays ra(stats, coef, rows, ws);
    int rc = SNNTC_OK;
    if (rows > 0)
        rc = launch_time_logp(times, type, tokens, a.weight, ra.logp, ra.stats, rows, J, static_cast<char*>(ws) + ra.bytes, stream);
    if (rc) return rc;
    {
        KernelTimerScope timer_("preference_pairs", stream);
        hipLaunchKernelGGL(preference_pairs_kernel, dim3((unsigned)P), dim3(kPairThreads), 0, stream, ra.logp, a, pair_loss, seq_logp, ra.coef,
                           P, (int)T);
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
