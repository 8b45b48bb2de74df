// One AdamW step over many tensors at once.  With g = share dw, share = min(1, max_norm / norm) where the gradients are clipped (else 1),
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,
//     w = w - lr decay w - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
// (the reference hands the update to the framework's optimizer, snntc/snntc-mnist.py:70).  One pass: every element is read once and
// written once, whatever its state is held in.
//
// States in 8 bits.  A block of 256 elements of a tensor has one float32 scale, its largest magnitude, which the largest code stands for;
// code 8 (E - 1) + k, k = 8 .. 15, is k 2^(E - 1) in units of that, codes below 8 are themselves (m: a sign and 7 bits, E to 15; v: 8 bits, E
// to 31, since v spans the square of m's range).  Two neighbours lie a 15th to an 8th apart, and a step
// changes v by 1 - b2 of itself: rounded to the nearest, an element whose gradients shrink while its block's do not would stand still for
// good.  So a value is rounded to either neighbour with the chance of its place between them, and on average a state moves as it should
// (4000 steps of gradients of constant variance: sqrt v off by 12 % of itself, by 1 on average).  The random bits are a function of seed, step, tensor
// and element.
// The two moments of an element are rounded apart.  One far below its block's largest can so keep a first moment (down to 2^-18 of the largest)
// and lose its second (below 2^-34): its next step without a gradient is then lr m / eps.  `paired` drops the first moment
// with the second.  Largest step in 200, gradients 1e-1 .. 1e-6 of their block's largest and half of them or 97 % 0: 320 .. 1830 lr without, 1.3 .. 2.0 lr
// with, 1.3 .. 1.8 lr of states in 32 bits.  It takes 2 % (68 M bf16 weights 155 -> 159 us).
// A double's upper word with 16 random bits and a half added below its third binary digit is that rounding.  Moments are therefore 64
// bits wide between the codes: next to a border a sum in 32 bits would leave another code than the definition.
// 16-bit weights are rounded in the same way and for the same reason: a step of a thousandth of a weight is less than half of what
// they can tell apart.
#include "../sequences.h"
#include "wave.h"

namespace snntc {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = SNNTC_STATE_BLOCK;                     // elements that share a scale: four to a lane
static_assert(kBlock == 4 * kWave, "a wavefront owns a block");
constexpr double kTopFirst = 15 << 14, kTopSecond = 15.0 * (1 << 30);

// A table of tensors travels in the kernel arguments, which hold 4 KiB.
constexpr int kMostTensors = 48;
struct AdamTable {
    void* w[kMostTensors];
    const void* g[kMostTensors];
    void* m[kMostTensors];
    void* v[kMostTensors];
    float* m_scale[kMostTensors];
    float* v_scale[kMostTensors];
    long long n[kMostTensors];
    unsigned first_block[kMostTensors + 1];
    int tensor[kMostTensors];                                 // its place in the caller's list, for the random bits
    int count;
};

// What depends on the step's number, from the host or (graphs) from the device.
struct AdamStep { double rate, second; unsigned step; };     // lr / (1 - b1^t), 1 / (1 - b2^t)
struct AdamScalars {
    double b1, b2, keep, eps, max_norm;                      // keep: 1 - lr decay
    const float* norm;                                        // NULL: not clipped
    const AdamStep* at;                                       // NULL: `step`
    AdamStep step;
    unsigned seed_low, seed_high;
    int paired;                                               // states in 8 bits: no first moment beside a second of 0
};

__device__ __forceinline__ unsigned mix(unsigned x) {
    x = (x ^ (x >> 16)) * 0x6A09E667u;
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}
__device__ __forceinline__ unsigned key_of(const AdamScalars& s, unsigned step, unsigned tensor) {
    return mix(s.seed_low + mix(s.seed_high + mix(step + mix(tensor))));
}
constexpr unsigned kElement = 0x9E3779B9u;
// place: the element's number times kElement.
__device__ __forceinline__ unsigned noise(unsigned key, unsigned place) { return mix(place ^ key); }
__device__ __forceinline__ unsigned third_noise(unsigned bits) { return bits * kElement >> 16; }

// Codes are the upper bits of numbers that begin to lose digits at 8: a code's bits below the sign of a float32 are value(code) 2^-129, codes
// below 8 being such that have fewer digits; and the upper word of y 2^-1025 as a double holds, from its 17th bit on, the code
// at or below y.
__device__ __forceinline__ double first_value(unsigned code) { return (double)__uint_as_float((code & 127u) << 20 | (code & 128u) << 24); }
__device__ __forceinline__ double second_value(unsigned code) { return (double)__uint_as_float(code << 20); }
constexpr double kFirstUnit = 0x1p129 / kTopFirst, kSecondUnit = 0x1p129 / kTopSecond;        // of a scale
// The code of y >= 0 (value(largest) for the largest magnitude), raised by (bits + 1/2) / 65536 of a step and cut off.
__device__ __forceinline__ unsigned code_of(double y, unsigned bits, unsigned most) {
    const unsigned c = ((unsigned)__double2hiint(ldexp(y, -1025)) + (bits << 1 | 1u)) >> 17;
    return c < most ? c : most;
}
// top / s for a scale s, 0 for a scale that is none: the hardware's reciprocal of 64 bits made exact by two steps (no such number is near
// the ends of the doubles).
__device__ __forceinline__ double per_scale(double top, float s) {
    const double d = (double)s;
    double r = __builtin_amdgcn_rcp(d);
    r = fma(fma(-d, r, 1.0), r, r);
    r = fma(fma(-d, r, 1.0), r, r);
    return s > 0.0f && s < INFINITY ? top * r : 0.0;
}

// float32 to a weight's type; 16-bit types to one of the two neighbours, the upper one if the place between them in 65536ths exceeds `bits`.
__device__ __forceinline__ void round_weight(float x, unsigned, float* to) { *to = x; }
__device__ __forceinline__ void round_weight(float x, unsigned bits, __bf16* to) {
    unsigned w = __float_as_uint(x);
    if (fabsf(x) < INFINITY) w += 0xFFFFu - bits;
    else if (w & 0xFFFFu) w |= 0x10000u;                      // (a NaN stays one)
    *to = __builtin_bit_cast(__bf16, (unsigned short)(w >> 16));
}
__device__ __forceinline__ void round_weight(float x, unsigned bits, _Float16* to) {
    if (!(fabsf(x) < 65504.0f)) { *to = (_Float16)x; return; }
    const int e = max((int)(__float_as_uint(x) >> 23 & 255) - 127, -14);
    const float y = ldexpf(fabsf(x), 10 - e), low = floorf(y);
    const float q = low + ((y - low) * 65536.0f > (float)bits ? 1.0f : 0.0f);
    *to = (_Float16)copysignf(ldexpf(q, e - 10), x);
}

// Four elements at any place of their type.
template <typename E> struct Four { E v[4]; };
typedef unsigned FourFloats __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned FourHalves __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned FourBytes __attribute__((aligned(1)));
template <typename E>
using Place = typename std::conditional<sizeof(E) == 4, FourFloats, typename std::conditional<sizeof(E) == 2, FourHalves, FourBytes>::type>::type;

// PAST: past the caches.  A call that touches more than they hold reads and writes weights and states so: what the norm has left of
// the gradients stays there, and the next call's gradients do not wait for this one's results (68 M float32 weights, 410 -> 333 us with
// the norm, which takes 85 and 47 of it; with states in 8 bits and their moments read back 385 -> 326).
// WHOLE: there are four elements from e on; else those at or behind n are the last one once more.  Not one load stands in a branch: the
// compiler waits for all that are under way where branches meet.
template <bool PAST, bool WHOLE, typename E>
__device__ __forceinline__ Four<E> load4(const E* from, long long e, long long n) {
    if constexpr (WHOLE) {
        const Place<E>* p = reinterpret_cast<const Place<E>*>(from + e);
        if constexpr (PAST) return __builtin_bit_cast(Four<E>, __builtin_nontemporal_load(p));
        return __builtin_bit_cast(Four<E>, *p);
    }
    Four<E> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.v[i] = from[min(e + i, n - 1)];
    return r;
}
template <bool PAST, bool WHOLE, typename E>
__device__ __forceinline__ void store4(E* to, long long e, long long n, const Four<E>& r) {
    if constexpr (WHOLE) {
        Place<E>* p = reinterpret_cast<Place<E>*>(to + e);
        if constexpr (PAST) __builtin_nontemporal_store(__builtin_bit_cast(Place<E>, r), p);
        else *p = __builtin_bit_cast(Place<E>, r);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (e + i < n) to[e + i] = r.v[i];
    }
}

// The tensor that a workgroup belongs to: all of the table's first workgroups are compared at once.
template <typename T>
__device__ __forceinline__ int tensor_of(const T& tab, unsigned block) {
    constexpr int kEntries = sizeof(tab.first_block) / sizeof(unsigned);
    const int lane = threadIdx.x % kWave;
    int t = -1;
#pragma unroll
    for (int i = 0; i < (kEntries + kWave - 1) / kWave; ++i) {
        const int at = i * kWave + lane;
        const unsigned first = tab.first_block[min(at, kEntries - 1)];
        t += __popcll(__ballot(at < tab.count && first <= block));
    }
    return t;
}

// What the gradients are scaled by; a norm that is no finite number: the step is left out.
__device__ __forceinline__ double share_of(const AdamScalars& s, bool* skip) {
    *skip = false;
    if (!s.norm) return 1.0;
    const float norm = *s.norm;
    *skip = !(norm < INFINITY);
    return (double)norm > s.max_norm ? s.max_norm / (double)norm : 1.0;
}

constexpr int kTimes = 2;                                      // blocks of 256 elements that a wavefront holds
constexpr int kChunk = kThreads * 4 * kTimes;
// A wavefront's first element in a tensor, of workgroup `block` of the tensor's.
__device__ __forceinline__ long long wave_begin(unsigned block) {
    return ((long long)block * (kThreads / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave)) *
           (kBlock * kTimes);
}

// First moments without those whose second moment's code is 0, four of each.
__device__ __forceinline__ Four<unsigned char> with_second(const Four<unsigned char>& m, const Four<unsigned char>& v) {
    const unsigned w = __builtin_bit_cast(unsigned, v), some = (((w & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | w) & 0x80808080u;      // 128 in a byte that is not 0
    return __builtin_bit_cast(Four<unsigned char>, __builtin_bit_cast(unsigned, m) & (some | (some - (some >> 7))));
}

// The hardware's root, off by a step; it takes no number below 2^-126, which a power of four brings up.
__device__ __forceinline__ float root(float x) {
    const bool small = x < 0x1p-96f;
    const float r = __builtin_amdgcn_sqrtf(small ? x * 0x1p96f : x);
    return small ? r * 0x1p-48f : r;
}
// A weight after the step.  Root and reciprocal are the hardware's, two steps of a change that is a small part of the weight.
__device__ __forceinline__ float stepped(float w, float m, float v, float keep, float rate, float second, float eps) {
    return fmaf(-rate * m, __builtin_amdgcn_rcpf(root(v * second) + eps), w * keep);
}

// States in float32.  Bound by memory: 281 us for 68 M float32 weights, 1909 MB at 6.8 TB/s; 231 for bf16 or f16 weights, 1500 MB at 6.5 TB/s.
template <bool WHOLE, typename E, bool PAST>
__device__ __forceinline__ void adamw_run(const AdamTable& tab, const AdamScalars& s, int t, long long begin) {
    const long long n = tab.n[t], e0 = begin + threadIdx.x % kWave * 4;
    E* __restrict__ w = static_cast<E*>(tab.w[t]);
    const E* __restrict__ g = static_cast<const E*>(tab.g[t]);
    float* __restrict__ m = static_cast<float*>(tab.m[t]);
    float* __restrict__ v = static_cast<float*>(tab.v[t]);
    Four<E> W[kTimes], G[kTimes];
    Four<float> M[kTimes], V[kTimes];
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const long long e = e0 + i * kBlock;
        W[i] = load4<PAST, WHOLE>(w, e, n); G[i] = load4<false, WHOLE>(g, e, n); M[i] = load4<PAST, WHOLE>(m, e, n); V[i] = load4<PAST, WHOLE>(v, e, n);
    }
    bool skip;
    const float share = (float)share_of(s, &skip);
    if (skip) return;
    const AdamStep at = s.at ? *s.at : s.step;
    const float b1 = (float)s.b1, b2 = (float)s.b2, new1 = (float)(1.0 - s.b1), new2 = (float)(1.0 - s.b2), keep = (float)s.keep,
                rate = (float)at.rate, second = (float)at.second, eps = (float)s.eps;
    const unsigned key = sizeof(E) == 2 ? key_of(s, at.step, tab.tensor[t]) : 0;
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const long long e = e0 + i * kBlock;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float d = (float)G[i].v[k] * share;
            M[i].v[k] = fmaf(b1, M[i].v[k], new1 * d);
            V[i].v[k] = fmaf(b2, V[i].v[k], new2 * d * d);
            const unsigned bits = sizeof(E) == 2 ? third_noise(noise(key, (unsigned)e * kElement + k * kElement)) : 0;
            round_weight(stepped((float)W[i].v[k], M[i].v[k], V[i].v[k], keep, rate, second, eps), bits, &W[i].v[k]);
        }
        store4<PAST, WHOLE>(w, e, n, W[i]); store4<PAST, WHOLE>(m, e, n, M[i]); store4<PAST, WHOLE>(v, e, n, V[i]);
    }
}
template <typename E, bool PAST>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(AdamTable tab, AdamScalars s) {
    const unsigned block = gridDim.x - 1 - blockIdx.x;                      // (the gradients that the norm has read last come first)
    const int t = tensor_of(tab, block);
    const long long begin = wave_begin(block - tab.first_block[t]), n = tab.n[t];
    if (begin + kBlock * kTimes <= n) adamw_run<true, E, PAST>(tab, s, t, begin);
    else if (begin < n) adamw_run<false, E, PAST>(tab, s, t, begin);
}

__device__ __forceinline__ unsigned wave_max(unsigned v) { return wave_join(v, 0u, [](unsigned a, unsigned b) { return max(a, b); }); }
// A magnitude's bits: ordered as magnitudes are, NaN above all.
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// States in 8 bits: a wavefront owns kTimes blocks of 256 elements.  Memory and vector instructions bind alike: 159 us for 68 M float32 weights, 1102 MB at
// 6.9 TB/s, with instructions in 84 % of the issue slots (75 for an element of each lane); instructions alone where weights are of 16 bits, 155 us (bf16) and 166
// (f16) for 682 MB.  Both blocks' maxima in one tree save a tenth of these, but
// hold 134 registers instead of 84, and the call is slower (322 -> 330 us with norm and moments).
// Copies of a tensor's last element leave a block's maxima as they are.
template <bool WHOLE, typename E, bool PAST>
__device__ __forceinline__ void adamw8_run(const AdamTable& tab, const AdamScalars& s, int t, long long begin) {
    const long long n = tab.n[t], e0 = begin + threadIdx.x % kWave * 4, b0 = begin / kBlock, last = (n - 1) / kBlock;
    E* __restrict__ w = static_cast<E*>(tab.w[t]);
    const E* __restrict__ g = static_cast<const E*>(tab.g[t]);
    unsigned char* __restrict__ m = static_cast<unsigned char*>(tab.m[t]);
    unsigned char* __restrict__ v = static_cast<unsigned char*>(tab.v[t]);
    float *__restrict__ ms = tab.m_scale[t], *__restrict__ vs = tab.v_scale[t];
    Four<E> W[kTimes], G[kTimes];
    Four<unsigned char> M[kTimes], V[kTimes];
    float m_scale[kTimes], v_scale[kTimes];
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const long long e = e0 + i * kBlock, b = WHOLE ? b0 + i : min(b0 + i, last);
        W[i] = load4<PAST, WHOLE>(w, e, n); G[i] = load4<false, WHOLE>(g, e, n); M[i] = load4<PAST, WHOLE>(m, e, n); V[i] = load4<PAST, WHOLE>(v, e, n);
        m_scale[i] = ms[b]; v_scale[i] = vs[b];
    }
    bool skip;
    const double share = share_of(s, &skip);
    if (skip) return;
    const AdamStep at = s.at ? *s.at : s.step;
    const float keep = (float)s.keep, rate = (float)at.rate, second = (float)at.second, eps = (float)s.eps;
    const double new1 = (1.0 - s.b1) * share, new2 = (1.0 - s.b2) * share * share;
    const unsigned key = key_of(s, at.step, tab.tensor[t]);
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const long long e = e0 + i * kBlock;
        if (!WHOLE && begin + i * kBlock >= n) return;        // (a whole wavefront)
        const double old1 = s.b1 * kFirstUnit * (double)m_scale[i], old2 = s.b2 * kSecondUnit * (double)v_scale[i];
        const unsigned place = (unsigned)e * kElement;
        double a[4], q[4];
        unsigned top1 = 0, top2 = 0, bits[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double d = (double)(float)G[i].v[k];
            a[k] = fma(new1, d, old1 * first_value(M[i].v[k]));
            q[k] = fma(new2 * d, d, old2 * second_value(V[i].v[k]));
            const float fa = (float)a[k], fq = (float)q[k];
            top1 = max(top1, magnitude(fa)); top2 = max(top2, magnitude(fq));
            bits[k] = noise(key, place + k * kElement);
            round_weight(stepped((float)W[i].v[k], fa, fq, keep, rate, second, eps), sizeof(E) == 2 ? third_noise(bits[k]) : 0, &W[i].v[k]);
        }
        store4<PAST, WHOLE>(w, e, n, W[i]);
        const float scale1 = __uint_as_float(wave_max(top1)), scale2 = __uint_as_float(wave_max(top2));
        const double unit1 = per_scale(kTopFirst, scale1), unit2 = per_scale(kTopSecond, scale2);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned c = code_of(fabs(a[k]) * unit1, bits[k] & 0xFFFFu, 127u);
            M[i].v[k] = (unsigned char)(c | ((unsigned)__double2hiint(a[k]) >> 24 & 128u));
            V[i].v[k] = (unsigned char)code_of(q[k] * unit2, bits[k] >> 16, 255u);
        }
        if (s.paired) M[i] = with_second(M[i], V[i]);         // (uniform)
        store4<PAST, WHOLE>(m, e, n, M[i]); store4<PAST, WHOLE>(v, e, n, V[i]);
        if (threadIdx.x % kWave == 0) { ms[b0 + i] = scale1; vs[b0 + i] = scale2; }
    }
}
template <typename E, bool PAST>
__global__ void __launch_bounds__(kThreads)
adamw8_kernel(AdamTable tab, AdamScalars s) {
    const unsigned block = gridDim.x - 1 - blockIdx.x;
    const int t = tensor_of(tab, block);
    const long long begin = wave_begin(block - tab.first_block[t]), n = tab.n[t];
    if (begin + kBlock * kTimes <= n) adamw8_run<true, E, PAST>(tab, s, t, begin);
    else if (begin < n) adamw8_run<false, E, PAST>(tab, s, t, begin);
}

// The number of a step that a graph replays: one more each time, and what follows from it.
__global__ void adamw_advance_kernel(long long* __restrict__ steps, AdamStep* __restrict__ at, double lr, double b1, double b2) {
    const long long t = *steps + 1;
    *steps = t;
    *at = AdamStep{lr / (1.0 - pow(b1, (double)t)), 1.0 / (1.0 - pow(b2, (double)t)), (unsigned)t};
}

// Both moments from their codes, float32.  Bound by memory: 111 us for 68 M, 691 MB at 6.2 TB/s.
struct MomentTable {
    const unsigned char* m[kMostTensors];
    const unsigned char* v[kMostTensors];
    const float* m_scale[kMostTensors];
    const float* v_scale[kMostTensors];
    float* first[kMostTensors];
    float* second[kMostTensors];
    long long n[kMostTensors];
    unsigned first_block[kMostTensors + 1];
    int count;
};
template <bool WHOLE, bool PAST>
__device__ __forceinline__ void moments_run(const MomentTable& tab, int t, long long begin) {
    const long long n = tab.n[t], e0 = begin + threadIdx.x % kWave * 4, b0 = begin / kBlock, last = (n - 1) / kBlock;
    Four<unsigned char> M[kTimes], V[kTimes];
    float m_scale[kTimes], v_scale[kTimes];
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const long long e = e0 + i * kBlock, b = WHOLE ? b0 + i : min(b0 + i, last);
        M[i] = load4<false, WHOLE>(tab.m[t], e, n); V[i] = load4<false, WHOLE>(tab.v[t], e, n);
        m_scale[i] = tab.m_scale[t][b]; v_scale[i] = tab.v_scale[t][b];
    }
#pragma unroll
    for (int i = 0; i < kTimes; ++i) {
        const long long e = e0 + i * kBlock;
        const double u1 = kFirstUnit * (double)m_scale[i], u2 = kSecondUnit * (double)v_scale[i];
        Four<float> a, q;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            a.v[k] = (float)(first_value(M[i].v[k]) * u1);
            q.v[k] = (float)(second_value(V[i].v[k]) * u2);
        }
        store4<PAST, WHOLE>(tab.first[t], e, n, a); store4<PAST, WHOLE>(tab.second[t], e, n, q);
    }
}
template <bool PAST>
__global__ void __launch_bounds__(kThreads)
moments_kernel(MomentTable tab) {
    const int t = tensor_of(tab, blockIdx.x);
    const long long begin = wave_begin(blockIdx.x - tab.first_block[t]), n = tab.n[t];
    if (begin + kBlock * kTimes <= n) moments_run<true, PAST>(tab, t, begin);
    else if (begin < n) moments_run<false, PAST>(tab, t, begin);
}

// ---- the norm over all gradients -------------------------------------------------------------------------------------------------

constexpr int kMostGrads = 96;
struct GradTable {
    const void* g[kMostGrads];
    long long n[kMostGrads];
    unsigned first_block[kMostGrads + 1];
    unsigned char type[kMostGrads];
    int count;
    long long chunk;                                          // elements of a workgroup
};

template <int THREADS>
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[THREADS / kWave];
    v = wave_sum(v);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < THREADS / kWave; ++i) v += part[i];
    return v;
}

// Squares in 64 bits: of 10^8 gradients neither the largest overflow nor the smallest vanish, and the sum's order does not show.
// Eight pieces of four elements are requested together (68 M float32 gradients 48 us, 5.7 TB/s).
constexpr int kPieces = 8;
template <typename E>
__device__ __forceinline__ double squares(const E* __restrict__ g, long long from, long long to) {
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
    const auto add = [&](const Four<E>& x) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const double d = (double)(float)x.v[k];
            sum[k] = fma(d, d, sum[k]);
        }
    };
    const auto pieces = [&](auto many) {
        constexpr int N = decltype(many)::value;
        for (; from + N * kThreads * 4 <= to; from += N * kThreads * 4) {
            Four<E> x[N];
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = load4<false, true>(g, from + (i * kThreads + threadIdx.x) * 4, to);
#pragma unroll
            for (int i = 0; i < N; ++i) add(x[i]);
        }
    };
    pieces(std::integral_constant<int, kPieces>());
    pieces(std::integral_constant<int, 2>());
    for (long long e = from + threadIdx.x * 4; e < to; e += kThreads * 4) {
        Four<E> x = load4<false, false>(g, e, to);
#pragma unroll
        for (int k = 0; k < 4; ++k) x.v[k] = e + k < to ? x.v[k] : (E)0.0f;
        add(x);
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}
__global__ void __launch_bounds__(kThreads)
grad_squares_kernel(GradTable tab, double* __restrict__ partial) {
    const int t = tensor_of(tab, blockIdx.x);
    const long long from = (long long)(blockIdx.x - tab.first_block[t]) * tab.chunk, to = min(from + tab.chunk, tab.n[t]);
    double s;
    if (tab.type[t] == SNNTC_F32) s = squares(static_cast<const float*>(tab.g[t]), from, to);
    else if (tab.type[t] == SNNTC_BF16) s = squares(static_cast<const __bf16*>(tab.g[t]), from, to);
    else s = squares(static_cast<const _Float16*>(tab.g[t]), from, to);
    s = block_sum<kThreads>(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}
__global__ void __launch_bounds__(1024)
grad_norm_kernel(const double* __restrict__ partial, float* __restrict__ norm, int n) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) s += partial[i];
    s = block_sum<1024>(s);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// Workgroups of one launch: 2^32 threads are too many.
constexpr int64_t kMostBlocks = (1 << 24) - 1;

// Elements of a workgroup: small calls spread over all CUs, large ones leave some thousand sums.
int64_t norm_chunk(int64_t total) { return total < (4 << 20) ? 2048 : 8192 * std::max<int64_t>(1, total / (8192ll * 4096)); }

}  // namespace

size_t grad_norm_workspace(const int64_t* n, int64_t count) {
    int64_t total = 0, blocks = 0;
    for (int64_t t = 0; t < count; ++t) total += n[t];
    const int64_t chunk = norm_chunk(total);
    for (int64_t t = 0; t < count; ++t) blocks += (n[t] + chunk - 1) / chunk;
    return align_up((size_t)blocks * sizeof(double));
}

int launch_grad_norm(const void* const* g, const int* types, const int64_t* n, int count, float* norm, void* ws, hipStream_t stream) {
    int64_t total = 0;
    for (int t = 0; t < count; ++t) total += n[t];
    double* partial = static_cast<double*>(ws);
    int64_t done = 0;
    for (int t = 0; t < count;) {
        GradTable tab;
        tab.count = 0;
        tab.chunk = norm_chunk(total);
        int64_t blocks = 0;
        for (; t < count && tab.count < kMostGrads; ++t) {
            if (n[t] == 0) continue;
            tab.g[tab.count] = g[t];
            tab.n[tab.count] = n[t];
            tab.type[tab.count] = (unsigned char)types[t];
            tab.first_block[tab.count] = (unsigned)blocks;
            blocks += (n[t] + tab.chunk - 1) / tab.chunk;
            ++tab.count;
        }
        if (tab.count == 0) continue;
        {
            KernelTimerScope timer_("grad_squares", stream);
            hipLaunchKernelGGL(grad_squares_kernel, dim3((unsigned)blocks), dim3(kThreads), 0, stream, tab, partial + done);
        }
        done += blocks;
    }
    {
        KernelTimerScope timer_("grad_norm", stream);
        hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(1024), 0, stream, partial, norm, (int)done);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

int launch_adamw(const AdamTensors& a, int count, const AdamNumbers& p, void* ws, hipStream_t stream) {
    AdamScalars s{};
    s.b1 = p.b1; s.b2 = p.b2; s.keep = 1.0 - p.lr * p.decay; s.eps = p.eps; s.max_norm = p.max_norm; s.norm = p.norm;
    s.seed_low = (unsigned)p.seed; s.seed_high = (unsigned)(p.seed >> 32);
    s.paired = p.paired;
    if (p.steps) {
        AdamStep* at = static_cast<AdamStep*>(ws);
        KernelTimerScope timer_("adamw_advance", stream);
        hipLaunchKernelGGL(adamw_advance_kernel, dim3(1), dim3(1), 0, stream, reinterpret_cast<long long*>(p.steps), at, p.lr, p.b1, p.b2);
        SNNTC_HIP_CHECK(hipGetLastError());
        s.at = at;
    } else {
        s.step = AdamStep{p.lr / (1.0 - pow(p.b1, (double)p.step)), 1.0 / (1.0 - pow(p.b2, (double)p.step)), (unsigned)p.step};
    }
    int64_t bytes = 0;
    for (int t = 0; t < count; ++t) bytes += a.n[t] * (3 * (int64_t)type_bytes(a.types[t]) + (a.m_scale ? 4 : 16));
    const bool past = bytes > kStreamBytes;
    for (int type = SNNTC_F32; type <= SNNTC_F16; ++type)
        for (int t = 0; t < count;) {
            AdamTable tab;
            tab.count = 0;
            int64_t blocks = 0;
            for (; t < count && tab.count < kMostTensors; ++t) {
                if (a.n[t] == 0 || a.types[t] != type) continue;
                const int64_t more = (a.n[t] + kChunk - 1) / kChunk;
                if (blocks + more > kMostBlocks) break;
                const int c = tab.count++;
                tab.w[c] = a.w[t]; tab.g[c] = a.g[t]; tab.m[c] = a.m[t]; tab.v[c] = a.v[t];
                tab.m_scale[c] = a.m_scale ? a.m_scale[t] : nullptr;
                tab.v_scale[c] = a.v_scale ? a.v_scale[t] : nullptr;
                tab.n[c] = a.n[t];
                tab.tensor[c] = t;
                tab.first_block[c] = (unsigned)blocks;
                blocks += more;
            }
            if (tab.count == 0) continue;
            with_type(type, [&](auto e) -> int {
                using E = decltype(e);
                KernelTimerScope timer_(a.m_scale ? "adamw8" : "adamw", stream);
                const auto kern = a.m_scale ? (past ? adamw8_kernel<E, true> : adamw8_kernel<E, false>) : past ? adamw_kernel<E, true> : adamw_kernel<E, false>;
                hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(kThreads), 0, stream, tab, s);
                return SNNTC_OK;
            });
            SNNTC_HIP_CHECK(hipGetLastError());
        }
    return SNNTC_OK;
}

int launch_adamw_moments(const uint8_t* const* m, const uint8_t* const* v, const float* const* m_scale, const float* const* v_scale,
                         float* const* first, float* const* second, const int64_t* n, int count, hipStream_t stream) {
    int64_t total = 0;
    for (int t = 0; t < count; ++t) total += n[t];
    for (int t = 0; t < count;) {
        MomentTable tab;
        tab.count = 0;
        int64_t blocks = 0;
        for (; t < count && tab.count < kMostTensors; ++t) {
            if (n[t] == 0) continue;
            const int64_t more = (n[t] + kChunk - 1) / kChunk;
            if (blocks + more > kMostBlocks) break;
            const int c = tab.count++;
            tab.m[c] = m[t]; tab.v[c] = v[t]; tab.m_scale[c] = m_scale[t]; tab.v_scale[c] = v_scale[t];
            tab.first[c] = first[t]; tab.second[c] = second[t]; tab.n[c] = n[t];
            tab.first_block[c] = (unsigned)blocks;
            blocks += more;
        }
        if (tab.count == 0) continue;
        KernelTimerScope timer_("adamw_moments", stream);
        hipLaunchKernelGGL(10 * total > kStreamBytes ? moments_kernel<true> : moments_kernel<false>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, tab);
        SNNTC_HIP_CHECK(hipGetLastError());
    }
    return SNNTC_OK;
}

}  // namespace snntc
