// Choices by rules.  A row of spike times t[J] stands for the distribution softmax(-t); rules change the times before a token is drawn
// or a loss is taken.  With c_j the occurrences of j in the row's part of a history of tokens and o_j those behind the prompt,
//     a_j = t_j r  (t_j > 0),  t_j / r  (t_j <= 0)       where c_j > 0,  t_j elsewhere
//     b_j = a_j + (presence + frequency o_j)             where o_j > 0,  a_j elsewhere
//     t'_j = b_j + delay_j  where j is allowed, +infinity elsewhere,         dt_j = dt'_j (1, r or 1 / r; 0 where not allowed)
// and a token is the first j with sum_{i <= j} exp(-(t'_i - min t') / T) > u sum_i exp(-(t'_i - min t') / T).
//
// A workgroup owns a slice of a row.  It marks the history's tokens that lie in the slice in a bitmap in LDS, a bit for each element; where
// occurrences count, the marked elements are numbered by their rank in the bitmap and counted in an array of at most the history's
// length.  So LDS holds a quarter of a byte for each element, whatever the vocabulary, and an element that no token names costs one bit test.
// The arithmetic of a ruled time is float32 without contraction: products and sums round one by one, as written above.  A
// token is drawn from the times as rule_times stores them, rounded to times' type, so that its log-probability is that of the ruled times.
#include "../sequences.h"

namespace snntc {
namespace {

constexpr float kLog2e = 1.44269504f;

// VEC elements, 16 bytes (or, of float32, 32), at any place of their type: the target loads and stores four words at any address.
template <typename E, int VEC>
struct Piece { E v[VEC]; };
typedef unsigned Words __attribute__((ext_vector_type(4)));
template <typename E>
struct __attribute__((packed, aligned(sizeof(E)))) Place { Words w; };
template <typename E, int VEC>
__device__ __forceinline__ Piece<E, VEC> read_piece(const E* at) {
    constexpr int N = VEC * sizeof(E) / sizeof(Words);
    struct All { Words w[N]; } all;
#pragma unroll
    for (int i = 0; i < N; ++i) all.w[i] = reinterpret_cast<const Place<E>*>(at)[i].w;
    return __builtin_bit_cast(Piece<E, VEC>, all);
}

// What is the same for a whole row.
struct RowRules {
    const long long* tokens;
    int seen, prompt;                                // tokens [0, seen) count, those from `prompt` on as occurrences
    float rep, inv, pres, freq;
    const float* delay;
    const unsigned* allowed;
};
__device__ __forceinline__ RowRules row_rules(const RuleArgs& a, int64_t r) {
    RowRules q{};
    q.rep = 1.0f;
    if (a.history) {
        const int64_t h = r / a.rows_per_history;
        q.tokens = reinterpret_cast<const long long*>(a.history) + h * a.L;
        const auto inside = [&](int64_t n) { return (int)(n < 0 ? 0 : n > a.L ? a.L : n); };
        q.seen = a.lengths ? inside(a.lengths[r]) : (int)a.L;
        q.prompt = a.prompts ? inside(a.prompts[h]) : 0;
        q.rep = a.repetition ? a.repetition[h] : a.rep;
        q.pres = a.presence ? a.presence[h] : a.pres;
        q.freq = a.frequency ? a.frequency[h] : a.freq;
        q.inv = 1.0f / q.rep;
    }
    q.delay = a.delay ? a.delay + r * a.delay_stride : nullptr;
    q.allowed = a.allowed ? a.allowed + r * a.allowed_stride : nullptr;
    return q;
}

extern __shared__ unsigned lds_marks[];

// The marks of a slice of WIDTH * PER elements in LDS: a bitmap, the marked elements before each of its words, and their occurrences.
template <int WIDTH, int PER>
struct Marks {
    static constexpr int kSlice = WIDTH * PER, kWords = kSlice / 32, kWaves = WIDTH / kWave;
    static_assert(kWords <= WIDTH, "a word for each thread");
    // (named by their place in LDS: kept as pointers they would be read as generic memory)
    __device__ __forceinline__ static unsigned& bits(int i) { return lds_marks[i]; }
    __device__ __forceinline__ static unsigned& before(int i) { return lds_marks[kWords + i]; }
    __device__ __forceinline__ static unsigned& count(int i) { return lds_marks[2 * kWords + i]; }

    // Returns whether there are any rules from the history; every thread of the workgroup calls it.
    __device__ __forceinline__ bool build(const RowRules& q, int64_t first, int J, int most, bool counts) {
        counts = counts && (q.pres != 0.0f || q.freq != 0.0f) && q.prompt < q.seen;
        if (q.seen == 0 || (q.rep == 1.0f && !counts)) return false;                   // (uniform)
        const int k = threadIdx.x, end = (int)min((int64_t)kSlice, J - first);
        if (k < kWords) { bits(k) = 0; before(k) = 0; }
        if (counts) for (int i = k; i < most; i += WIDTH) count(i) = 0;
        __syncthreads();
        for (int i = k; i < q.seen; i += WIDTH) {
            const int64_t j = q.tokens[i] - first;
            if (j >= 0 && j < end) atomicOr(&bits(j >> 5), 1u << (j & 31));
        }
        __syncthreads();
        if (!counts) return true;
        __shared__ unsigned total[kWaves];
        const int mine = k < kWords ? __popc(bits(k)) : 0;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const int other = __shfl_up(sum, d, kWave);
            if (k % kWave >= d) sum += other;
        }
        if (kWaves > 1) {
            if (k % kWave == kWave - 1) total[k / kWave] = sum;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                if (w < k / kWave) sum += total[w];
        }
        if (k < kWords) before(k) = sum - mine;
        __syncthreads();
        for (int i = q.prompt + k; i < q.seen; i += WIDTH) {
            const int64_t j = q.tokens[i] - first;
            if (j >= 0 && j < end) atomicAdd(&count(slot((int)j)), 1u);
        }
        __syncthreads();
        return true;
    }
    __device__ __forceinline__ int slot(int j) const { return before(j >> 5) + __popc(bits(j >> 5) & ((1u << (j & 31)) - 1)); }
    __device__ __forceinline__ unsigned marked(int j, int vec) const { return bits(j >> 5) >> (j & 31) & ((1u << vec) - 1); }
    __device__ __forceinline__ bool counted(const RowRules& q) const { return (q.pres != 0.0f || q.freq != 0.0f) && q.prompt < q.seen; }
};

// A marked element's time before the delay.
__device__ __forceinline__ float ruled(float t, unsigned occurrences, const RowRules& q) {
#pragma clang fp contract(off)
    if (q.rep != 1.0f) {
        if (t > 0.0f) t = t * q.rep;
        else t = t / q.rep;                                            // (a branch of its own: seldom taken, and a long division)
    }
    if (occurrences) {
        const float more = q.freq * (float)occurrences;
        t = t + (q.pres + more);
    }
    return t;
}

// The ruled times of one piece: VEC elements from j on, of which n are in the row.
template <typename E, int VEC, typename M>
__device__ __forceinline__ void rule_piece(float (&t)[VEC], const M& marks, bool from_history, const RowRules& q, int64_t first, int local, int n) {
    const int64_t j = first + local;
    if (from_history) {
        const unsigned m = marks.marked(local, VEC);
        if (m) {
            const bool counted = marks.counted(q);
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (m >> v & 1) t[v] = ruled(t[v], counted ? marks.count(marks.slot(local + v)) : 0, q);
        }
    }
    if (q.delay) {
        if (n == VEC) {
            const Piece<float, VEC> d = read_piece<float, VEC>(q.delay + j);
#pragma unroll
            for (int v = 0; v < VEC; ++v) t[v] += d.v[v];
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (v < n) t[v] += q.delay[j + v];
        }
    }
    if (q.allowed) {
        const unsigned a = q.allowed[j >> 5] >> (j & 31);
#pragma unroll
        for (int v = 0; v < VEC; ++v) t[v] = a >> v & 1 ? t[v] : INFINITY;
    }
}

template <typename E, int VEC>
__device__ __forceinline__ Piece<E, VEC> load_piece(const E* t, int n, E fill) {
    Piece<E, VEC> p;
    if (n == VEC) return read_piece<E, VEC>(t);
#pragma unroll
    for (int v = 0; v < VEC; ++v) p.v[v] = v < n ? t[v] : fill;
    return p;
}
template <typename E, int VEC>
__device__ __forceinline__ void store_piece(E* t, const Piece<E, VEC>& p, int n) {
    if (n == VEC) {
        reinterpret_cast<Place<E>*>(t)->w = __builtin_bit_cast(Words, p);
        return;
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v)
        if (v < n) t[v] = p.v[v];
}

// Ruled times, or (GRAD) the gradient by the times: in = times or the upstream gradient.  The gradient reads times where a token
// repeats only: their sign is all it needs.
template <typename E, int VEC, int WIDTH, int R, bool GRAD>
__global__ void __launch_bounds__(WIDTH)
rule_kernel(const E* __restrict__ in, const E* __restrict__ times, E* __restrict__ out, RuleArgs a, int64_t rows, int J, int slices) {
    using M = Marks<WIDTH, VEC * R>;
    const int64_t block = workgroup(), r = block / slices;
    if (r >= rows) return;
    const int64_t first = (block % slices) * (int64_t)M::kSlice;
    const int end = (int)min((int64_t)M::kSlice, J - first);
    const E* __restrict__ x = in + r * J + first;
    E* __restrict__ y = out + r * J + first;
    Piece<E, VEC> held[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int local = (i * WIDTH + (int)threadIdx.x) * VEC;
        if (local < end) held[i] = load_piece<E, VEC>(x + local, min(VEC, end - local), (E)0.0f);
    }
    const RowRules q = row_rules(a, r);
    M marks;
    const bool from_history = marks.build(q, first, J, a.most, !GRAD);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int local = (i * WIDTH + (int)threadIdx.x) * VEC;
        if (local >= end) continue;
        const int n = min(VEC, end - local);
        float t[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) t[v] = (float)held[i].v[v];
        if constexpr (GRAD) {
            const unsigned m = from_history ? marks.marked(local, VEC) : 0;
            if (m) {
                const E* __restrict__ at = times + r * J + first + local;
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    if (m >> v & 1) t[v] *= (float)at[v] > 0.0f ? q.rep : q.inv;
            }
            if (q.allowed) {
                const int64_t j = first + local;
                const unsigned w = q.allowed[j >> 5] >> (j & 31);
#pragma unroll
                for (int v = 0; v < VEC; ++v) t[v] = w >> v & 1 ? t[v] : 0.0f;
            }
        } else {
            rule_piece<E, VEC>(t, marks, from_history, q, first, local, n);
        }
        Piece<E, VEC> p;
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.v[v] = (E)t[v];
        store_piece<E, VEC>(y + local, p, n);
    }
}

// A part of a row: the largest negated time m, sum of exp((-t' - m) / T), and the first index that attains m.
struct Part { double s; float m; int arg; };

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, kWave));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, kWave);
    return v;
}
__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) v = min(v, __shfl_xor(v, d, kWave));
    return v;
}
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
// exp(v / T), k = log2(e) / T.  The argument is a difference from a maximum: what its rounding loses is its own size in half
// steps, of a term that shrinks faster than that grows.
__device__ __forceinline__ float soft(float v, float k) { return __builtin_amdgcn_exp2f(v * k); }
__device__ __forceinline__ double weight_of(const Part& p, float m, float k) { return p.s * (double)soft(p.m - base_of(m), k); }

// Where a part of a list begins, and the list's maximum and sum.  Parts in order; k: log2(e) / T.
struct Chosen { int part; double rest; float m; double total; };

// A row's elements as a wavefront holds them: R pieces, WIDTH / 64 wavefronts one behind the other, so that each has a run of the slice.
template <typename E, int VEC, int WIDTH, int R>
struct Run {
    float v[R][VEC];                                 // negated ruled times; -infinity: not allowed, or behind the row
    __device__ __forceinline__ static int local(int i) {
        return (((int)threadIdx.x / kWave * R + i) * kWave + (int)threadIdx.x % kWave) * VEC;
    }
    __device__ __forceinline__ void load(const E* times, const RuleArgs& a, const RowRules& q, int64_t first, int J) {
        const int end = (int)min((int64_t)WIDTH * VEC * R, J - first);
        Piece<E, VEC> held[R];
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (local(i) < end) held[i] = load_piece<E, VEC>(times + first + local(i), min(VEC, end - local(i)), (E)0.0f);
        Marks<WIDTH, VEC * R> marks;
        const bool from_history = marks.build(q, first, J, a.most, true);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (local(i) >= end) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] = -INFINITY;
                continue;
            }
            const int n = min(VEC, end - local(i));
            float t[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = (float)held[i].v[e];
            rule_piece<E, VEC>(t, marks, from_history, q, first, local(i), n);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = e < n ? -(float)(E)t[e] : -INFINITY;
        }
    }
    __device__ __forceinline__ Part part(float k, bool greedy) const {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) m = fmaxf(m, v[i][e]);
        m = wave_max(m);
        const float base = base_of(m);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += soft(v[i][e] - base, k);
        Part p{(double)wave_sum(sum), m, 0};
        if (greedy) {                                                  // (uniform)
            int at = INT32_MAX;
#pragma unroll
            for (int i = R - 1; i >= 0; --i)
#pragma unroll
                for (int e = VEC - 1; e >= 0; --e)
                    if (v[i][e] == m) at = local(i) + e;
            p.arg = wave_min(at);
        }
        return p;
    }
    // The first element whose running sum exceeds `rest`, the last possible one where rounding leaves none; -1 in a run without any.
    __device__ __forceinline__ int pick(double rest, float m, float k, float* value) const {
        const float base = base_of(m);
        const int lane = threadIdx.x % kWave;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float e[VEC], sum = 0.0f;
#pragma unroll
            for (int x = 0; x < VEC; ++x) sum += e[x] = soft(v[i][x] - base, k);
            float run = sum;
#pragma unroll
            for (int d = 1; d < kWave; d <<= 1) {
                const float other = __shfl_up(run, d, kWave);
                if (lane >= d) run += other;
            }
            const float all = __shfl(run, kWave - 1, kWave);
            if (!((double)all > rest)) { rest -= all; continue; }
            const unsigned long long over = __ballot((double)run > rest);
            const int owner = __ffsll(over) - 1;
            double left = rest - (double)(run - sum);
            int at = -1, last = 0;
#pragma unroll
            for (int x = 0; x < VEC; ++x) {
                if (e[x] > 0.0f) last = x;
                if (at < 0) { if ((double)e[x] > left) at = x; else left -= e[x]; }
            }
            at = at < 0 ? last : at;
            float mine = v[i][0];
#pragma unroll
            for (int x = 1; x < VEC; ++x) mine = at == x ? v[i][x] : mine;
            *value = __shfl(mine, owner, kWave);
            return __shfl(local(i) + at, owner, kWave);
        }
#pragma unroll
        for (int i = R - 1; i >= 0; --i) {
            int last = -1;
            float mine = 0.0f;
#pragma unroll
            for (int x = 0; x < VEC; ++x)
                if (soft(v[i][x] - base, k) > 0.0f) { last = local(i) + x; mine = v[i][x]; }
            const unsigned long long any = __ballot(last >= 0);
            if (!any) continue;
            const int owner = 63 - __clzll(any);
            *value = __shfl(mine, owner, kWave);
            return __shfl(last, owner, kWave);
        }
        return -1;
    }
};

struct Heat { float k; bool greedy, valid; double t; };
// Temperatures below 1e-37 count as 0: log2(e) / T has to be a number.
__device__ __forceinline__ Heat heat_of(const ChooseArgs& a, int64_t r) {
    const float t = a.temperature ? a.temperature[r] : a.heat;
    Heat h;
    h.valid = t >= 0.0f && t < INFINITY;
    h.greedy = t < 1e-37f;
    h.k = h.greedy || !h.valid ? kLog2e : kLog2e / t;
    h.t = h.greedy || !h.valid ? 1.0 : (double)t;
    return h;
}
__device__ __forceinline__ void store_choice(const ChooseArgs& a, int64_t r, const Heat& h, int64_t token, float value, float m, double total) {
    a.tokens[r] = token;
    a.logp[r] = token < 0 ? NAN : (float)(((double)value - (double)m) / h.t - log(total));
}

// One slice of a row: its part to `parts`, or (WHOLE: the slice is the row) the row's token.
// Bound by memory and, in a call of few rows, by the way from the history's tokens through LDS to the sums.
template <typename E, int VEC, int WIDTH, int R, bool WHOLE>
__global__ void __launch_bounds__(WIDTH)
choose_slice_kernel(const E* __restrict__ times, RuleArgs a, ChooseArgs c, Part* __restrict__ parts, int64_t rows, int J, int slices) {
    constexpr int kWaves = WIDTH / kWave;
    const int64_t block = workgroup(), r = WHOLE ? block : block / slices;
    if (r >= rows) return;
    const int slice = WHOLE ? 0 : block % slices;
    const int64_t first = (int64_t)slice * (WIDTH * VEC * R);
    const RowRules q = row_rules(a, r);
    const Heat h = heat_of(c, r);
    Run<E, VEC, WIDTH, R> run;
    run.load(times + r * J, a, q, first, J);
    Part mine = run.part(h.k, h.greedy);
    __shared__ Part part[kWaves];
    if (kWaves > 1) {
        if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = mine;
        __syncthreads();
    }
    float m = mine.m;
    double total = mine.s;
    int arg = mine.arg;
    if (kWaves > 1) {
        m = part[0].m;
#pragma unroll
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, part[w].m);
        total = 0.0;
        arg = INT32_MAX;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            total += weight_of(part[w], m, h.k);
            if (part[w].m == m) arg = min(arg, part[w].arg);
        }
    }
    if constexpr (!WHOLE) {
        if (threadIdx.x == 0) parts[r * slices + slice] = Part{total, m, arg};
        return;
    }
    if (!(total > 0.0) || !h.valid) {                                   // nothing possible, or no numbers
        if (threadIdx.x == 0) store_choice(c, r, h, -1, 0.0f, m, total);
        return;
    }
    if (h.greedy) {
        if (threadIdx.x == 0) store_choice(c, r, h, arg, m, m, total);
        return;
    }
    const float u = c.uniform[r];
    double rest = total * (double)(u > 0.0f ? u : 0.0f);
    int owner = -1, last = 0;
    if (kWaves > 1) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const double s = weight_of(part[w], m, h.k);
            if (s > 0.0) last = w;
            if (owner < 0) { if (s > rest) owner = w; else rest -= s; }
        }
        if (owner < 0) { owner = last; rest = INFINITY; }
        if ((int)threadIdx.x / kWave != owner) return;
        rest /= (double)soft(mine.m - base_of(m), h.k);
    }
    float value = 0.0f;
    const int at = run.pick(rest, mine.m, h.k, &value);
    if (threadIdx.x % kWave == 0) store_choice(c, r, h, at, value, m, total);
}

// A row's slices joined in order, and the token found in the one that it lies in: that slice is read once more.
template <typename E, int VEC, int WIDTH, int R>
__global__ void __launch_bounds__(WIDTH)
choose_join_kernel(const E* __restrict__ times, RuleArgs a, ChooseArgs c, const Part* __restrict__ parts, int J, int slices) {
    constexpr int kWaves = WIDTH / kWave;
    const int64_t r = blockIdx.x;
    const Heat h = heat_of(c, r);
    const Part* __restrict__ p = parts + r * slices;
    const int lane = threadIdx.x % kWave;
    // every wavefront joins the slices by itself
    float m = -INFINITY;
    for (int i = lane; i < slices; i += kWave) m = fmaxf(m, p[i].m);
    m = wave_max(m);
    double total = 0.0;
    int best = INT32_MAX;
    for (int i = lane; i < slices; i += kWave) {
        total += weight_of(p[i], m, h.k);
        if (p[i].m == m) best = min(best, i);
    }
#pragma unroll
    for (int d = kWave / 2; d > 0; d >>= 1) total += __shfl_xor(total, d, kWave);
    best = wave_min(best);
    if (!(total > 0.0) || !h.valid) {
        if (threadIdx.x == 0) store_choice(c, r, h, -1, 0.0f, m, total);
        return;
    }
    if (h.greedy) {
        if (threadIdx.x == 0) store_choice(c, r, h, (int64_t)best * (WIDTH * VEC * R) + p[best].arg, m, m, total);
        return;
    }
    const float u = c.uniform[r];
    double rest = total * (double)(u > 0.0f ? u : 0.0f);
    int slice = -1, last = 0;
    for (int i0 = 0; i0 < slices && slice < 0; i0 += kWave) {
        const double s = i0 + lane < slices ? weight_of(p[i0 + lane], m, h.k) : 0.0;
        double run = s;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const double other = __shfl_up(run, d, kWave);
            if (lane >= d) run += other;
        }
        const unsigned long long any = __ballot(s > 0.0), over = __ballot(run > rest && s > 0.0);
        if (any) last = i0 + 63 - __clzll(any);
        if (over) {
            const int owner = __ffsll(over) - 1;
            slice = i0 + owner;
            rest -= __shfl(run - s, owner, kWave);
        } else {
            rest -= __shfl(run, kWave - 1, kWave);
        }
    }
    if (slice < 0) { slice = last; rest = INFINITY; }
    rest = fmax(rest, 0.0);
    const Part part = p[slice];
    rest /= (double)soft(part.m - base_of(m), h.k);
    const int64_t first = (int64_t)slice * (WIDTH * VEC * R);
    const RowRules q = row_rules(a, r);
    Run<E, VEC, WIDTH, R> run;
    run.load(times + r * J, a, q, first, J);
    const Part mine = run.part(h.k, false);
    float base = mine.m;
    if (kWaves > 1) {
        __shared__ Part wave[kWaves];
        if (lane == 0) wave[threadIdx.x / kWave] = mine;
        __syncthreads();
        int owner = -1, back = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const double s = weight_of(wave[w], part.m, h.k);
            if (s > 0.0) back = w;
            if (owner < 0) { if (s > rest) owner = w; else rest -= s; }
        }
        if (owner < 0) { owner = back; rest = INFINITY; }
        if ((int)threadIdx.x / kWave != owner) return;
        rest /= (double)soft(mine.m - base_of(part.m), h.k);
    }
    float value = 0.0f;
    const int at = run.pick(rest, base, h.k, &value);
    if (lane == 0) store_choice(c, r, h, at < 0 ? -1 : first + at, value, m, total);
}

// ---- launches --------------------------------------------------------------------------------------------------------------------

// Bytes of LDS of a slice's marks; a slice counts at most min(slice, L) elements.
template <int SLICE>
size_t marks_bytes(const RuleArgs& a) { return a.history ? (size_t)SLICE / 4 + 4 * (size_t)a.most : 0; }

template <typename E, int WIDTH, int R, bool GRAD>
int launch_rule_slices(const void* in, const void* times, void* out, RuleArgs a, int64_t rows, int64_t J, hipStream_t stream) {
    constexpr int VEC = 16 / sizeof(E), kSlice = WIDTH * VEC * R;
    const int slices = (int)((J + kSlice - 1) / kSlice);
    a.most = a.history && !GRAD ? (int)std::min<int64_t>(a.L, kSlice) : 0;
    {
        KernelTimerScope timer_(GRAD ? "rule_times_backward" : "rule_times", stream);
        hipLaunchKernelGGL((rule_kernel<E, VEC, WIDTH, R, GRAD>), wide_grid(rows * slices, WIDTH), dim3(WIDTH), marks_bytes<kSlice>(a), stream,
                           static_cast<const E*>(in), static_cast<const E*>(times), static_cast<E*>(out), a, rows, (int)J, slices);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

template <bool GRAD>
int launch_rules(const void* in, const void* times, int type, const RuleArgs& a, void* out, int64_t rows, int64_t J, hipStream_t stream) {
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        constexpr int VEC = 16 / sizeof(E);
        if (J <= 64 * VEC) return launch_rule_slices<E, 64, 1, GRAD>(in, times, out, a, rows, J, stream);
        return launch_rule_slices<E, 256, 4, GRAD>(in, times, out, a, rows, J, stream);
    });
}

template <typename E, int WIDTH, int R>
int launch_choose_slices(const void* times, RuleArgs a, const ChooseArgs& c, int64_t rows, int64_t J, void* ws, hipStream_t stream) {
    constexpr int VEC = 16 / sizeof(E), kSlice = WIDTH * VEC * R;
    const int slices = (int)((J + kSlice - 1) / kSlice);
    const E* t = static_cast<const E*>(times);
    Part* parts = static_cast<Part*>(ws);
    a.most = a.history ? (int)std::min<int64_t>(a.L, kSlice) : 0;
    if (slices == 1) {
        KernelTimerScope timer_("choose", stream);
        hipLaunchKernelGGL((choose_slice_kernel<E, VEC, WIDTH, R, true>), wide_grid(rows, WIDTH), dim3(WIDTH), marks_bytes<kSlice>(a), stream, t, a, c,
                           nullptr, rows, (int)J, 1);
    } else {
        {
            KernelTimerScope timer_("choose_slice", stream);
            hipLaunchKernelGGL((choose_slice_kernel<E, VEC, WIDTH, R, false>), wide_grid(rows * slices, WIDTH), dim3(WIDTH), marks_bytes<kSlice>(a),
                               stream, t, a, c, parts, rows, (int)J, slices);
        }
        KernelTimerScope timer_("choose_join", stream);
        hipLaunchKernelGGL((choose_join_kernel<E, VEC, WIDTH, R>), dim3((unsigned)rows), dim3(WIDTH), marks_bytes<kSlice>(a), stream, t, a, c, parts,
                           (int)J, slices);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

constexpr int kChooseSlice = 256 * 32;

}  // namespace

size_t choose_workspace(int64_t rows, int64_t J) {
    return J > kChooseSlice ? align_up((size_t)rows * (size_t)((J + kChooseSlice - 1) / kChooseSlice) * sizeof(Part)) : 0;
}

int launch_rule_times(const void* times, int type, const RuleArgs& a, void* out, int64_t rows, int64_t J, hipStream_t stream) {
    return launch_rules<false>(times, nullptr, type, a, out, rows, J, stream);
}

int launch_rule_times_backward(const void* grad, const void* times, int type, const RuleArgs& a, void* dtimes, int64_t rows, int64_t J,
                               hipStream_t stream) {
    return launch_rules<true>(grad, times, type, a, dtimes, rows, J, stream);
}

int launch_choose(const void* times, int type, const RuleArgs& a, const ChooseArgs& c, int64_t rows, int64_t J, void* ws, hipStream_t stream) {
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        constexpr int VEC = 16 / sizeof(E);
        if (J <= 64 * VEC) return launch_choose_slices<E, 64, 1>(times, a, c, rows, J, ws, stream);
        return launch_choose_slices<E, 256, 32 / VEC>(times, a, c, rows, J, ws, stream);
    });
}

}  // namespace snntc
