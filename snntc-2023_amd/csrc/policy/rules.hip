// Choices by rules.  A row of spike times t[J] stands for the distribution softmax(-t); rules change the times before a token is drawn
// or a loss is taken.  With c_j the occurrences of j in the row's part of a history of tokens and o_j those behind the prompt,
//     a_j = t_j r  (t_j > 0),  t_j / r  (t_j <= 0)       where c_j > 0,  t_j elsewhere
//     b_j = a_j + (presence + frequency o_j)             where o_j > 0,  a_j elsewhere
//     t'_j = b_j + delay_j  where j is allowed, +infinity elsewhere,         dt_j = dt'_j (1, r or 1 / r; 0 where not allowed)
// and a token is the first j with sum_{i <= j} exp(-(t'_i - min t') / T) > u sum_i exp(-(t'_i - min t') / T).
//
// A workgroup owns a slice of a row.  It marks the history's tokens that lie in the slice in a bitmap in LDS, a bit for each element, and
// counts the occurrences of marked elements: an element that no token names costs one bit test.
// The arithmetic of a ruled time is float32 without contraction: products and sums round one by one, as written above.  A
// token is drawn from the times as rule_times stores them, rounded to times' type, so that its log-probability is that of the ruled times.
#include "../sequences.h"
#include "wave.h"

namespace snntc {
namespace {

constexpr float kLog2e = 1.44269504f;
constexpr float kColdest = 1e-30f;                   // temperatures below count as 0: log2(e) / T has to leave room for a time
// VEC elements, 16 bytes (or, of float32, 32), at any place of their type: the target loads and stores four words at any address.
template <typename E, int VEC>
struct Piece { E v[VEC]; };
typedef unsigned Words __attribute__((ext_vector_type(4)));
typedef unsigned WordsAt2 __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned WordsAt4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename E>
using Place = typename std::conditional<sizeof(E) == 2, WordsAt2, WordsAt4>::type;
template <typename E, int VEC>
__device__ __forceinline__ Piece<E, VEC> read_piece(const E* at) {
    if constexpr (VEC == 1) return Piece<E, 1>{{*at}};
    constexpr int N = VEC * sizeof(E) / sizeof(Words) + (VEC == 1);
    struct All { Words w[N]; } all;
#pragma unroll
    for (int i = 0; i < N; ++i) all.w[i] = reinterpret_cast<const Place<E>*>(at)[i];
    if constexpr (VEC > 1) return __builtin_bit_cast(Piece<E, VEC>, all);
}
template <bool STREAM, typename E, int VEC>
__device__ __forceinline__ void store_piece(E* at, const Piece<E, VEC>& p) {
    if constexpr (VEC == 1) *at = p.v[0];
    else if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(Words, p), reinterpret_cast<Place<E>*>(at));
    else *reinterpret_cast<Place<E>*>(at) = __builtin_bit_cast(Words, p);
}
// VEC numbers rounded to E, two by one instruction.
template <typename E, int VEC>
__device__ __forceinline__ Piece<E, VEC> round_piece(const float (&t)[VEC]) {
    Piece<E, VEC> p;
    if constexpr (VEC == 1 || sizeof(E) == 4) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.v[v] = (E)t[v];
    } else {
        typedef float Pair __attribute__((ext_vector_type(2)));
        typedef E Two __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int v = 0; v < VEC; v += 2) {
            const Two two = __builtin_convertvector((Pair{t[v], t[v + 1]}), Two);
            p.v[v] = two.x; p.v[v + 1] = two.y;
        }
    }
    return p;
}

// A launch's workgroup among fewer than 2^32: 2^24 rows, and as many slices as their times' memory has place for.
__device__ __forceinline__ unsigned place() { return (unsigned)workgroup(); }

// (named as device memory: a choice between two pointers would be read as generic memory)
template <typename T>
using Device = const T __attribute__((address_space(1)))*;
// An element of an array by its offset in 32 bits, which the instructions add to a common address: an address of its own takes two registers (with them
// 4096 draws from 1000 float32 times take 16.3 us, without 13.5).
template <typename T>
__device__ __forceinline__ Device<T> place_in(Device<T> array, unsigned i) {
    return (Device<T>)((Device<char>)array + (unsigned)(i * sizeof(T)));
}

// What is the same for a whole row.
struct RowRules {
    const long long* tokens;
    int seen, prompt;                                // tokens [0, seen) count, those from `prompt` on as occurrences
    float rep, inv, pres, freq;
    const float* delay;
    const unsigned* allowed;
};
__device__ __forceinline__ RowRules row_rules(const RuleArgs& a, unsigned r) {
    RowRules q{};
    q.rep = 1.0f;
    if (a.history) {
        const int64_t h = r / (unsigned)a.rows_per_history;
        q.tokens = reinterpret_cast<const long long*>(a.history) + h * a.L;
        const auto inside = [&](int64_t n) { return (int)(n < 0 ? 0 : n > a.L ? a.L : n); };
        q.seen = a.lengths ? inside(a.lengths[r]) : (int)a.L;
        q.prompt = a.prompts ? inside(a.prompts[h]) : 0;
        q.rep = a.repetition ? a.repetition[h] : a.rep;
        q.pres = a.presence ? a.presence[h] : a.pres;
        q.freq = a.frequency ? a.frequency[h] : a.freq;
        q.inv = 1.0f / q.rep;
    }
    q.delay = a.delay ? a.delay + (int64_t)r * a.delay_stride : nullptr;
    q.allowed = a.allowed ? a.allowed + (int64_t)r * a.allowed_stride : nullptr;
    return q;
}

// The marks of a slice of WIDTH * PER elements in LDS: a bitmap and, for COUNT (16-bit or 32-bit integers), occurrences; only those of
// marked elements are ever cleared or read.
template <int SLICE, typename COUNT>
struct MarkMemory { unsigned bits[SLICE / 32 + 1]; COUNT count[SLICE]; };
// For the gradient: `late` marked elements have a time above 0.
template <int SLICE>
struct MarkMemory<SLICE, void> { unsigned bits[SLICE / 32 + 1], late[SLICE / 32 + 1]; };

template <int WIDTH, int PER, typename COUNT>
struct Marks {
    static constexpr int kSlice = WIDTH * PER, kWords = kSlice / 32, kHeld = 1024 / WIDTH < 2 ? 2 : 1024 / WIDTH > 8 ? 8 : 1024 / WIDTH;
    static constexpr bool kCounts = !std::is_void<COUNT>::value;
    using Memory = MarkMemory<kSlice, COUNT>;
    long long held[kHeld];                           // the thread's first tokens, as they come: what is done with them waits for them

    // The thread's tokens of a batch, the last of `n` once more behind them.
    __device__ __forceinline__ static void batch(long long (&to)[kHeld], const long long* tokens, int64_t n) {
        const int last = (int)min(n, (int64_t)kHeld * WIDTH) - 1;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) to[i] = *place_in((Device<long long>)tokens, min(i * WIDTH + (int)threadIdx.x, last));
    }
    // Before the row's numbers are known: the two do not wait for each other.
    __device__ __forceinline__ void request(const RuleArgs& a, const RowRules& q) {
        if (a.history) batch(held, q.tokens, a.L);
    }
    // Where the thread's tokens of the batch at `base` lie in the slice; -1: nowhere, or the row does not see them.
    __device__ __forceinline__ static void places(int (&j)[kHeld], const long long (&tok)[kHeld], int base, const RowRules& q, int first, int end) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const unsigned long long to = (unsigned long long)tok[i] - (unsigned)first;
            j[i] = base + i * WIDTH + (int)threadIdx.x < q.seen && to < (unsigned)end ? (int)to : -1;
        }
    }
    // f(places, batch's first token, live) of the batches behind the first from the one with token `from` on.
    template <typename F>
    __device__ __forceinline__ static void others(const RowRules& q, int from, int first, int end, F&& f) {
        constexpr int kBatch = kHeld * WIDTH;
        for (int base = max(from / kBatch, 1) * kBatch; base < q.seen; base += kBatch) {
            long long tok[kHeld];
            int j[kHeld];
            batch(tok, q.tokens + base, q.seen - base);
            places(j, tok, base, q, first, end);
            f(j, base, std::integral_constant<int, kHeld>());
        }
    }
    // Returns whether there are any rules from the history; every thread of the workgroup calls it.  times: of the slice, for the signs.
    template <typename E>
    __device__ __forceinline__ bool build(Memory& lds, const RowRules& q, int64_t first, int end, const E* times) const {
        const bool counts = counted(q);
        if (q.seen == 0 || (q.rep == 1.0f && !counts)) return false;                   // (uniform)
        const int k = threadIdx.x;
#pragma unroll
        for (int w = 0; w < (kWords + WIDTH - 1) / WIDTH; ++w)
            if (w * WIDTH + k < kWords) {
                lds.bits[w * WIDTH + k] = 0;
                if constexpr (!kCounts) lds.late[w * WIDTH + k] = 0;
            }
        __syncthreads();
        // (of a first batch that is not full only the first `live` of a thread's tokens are looked at: rows of 5003 with some 100 tokens 31.5 -> 29.3 us)
        const int full = (q.seen + WIDTH - 1) / WIDTH;                                 // (uniform)
        int mine[kHeld];
        places(mine, held, 0, q, (int)first, end);
        const auto mark = [&](const int (&j)[kHeld], int, auto live) {
            float t[kHeld];
            if constexpr (!kCounts) {
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    if (i >= live) break;
                    t[i] = j[i] >= 0 ? (float)times[j[i]] : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (i >= live) break;
                if (j[i] < 0) continue;
                atomicOr(&lds.bits[j[i] >> 5], 1u << (j[i] & 31));
                if constexpr (kCounts) lds.count[j[i]] = 0;
                else if (t[i] > 0.0f) atomicOr(&lds.late[j[i] >> 5], 1u << (j[i] & 31));
            }
        };
        mark(mine, 0, full);
        others(q, 0, (int)first, end, mark);
        __syncthreads();
        if constexpr (kCounts) {
            if (!counts) return true;
            const auto count = [&](const int (&j)[kHeld], int base, auto live) {
#pragma unroll
                for (int i = 0; i < kHeld; ++i) {
                    if (i >= live) break;
                    if (j[i] < 0 || base + i * WIDTH + k < q.prompt) continue;
                    const unsigned at = j[i];
                    if constexpr (sizeof(COUNT) == 2)                                  // (at most 2^16 - 1 of a token: no carry to the neighbour)
                        atomicAdd(reinterpret_cast<unsigned*>(&lds.count[at & ~1u]), at & 1 ? 1u << 16 : 1u);
                    else
                        atomicAdd(&lds.count[at], (COUNT)1);
                }
            };
            count(mine, 0, full);
            others(q, q.prompt, (int)first, end, count);
            __syncthreads();
        }
        return true;
    }
    // Bits of the elements from j on, at any place in their words (there is a word behind the last one).
    __device__ __forceinline__ static unsigned from(const unsigned* bits, int j) { return __builtin_amdgcn_alignbit(bits[(j >> 5) + 1], bits[j >> 5], j & 31); }
    __device__ __forceinline__ static unsigned marked(const Memory& lds, int j, int vec) { return from(lds.bits, j) & ((1u << vec) - 1); }
    __device__ __forceinline__ static unsigned late(const Memory& lds, int j) { return from(lds.late, j); }
    __device__ __forceinline__ static bool counted(const RowRules& q) {
        return kCounts && (q.pres != 0.0f || q.freq != 0.0f) && q.prompt < q.seen;
    }
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

// t where bit `at` of a mask is set, `other` elsewhere: a sign-extended bit selects.
__device__ __forceinline__ float where_bit(unsigned mask, int at, float t, float other) {
    const unsigned m = (unsigned)__builtin_amdgcn_sbfe((int)mask, at, 1);
    return __uint_as_float((__float_as_uint(t) & m) | (__float_as_uint(other) & ~m));
}

// Keeps the compiler from carrying a piece's elements in float32 from one use to the next, which takes half of the wavefronts' registers.
template <typename P>
__device__ __forceinline__ void forget(P& p) {
    if constexpr (sizeof(P) == sizeof(Words)) {
        Words w = __builtin_bit_cast(Words, p);
        asm volatile("" : "+v"(w));
        p = __builtin_bit_cast(P, w);
    }
}

// Loads return in order, and the compiler counts on how many are behind the one it waits for: only where none of them is in a branch.
// So every lane loads whole pieces: behind the end of a slice its last VEC elements once more (a slice that would have fewer begins earlier),
// and where a row has no delays or mask, these.
__device__ const float kNoDelay[8] = {};
__device__ const unsigned kAllAllowed[1] = {~0u};

// Words of a mask that hold a piece's bits.
struct Allowed { unsigned low, high; };

// A slice of a row: elements [first, first + end).
struct Slice { int64_t first; int end; };
template <int SLICE, int VEC>
__device__ __forceinline__ Slice slice_of(unsigned slice, int J) {
    const int64_t latest = J > VEC ? (J - VEC) & ~31 : 0;
    Slice s;
    s.first = min((int64_t)slice * SLICE, latest);
    s.end = (int)min((int64_t)SLICE, J - s.first);
    return s;
}
// What there is of a slice, by elements of the slice; its first element has the lowest bit of a word of `allowed`.
template <typename E, int VEC>
struct Reader {
    Device<E> times;
    Device<float> delay;
    Device<unsigned> allowed;
    unsigned any_delay, last_word;                   // (0: where there is no array)
    __device__ __forceinline__ Reader(const E* row, const RowRules& q, const Slice& s)
        : times((Device<E>)row + s.first), delay(q.delay ? (Device<float>)q.delay + s.first : (Device<float>)kNoDelay),
          allowed(q.allowed ? (Device<unsigned>)q.allowed + (s.first >> 5) : (Device<unsigned>)kAllAllowed),
          any_delay(q.delay ? ~0u : 0), last_word(q.allowed ? (unsigned)(s.end - 1) >> 5 : 0) {}
    __device__ __forceinline__ Piece<E, VEC> piece(int j) const { return read_piece<E, VEC>((const E*)place_in(times, j)); }
    __device__ __forceinline__ Piece<float, VEC> delays(int j) const { return read_piece<float, VEC>((const float*)place_in(delay, j & any_delay)); }
    __device__ __forceinline__ Allowed words(int j) const {
        const unsigned at = (unsigned)j >> 5;
        return Allowed{*place_in(allowed, min(at, last_word)), *place_in(allowed, min(at + 1, last_word))};
    }
};
__device__ __forceinline__ unsigned allowed_from(const Allowed& w, int j) { return __builtin_amdgcn_alignbit(w.high, w.low, (unsigned)j & 31); }

// The ruled times of one piece.  Marked elements are few: one at a time and lane, instead of a test for each.
template <typename E, int VEC, typename M>
__device__ __forceinline__ void rule_piece(Piece<E, VEC>& p, const typename M::Memory& lds, bool from_history, const RowRules& q,
                                           const Piece<float, VEC>& delay, unsigned allowed, int local) {
    unsigned m = from_history ? M::marked(lds, local, VEC) : 0;
    if (!m && !q.delay && !q.allowed) return;
    float t[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) t[v] = (float)p.v[v];
    const bool counted = M::counted(q);
    while (m) {
        const int at = __ffs(m) - 1;
        m &= m - 1;
        float y = t[0];
#pragma unroll
        for (int v = 1; v < VEC; ++v) y = at == v ? t[v] : y;
        y = ruled(y, counted ? (unsigned)lds.count[local + at] : 0, q);
#pragma unroll
        for (int v = 0; v < VEC; ++v) t[v] = at == v ? y : t[v];
    }
    if (q.delay) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) t[v] += delay.v[v];
    }
    if (q.allowed) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) t[v] = where_bit(allowed, v, t[v], INFINITY);
    }
    p = round_piece<E, VEC>(t);
}

// Ruled times, or (GRAD) the gradient by the times: in = times or the upstream gradient.  The gradient reads times where a token
// repeats only: their sign is all it needs.  Bound by memory: 4096 rows of 32000 bf16 times forward 111 us (545 MB, 4.9 TB/s; a copy of the times takes 98),
// gradient 110 us (636 MB, 5.8 TB/s: lines of scattered times for their signs are 91 MB of it).
template <typename E, int VEC, int WIDTH, int R, typename COUNT, bool STREAM>
__global__ void __launch_bounds__(WIDTH)
rule_kernel(const E* __restrict__ in, const E* __restrict__ times, E* __restrict__ out, RuleArgs a, int64_t rows, int J, int slices) {
    using M = Marks<WIDTH, VEC * R, COUNT>;
    constexpr bool GRAD = !M::kCounts;
    __shared__ typename M::Memory lds;
    const unsigned block = place(), r = block / (unsigned)slices;
    if (r >= rows) return;
    const Slice s = slice_of<M::kSlice, VEC>(block - r * (unsigned)slices, J);
    const int64_t at = (int64_t)r * J + s.first;
    const RowRules q = row_rules(a, r);
    const Reader<E, VEC> from(in + (int64_t)r * J, q, s);
    M marks;
    marks.request(a, q);
    const auto local = [&](int i) { return min((i * WIDTH + (int)threadIdx.x) * VEC, s.end - VEC); };
    Piece<E, VEC> held[R];
    Allowed allowed[R];
    Piece<float, VEC> delay[2];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        held[i] = from.piece(local(i));
        allowed[i] = from.words(local(i));
    }
    if constexpr (!GRAD) delay[0] = from.delays(local(0));
    const bool from_history = marks.build(lds, q, s.first, s.end, GRAD ? times + at : nullptr);
#pragma unroll
    for (int i = 0; i < R; ++i) {
        if ((i * WIDTH + ((int)threadIdx.x & -kWave)) * VEC >= s.end) break;              // (a whole wavefront)
        if constexpr (GRAD) {
            const unsigned m = from_history ? M::marked(lds, local(i), VEC) : 0;
            if (m) {
                const unsigned late = M::late(lds, local(i));
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float t = (float)held[i].v[v] * where_bit(late, v, q.rep, q.inv);
                    held[i].v[v] = m >> v & 1 ? (E)t : held[i].v[v];
                }
            }
            if (q.allowed) {
                const unsigned w = allowed_from(allowed[i], local(i));
#pragma unroll
                for (int v = 0; v < VEC; ++v) held[i].v[v] = w >> v & 1 ? held[i].v[v] : (E)0.0f;
            }
        } else {
            if (i + 1 < R) delay[(i + 1) % 2] = from.delays(local(i + 1));
            rule_piece<E, VEC, M>(held[i], lds, from_history, q, delay[i % 2], allowed_from(allowed[i], local(i)), local(i));
        }
        store_piece<STREAM, E, VEC>(out + at + local(i), held[i]);
    }
}

// A wavefront's run of a row: the largest negated time m, the sum of exp((-t' - m) / T), and the first index in the run that attains m (where
// it is asked for).
struct Part { float s, m; int arg, unused; };

__device__ __forceinline__ float wave_max(float v) { return wave_join(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); }); }
__device__ __forceinline__ int wave_min(int v) { return wave_join(v, INT32_MAX, [](int a, int b) { return min(a, b); }); }
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.0f : m; }
// exp(d / T), k = log2(e) / T, of a difference from a maximum: what the argument's rounding loses is its own size in half steps, of a
// term that shrinks faster than that grows, and equal times have terms of exactly 1.
__device__ __forceinline__ float term(float d, float k) { return __builtin_amdgcn_exp2f(d * k); }
__device__ __forceinline__ double weight_of(const Part& p, float m, float k) { return (double)p.s * (double)term(p.m - base_of(m), k); }

// A row's elements as a wavefront holds them: R pieces, WIDTH / 64 wavefronts one behind the other, so that each has a run of the slice.
template <typename E, int VEC, int R>
struct Run {
    static constexpr int kLength = kWave * VEC * R;
    Piece<E, VEC> t[R];                              // ruled times; +infinity: not allowed, or behind the row
    Allowed allowed[R];
    Piece<float, VEC> delay[2];
    int end;                                         // of the slice
    __device__ __forceinline__ int origin() const { return (int)threadIdx.x / kWave * kLength; }      // of the wavefront's run in the slice
    __device__ __forceinline__ int proper(int i) const { return origin() + (i * kWave + (int)threadIdx.x % kWave) * VEC; }
    __device__ __forceinline__ int local(int i) const { return min(proper(i), end - VEC); }
    __device__ __forceinline__ int in_run(int i) const { return local(i) - origin(); }
    __device__ __forceinline__ float v(int i, int e) const { return -(float)t[i].v[e]; }
    __device__ __forceinline__ void request(const Reader<E, VEC>& from, const Slice& s) {
        end = s.end;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            t[i] = from.piece(local(i));
            allowed[i] = from.words(local(i));
        }
        delay[0] = from.delays(local(0));
    }
    // M: the marks of the slice.  own: elements of the slice before this one have been the last slice's.
    template <typename M>
    __device__ __forceinline__ void rule(const typename M::Memory& lds, bool from_history, const RowRules& q, const Reader<E, VEC>& from, int own) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (i + 1 < R) delay[(i + 1) % 2] = from.delays(local(i + 1));
            rule_piece<E, VEC, M>(t[i], lds, from_history, q, delay[i % 2], allowed_from(allowed[i], local(i)), local(i));
            const int skip = max(proper(i), own) - local(i);
            if (skip > 0) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) t[i].v[e] = e < skip ? (E)INFINITY : t[i].v[e];
            }
        }
    }
    __device__ __forceinline__ Part part(float k, bool greedy) {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) m = fmaxf(m, v(i, e));
        m = wave_max(m);
        const float base = base_of(m);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            forget(t[i]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum += term(v(i, e) - base, k);
        }
        Part p{wave_sum(sum), m, 0, 0};
        if (greedy) {                                                  // (uniform)
            int at = INT32_MAX;
#pragma unroll
            for (int i = R - 1; i >= 0; --i) {
                forget(t[i]);
#pragma unroll
                for (int e = VEC - 1; e >= 0; --e)
                    if (v(i, e) == m) at = in_run(i) + e;
            }
            p.arg = wave_min(at);
        }
        return p;
    }
    // The first element of the run whose running sum exceeds `rest`, the last possible one where rounding leaves none; -1 in
    // a run without any.  Sums over lanes are rounded in an order of their own: `run` may rise at a lane without a term, and run - sum need not
    // be the lane before's `run`.  So only lanes and elements with a term are asked, and what is left in a lane is no less than 0.
    __device__ __forceinline__ int pick(double rest, float m, float k, float* value) {
        const float base = base_of(m);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            forget(t[i]);
            float e[VEC], sum = 0.0f;
#pragma unroll
            for (int x = 0; x < VEC; ++x) sum += e[x] = term(v(i, x) - base, k);
            const float run = wave_scan(sum), all = of_lane(run, kWave - 1);
            if (!((double)all > rest)) { rest -= all; continue; }
            const unsigned long long any = __ballot(sum > 0.0f), over = __ballot(sum > 0.0f && (double)run > rest);
            const int owner = over ? __ffsll(over) - 1 : 63 - __clzll(any);
            double left = fmax(rest - (double)(run - sum), 0.0);
            int at = -1, last = 0;
#pragma unroll
            for (int x = 0; x < VEC; ++x) {
                if (e[x] > 0.0f) last = x;
                if (at < 0) { if ((double)e[x] > left) at = x; else left -= e[x]; }
            }
            at = at < 0 ? last : at;
            float mine = v(i, 0);
#pragma unroll
            for (int x = 1; x < VEC; ++x) mine = at == x ? v(i, x) : mine;
            *value = of_lane(mine, owner);
            return of_lane(in_run(i) + at, owner);
        }
#pragma unroll
        for (int i = R - 1; i >= 0; --i) {
            forget(t[i]);
            int last = -1;
            float mine = 0.0f;
#pragma unroll
            for (int x = 0; x < VEC; ++x)
                if (term(v(i, x) - base, k) > 0.0f) { last = in_run(i) + x; mine = v(i, x); }
            const unsigned long long any = __ballot(last >= 0);
            if (!any) continue;
            const int owner = 63 - __clzll(any);
            *value = of_lane(mine, owner);
            return of_lane(last, owner);
        }
        return -1;
    }
};

struct Heat { float k; bool greedy, valid; double t; };
__device__ __forceinline__ Heat heat_of(const ChooseArgs& a, unsigned r) {
    const float t = a.temperature ? a.temperature[r] : a.heat;
    Heat h;
    h.valid = t >= 0.0f && t < INFINITY;
    h.greedy = t < kColdest;
    h.k = h.greedy || !h.valid ? kLog2e : kLog2e / t;
    h.t = h.greedy || !h.valid ? 1.0 : (double)t;
    return h;
}

// A row's n parts joined by a wavefront, and the part that the row's token lies in: part -1: there is none.
struct Found { int part; double rest, total; float m; Part at; };
__device__ __forceinline__ Found find_part(const Part* parts, int n, const Heat& h, const float* uniform, unsigned r) {
    const int lane = threadIdx.x % kWave;
    const Part none{0.0f, -INFINITY, 0, 0}, mine = lane < n ? parts[lane] : none;       // (mostly all there are)
    const auto get = [&](int i0) { return i0 == 0 ? mine : i0 + lane < n ? parts[i0 + lane] : none; };
    const float u = h.greedy || !h.valid ? 0.0f : uniform[r];
    float m = -INFINITY;
    for (int i0 = 0; i0 < n; i0 += kWave) m = fmaxf(m, get(i0).m);
    m = wave_max(m);
    double total = 0.0;
    int best = INT32_MAX;
    for (int i0 = 0; i0 < n; i0 += kWave) {
        const Part p = get(i0);
        total += weight_of(p, m, h.k);
        if (p.m == m) best = min(best, i0 + lane);
    }
    total = wave_sum(total);
    Found f{-1, 0.0, total, m, none};
    if (!(total > 0.0) || !h.valid) return f;                           // nothing possible, or no numbers
    if (h.greedy) {
        f.part = wave_min(best);
        f.at = parts[f.part];
        return f;
    }
    double rest = total * (double)(u > 0.0f ? u : 0.0f);
    int last = 0;
    for (int i0 = 0; i0 < n && f.part < 0; i0 += kWave) {
        const double s = weight_of(get(i0), m, h.k), run = wave_scan(s);
        const unsigned long long any = __ballot(s > 0.0), over = __ballot(run > rest && s > 0.0);
        if (any) last = i0 + 63 - __clzll(any);
        if (over) {
            const int owner = __ffsll(over) - 1;
            f.part = i0 + owner;
            rest -= of_lane(run - s, owner);
        } else {
            rest -= of_lane(run, kWave - 1);
        }
    }
    if (f.part < 0) { f.part = last; rest = INFINITY; }
    f.at = parts[f.part];
    // (in units of the part's own sum, which the choice of the part keeps above 0)
    f.rest = fmax(rest, 0.0) / (double)term(f.at.m - base_of(m), h.k);
    return f;
}

__device__ __forceinline__ void store_choice(const ChooseArgs& a, unsigned r, const Heat& h, int64_t token, float value, const Found& f) {
    a.tokens[r] = token;
    a.logp[r] = token < 0 ? NAN : (float)(((double)value - (double)f.m) / h.t - log(f.total));
}

// A slice of a row.  WHOLE: the slice is the row, and the row's token is found; else its wavefronts' parts go to `parts`.  Bound by vector instructions:
// 4096 rows of 32000 bf16 times with delays and 256 tokens each take 77 us (281 MB, 3.7 TB/s, 84 % of the issue slots and the exponentials besides),
// without rules 58 with the join.
template <typename E, int VEC, int WIDTH, int R, typename COUNT, bool WHOLE>
__global__ void __launch_bounds__(WIDTH)
choose_slice_kernel(const E* __restrict__ times, RuleArgs a, ChooseArgs c, Part* __restrict__ parts, int64_t rows, int J, int slices) {
    using M = Marks<WIDTH, VEC * R, COUNT>;
    using Mine = Run<E, VEC, R>;
    constexpr int kWaves = WIDTH / kWave;
    __shared__ typename M::Memory lds;
    __shared__ Part part[kWaves];
    const unsigned block = place(), r = WHOLE ? block : block / (unsigned)slices;
    if (r >= rows) return;
    const unsigned slice = WHOLE ? 0 : block - r * (unsigned)slices, wave = threadIdx.x / kWave;
    const Slice s = slice_of<M::kSlice, VEC>(slice, J);
    const E* __restrict__ row = times + (int64_t)r * J;
    const RowRules q = row_rules(a, r);
    M marks;
    marks.request(a, q);
    const Reader<E, VEC> from(row, q, s);
    Mine run;
    run.request(from, s);
    const Heat h = heat_of(c, r);
    const bool from_history = marks.build(lds, q, s.first, s.end, row);
    run.template rule<M>(lds, from_history, q, from, (int)((int64_t)slice * M::kSlice - s.first));
    const Part mine = run.part(h.k, h.greedy);
    if constexpr (!WHOLE) {
        // (an index from where the run has its place, wherever the slice begins)
        if (threadIdx.x % kWave == 0)
            parts[((int64_t)r * slices + slice) * kWaves + wave] = Part{mine.s, mine.m, mine.arg - (int)((int64_t)slice * M::kSlice - s.first), 0};
        return;
    }
    if (threadIdx.x % kWave == 0) part[wave] = mine;
    __syncthreads();
    const Found f = find_part(part, kWaves, h, c.uniform, r);
    if (wave != (f.part < 0 ? 0u : (unsigned)f.part)) return;
    int at = -1;
    float value = 0.0f;
    if (f.part >= 0 && h.greedy) { at = mine.arg; value = mine.m; }
    else if (f.part >= 0) at = run.pick(f.rest, mine.m, h.k, &value);
    if (threadIdx.x % kWave == 0) store_choice(c, r, h, at < 0 ? -1 : run.origin() + at, value, f);
}

// A row's parts joined in order, and the run that the token lies in read once more: by the first wavefront, while all go through
// the history, which was requested before the run was known.
template <typename E, int VEC, int R, typename COUNT, int kJoinThreads>
__global__ void __launch_bounds__(kJoinThreads)
choose_join_kernel(const E* __restrict__ times, RuleArgs a, ChooseArgs c, const Part* __restrict__ parts, int64_t rows, int J, int count) {
    using Mine = Run<E, VEC, R>;
    using M = Marks<kJoinThreads, Mine::kLength / kJoinThreads, COUNT>;
    __shared__ typename M::Memory lds;
    const unsigned r = place();
    if (r >= rows) return;
    const RowRules q = row_rules(a, r);
    const Heat h = heat_of(c, r);
    M marks;
    if (!h.greedy) marks.request(a, q);
    const Found f = find_part(parts + (int64_t)r * count, count, h, c.uniform, r);
    const int64_t begin = (int64_t)f.part * Mine::kLength;
    int64_t token = -1;
    float value = 0.0f;
    if (f.part >= 0 && h.greedy) {
        token = begin + f.at.arg;
        value = f.at.m;
    } else if (f.part >= 0) {
        const E* __restrict__ row = times + (int64_t)r * J;
        const Slice s = slice_of<Mine::kLength, VEC>(f.part, J);
        const Reader<E, VEC> from(row, q, s);
        Mine run;
        if (threadIdx.x < kWave) run.request(from, s);
        const bool from_history = marks.build(lds, q, s.first, s.end, row);
        if (threadIdx.x >= kWave) return;
        run.template rule<M>(lds, from_history, q, from, (int)(begin - s.first));
        const int at = run.pick(f.rest, f.at.m, h.k, &value);
        token = at < 0 ? -1 : s.first + at;
    }
    if (threadIdx.x == 0) store_choice(c, r, h, token, value, f);
}

// ---- launches --------------------------------------------------------------------------------------------------------------------

template <typename E, int WIDTH, int R, typename COUNT, bool STREAM, int VEC = 16 / sizeof(E)>
int launch_rule_slices(const void* in, const void* times, void* out, const RuleArgs& a, int64_t rows, int64_t J, hipStream_t stream) {
    constexpr int kSlice = WIDTH * VEC * R;
    const int slices = (int)((J + kSlice - 1) / kSlice);
    {
        KernelTimerScope timer_(std::is_void<COUNT>::value ? "rule_times_backward" : "rule_times", stream);
        hipLaunchKernelGGL((rule_kernel<E, VEC, WIDTH, R, COUNT, STREAM>), wide_grid(rows * slices, WIDTH), dim3(WIDTH), 0, stream,
                           static_cast<const E*>(in), static_cast<const E*>(times), static_cast<E*>(out), a, rows, (int)J, slices);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

// Slices of 4096 elements, four wavefronts each, and of 2048 by one in rows of up to 8192 elements (a border between the two lengths that were measured).
// Rows with their gradient:
//     slices                        2048, 1 wavefront   4096, 4   8192, 4   8192, 8
//     2328 rows of 5003 f16 times         29.1 us         35.3
//     4096 rows of 32000 bf16 times      230             219       224       218
template <typename COUNT>
int launch_rules(const void* in, const void* times, int type, const RuleArgs& a, void* out, int64_t rows, int64_t J, hipStream_t stream) {
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        constexpr int VEC = 16 / sizeof(E);
        if (J < VEC) return launch_rule_slices<E, 64, 1, COUNT, false, 1>(in, times, out, a, rows, J, stream);
        if (J <= 64 * VEC) return launch_rule_slices<E, 64, 1, COUNT, false>(in, times, out, a, rows, J, stream);
        if (J <= 8192) return launch_rule_slices<E, 64, 32 / VEC, COUNT, false>(in, times, out, a, rows, J, stream);
        // (4096 rows of 32000 bf16 times with their gradient: 235 us through the caches, 220 past them)
        if (2 * rows * J * (int64_t)sizeof(E) > kStreamBytes) return launch_rule_slices<E, 256, 16 / VEC, COUNT, true>(in, times, out, a, rows, J, stream);
        return launch_rule_slices<E, 256, 16 / VEC, COUNT, false>(in, times, out, a, rows, J, stream);
    });
}

template <typename E, int WIDTH, int R, typename COUNT, int VEC = 16 / sizeof(E)>
int launch_choose_whole(const void* times, const RuleArgs& a, const ChooseArgs& c, int64_t rows, int64_t J, hipStream_t stream) {
    {
        KernelTimerScope timer_("choose", stream);
        hipLaunchKernelGGL((choose_slice_kernel<E, VEC, WIDTH, R, COUNT, true>), wide_grid(rows, WIDTH), dim3(WIDTH), 0, stream,
                           static_cast<const E*>(times), a, c, nullptr, rows, (int)J, 1);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

template <typename E, int WIDTH, int R, typename COUNT>
int launch_choose_slices(const void* times, const RuleArgs& a, const ChooseArgs& c, int64_t rows, int64_t J, Part* parts, hipStream_t stream) {
    constexpr int VEC = 16 / sizeof(E), kSlice = WIDTH * VEC * R, kWaves = WIDTH / kWave;
    const int slices = (int)((J + kSlice - 1) / kSlice);
    {
        KernelTimerScope timer_("choose_slice", stream);
        hipLaunchKernelGGL((choose_slice_kernel<E, VEC, WIDTH, R, COUNT, false>), wide_grid(rows * slices, WIDTH), dim3(WIDTH), 0, stream,
                           static_cast<const E*>(times), a, c, parts, rows, (int)J, slices);
    }
    {
        KernelTimerScope timer_("choose_join", stream);
        // (a call on 4096 rows of 32000: 89 us with a wavefront for each, 93 with four; on 64 of 131072 with 2048 tokens: 23.2 and 20.4; the border,
        // a row for each CU, lies between them)
        if (rows >= 256)
            hipLaunchKernelGGL((choose_join_kernel<E, VEC, R, COUNT, 64>), wide_grid(rows, 64), dim3(64), 0, stream,
                               static_cast<const E*>(times), a, c, parts, rows, (int)J, slices * kWaves);
        else
            hipLaunchKernelGGL((choose_join_kernel<E, VEC, R, COUNT, 256>), wide_grid(rows, 256), dim3(256), 0, stream,
                               static_cast<const E*>(times), a, c, parts, rows, (int)J, slices * kWaves);
    }
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

// Occurrences are counted in 16 bits where no token can have more.
bool narrow(const RuleArgs& a) { return !a.history || a.L < (1 << 16); }

}  // namespace

// Every wavefront of a row's slices leaves a part; the shortest slices are of 4096 elements and four wavefronts.
size_t choose_workspace(int64_t rows, int64_t J) { return J > 4096 ? align_up((size_t)rows * (size_t)((J + 4095) / 4096 * 4) * sizeof(Part)) : 0; }

int launch_rule_times(const void* times, int type, const RuleArgs& a, void* out, int64_t rows, int64_t J, hipStream_t stream) {
    return narrow(a) ? launch_rules<unsigned short>(times, nullptr, type, a, out, rows, J, stream)
                     : launch_rules<unsigned>(times, nullptr, type, a, out, rows, J, stream);
}

int launch_rule_times_backward(const void* grad, const void* times, int type, const RuleArgs& a, void* dtimes, int64_t rows, int64_t J,
                               hipStream_t stream) {
    return launch_rules<void>(grad, times, type, a, dtimes, rows, J, stream);
}

int launch_choose(const void* times, int type, const RuleArgs& a, const ChooseArgs& c, int64_t rows, int64_t J, void* ws, hipStream_t stream) {
    Part* parts = static_cast<Part*>(ws);
    return with_type(type, [&](auto e) -> int {
        using E = decltype(e);
        constexpr int VEC = 16 / sizeof(E), R = 32 / VEC;
        if (!narrow(a)) {
            if (J < VEC) return launch_choose_whole<E, 64, 1, unsigned, 1>(times, a, c, rows, J, stream);
            if (J <= 256 * 16) return launch_choose_whole<E, 256, R / 2, unsigned>(times, a, c, rows, J, stream);
            return launch_choose_slices<E, 256, R / 2, unsigned>(times, a, c, rows, J, parts, stream);
        }
        using C = unsigned short;
        if (J < VEC) return launch_choose_whole<E, 64, 1, C, 1>(times, a, c, rows, J, stream);
        if (J <= 64 * VEC) return launch_choose_whole<E, 64, 1, C>(times, a, c, rows, J, stream);
        if (J <= 64 * 32) return launch_choose_whole<E, 64, R, C>(times, a, c, rows, J, stream);
        if (J <= 256 * 32) return launch_choose_whole<E, 256, R, C>(times, a, c, rows, J, stream);
        // One launch of a workgroup for each row, or shorter workgroups that overlap better where there are many.  Of bf16 times, in us:
        //     rows         256 of 10000   256 of 32000   512 of 10000   512 of 32000   1024 of 32000   4096 of 32000
        //     one launch        11.2           12.2           19.8           20.8            36.7           138
        //     slices            14.4           17.1           17.2           22.2            31.7            89
        if (J <= 1024 * 32 && (rows <= 256 || (rows <= 512 && J > 1024 * 16)))
            return launch_choose_whole<E, 1024, R, C>(times, a, c, rows, J, stream);
        if (J <= 1024 * 32) return launch_choose_slices<E, 512, R, C>(times, a, c, rows, J, parts, stream);
        return launch_choose_slices<E, 256, R, C>(times, a, c, rows, J, parts, stream);
    });
}

}  // namespace snntc
