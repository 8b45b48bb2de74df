// Spike times of tokens, and the gradient of their table.
//     z[n,:] = scale E[tok_n,:]   or, encoded like an image's intensities, exp(1 - scale E[tok_n,:])
//     dE[v,:] = k_v sum over the n with tok_n = v of g[n,:],   k_v = scale, or -scale exp(1 - scale E[v,:])
// The gradient is a sum of rows by token.  Atomic adds would make its last digits depend on the order in which workgroups run;
// here the tokens are sorted first (by token, then by position), and the rows are added in that order.
#include <algorithm>

#include "sequences.h"

namespace snntc {
namespace {

constexpr int kCols = 4;                            // columns of a lane
constexpr int kSlice = kCols * kWave;               // columns of a wavefront

// Column q of a lane: four neighbours (VEC: one access for all of them) or one of every 64.
template <bool VEC>
__device__ __forceinline__ int column(int slice, int lane, int q) { return slice * kSlice + (VEC ? lane * kCols + q : q * kWave + lane); }

template <typename E>
struct alignas(kCols * sizeof(E)) Four { E v[kCols]; };

// STREAM: past the caches, for more than they hold.
template <typename E, bool VEC, bool STREAM = false>
__device__ __forceinline__ void load_cols(const E* row, int slice, int lane, int D, float (&v)[kCols]) {
    if (VEC) {
        const int d = column<true>(slice, lane, 0);
        typedef E Words __attribute__((ext_vector_type(kCols)));
        Words f{};
        if (d < D) f = STREAM ? __builtin_nontemporal_load(reinterpret_cast<const Words*>(row + d)) : *reinterpret_cast<const Words*>(row + d);
#pragma unroll
        for (int q = 0; q < kCols; ++q) v[q] = (float)f[q];
    } else {
#pragma unroll
        for (int q = 0; q < kCols; ++q) {
            const int d = column<false>(slice, lane, q);
            v[q] = d >= D ? 0.0f : STREAM ? (float)__builtin_nontemporal_load(row + d) : (float)row[d];
        }
    }
}

// The same as they stand in memory.
template <typename E>
struct Raw { E v[kCols]; };
template <typename E, bool VEC>
__device__ __forceinline__ Raw<E> load_raw(const E* row, int slice, int lane, int D) {
    Raw<E> r{};
    if (VEC) {
        const int d = column<true>(slice, lane, 0);
        Four<E> f{};
        if (d < D) f = *reinterpret_cast<const Four<E>*>(row + d);
#pragma unroll
        for (int q = 0; q < kCols; ++q) r.v[q] = f.v[q];
    } else {
#pragma unroll
        for (int q = 0; q < kCols; ++q) {
            const int d = column<false>(slice, lane, q);
            if (d < D) r.v[q] = row[d];
        }
    }
    return r;
}

template <typename E, bool VEC, bool STREAM = false>
__device__ __forceinline__ void store_cols(E* row, int slice, int lane, int D, const float (&v)[kCols]) {
    if (VEC) {
        const int d = column<true>(slice, lane, 0);
        typedef E Words __attribute__((ext_vector_type(kCols)));
        Words f;
#pragma unroll
        for (int q = 0; q < kCols; ++q) f[q] = (E)v[q];
        if (d < D) {
            if (STREAM) __builtin_nontemporal_store(f, reinterpret_cast<Words*>(row + d));
            else *reinterpret_cast<Words*>(row + d) = f;
        }
    } else {
#pragma unroll
        for (int q = 0; q < kCols; ++q) {
            const int d = column<false>(slice, lane, q);
            if (d < D) row[d] = (E)v[q];
        }
    }
}

// Whether rows of D elements from p on can be accessed four elements at a time.
inline bool fours(const void* p, int64_t D, size_t element) { return D % kCols == 0 && (uintptr_t)p % (kCols * element) == 0; }

// ---- forward -------------------------------------------------------------------------------------

__device__ __forceinline__ float time_of(float e, float scale, bool encode) {
    return encode ? exp_close(1.0f - scale * e) : scale * e;
}

// A wavefront owns 256 columns of TOKENS consecutive tokens and requests their rows together.  Bound by memory: 131072 tokens of 1024
// columns from a 16-bit table 95 us, 6.9 TB/s; 8192 of 800 from float32 9.0 us, 4.5 TB/s.
template <typename E, typename I, bool VEC, int TOKENS, bool STREAM>
__global__ void __launch_bounds__(256)
embed_forward_kernel(const I* __restrict__ tokens, const E* __restrict__ table, float* __restrict__ z, int N, int V, int D, int slices,
                     int64_t units, float scale, bool encode) {
    const int64_t unit = workgroup() * (256 / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (unit >= units) return;
    const int64_t n0 = unit / slices * TOKENS;
    const int slice = (int)(unit % slices), lane = threadIdx.x % kWave;
    float v[TOKENS][kCols];
    bool known[TOKENS];
#pragma unroll
    for (int k = 0; k < TOKENS; ++k) {
        const long long tok = tokens[min(n0 + k, (int64_t)N - 1)];
        known[k] = tok >= 0 && tok < V;
        load_cols<E, VEC>(table + (size_t)(known[k] ? tok : 0) * D, slice, lane, D, v[k]);
    }
#pragma unroll
    for (int k = 0; k < TOKENS; ++k) {
        if (n0 + k >= N) return;
#pragma unroll
        for (int q = 0; q < kCols; ++q) v[k][q] = known[k] ? time_of(v[k][q], scale, encode) : NAN;
        store_cols<float, VEC, STREAM>(z + (size_t)(n0 + k) * D, slice, lane, D, v[k]);
    }
}

// ---- gradient ------------------------------------------------------------------------------------
//
// 1. The positions are put in the order (token, position).  Up to kRankMost of them by counting, for each, those that come
//    before it: N^2 compares spread over the whole chip in one launch, 64 in one instruction and a scalar count of its mask,
//    where a sort that works by passes is several launches.  8192 positions take 11 us, 16384 33 us.  More go by stable radix
//    passes of at most nine bits, two launches each: 16384 positions 24 us.  The same first launch clears dtable (at 6 TB/s): rows of
//    tokens that do not occur stay like that.
// 2. The sorted positions are cut into chunks of equal length, whatever the tokens' frequencies are; a wavefront owns a chunk and
//    256 columns.  It adds up the rows of each token in order; a token that lies wholly in the chunk is finished there, the
//    first and last one may reach beyond it and leave partial sums.  131072 rows of 1024: 624 MB in 124 us, 5.0 TB/s.
// 3. Partial sums of one token are added in the order of their chunks.

constexpr int kRankThreads = 1024;
constexpr int kRankWaves = kRankThreads / kWave;
constexpr int kRankOwn = 32;                        // positions a workgroup ranks
constexpr int kRankMost = 12 * kRankThreads;

// Positions whose token lies outside the table count as token V and end up last.
template <typename I>
__device__ __forceinline__ int token_key(const I* tokens, int i, int V) {
    const long long t = tokens[i];
    return t >= 0 && t < V ? (int)t : V;
}

// What clears a tensor: workgroups from first_block on, 16 bytes a thread and step; the bytes before the first 16-byte boundary and
// behind the last one by themselves.
struct ClearArgs {
    char* p;
    int64_t bytes;
    int first_block;
    __device__ __forceinline__ bool mine() const { return (int)blockIdx.x >= first_block; }
    __device__ __forceinline__ void run() const {
        const int64_t block = blockIdx.x - first_block, blocks = gridDim.x - first_block;
        const int64_t lead = min(bytes, (int64_t)(-(uintptr_t)p & 15)), n16 = (bytes - lead) / 16, tail = lead + n16 * 16;
        uint4* q = reinterpret_cast<uint4*>(p + lead);
        for (int64_t e = block * blockDim.x + threadIdx.x; e < n16; e += blocks * blockDim.x) q[e] = uint4{0, 0, 0, 0};
        if (block == 0 && (int64_t)threadIdx.x < lead) p[threadIdx.x] = 0;
        if (block == 0 && tail + threadIdx.x < bytes) p[tail + threadIdx.x] = 0;
    }
};
// A wavefront holds R x 64 tokens, the workgroup all of them; each of its kRankOwn positions is compared with all.  Equal tokens
// count where their position is lower: a token before the owned positions is held as 2 token, one behind them as 2 token + 1, and
// both count where they lie below 2 own + 1.  The owned ones among themselves are counted apart.
template <typename I, int R>
__global__ void __launch_bounds__(kRankThreads)
token_rank_kernel(const I* __restrict__ tokens, int* __restrict__ sorted_token, int* __restrict__ sorted_pos, int N, int V, ClearArgs clear) {
    if (clear.mine()) { clear.run(); return; }
    __shared__ int part[kRankWaves][kRankOwn];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n0 = blockIdx.x * kRankOwn;
    const int loaded = token_key(tokens, min(n0 + lane % kRankOwn, N - 1), V);
    const int own = n0 + lane % kRankOwn < N ? loaded : V;               // (places behind the last position count as behind everything)
    unsigned held[R];
#pragma unroll
    for (int r = 0; r < R; ++r) held[r] = token_key(tokens, min((wave * R + r) * kWave + lane, N - 1), V);      // all requested together
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = (wave * R + r) * kWave + lane;
        held[r] = i >= N || (i >= n0 && i < n0 + kRankOwn) ? ~0u : 2u * held[r] + (i >= n0);
    }
    int before = 0;
#pragma unroll 4
    for (int k = 0; k < kRankOwn; ++k) {
        const unsigned bound = 2u * (unsigned)__builtin_amdgcn_readlane(own, k) + 1u;
        int count = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) count += __popcll(__ballot(held[r] < bound));
        before = lane == k ? count : before;
    }
    if (lane < kRankOwn) part[wave][lane] = before;
    __syncthreads();
    if (wave == 0) {
        int rank = 0;
#pragma unroll
        for (int w = 0; w < kRankWaves; ++w) rank += part[w][lane % kRankOwn];
        for (int k = 0; k < kRankOwn; ++k) {
            const int other = __builtin_amdgcn_readlane(own, k);
            rank += other < own || (other == own && k < lane);
        }
        if (lane < kRankOwn && n0 + lane < N) {
            sorted_token[rank] = own;
            sorted_pos[rank] = n0 + lane;
        }
    }
}

// One pass of the radix sort: digits of `bits` bits from bit `shift` on.  A workgroup owns `chunk` consecutive entries; counts[g][d]
// is how often digit d occurs in chunk g.  The first pass reads tokens (and positions are its indices), later ones key and pos.
constexpr int kRadixThreads = 1024;
constexpr int kRadixWaves = kRadixThreads / kWave;
constexpr int kRadixBits = 9;
constexpr int kRadixChunk = 2048, kRadixChunks = 256;

template <typename I, bool FIRST>
__device__ __forceinline__ int entry_key(const I* tokens, const int* key, int i, int V) {
    return FIRST ? token_key(tokens, i, V) : key[i];
}

template <typename I, bool FIRST>
__global__ void __launch_bounds__(kRadixThreads)
radix_count_kernel(const I* __restrict__ tokens, const int* __restrict__ key, int* __restrict__ counts, int N, int V, int shift, int bits,
                   int chunk, ClearArgs clear) {
    if (clear.mine()) { clear.run(); return; }
    __shared__ int hist[1 << kRadixBits];
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += kRadixThreads) hist[d] = 0;
    __syncthreads();
    const int64_t i0 = (int64_t)blockIdx.x * chunk;
    const int i1 = (int)min((int64_t)N, i0 + chunk);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += kRadixThreads)
        atomicAdd(&hist[(entry_key<I, FIRST>(tokens, key, (int)i, V) >> shift) & (bins - 1)], 1);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kRadixThreads) counts[(size_t)blockIdx.x * bins + d] = hist[d];
}

// What the lanes of a wavefront have read and written in LDS before comes before what they do after.
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename I, bool FIRST>
__global__ void __launch_bounds__(kRadixThreads)
radix_place_kernel(const I* __restrict__ tokens, const int* __restrict__ key, const int* __restrict__ pos, const int* __restrict__ counts,
                   int* __restrict__ out_key, int* __restrict__ out_pos, int N, int V, int shift, int bits, int chunk, int chunks) {
    __shared__ int total[1 << kRadixBits], start[1 << kRadixBits], seen[kRadixWaves][1 << kRadixBits], wave_sum[kRadixWaves];
    const int bins = 1 << bits, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int g = blockIdx.x;
    // where digit d of this chunk begins: all lower digits, and the same digit in earlier chunks; a digit's counts are read by
    // several threads, each of which requests sixteen chunks together
    for (int d = threadIdx.x; d < bins; d += kRadixThreads) total[d] = start[d] = 0;
    for (int e = threadIdx.x; e < (kRadixWaves << bits); e += kRadixThreads) seen[e >> bits][e & (bins - 1)] = 0;
    __syncthreads();
    {
        const int d = threadIdx.x & (bins - 1), parts = kRadixThreads >> bits;
        int all = 0, earlier = 0;
#pragma unroll 16
        for (int h = threadIdx.x >> bits; h < chunks; h += parts) {
            const int c = counts[((size_t)h << bits) + d];
            all += c;
            earlier += h < g ? c : 0;
        }
        atomicAdd(&total[d], all);
        atomicAdd(&start[d], earlier);
    }
    __syncthreads();
    const int own = (int)threadIdx.x < bins ? total[threadIdx.x] : 0;
    int upto = own;
#pragma unroll
    for (int s = 1; s < kWave; s <<= 1) {
        const int v = __shfl_up(upto, s, kWave);
        if (lane >= s) upto += v;
    }
    if (lane == kWave - 1) wave_sum[wave] = upto;
    __syncthreads();
    if ((int)threadIdx.x < bins) {
        int base = upto - own;
        for (int w = 0; w < wave; ++w) base += wave_sum[w];
        start[threadIdx.x] += base;
    }
    // each wavefront takes a consecutive part of the chunk, 64 entries at a time: first to count its digits, then, knowing what the
    // wavefronts before it hold, to place them
    const int64_t w0 = (int64_t)g * chunk + (int64_t)wave * (chunk / kRadixWaves);
    const int64_t end = min((int64_t)N, w0 + chunk / kRadixWaves);
    auto same_digit = [&](int digit, bool there) {
        unsigned long long same = __ballot(there);
        for (int b = 0; b < bits; ++b) {
            const unsigned long long ones = __ballot((digit >> b) & 1);
            same &= (digit >> b) & 1 ? ones : ~ones;
        }
        return same;
    };
    for (int64_t i = w0; i < end; i += kWave) {
        const bool there = i + lane < end;
        const int digit = there ? (entry_key<I, FIRST>(tokens, key, (int)(i + lane), V) >> shift) & (bins - 1) : 0;
        if (there) atomicAdd(&seen[wave][digit], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kRadixThreads) {
        int at = start[d];
#pragma unroll
        for (int w = 0; w < kRadixWaves; ++w) {
            const int c = seen[w][d];
            seen[w][d] = at;
            at += c;
        }
    }
    __syncthreads();
    for (int64_t i = w0; i < end; i += kWave) {
        const bool there = i + lane < end;
        const int k = there ? entry_key<I, FIRST>(tokens, key, (int)(i + lane), V) : 0;
        const int digit = (k >> shift) & (bins - 1);
        const unsigned long long same = same_digit(digit, there);
        const int ahead = __popcll(same & ((1ull << lane) - 1));
        int at = 0;
        if (there) {
            at = seen[wave][digit] + ahead;
            out_key[at] = k;
            out_pos[at] = FIRST ? (int)(i + lane) : pos[i + lane];
        }
        // the last of equal digits moves the mark on, after all have read it and before they read again: one wavefront's LDS accesses are
        // done in order, and the barriers (no instructions) keep the compiler from changing it
        wave_order();
        if (there && (same >> lane) == 1) seen[wave][digit] = at + 1;
        wave_order();
    }
}

// ---- sums of rows

constexpr int kBatch = 8;                           // rows requested together

// The sum s of a table row's gradients becomes the row's own; e: the row's elements, needed where they are encoded.
__device__ __forceinline__ void finish_row(float scale, bool encode, const float (&e)[kCols], float (&s)[kCols]) {
#pragma unroll
    for (int q = 0; q < kCols; ++q) s[q] *= encode ? -scale * exp_close(1.0f - scale * e[q]) : scale;
}
template <typename E, bool VEC>
__device__ __forceinline__ void store_row(E* dtable, const E* table, int v, int slice, int lane, int D, float scale, bool encode,
                                          float (&s)[kCols]) {
    float e[kCols] = {};
    if (encode) load_cols<E, VEC>(table + (size_t)v * D, slice, lane, D, e);
    finish_row(scale, encode, e, s);
    store_cols<E, VEC>(dtable + (size_t)v * D, slice, lane, D, s);
}

// partial[chunk][0]: what a chunk adds to the token that began before it; [1]: the token that begins in it and goes on behind it.
template <typename E, bool VEC, bool STREAM>
__global__ void __launch_bounds__(256)
embed_sums_kernel(const float* __restrict__ grad, const int* __restrict__ sorted_token, const int* __restrict__ sorted_pos,
                  const E* __restrict__ table, E* __restrict__ dtable, float* __restrict__ partial, int N, int V, int D, int chunk,
                  int slices, int64_t units, float scale, bool encode) {
    const int64_t unit = (int64_t)blockIdx.x * (256 / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (unit >= units) return;
    const int c = (int)(unit / slices), slice = (int)(unit % slices), lane = threadIdx.x % kWave;
    const int i0 = c * chunk, i1 = min(N, i0 + chunk);                   // (N is at most 2^30)
    float s[kCols] = {0.0f, 0.0f, 0.0f, 0.0f};
    bool head = i0 > 0 && sorted_token[i0 - 1] == sorted_token[i0];      // the first token began before
    int tok = V;
    for (int g = i0; g < i1; g += kWave) {
        // 64 entries at a time: lane k holds the token and the row of entry g + k, and whether the token ends there
        const int here = min(kWave, i1 - g), at = min(g + lane, i1 - 1);
        const int token = sorted_token[at], row = sorted_pos[at], follows = at + 1 < N ? sorted_token[at + 1] : V;
        const unsigned long long ends = __ballot(token != follows), known = __ballot(lane < here && token < V);
        const int rows = __popcll(known);                                // (tokens outside the table come last)
        float next[kBatch][kCols];
        auto request = [&](int k0) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
                load_cols<float, VEC, STREAM>(grad + (size_t)__builtin_amdgcn_readlane(row, min(k0 + k, kWave - 1)) * D, slice, lane, D, next[k]);
        };
        if (rows > 0) request(0);
        for (int k0 = 0; k0 < rows; k0 += kBatch) {
            float v[kBatch][kCols];
            Raw<E> e[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
#pragma unroll
                for (int q = 0; q < kCols; ++q) v[k][q] = next[k][q];
            // the table's rows of the tokens that end in this batch, together: one by one, each would cost a trip to memory
            if (encode) {
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if (k0 + k < rows && (ends >> (k0 + k)) & 1)
                        e[k] = load_raw<E, VEC>(table + (size_t)__builtin_amdgcn_readlane(token, k0 + k) * D, slice, lane, D);
            }
            if (k0 + kBatch < rows) request(k0 + kBatch);
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
                if (k0 + k >= rows) break;
#pragma unroll
                for (int q = 0; q < kCols; ++q) s[q] += v[k][q];
                tok = __builtin_amdgcn_readlane(token, k0 + k);
                if ((ends >> (k0 + k)) & 1) {                            // (uniform)
                    if (head) store_cols<float, VEC>(partial + (size_t)c * 2 * D, slice, lane, D, s);
                    else {
                        float row_of[kCols];
#pragma unroll
                        for (int q = 0; q < kCols; ++q) row_of[q] = (float)e[k].v[q];
                        finish_row(scale, encode, row_of, s);
                        store_cols<E, VEC>(dtable + (size_t)tok * D, slice, lane, D, s);
                    }
                    head = false;
                    tok = V;
#pragma unroll
                    for (int q = 0; q < kCols; ++q) s[q] = 0.0f;
                }
            }
        }
        if (rows < here) return;
    }
    if (tok < V)                                                         // it goes on behind this chunk
        store_cols<float, VEC>(partial + ((size_t)c * 2 + (head ? 0 : 1)) * D, slice, lane, D, s);
}

// A workgroup joins the token that begins in chunk c and goes on behind it, if there is one.  Its sixteen wavefronts share the
// slices of 256 columns, and where those are fewer the chunks of a slice, each a consecutive part; the parts are added in order.
constexpr int kJoinWaves = 16;
template <typename E, bool VEC>
__global__ void __launch_bounds__(kJoinWaves * kWave)
embed_join_kernel(const float* __restrict__ partial, const int* __restrict__ sorted_token, const E* __restrict__ table, E* __restrict__ dtable,
                  int N, int V, int D, int chunk, int chunks, int slices, float scale, bool encode) {
    __shared__ float part[kJoinWaves][kCols][kWave];
    const int c = blockIdx.x, lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t i0 = (int64_t)c * chunk, i1 = i0 + chunk;
    const int tok = sorted_token[i1], ends = sorted_token[i1 - 1], before = sorted_token[i0 > 0 ? i0 - 1 : 0];
    if (tok >= V || ends != tok) return;                                 // nothing goes on behind this chunk
    if (i0 > 0 && before == tok) return;                                 // it began earlier
    int last = c + 1;                                                    // the last chunk that begins with this token
    while (last + 1 < chunks) {
        const int at = last + 1 + lane;
        const unsigned long long more = __ballot(at < chunks && sorted_token[(int64_t)min(at, chunks - 1) * chunk] == tok);
        const int run = more == ~0ull ? kWave : __ffsll((long long)~more) - 1;
        last += run;
        if (run < kWave) break;
    }
    const int rows = last - c + 1;                                       // partial sums: the begun one, then one a chunk
    int parts = 1;
    while (parts * 2 * slices <= kJoinWaves) parts *= 2;
    const int together = kJoinWaves / parts;                             // slices at a time
    const int per = (rows + parts - 1) / parts, p = wave / together, r0 = min(rows, p * per), r1 = min(rows, r0 + per);
    for (int first = 0; first < slices; first += together) {
        const int slice = first + wave % together;
        float s[kCols] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (slice < slices) {
#pragma unroll 8
            for (int r = r0; r < r1; ++r) {
                float v[kCols];
                load_cols<float, VEC>(partial + ((size_t)(c + r) * 2 + (r == 0)) * D, slice, lane, D, v);
#pragma unroll
                for (int q = 0; q < kCols; ++q) s[q] += v[q];
            }
        }
#pragma unroll
        for (int q = 0; q < kCols; ++q) part[wave][q][lane] = s[q];
        __syncthreads();
        if (p == 0 && slice < slices) {
            for (int other = 1; other < parts && other * per < rows; ++other)
#pragma unroll
                for (int q = 0; q < kCols; ++q) s[q] += part[other * together + wave][q][lane];
            store_row<E, VEC>(dtable, table, tok, slice, lane, D, scale, encode, s);
        }
        __syncthreads();
    }
}

// Few positions: no order has to be made, and one launch does it all.  Every wavefront holds all tokens (lane k: positions k, k + 64, ...)
// and walks over its share of the table's rows: a compare gives the mask of a row's positions, an empty one clears it, else they
// are added from the lowest on.  (100 rows of 958 columns, 33 positions: 8 us where sorting, adding and joining take 14.)
constexpr int kFewHeld = 4, kFew = kFewHeld * kWave;
template <typename E, typename I, bool VEC>
__global__ void __launch_bounds__(256)
embed_few_kernel(const float* __restrict__ grad, const I* __restrict__ tokens, const E* __restrict__ table, E* __restrict__ dtable, int N, int V,
                 int D, int rows, int slices, int64_t units, float scale, bool encode) {
    const int64_t unit = (int64_t)blockIdx.x * (256 / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (unit >= units) return;
    const int slice = (int)(unit % slices), lane = threadIdx.x % kWave;
    const int64_t v0 = unit / slices * rows, v1 = min((int64_t)V, v0 + rows);
    int held[kFewHeld];
#pragma unroll
    for (int h = 0; h < kFewHeld; ++h) held[h] = N > 0 ? token_key(tokens, min(h * kWave + lane, N - 1), V) : V;      // (requested together)
#pragma unroll
    for (int h = 0; h < kFewHeld; ++h) held[h] = h * kWave + lane < N ? held[h] : V;
    for (int64_t v = v0; v < v1; ++v) {
        unsigned long long here[kFewHeld], any = 0;
#pragma unroll
        for (int h = 0; h < kFewHeld; ++h) any |= here[h] = __ballot(held[h] == (int)v);
        float s[kCols] = {0.0f, 0.0f, 0.0f, 0.0f}, e[kCols] = {};
        if (any) {
            if (encode) load_cols<E, VEC>(table + (size_t)v * D, slice, lane, D, e);
#pragma unroll
            for (int h = 0; h < kFewHeld; ++h) {
                unsigned long long mask = here[h];
                while (mask) {
                    float r[kBatch][kCols];
                    const int count = min(kBatch, __popcll(mask));
#pragma unroll
                    for (int k = 0; k < kBatch; ++k)
                        if (k < count) {
                            load_cols<float, VEC>(grad + (size_t)(h * kWave + __ffsll((long long)mask) - 1) * D, slice, lane, D, r[k]);
                            mask &= mask - 1;
                        }
#pragma unroll
                    for (int k = 0; k < kBatch; ++k)
                        if (k < count)
#pragma unroll
                            for (int q = 0; q < kCols; ++q) s[q] += r[k][q];
                }
            }
            finish_row(scale, encode, e, s);
        }
        store_cols<E, VEC>(dtable + (size_t)v * D, slice, lane, D, s);
    }
}

// How the sorted positions are cut: chunks long enough that few tokens are cut, short enough that some 4096 wavefronts are at work; at the
// least 16 rows, or 8 where that leaves most SIMDs without one (1000 x 233: 22 / 18 us, 8192 x 800: 30 / 33 us).
struct SumPlan { int chunk, chunks, slices; };
SumPlan sum_plan(int64_t N, int64_t D) {
    SumPlan p;
    p.slices = (int)((D + kSlice - 1) / kSlice);
    int64_t chunk = N * p.slices / 4096;
    chunk = (chunk + kBatch - 1) / kBatch * kBatch;
    const int64_t least = N * p.slices <= 8192 ? 8 : 16;
    chunk = chunk < least ? least : chunk > 256 ? 256 : chunk;
    p.chunk = (int)chunk;
    p.chunks = (int)((N + chunk - 1) / chunk);
    return p;
}

struct RadixPlan { int passes, bits, chunk, chunks; };
RadixPlan radix_plan(int64_t N, int64_t V) {
    RadixPlan p;
    int bits = 1;
    while (bits < 32 && (V >> bits) > 0) ++bits;                         // of keys 0 .. V
    p.passes = (bits + kRadixBits - 1) / kRadixBits;
    p.bits = (bits + p.passes - 1) / p.passes;
    int64_t chunk = (N + kRadixChunks - 1) / kRadixChunks;
    chunk = (chunk + kRadixThreads - 1) / kRadixThreads * kRadixThreads;
    p.chunk = (int)(chunk < kRadixChunk ? kRadixChunk : chunk);
    p.chunks = (int)((N + p.chunk - 1) / p.chunk);
    return p;
}

struct SortWs {
    int *token, *pos, *other_token, *other_pos, *counts;
    float* partial;
    size_t bytes;
    SortWs(void* ws, int64_t N, int64_t V, int64_t D) {
        char* base = static_cast<char*>(ws);
        size_t used = 0;
        auto take = [&](size_t b) { char* p = base + used; used += align_up(b); return p; };
        token = reinterpret_cast<int*>(take(N * sizeof(int)));
        pos = reinterpret_cast<int*>(take(N * sizeof(int)));
        const SumPlan s = sum_plan(N, D);
        partial = reinterpret_cast<float*>(take((size_t)s.chunks * 2 * D * sizeof(float)));
        other_token = other_pos = counts = nullptr;
        if (N > kRankMost) {
            const RadixPlan r = radix_plan(N, V);
            other_token = reinterpret_cast<int*>(take(N * sizeof(int)));
            other_pos = reinterpret_cast<int*>(take(N * sizeof(int)));
            counts = reinterpret_cast<int*>(take((size_t)r.chunks * (1 << r.bits) * sizeof(int)));
        }
        bytes = used;
    }
};

template <typename I>
int sort_tokens(const I* tokens, const SortWs& w, int64_t N, int64_t V, void* dtable, int64_t table_bytes, hipStream_t stream) {
    // workgroups that clear: 16 KiB a workgroup and step, up to four a CU
    const int64_t clear_blocks = std::max<int64_t>(1, std::min<int64_t>(1024, table_bytes / (16 * 1024)));
    if (N <= kRankMost) {
        const int blocks = (int)((N + kRankOwn - 1) / kRankOwn);
        const dim3 grid((unsigned)(blocks + clear_blocks));
        const ClearArgs clear{static_cast<char*>(dtable), table_bytes, blocks};
        const int held = (int)((N + kRankThreads - 1) / kRankThreads);
        KernelTimerScope timer_("token_rank", stream);
        auto kern = held <= 1 ? token_rank_kernel<I, 1> : held <= 2 ? token_rank_kernel<I, 2> : held <= 4 ? token_rank_kernel<I, 4>
                    : held <= 8 ? token_rank_kernel<I, 8> : token_rank_kernel<I, 16>;
        hipLaunchKernelGGL(kern, grid, dim3(kRankThreads), 0, stream, tokens, w.token, w.pos, (int)N, (int)V, clear);
        SNNTC_HIP_CHECK(hipGetLastError());
        return SNNTC_OK;
    }
    const RadixPlan r = radix_plan(N, V);
    // the last pass ends in token / pos
    int *to_key = r.passes % 2 ? w.token : w.other_token, *to_pos = r.passes % 2 ? w.pos : w.other_pos;
    const int *key = nullptr, *pos = nullptr;
    for (int pass = 0; pass < r.passes; ++pass) {
        const int shift = pass * r.bits;
        const ClearArgs clear{static_cast<char*>(dtable), table_bytes, r.chunks};
        {
            KernelTimerScope timer_("radix_count", stream);
            if (pass == 0)
                hipLaunchKernelGGL((radix_count_kernel<I, true>), dim3((unsigned)(r.chunks + clear_blocks)), dim3(kRadixThreads), 0, stream,
                                   tokens, key, w.counts, (int)N, (int)V, shift, r.bits, r.chunk, clear);
            else
                hipLaunchKernelGGL((radix_count_kernel<I, false>), dim3((unsigned)r.chunks), dim3(kRadixThreads), 0, stream, tokens, key,
                                   w.counts, (int)N, (int)V, shift, r.bits, r.chunk, clear);
        }
        SNNTC_HIP_CHECK(hipGetLastError());
        {
            KernelTimerScope timer_("radix_place", stream);
            if (pass == 0)
                hipLaunchKernelGGL((radix_place_kernel<I, true>), dim3((unsigned)r.chunks), dim3(kRadixThreads), 0, stream, tokens, key, pos,
                                   w.counts, to_key, to_pos, (int)N, (int)V, shift, r.bits, r.chunk, r.chunks);
            else
                hipLaunchKernelGGL((radix_place_kernel<I, false>), dim3((unsigned)r.chunks), dim3(kRadixThreads), 0, stream, tokens, key, pos,
                                   w.counts, to_key, to_pos, (int)N, (int)V, shift, r.bits, r.chunk, r.chunks);
        }
        SNNTC_HIP_CHECK(hipGetLastError());
        key = to_key; pos = to_pos;
        to_key = key == w.token ? w.other_token : w.token;
        to_pos = pos == w.pos ? w.other_pos : w.pos;
    }
    return SNNTC_OK;
}

}  // namespace

// Whether times and the gradient that comes back for them are more than the caches hold (kStreamBytes): forward and gradient of N x 1024 from
// 32768 rows of 16 bits, us, through the caches / past them, N = 20000 81 / 83, 33000 127 / 109, 40000 142 / 119, 60000 203 / 159, 131072 366 / 275.
static bool beyond_caches(int64_t N, int64_t D) { return 2 * N * D * (int64_t)sizeof(float) > kStreamBytes; }

int launch_embed_forward(const void* tokens, int token_bytes, const void* table, int type, float* z, int64_t N, int64_t V, int64_t D,
                         float scale, bool encode, hipStream_t stream) {
    const int slices = (int)((D + kSlice - 1) / kSlice);
    // four rows in flight a wavefront once that still leaves every SIMD two of them, eight where they stream past the caches (131072 x
    // 1024 with the table thrown out of the caches by gradients 136 us with four, 127 with eight)
    const bool stream_out = beyond_caches(N, D);
    const bool vec = fours(table, D, type_bytes(type)) && fours(z, D, sizeof(float));
    const int each = vec && stream_out ? 8 : N * slices >= 8192 ? 4 : 1;
    const int64_t units = (N + each - 1) / each * slices, blocks = (units + 3) / 4;
    with_type(type, [&](auto e) {
        using E = decltype(e);
        KernelTimerScope timer_("embed_forward", stream);
        auto launch = [&](auto i) {
            using I = decltype(i);
            auto kern = !vec ? (each == 4 ? embed_forward_kernel<E, I, false, 4, false> : embed_forward_kernel<E, I, false, 1, false>)
                        : each == 8 ? embed_forward_kernel<E, I, true, 8, true>
                        : each == 4 ? embed_forward_kernel<E, I, true, 4, false> : embed_forward_kernel<E, I, true, 1, false>;
            hipLaunchKernelGGL(kern, wide_grid(blocks, 256), dim3(256), 0, stream, static_cast<const I*>(tokens),
                               static_cast<const E*>(table), z, (int)N, (int)V, (int)D, slices, units, scale, encode);
        };
        if (token_bytes == 8) launch(int64_t{});
        else launch(int32_t{});
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

size_t embed_backward_workspace(int64_t N, int64_t V, int64_t D) { return N > kFew ? SortWs(nullptr, N, V, D).bytes : 0; }

int launch_embed_backward(const float* grad, const void* tokens, int token_bytes, const void* table, int type, void* dtable, int64_t N,
                          int64_t V, int64_t D, float scale, bool encode, void* ws, hipStream_t stream) {
    const int64_t table_bytes = V * D * (int64_t)type_bytes(type);
    const size_t element = type_bytes(type);
    const bool vec = fours(grad, D, sizeof(float)) && fours(dtable, D, element) && (!encode || fours(table, D, element));
    if (N <= kFew) {
        // some 8192 wavefronts, each with up to 64 rows
        const int slices = (int)((D + kSlice - 1) / kSlice);
        const int rows = (int)std::max<int64_t>(1, std::min<int64_t>(64, V * slices / 8192));
        const int64_t units = (V + rows - 1) / rows * slices, blocks = (units + 3) / 4;
        if (blocks > (1 << 24) - 1) return fail(SNNTC_ERR_TOO_LARGE, "embed: too many table elements");
        with_type(type, [&](auto e) {
            using E = decltype(e);
            KernelTimerScope timer_("embed_few", stream);
            auto launch = [&](auto i) {
                using I = decltype(i);
                auto kern = vec ? embed_few_kernel<E, I, true> : embed_few_kernel<E, I, false>;
                hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, grad, static_cast<const I*>(tokens),
                                   static_cast<const E*>(table), static_cast<E*>(dtable), (int)N, (int)V, (int)D, rows, slices, units, scale,
                                   encode);
            };
            if (token_bytes == 8) launch(int64_t{});
            else launch(int32_t{});
            return 0;
        });
        SNNTC_HIP_CHECK(hipGetLastError());
        return SNNTC_OK;
    }
    const SumPlan p = sum_plan(N, D);
    const int64_t units = (int64_t)p.chunks * p.slices, blocks = (units + 3) / 4;
    if (blocks > (1 << 24) - 1) return fail(SNNTC_ERR_TOO_LARGE, "embed: too many rows of gradients");
    const SortWs w(ws, N, V, D);
    int rc = token_bytes == 8 ? sort_tokens(static_cast<const int64_t*>(tokens), w, N, V, dtable, table_bytes, stream)
                              : sort_tokens(static_cast<const int32_t*>(tokens), w, N, V, dtable, table_bytes, stream);
    if (rc) return rc;
    with_type(type, [&](auto e) {
        using E = decltype(e);
        {
            KernelTimerScope timer_("embed_sums", stream);
            const bool past = beyond_caches(N, D);                       // (131072 x 777 352 -> 306 us)
            auto kern = vec ? (past ? embed_sums_kernel<E, true, true> : embed_sums_kernel<E, true, false>)
                            : (past ? embed_sums_kernel<E, false, true> : embed_sums_kernel<E, false, false>);
            hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(256), 0, stream, grad, w.token, w.pos, static_cast<const E*>(table),
                               static_cast<E*>(dtable), w.partial, (int)N, (int)V, (int)D, p.chunk, p.slices, units, scale, encode);
        }
        if (p.chunks > 1) {
            KernelTimerScope timer_("embed_join", stream);
            auto kern = vec ? embed_join_kernel<E, true> : embed_join_kernel<E, false>;
            hipLaunchKernelGGL(kern, dim3((unsigned)(p.chunks - 1)), dim3(kJoinWaves * kWave), 0, stream, w.partial, w.token,
                               static_cast<const E*>(table), static_cast<E*>(dtable), (int)N, (int)V, (int)D, p.chunk, p.chunks, p.slices,
                               scale, encode);
        }
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

}  // namespace snntc
