// Gated running mean along a sequence, per channel:
//     a_t = sigmoid(gate_t),   h_t = a_t h_{t-1} + (1 - a_t) x_t,   y_t = h_t
// and its gradient, with u the gradient that reaches h_t:
//     u_t = dy_t + a_{t+1} u_{t+1}  (the last step of a sequence: dy_t + dfinal)
//     dx_t = (1 - a_t) u_t,   dgate_t = u_t (h_{t-1} - x_t) a_t (1 - a_t),   dstate = a_1 u_1
// A step mixes two spike times, so what comes out lies between those that went in and is a spike time itself.  That needs a and 1 - a
// to add up to one.  In float32 the half steps of each leave them off, by as much in every step alike where a gate stays, which the
// 1 / (1 - a) steps of the mean add up: a constant came back 0.05 % off at gates of 10, 0.2 % at 12.  Gates, the state along a sequence and the maps
// of its runs are therefore held in 64 bits, where they add up to one within 2^-46 (below: half a step of a result after 10^6 steps), and a
// result is rounded to 32 once.  (What that costs, forward + backward in us, 32 bits / 64:
// 32 x 256 x 800 14.4 + 26.1 / 15.7 + 26.2, 24 x 333 x 777 17.1 + 28.2 / 20.4 + 30.1, 16 x 6400 x 1024 200 + 430 / 201 + 429,
// 16 x 32768 x 16 56 + 78 / 71 + 90.)
#include <algorithm>

#include "sequences.h"

namespace snntc {
namespace {

// a = sigmoid(g) and 1 - a: with e = exp(-g), a = 1 / (1 + e) and 1 - a = e a, each to its own precision.  e is a float32 number, off by
// a step and a half at most, which moves both together; the reciprocal in 32 bits is off by a step, after a step of Newton's method in 64 by the
// square of that, 2^-46, and so is a + (1 - a) from one.  (Below -80, where 1 - a is 1 and a below 2e-35, e is held finite.  A NaN stays one.)
struct Gate {
    float e, near;                                  // near: a, off by a step
    __device__ __forceinline__ explicit Gate(float g) : e(exp_close(g < -80.0f ? 80.0f : -g)), near(__builtin_amdgcn_rcpf(1.0f + e)) {}
    __device__ __forceinline__ double a() const {
        const double whole = 1.0 + (double)e, r = (double)near;
        return fma(r, fma(-whole, r, 1.0), r);
    }
};

constexpr float kKeep = INFINITY;                   // the gate that leaves the state as it is: a = 1, 1 - a = 0

__device__ __forceinline__ int length_of(const int64_t* lengths, int64_t b, int64_t T) {
    if (!lengths) return (int)T;
    const int64_t n = lengths[b];
    return (int)(n < 0 ? 0 : n > T ? T : n);
}

// A workgroup owns W (64) neighbouring channels of a sequence and walks along it in tiles of kWaves x kSteps steps: each wavefront holds
// kSteps of them in registers (lane = channel).  A run of steps maps the state it is given to A h + H, so the wavefronts exchange
// (A, H) of their runs through LDS, every one composes those before its own, and goes through its steps a second time with the
// right start.  The next tile's loads are under way meanwhile; every value is read once and written once.  Bound by memory, and in short
// sequences by the instructions between two tiles' loads: 32 x 256 x 800 17.1 us forward and 28.5 backward, 4.6 and 5.5 TB/s; 32768 x 1024
// cut along time 40 + 57 and 38 + 104, 5.0 to 6.5 TB/s.
//
// Where that makes fewer than kFill workgroups, long sequences (more than kShort tiles) are also cut along time: a first kernel composes
// (A, H) of each part, and a workgroup starts from the composition of the parts before its own.  The order of composition depends on
// sizes alone.  Forward + backward in us, sequences whole / cut, 16-bit gates: 4096 steps, 16 groups of 64 channels 99 + 155 / 18 + 25,
// 192 groups 122 + 220 / 145 + 225.
// As few that are not cut become groups of 32 channels: each half of a wavefront has eight steps of its own, a tile twice as many.  Groups
// of 64 / 32, us: 4 x 256 x 1024 9 + 13 / 7 + 8, 32 x 200 x 200 9 + 13 / 7 + 9; 160 groups alike (10 x 256 x 1024 10 + 15 / 10 + 16),
// 32 x 256 x 800 14 + 23 / 17 + 33.  One workgroup of 32 channels a CU, or a little less (kMany groups of 64 and more), is not cut however
// long: cut / in groups of 32, us, 2048 steps, 128 groups 48 + 77 / 34 + 57, 96 groups 40 + 56 / 33 + 48, 80 groups 35 + 51 / 32 + 47, 144 groups
// 52 + 85 / 51 + 98; 8192 steps, 128 groups 194 + 293 / 147 + 308; 384 steps, 32 groups 11 + 12 / 8 + 11; 512 steps, 32 groups 12 + 12 / 10 + 13,
// 16 groups 12 + 12 / 10 + 13.
//
// Workgroups are dealt to the dies in turn.  Where neighbours share lines they go to one die, whose cache then holds those: where rows, those
// of the gates among them, are not whole lines (in turn / neighbours together, 24 x 333 x 777 22 + 36 / 19 + 29 us, 16 x 2530 x 777
// 94 + 180 / 82 + 152, 16 x 8434 x 777 313 + 612 / 269 + 507, 16 x 32768 x 200 464 + 827 / 416 + 712), and where 32 channels of 16-bit gates are
// half a line (8 x 1024 x 1024 21.4 + 32.8 / 20.2 + 30.2, 8 x 4096 x 1024 66 + 154 / 63 + 155, 2 x 8192 x 4096 146 + 294 / 143 + 287).  Else in turn:
// 32768 x 1024, cut, 110 + 152 / 111 + 157, others the same.
// Calls that touch more than the caches hold store past them, where rows are whole lines (the ends of a row that is none are stored by two groups
// that need not run at one time): through / past, 8 x 4096 x 1024 76 + 160 / 66 + 157, 16 x 1920 x 1024 61 + 132 / 52 + 125, 16 x 6400 x 1024 alike;
// 16 x 8434 x 777 269 + 507 / 291 + 586.  Half lines of 16-bit gates are among them, whose two halves neighbours on one die store together
// (through the caches 8 x 4096 x 1024 78 + 159, 2 x 2048 x 4096 35 + 75 for 35 + 57).
// Where sequences are cut, they load past them too, in the second and last reading (all through the caches / stores past / loads too,
// 16 x 102400 x 64 338 + 542 / 321 + 521 / 301 + 471, 16 x 30720 x 64 89 + 154 / 87 + 141 / 94 + 135, 32768 x 1024 101 + 170 / 98 + 159 / 109 + 152);
// whole ones gain less (16 x 6400 x 1024 202 + 421 / 195 + 414) or lose what a cache still holds for a call that follows (8 x 4096 x 1024, the
// gradient right after the forward pass, 211 / 243).
constexpr int kWaves = 8, kSteps = 8, kTile = kWaves * kSteps;
constexpr int kThreads = kWaves * kWave;
constexpr int kDies = 8;
constexpr int kFill = 160, kMany = 96, kUnits = 256, kShort = 6, kCutFill = 1024, kHalf = kWave / 2;

struct Map { double A, H; };                        // h -> A h + H
__device__ __forceinline__ Map then(const Map& first, const Map& second) { return Map{first.A * second.A, fma(second.A, first.H, second.H)}; }

struct Geometry {
    int B, T, D, groups, parts, part;               // groups of 64 (or 32) channels, parts of `part` steps (a multiple of kTile)
    bool half;                                      // groups of 32
    bool whole_lines;                               // rows are
    bool together;                                  // neighbouring groups share lines: they go to one die
};
// What goes past the caches.
enum Past { NONE, STORES, BOTH };
template <Past PAST, typename E>
__device__ __forceinline__ E get(const E* from) {
    if constexpr (PAST == BOTH) return __builtin_nontemporal_load(from);
    else return *from;
}
template <Past PAST, typename E>
__device__ __forceinline__ void put(E* to, E v) {
    if constexpr (PAST != NONE) __builtin_nontemporal_store(v, to);
    else *to = v;
}
struct Place {
    int64_t b;
    int d, s, lane, run;                            // run: the wavefront, or half of one where groups are 32 channels
    bool valid;                                     // lanes behind the last channel repeat it and store nothing
};
template <int W>
__device__ __forceinline__ Place place_of(const Geometry& g) {
    int block = blockIdx.x;
    if (g.together) {
        const int die = blockIdx.x % kDies, each = gridDim.x / kDies, more = gridDim.x % kDies;
        block = die * each + min(die, more) + blockIdx.x / kDies;
    }
    Place p;
    p.lane = threadIdx.x % W;
    p.run = W == kWave ? __builtin_amdgcn_readfirstlane(threadIdx.x / W) : threadIdx.x / W;
    const int rest = block / g.groups, d = block % g.groups * W + p.lane;
    p.valid = d < g.D;
    p.d = p.valid ? d : g.D - 1;
    p.s = rest % g.parts;
    p.b = rest / g.parts;
    return p;
}

// Composition of maps[w][lane] over the wavefronts, w ascending (or descending) from the state h: what comes in at wavefront `wave`
// and what goes out at the end.
template <bool DOWN, int W>
__device__ __forceinline__ double through(const Map (*maps)[W], const Place& p, double h, double* in) {
    constexpr int kRuns = kThreads / W;
#pragma unroll
    for (int k = 0; k < kRuns; ++k) {
        const int w = DOWN ? kRuns - 1 - k : k;
        if (w == p.run) *in = h;
        const Map m = maps[w][p.lane];
        h = fma(m.A, h, m.H);
    }
    return h;
}

// The state with which part s begins, from the maps of the parts on its way: each wavefront composes a consecutive share of them.
template <bool DOWN>
__device__ __forceinline__ double enter_part(const Map* parts, const Geometry& g, const Place& p, Map (*maps)[kWave], double h) {
    const int count = DOWN ? g.parts - 1 - p.s : p.s;
    if (count == 0) return h;
    const int first = DOWN ? p.s + 1 : 0, per = (count + kWaves - 1) / kWaves;
    const int r0 = min(count, p.run * per), r1 = min(count, r0 + per);
    Map m{1.0, 0.0};
#pragma unroll 8
    for (int r = r0; r < r1; ++r) {
        // ascending in time; going down, the later part acts first
        const Map next = parts[((size_t)p.b * g.parts + first + r) * g.D + p.d];
        m = DOWN ? then(next, m) : then(m, next);
    }
    maps[p.run][p.lane] = m;
    __syncthreads();
    double unused;
    h = through<DOWN, kWave>(maps, p, h, &unused);
    __syncthreads();
    return h;
}

template <typename G, Past PAST, int W>
__global__ void __launch_bounds__(kThreads)
gated_scan_forward_kernel(const float* __restrict__ x, const G* __restrict__ gate, const float* __restrict__ state,
                          const int64_t* __restrict__ lengths, float* __restrict__ y, float* __restrict__ final_state,
                          const Map* __restrict__ parts, Geometry g) {
    constexpr int kSpan = kThreads / W * kSteps;                         // steps of a tile
    __shared__ Map maps[2][kThreads / W][W];
    const Place p = place_of<W>(g);
    const int t0 = p.s * g.part, t1 = min(g.T, t0 + g.part);
    const int n = min(length_of(lengths, p.b, g.T), t1);                 // steps from n on are not there
    double h = state ? (double)state[p.b * g.D + p.d] : 0.0;
    if constexpr (W == kWave) h = enter_part<false>(parts, g, p, maps[0], h);
    const size_t base = (size_t)p.b * g.T * g.D + p.d;
    float xn[kSteps];
    G gn[kSteps];
    auto request = [&](int t) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const size_t e = base + (size_t)max(0, min(t + i, n - 1)) * g.D;
            xn[i] = get<PAST>(x + e);
            gn[i] = get<PAST>(gate + e);
        }
    };
    int buffer = 0;
    if (t0 < n) request(t0 + p.run * kSteps);
    for (int tile = t0; tile < t1; tile += kSpan) {
        const int t = tile + p.run * kSteps;
        float* __restrict__ out = y + base;
        if (tile >= n) {                                                 // (uniform) nothing there any more
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                if (t + i < t1 && p.valid) put<PAST>(out + (size_t)(t + i) * g.D, 0.0f);
            continue;
        }
        double a[kSteps], b[kSteps];
        Map m{1.0, 0.0};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const Gate q(t + i < n ? (float)gn[i] : kKeep);
            a[i] = q.a();
            b[i] = (double)q.e * a[i] * (double)(t + i < n ? xn[i] : 0.0f);
            m.H = fma(a[i], m.H, b[i]);
            m.A *= a[i];
        }
        maps[buffer][p.run][p.lane] = m;
        if (tile + kSpan < n) request(t + kSpan);
        __syncthreads();
        double in = h;
        h = through<false, W>(maps[buffer], p, h, &in);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            in = fma(a[i], in, b[i]);
            if (t + i < t1 && p.valid) put<PAST>(out + (size_t)(t + i) * g.D, t + i < n ? (float)in : 0.0f);
        }
        buffer ^= 1;                                                     // (the other half is written behind the next barrier's readers)
    }
    if (final_state && p.s == g.parts - 1 && p.run == 0 && p.valid) final_state[p.b * g.D + p.d] = (float)h;
}

// (A, H) of every part but the last on the way: forward of x and the gates, backward (DOWN) of the gradients v_t = a_t (dy_t + v_{t+1}).
template <typename G, bool DOWN>
__global__ void __launch_bounds__(kThreads)
gated_scan_parts_kernel(const float* __restrict__ x, const G* __restrict__ gate, const int64_t* __restrict__ lengths, Map* __restrict__ parts,
                        Geometry g) {
    __shared__ Map maps[kWaves][kWave];
    // the grid leaves out the last part on the way: renumbered over parts - 1
    Geometry less = g;
    less.parts = g.parts - 1;
    Place p = place_of<kWave>(less);
    if (DOWN) ++p.s;
    const int t0 = p.s * g.part, t1 = min(g.T, t0 + g.part);
    const int n = min(length_of(lengths, p.b, g.T), t1);
    const size_t base = (size_t)p.b * g.T * g.D + p.d;
    // each wavefront composes a consecutive share of the part's steps; shares are joined once
    const int share = g.part / kWaves, w0 = t0 + p.run * share, w1 = min(n, w0 + share);
    Map m{1.0, 0.0};
    float xn[kSteps];
    G gn[kSteps];
    auto at = [&](int i) { return DOWN ? w1 - 1 - i : w0 + i; };        // the i-th step on the way
    const int count = w1 - w0;
    auto request = [&](int i0) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const size_t e = base + (size_t)at(min(i0 + i, count - 1)) * g.D;
            xn[i] = x ? x[e] : 0.0f;
            gn[i] = gate[e];
        }
    };
    if (count > 0) request(0);
    for (int i0 = 0; i0 < count; i0 += kSteps) {
        float xv[kSteps];
        G gv[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) { xv[i] = xn[i]; gv[i] = gn[i]; }
        if (i0 + kSteps < count) request(i0 + kSteps);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            if (i0 + i >= count) break;
            const Gate q((float)gv[i]);
            const double a = q.a();
            m.H = DOWN ? a * (m.H + (double)xv[i]) : fma(a, m.H, (double)q.e * a * (double)xv[i]);
            m.A *= a;
        }
    }
    maps[p.run][p.lane] = m;
    __syncthreads();
    if (p.run != 0) return;
    m = maps[DOWN ? kWaves - 1 : 0][p.lane];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) m = then(m, maps[DOWN ? kWaves - 1 - k : k][p.lane]);
    if (p.valid) parts[((size_t)p.b * g.parts + p.s) * g.D + p.d] = m;
}

// The same walk from the end: v_t = a_t u_t, u_t = dy_t + v_{t+1}, v behind the last step = dfinal.
template <typename G, Past PAST, int W>
__global__ void __launch_bounds__(kThreads)
gated_scan_backward_kernel(const float* __restrict__ dy, const float* __restrict__ dfinal, const float* __restrict__ x,
                           const G* __restrict__ gate, const float* __restrict__ y, const float* __restrict__ state,
                           const int64_t* __restrict__ lengths, float* __restrict__ dx, G* __restrict__ dgate, float* __restrict__ dstate,
                           const Map* __restrict__ parts, Geometry g) {
    constexpr int kSpan = kThreads / W * kSteps;                         // steps of a tile
    __shared__ Map maps[2][kThreads / W][W];
    const Place p = place_of<W>(g);
    const int t0 = p.s * g.part, t1 = min(g.T, t0 + g.part);
    const int n = min(length_of(lengths, p.b, g.T), t1);
    double v = dfinal ? (double)dfinal[p.b * g.D + p.d] : 0.0;
    if constexpr (W == kWave) v = enter_part<true>(parts, g, p, maps[0], v);
    const float start = state ? state[p.b * g.D + p.d] : 0.0f;
    const size_t base = (size_t)p.b * g.T * g.D + p.d;
    float un[kSteps], xn[kSteps], hn[kSteps];
    G gn[kSteps];
    auto request = [&](int t) {
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int at = max(0, min(t + i, n - 1));
            const size_t e = base + (size_t)at * g.D;
            gn[i] = get<PAST>(gate + e);
            un[i] = dy ? get<PAST>(dy + e) : 0.0f;
            xn[i] = get<PAST>(x + e);
            hn[i] = get<PAST>(y + (at > 0 ? e - g.D : e));
        }
    };
    int buffer = 0;
    const int last = t0 + (t1 - t0 - 1) / kSpan * kSpan;
    bool asked = false;
    for (int tile = last; tile >= t0; tile -= kSpan) {
        const int t = tile + p.run * kSteps;
        if (tile >= n) {                                                 // (uniform) nothing there
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                if (t + i < t1 && p.valid) {
                    const size_t e = base + (size_t)(t + i) * g.D;
                    if (dx) put<PAST>(dx + e, 0.0f);
                    if (dgate) put<PAST>(dgate + e, (G)0.0f);
                }
            continue;
        }
        if (!asked) request(t);
        asked = true;
        double a[kSteps];
        float rest[kSteps], up[kSteps], slope[kSteps];               // slope: (h_{t-1} - x_t) a_t (1 - a_t)
        Map m{1.0, 0.0};
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            const Gate q(t + i < n ? (float)gn[i] : kKeep);
            a[i] = q.a();
            rest[i] = q.e * q.near;
            up[i] = t + i < n ? un[i] : 0.0f;
            slope[i] = ((t + i > 0 ? hn[i] : start) - xn[i]) * (rest[i] * q.near);
            m.H = a[i] * (m.H + (double)up[i]);
            m.A *= a[i];
        }
        maps[buffer][p.run][p.lane] = m;
        if (tile > t0) request(t - kSpan);
        __syncthreads();
        double in = v;
        v = through<true, W>(maps[buffer], p, v, &in);
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            const double sum = (double)up[i] + in;
            const float u = (float)sum;
            in = a[i] * sum;
            if (t + i < t1 && p.valid) {
                const size_t e = base + (size_t)(t + i) * g.D;
                if (dx) put<PAST>(dx + e, t + i < n ? rest[i] * u : 0.0f);
                if (dgate) put<PAST>(dgate + e, (G)(t + i < n ? u * slope[i] : 0.0f));
            }
        }
        buffer ^= 1;
    }
    if (dstate && p.s == 0 && p.run == 0 && p.valid) dstate[p.b * g.D + p.d] = (float)v;
}

template <typename G>
__global__ void __launch_bounds__(256)
gated_step_kernel(const float* x, const G* gate, const float* state, float* out, long long n) {
    const long long e = workgroup() * 256 + threadIdx.x;
    if (e >= n) return;
    const Gate g((float)gate[e]);
    const double a = g.a();
    out[e] = (float)fma(a, state ? (double)state[e] : 0.0, (double)g.e * a * (double)x[e]);
}

}  // namespace

namespace {
constexpr int kLine = 128;
Geometry geometry(int64_t B, int64_t T, int64_t D, int gate_bytes = 4) {
    Geometry g{(int)B, (int)T, (int)D, (int)((D + kWave - 1) / kWave), 1, 0, false, D * gate_bytes % kLine == 0, false};
    const int64_t rows = B * g.groups, tiles = (T + kTile - 1) / kTile, halves = B * ((D + kHalf - 1) / kHalf);
    if (rows < kFill && tiles > kShort && (rows < kMany || halves > kUnits)) g.parts = (int)std::min(tiles, (kCutFill + rows - 1) / rows);
    g.half = rows < kFill && tiles > 1 && g.parts == 1;
    if (g.half) g.groups = (int)((D + kHalf - 1) / kHalf);
    g.together = !g.whole_lines || (g.half && kHalf * gate_bytes % kLine != 0);
    g.part = (int)((tiles + g.parts - 1) / g.parts * kTile);
    g.parts = T > 0 ? (int)((T + g.part - 1) / g.part) : 1;
    return g;
}
}  // namespace

size_t gated_scan_workspace(int64_t B, int64_t T, int64_t D) {
    const Geometry g = geometry(B, T, D);
    return g.parts > 1 ? align_up((size_t)B * g.parts * D * sizeof(Map)) : 0;
}

int launch_gated_scan_forward(const float* x, const void* gate, int type, const float* state, const int64_t* lengths, float* y,
                              float* final_state, int64_t B, int64_t T, int64_t D, void* ws, hipStream_t stream) {
    const Geometry g = geometry(B, T, D, (int)type_bytes(type));
    const int64_t rows = B * g.groups;
    with_type(type, [&](auto e) {
        using G = decltype(e);
        if (g.parts > 1) {
            KernelTimerScope timer_("gated_scan_parts", stream);
            hipLaunchKernelGGL((gated_scan_parts_kernel<G, false>), dim3((unsigned)(rows * (g.parts - 1))), dim3(kThreads), 0, stream, x,
                               static_cast<const G*>(gate), lengths, static_cast<Map*>(ws), g);
        }
        KernelTimerScope timer_("gated_scan_forward", stream);
        const bool past = B * T * D * (int64_t)(2 * sizeof(float) + sizeof(G)) > kStreamBytes && g.whole_lines;      // x, y, gates
        auto kern = g.half ? (past ? gated_scan_forward_kernel<G, STORES, kHalf> : gated_scan_forward_kernel<G, NONE, kHalf>)
                    : !past ? gated_scan_forward_kernel<G, NONE, kWave>
                    : g.parts > 1 ? gated_scan_forward_kernel<G, BOTH, kWave> : gated_scan_forward_kernel<G, STORES, kWave>;
        hipLaunchKernelGGL(kern, dim3((unsigned)(rows * g.parts)), dim3(kThreads), 0, stream, x,
                           static_cast<const G*>(gate), state, lengths, y, final_state, static_cast<const Map*>(ws), g);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

int launch_gated_scan_backward(const float* dy, const float* dfinal, const float* x, const void* gate, int type, const float* y,
                               const float* state, const int64_t* lengths, float* dx, void* dgate, float* dstate, int64_t B, int64_t T,
                               int64_t D, void* ws, hipStream_t stream) {
    const Geometry g = geometry(B, T, D, (int)type_bytes(type));
    const int64_t rows = B * g.groups;
    with_type(type, [&](auto e) {
        using G = decltype(e);
        if (g.parts > 1) {
            KernelTimerScope timer_("gated_scan_parts_down", stream);
            hipLaunchKernelGGL((gated_scan_parts_kernel<G, true>), dim3((unsigned)(rows * (g.parts - 1))), dim3(kThreads), 0, stream, dy,
                               static_cast<const G*>(gate), lengths, static_cast<Map*>(ws), g);
        }
        KernelTimerScope timer_("gated_scan_backward", stream);
        const bool past = B * T * D * (int64_t)(4 * sizeof(float) + 2 * sizeof(G)) > kStreamBytes && g.whole_lines;  // dy, x, y, dx, gates, dgate
        auto kern = g.half ? (past ? gated_scan_backward_kernel<G, STORES, kHalf> : gated_scan_backward_kernel<G, NONE, kHalf>)
                    : !past ? gated_scan_backward_kernel<G, NONE, kWave>
                    : g.parts > 1 ? gated_scan_backward_kernel<G, BOTH, kWave> : gated_scan_backward_kernel<G, STORES, kWave>;
        hipLaunchKernelGGL(kern, dim3((unsigned)(rows * g.parts)), dim3(kThreads), 0, stream, dy, dfinal, x,
                           static_cast<const G*>(gate), y, state, lengths, dx, static_cast<G*>(dgate), dstate, static_cast<const Map*>(ws),
                           g);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

int launch_gated_step(const float* x, const void* gate, int type, const float* state, float* out, int64_t n, hipStream_t stream) {
    const int64_t blocks = (n + 255) / 256;
    with_type(type, [&](auto g) {
        using G = decltype(g);
        KernelTimerScope timer_("gated_step", stream);
        hipLaunchKernelGGL(gated_step_kernel<G>, wide_grid(blocks, 256), dim3(256), 0, stream, x, static_cast<const G*>(gate), state, out,
                           (long long)n);
        return 0;
    });
    SNNTC_HIP_CHECK(hipGetLastError());
    return SNNTC_OK;
}

}  // namespace snntc
