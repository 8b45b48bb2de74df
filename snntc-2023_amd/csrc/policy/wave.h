// Sums and maxima over a wavefront in the registers' own network, for the kernels of this folder.
#pragma once

#include "../snntc_common.h"

namespace snntc {
namespace {

// v of the lane that CTRL names; `none` where there is no such lane, or MASK leaves a row of 16 out.
template <int CTRL, int MASK, typename T>
__device__ __forceinline__ T from_lane(T none, T v) {
    struct Halves { int h[sizeof(T) / 4]; };
    const Halves n = __builtin_bit_cast(Halves, none);
    Halves x = __builtin_bit_cast(Halves, v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) x.h[i] = __builtin_amdgcn_update_dpp(n.h[i], x.h[i], CTRL, MASK, 0xF, false);
    return __builtin_bit_cast(T, x);
}
// The same where every lane has one: part of the instruction that uses it.
template <int CTRL, typename T>
__device__ __forceinline__ T exchanged(T v) {
    struct Halves { int h[sizeof(T) / 4]; };
    Halves x = __builtin_bit_cast(Halves, v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) x.h[i] = __builtin_amdgcn_mov_dpp(x.h[i], CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(T, x);
}
// A lane's value for all; the lane is the same for all.
template <typename T>
__device__ __forceinline__ T of_lane(T v, int lane) {
    struct Halves { int h[sizeof(T) / 4]; };
    Halves x = __builtin_bit_cast(Halves, v);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) x.h[i] = __builtin_amdgcn_readlane(x.h[i], lane);
    return __builtin_bit_cast(T, x);
}
// All of a wavefront's values joined, in the registers' own network: pairs, quads, eights and sixteens by exchange, then lane 15 of a row to
// the next one and lane 31 to the upper half; the last lane has them all.
template <typename T, typename F>
__device__ __forceinline__ T wave_join(T v, T none, F&& f) {
    v = f(v, exchanged<0xB1>(v));
    v = f(v, exchanged<0x4E>(v));
    v = f(v, exchanged<0x141>(v));
    v = f(v, exchanged<0x140>(v));
    v = f(v, from_lane<0x142, 0xA>(none, v));
    v = f(v, from_lane<0x143, 0xC>(none, v));
    return of_lane(v, kWave - 1);
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) { return wave_join(v, (T)0, [](T a, T b) { return a + b; }); }
// The sum of the lanes up to and with each.
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v += from_lane<0x111, 0xF>((T)0, v);
    v += from_lane<0x112, 0xF>((T)0, v);
    v += from_lane<0x114, 0xF>((T)0, v);
    v += from_lane<0x118, 0xF>((T)0, v);
    v += from_lane<0x142, 0xA>((T)0, v);
    v += from_lane<0x143, 0xC>((T)0, v);
    return v;
}
}  // namespace
}  // namespace snntc
