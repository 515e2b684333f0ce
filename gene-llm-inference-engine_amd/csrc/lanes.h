// Reductions and prefix sums over the lanes of a wave in vector registers, without the trip through LDS that a shuffle is: of a small kernel's time much is the wait for such steps (three kernels with seven of them, each
// 32 to 64 bits, took 19.7 us by shuffles, 18.6 so).  The order of additions is fixed by the lane numbers alone.
#pragma once
#include "common.h"

template <typename T> struct Words { int w[sizeof(T) / 4]; };

// op(v of lane l, v of lane l ^ BY); for BY below 16, where v has to be the same every 2 BY lanes of sixteen, a rotation does.
template <int BY, typename T, typename Op>
__device__ __forceinline__ T with_lane(T v, Op op) {
    Words<T> a = __builtin_bit_cast(Words<T>, v), b;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 4; ++i) {
        if constexpr (BY == 32) {                                   // halves swapped between two copies: the lower ones in both halves of one, the upper ones in the other
            const auto both = __builtin_amdgcn_permlane32_swap(a.w[i], a.w[i], false, false);
            a.w[i] = both[0];
            b.w[i] = both[1];
        } else if constexpr (BY == 16) {
            const auto both = __builtin_amdgcn_permlane16_swap(a.w[i], a.w[i], false, false);
            a.w[i] = both[0];
            b.w[i] = both[1];
        } else {
            b.w[i] = __builtin_amdgcn_update_dpp(0, a.w[i], 0x120 + BY, 0xf, 0xf, false);        // (rotated within sixteen)
        }
    }
    return op(__builtin_bit_cast(T, a), __builtin_bit_cast(T, b));
}
// Every lane ends with the same value: of its sixteen, of the wave.
template <typename T, typename Op> __device__ __forceinline__ T over_16(T v, Op op) { return with_lane<1>(with_lane<2>(with_lane<4>(with_lane<8>(v, op), op), op), op); }
template <typename T, typename Op> __device__ __forceinline__ T over_wave(T v, Op op) { return over_16(with_lane<16>(with_lane<32>(v, op), op), op); }
struct Add { template <typename T> __device__ T operator()(T a, T b) const { return a + b; } };
struct Larger { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Lesser { __device__ int operator()(int a, int b) const { return min(a, b); } };

// v of another lane: CTRL says which, ROWS in which sixteens; 0 elsewhere and where there is none.
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T moved(T v) {
    Words<T> a = __builtin_bit_cast(Words<T>, v);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 4; ++i) a.w[i] = __builtin_amdgcn_update_dpp(0, a.w[i], CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(T, a);
}
template <typename T> __device__ __forceinline__ T lane_before(T v) { return moved<0x138, 0xf>(v); }
template <typename T>
__device__ __forceinline__ T of_lane(T v, int lane) {       // (the same lane for the wave)
    lane = __builtin_amdgcn_readfirstlane(lane);
    Words<T> a = __builtin_bit_cast(Words<T>, v);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 4; ++i) a.w[i] = __builtin_amdgcn_readlane(a.w[i], lane);
    return __builtin_bit_cast(T, a);
}
// The sum of the lanes up to each: within sixteen by lanes 1, 2, 4 and 8 before, then the sixteen before, then the 32 before.
template <typename T>
__device__ __forceinline__ T sum_up_to(T v) {
    v += moved<0x111, 0xf>(v);
    v += moved<0x112, 0xf>(v);
    v += moved<0x114, 0xf>(v);
    v += moved<0x118, 0xf>(v);
    v += moved<0x142, 0xa>(v);                              // (the last of the sixteen before, in the second and the fourth)
    return v + moved<0x143, 0xc>(v);                        // (the last of the first half, in the second)
}
