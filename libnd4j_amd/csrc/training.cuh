// Device helpers shared by the kernels behind training.h.
#pragma once

#include <hip/hip_runtime.h>

#include "elementwise.cuh"
#include "training.h"

namespace nd4j_amd {
namespace tr {

static constexpr int kWaveLanes = 64;

template <typename C> __device__ __forceinline__ C laneFrom(C v, int lane) {
    static_assert(sizeof(C) % 4 == 0, "a multiple of 4 bytes");
    constexpr int W = sizeof(C) / 4;
    struct Words { int w[W]; };
    Words in = __builtin_bit_cast(Words, v), out;
#pragma unroll
    for (int i = 0; i < W; i++) out.w[i] = __shfl(in.w[i], lane);
    return __builtin_bit_cast(C, out);
}
template <typename C> __device__ __forceinline__ C laneXorOf(C v, int mask) {
    static_assert(sizeof(C) % 4 == 0, "a multiple of 4 bytes");
    constexpr int W = sizeof(C) / 4;
    struct Words { int w[W]; };
    Words in = __builtin_bit_cast(Words, v), out;
#pragma unroll
    for (int i = 0; i < W; i++) out.w[i] = __shfl_xor(in.w[i], mask);
    return __builtin_bit_cast(C, out);
}
struct Add {
    template <typename C> __device__ __forceinline__ C operator()(C a, C b) const { return a + b; }
};
struct Largest {  // a NaN loses against anything
    __device__ __forceinline__ float operator()(float a, float b) const { return ::fmaxf(a, b); }
    __device__ __forceinline__ double operator()(double a, double b) const { return ::fmax(a, b); }
};
// every lane of a group of LANES neighbouring lanes gets the group's value
template <int LANES, class Op, typename C> __device__ __forceinline__ C waveAll(C v, Op op) {
#pragma unroll
    for (int d = LANES / 2; d >= 1; d >>= 1) v = op(v, laneXorOf(v, d));
    return v;
}
// every thread of a block of THREADS threads gets the block's value; smem: one C per wave, free for reuse behind the
// next barrier the caller passes
template <int THREADS, class Op, typename C> __device__ __forceinline__ C blockAll(C v, Op op, C *smem) {
    v = waveAll<kWaveLanes>(v, op);
    if (THREADS == kWaveLanes) return v;
    __syncthreads();  // smem may still be read from the round before
    if (threadIdx.x % kWaveLanes == 0) smem[threadIdx.x / kWaveLanes] = v;
    __syncthreads();
    v = smem[0];
#pragma unroll
    for (int w = 1; w < THREADS / kWaveLanes; w++) v = op(v, smem[w]);
    return v;
}

__device__ __forceinline__ float sqrtOf(float v) { return ::sqrtf(v); }
__device__ __forceinline__ double sqrtOf(double v) { return ::sqrt(v); }
template <typename C> __device__ __forceinline__ C notANumber() { return (C)__builtin_nanf(""); }
template <typename C> __device__ __forceinline__ C infinite() { return (C)__builtin_inff(); }

}  // namespace tr
}  // namespace nd4j_amd
