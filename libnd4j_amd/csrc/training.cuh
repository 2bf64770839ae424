// Device helpers shared by the kernels behind training.h.
#pragma once

#include <hip/hip_runtime.h>

#include "elementwise.cuh"
#include "training.h"

namespace nd4j_amd {
namespace tr {

static constexpr int kWaveLanes = 64;

struct Add {
    template <typename C> __device__ __forceinline__ C operator()(C a, C b) const { return a + b; }
};
struct Largest {  // a NaN loses against anything
    __device__ __forceinline__ float operator()(float a, float b) const { return ::fmaxf(a, b); }
    __device__ __forceinline__ double operator()(double a, double b) const { return ::fmax(a, b); }
};
// The value of another lane of the same 16, by the data path of the vector unit itself (a shuffle goes through LDS).
// CTRL: 0xb1 and 0x4e swap neighbours and pairs, 0x141 and 0x140 mirror 8 and 16 lanes.
template <int CTRL, typename C> __device__ __forceinline__ C laneDpp(C v) {
    constexpr int W = sizeof(C) / 4;
    struct Words { int w[W]; };
    Words in = __builtin_bit_cast(Words, v), out;
#pragma unroll
    for (int i = 0; i < W; i++) out.w[i] = __builtin_amdgcn_update_dpp(in.w[i], in.w[i], CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(C, out);
}
// Lane i's value beside that of the lane 16 (32) away: every lane gets both values of its pair, in the same order.
template <int APART, typename C> __device__ __forceinline__ void lanePair(C v, C &a, C &b) {
    static_assert(APART == 16 || APART == 32, "rows or halves of a wave");
    constexpr int W = sizeof(C) / 4;
    struct Words { unsigned w[W]; };
    Words in = __builtin_bit_cast(Words, v), x, y;
#pragma unroll
    for (int i = 0; i < W; i++) {
        auto both = APART == 16 ? __builtin_amdgcn_permlane16_swap(in.w[i], in.w[i], false, false)
                                : __builtin_amdgcn_permlane32_swap(in.w[i], in.w[i], false, false);
        x.w[i] = both[0];
        y.w[i] = both[1];
    }
    a = __builtin_bit_cast(C, x);
    b = __builtin_bit_cast(C, y);
}
// every lane of a group of LANES neighbouring lanes gets the group's value; op commutes
template <int LANES, class Op, typename C> __device__ __forceinline__ C waveAll(C v, Op op) {
    static_assert(LANES == 16 || LANES == 32 || LANES == 64, "whole rows of a wave");
    v = op(v, laneDpp<0xb1>(v));
    v = op(v, laneDpp<0x4e>(v));
    v = op(v, laneDpp<0x141>(v));
    v = op(v, laneDpp<0x140>(v));
    C a, b;
    if (LANES >= 32) {
        lanePair<16>(v, a, b);
        v = op(a, b);
    }
    if (LANES == 64) {
        lanePair<32>(v, a, b);
        v = op(a, b);
    }
    return v;
}
// every thread of a team of THREADS neighbouring threads gets the team's value (all teams of the block call it together);
// smem: one C per wave of the team, free for reuse behind the next barrier the caller passes
template <int THREADS, class Op, typename C> __device__ __forceinline__ C blockAll(C v, Op op, C *smem) {
    v = waveAll<kWaveLanes>(v, op);
    if (THREADS == kWaveLanes) return v;
    __syncthreads();  // smem may still be read from the round before
    if (threadIdx.x % kWaveLanes == 0) smem[threadIdx.x % THREADS / kWaveLanes] = v;
    __syncthreads();
    v = smem[0];
#pragma unroll
    for (int w = 1; w < THREADS / kWaveLanes; w++) v = op(v, smem[w]);
    return v;
}

// The sum over a team of LANES lanes (a part of a wave, waves == 1) or of `waves` whole waves; all teams of a block call it
// together, turn after turn.  smem: two values per wave of the team, for even and odd turns, so that one barrier a turn is
// enough.  VALUES sums at once.
template <int LANES, int VALUES, typename C>
__device__ __forceinline__ void teamSums(C (&v)[VALUES], C *smem, int waves, int &turn) {
#pragma unroll
    for (int i = 0; i < VALUES; i++) v[i] = waveAll<LANES>(v[i], Add());
    if (LANES < kWaveLanes || waves == 1) return;
    C *mine = smem + (turn & 1) * VALUES * waves;
    turn++;
    const int wave = threadIdx.x / kWaveLanes % waves;
    if (threadIdx.x % kWaveLanes == 0) {
#pragma unroll
        for (int i = 0; i < VALUES; i++) mine[wave * VALUES + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VALUES; i++) v[i] = mine[i];
    for (int w = 1; w < waves; w++) {
#pragma unroll
        for (int i = 0; i < VALUES; i++) v[i] += mine[w * VALUES + i];
    }
}
__device__ __forceinline__ float fused(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return __builtin_fma(a, b, c); }

__device__ __forceinline__ float sqrtOf(float v) { return ::sqrtf(v); }
__device__ __forceinline__ double sqrtOf(double v) { return ::sqrt(v); }
template <typename C> __device__ __forceinline__ C notANumber() { return (C)__builtin_nanf(""); }
template <typename C> __device__ __forceinline__ C infinite();
template <> __device__ __forceinline__ float infinite<float>() { return __builtin_inff(); }
// (From a register that the compiler does not see into: it moves a 64-bit constant into a pair of scalar registers in one
// instruction here, of which the hardware takes 32 bits, and a list that begins with minus infinity began with 0.)
template <> __device__ __forceinline__ double infinite<double>() {
    unsigned high = 0x7ff00000u;
    asm("" : "+v"(high));
    return __builtin_bit_cast(double, (unsigned long long)high << 32);
}

}  // namespace tr
}  // namespace nd4j_amd
