// Layer norm over the rows of a view, forward and backward.
//
//   mean = sum x / D,  v = sum (x - mean)^2 / D,  s = 1 / sqrt(v + epsilon),  h = (x - mean) s,  z = h gain + bias
//   a = dz gain,  dx = s (a - sum(a) / D - h sum(a h) / D),  dGain = sum over rows of dz h,  dBias = sum over rows of dz
//
// The variance is taken around the mean (two sweeps of the row), not from the sum of squares, which cancels.
// Statistics and sums are held in the compute type (float for half); a result is rounded to its type once.
#include "launch.h"
#include "training.cuh"

namespace nd4j_amd {
namespace {

using namespace tr;

constexpr int kRowThreads = 256;

// Steps in a form that takes a half operand as it is: one instruction converts it, multiplies and adds, where a conversion of
// its own and the two operations would be three.
// acc + v (times a 1 that the compiler does not see: of the constant it makes a conversion and an addition)
template <typename T> __device__ __forceinline__ typename Compute<T>::type plus(typename Compute<T>::type acc, T v) {
    if constexpr (sizeof(T) == 2) {
        float one = 1.0f;
        asm("" : "+s"(one));
        return fused(toCompute(v), one, acc);
    } else {
        return acc + toCompute(v);
    }
}
// v - mu, which is taken before anything else is: where a row's values are near each other v s and mu s are far larger than
// their difference, and a rounding of mu s on its own is an error of that size (a constant row of 30000 came out as 0.5).
template <typename T> __device__ __forceinline__ typename Compute<T>::type less(T v, typename Compute<T>::type mu) { return plus(-mu, v); }
// what is known to be no NaN
__device__ __forceinline__ float16 fromNumber(float v) {
    float16 h;
    h.x = __builtin_bit_cast(unsigned short, (_Float16)v);
    return h;
}
// a b
template <typename T> __device__ __forceinline__ typename Compute<T>::type times(T a, T b) {
    if constexpr (sizeof(T) == 2) return fused(toCompute(a), toCompute(b), 0.0f);
    else return toCompute(a) * toCompute(b);
}

// Rows too long for the kernel below, and views of any strides: a block per row, in three sweeps of which the second and
// third find the row in the caches.  UNIT: contiguous elements, in vectors.
constexpr int kLongThreads = 1024;
template <typename T, bool UNIT, typename F> __device__ __forceinline__ void sweep(const T *row, Long el, Long length, F f) {
    constexpr int N = Pack<T>::N;
    if constexpr (UNIT) {
        const Long whole = length / N * N;
#pragma unroll 2
        for (Long c = (Long)threadIdx.x * N; c < whole; c += kLongThreads * N) {
            const Pack<T> v = loadPackAnywhere(row + c);
#pragma unroll
            for (int e = 0; e < N; e++) f(c + e, v.v[e]);
        }
        if (whole + threadIdx.x < length) f(whole + threadIdx.x, row[whole + threadIdx.x]);
    } else {
#pragma unroll 4
        for (Long c = threadIdx.x; c < length; c += kLongThreads) f(c, row[c * el]);
    }
}
template <typename T, bool UNIT>
__global__ void __launch_bounds__(kLongThreads) layerNormAnyKernel(const T *x, RowView xv, const T *gain, const T *bias, T *z, RowView zv,
                                                                   typename Compute<T>::type *mean, typename Compute<T>::type *invStd,
                                                                   typename Compute<T>::type epsilon) {
    typedef typename Compute<T>::type C;
    __shared__ C smem[kLongThreads / kWaveLanes];
    for (Long r = blockIdx.x; r < xv.rows; r += gridDim.x) {
        const T *xr = x + r * xv.row;
        T *zr = z + r * zv.row;
        C sum = (C)0;
        sweep<T, UNIT>(xr, xv.el, xv.length, [&](Long, T v) { sum += toCompute(v); });
        const C mu = blockAll<kLongThreads>(sum, Add(), smem) / (C)xv.length;
        C squares = (C)0;
        sweep<T, UNIT>(xr, xv.el, xv.length, [&](Long, T v) {
            const C d = toCompute(v) - mu;
            squares += d * d;
        });
        const C s = (C)1 / sqrtOf(blockAll<kLongThreads>(squares, Add(), smem) / (C)xv.length + epsilon);
        if (threadIdx.x == 0) {
            if (mean != nullptr) mean[r] = mu;
            if (invStd != nullptr) invStd[r] = s;
        }
        // (stores element by element, which the compiler may not join: z may be x)
        sweep<T, UNIT>(xr, xv.el, xv.length, [&](Long c, T v) {
            C h = (toCompute(v) - mu) * s;
            if (gain != nullptr) h *= toCompute(gain[c]);
            if (bias != nullptr) h += toCompute(bias[c]);
            zr[c * zv.el] = fromCompute<T>(h);
        });
    }
}

// Views whose rows lie nearer to each other than a row's elements (an f-order matrix): lanes take neighbouring rows, the
// waves of a block share the columns.
constexpr int kAcrossThreads = 1024, kAcrossGroups = kAcrossThreads / kWaveLanes;
template <typename C> __device__ __forceinline__ C acrossSum(C v, C (*smem)[kWaveLanes]) {
    const int lane = threadIdx.x % kWaveLanes, group = threadIdx.x / kWaveLanes;
    __syncthreads();
    smem[group][lane] = v;
    __syncthreads();
    v = smem[0][lane];
#pragma unroll
    for (int g = 1; g < kAcrossGroups; g++) v += smem[g][lane];
    return v;
}
template <typename T>
__global__ void __launch_bounds__(kAcrossThreads) layerNormAcrossKernel(const T *x, RowView xv, const T *gain, const T *bias, T *z, RowView zv,
                                                                        typename Compute<T>::type *mean, typename Compute<T>::type *invStd,
                                                                        typename Compute<T>::type epsilon) {
    typedef typename Compute<T>::type C;
    __shared__ C smem[kAcrossGroups][kWaveLanes];
    const int lane = threadIdx.x % kWaveLanes, group = threadIdx.x / kWaveLanes;
    for (Long r0 = (Long)blockIdx.x * kWaveLanes; r0 < xv.rows; r0 += (Long)gridDim.x * kWaveLanes) {
        const bool live = r0 + lane < xv.rows;
        const Long r = live ? r0 + lane : r0;
        const T *xr = x + r * xv.row;
        C sum = (C)0;
#pragma unroll 8
        for (Long c = group; c < xv.length; c += kAcrossGroups) sum += toCompute(xr[c * xv.el]);
        const C mu = acrossSum(sum, smem) / (C)xv.length;
        C squares = (C)0;
#pragma unroll 8
        for (Long c = group; c < xv.length; c += kAcrossGroups) {
            const C d = toCompute(xr[c * xv.el]) - mu;
            squares += d * d;
        }
        const C s = (C)1 / sqrtOf(acrossSum(squares, smem) / (C)xv.length + epsilon);
        if (!live) continue;
        if (group == 0) {
            if (mean != nullptr) mean[r] = mu;
            if (invStd != nullptr) invStd[r] = s;
        }
#pragma unroll 4
        for (Long c = group; c < xv.length; c += kAcrossGroups) {
            C h = (toCompute(xr[c * xv.el]) - mu) * s;
            if (gain != nullptr) h *= toCompute(gain[c]);
            if (bias != nullptr) h += toCompute(bias[c]);
            z[r * zv.row + c * zv.el] = fromCompute<T>(h);
        }
    }
}

// Rows of contiguous elements that a team holds in its registers: a team is LANES lanes of a wave or as many whole waves as
// the row needs with PACKS vectors of 16 bytes a lane, and the elements behind the last whole vector go one a lane.  One
// read of x, one write of z, the next row on its way while one is worked on; gain and bias stay in registers over the
// team's rows (HELD).  [16384, 1024] halves 13.6 us, 4.9 TB/s, where a copy takes 10.5: 24 vector instructions an element hold the
// SIMDs for 10.1 us of it, and a row has two sums, one after the other.  (The multiplication by s behind the subtraction is 0.3 us of
// it.)  Stores have the streaming policy (a tenth longer without it, and with it for the loads too).
// Loads are unconditional (a vector that is not there re-reads the row's first place, see `at`).
template <typename T, int LANES, int PACKS>
__global__ void __launch_bounds__(1024)
    layerNormRowsKernel(const T *x, RowView xv, const T *gain, const T *bias, T *z, RowView zv, typename Compute<T>::type *mean,
                        typename Compute<T>::type *invStd, typename Compute<T>::type epsilon, int teamWaves) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N;
    constexpr bool HELD = PACKS <= 2;  // a lane of a block of 1024 has 128 registers, which more of the row needs
    __shared__ C sums[2 * (1024 / kWaveLanes)];
    const int size = LANES < kWaveLanes ? LANES : teamWaves * kWaveLanes, teams = blockDim.x / size;
    const int team = threadIdx.x / size, lane = threadIdx.x - team * size;
    C *smem = sums + 2 * team * teamWaves;
    int turn = 0;
    const int length = (int)xv.length, vectors = length / N, rest = vectors * N + lane;
    int at[PACKS];
    Pack<T> g[PACKS], b[PACKS];
    C gRest = (C)1, bRest = (C)0;
#pragma unroll
    for (int j = 0; j < PACKS; j++) {
        at[j] = lane + j * size < vectors ? (lane + j * size) * N : 0;
        if (HELD && vectors > 0 && gain != nullptr) g[j] = loadPackAnywhere(gain + at[j]);
        if (HELD && vectors > 0 && bias != nullptr) b[j] = loadPackAnywhere(bias + at[j]);
    }
    if (rest < length) {
        if (gain != nullptr) gRest = toCompute(gain[rest]);
        if (bias != nullptr) bRest = toCompute(bias[rest]);
    }
    Pack<T> v[PACKS], next[PACKS];
    C vRest = (C)0, nextRest = (C)0;
    const Long step = (Long)gridDim.x * teams;
    auto ask = [&](Long r0) {
        const T *xr = x + (team < teams && r0 + team < xv.rows ? r0 + team : r0) * xv.row;
        if (vectors > 0) {
#pragma unroll
            for (int j = 0; j < PACKS; j++) next[j] = loadPackAnywhere(xr + at[j]);
        }
        if (rest < length) nextRest = toCompute(xr[rest]);
    };
    ask((Long)blockIdx.x * teams);
    for (Long r0 = (Long)blockIdx.x * teams; r0 < xv.rows; r0 += step) {
        const Long r = r0 + team;
        const bool live = team < teams && r < xv.rows;
#pragma unroll
        for (int j = 0; j < PACKS; j++) v[j] = next[j];
        vRest = nextRest;
        if (r0 + step < xv.rows) ask(r0 + step);
        C sum[1] = {vRest};
#pragma unroll
        for (int j = 0; j < PACKS; j++)
            if (lane + j * size < vectors) {
#pragma unroll
                for (int e = 0; e < N; e++) sum[0] = plus(sum[0], v[j].v[e]);
            }
        teamSums<LANES>(sum, smem, teamWaves, turn);
        const C mu = sum[0] / (C)length;
        C squares[1] = {rest < length ? (vRest - mu) * (vRest - mu) : (C)0};
#pragma unroll
        for (int j = 0; j < PACKS; j++)
            if (lane + j * size < vectors) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const C d = less(v[j].v[e], mu);
                    squares[0] = fused(d, d, squares[0]);
                }
            }
        teamSums<LANES>(squares, smem, teamWaves, turn);
        const C s = (C)1 / sqrtOf(squares[0] / (C)length + epsilon);
        if (!live) continue;
        if (lane == 0) {
            if (mean != nullptr) mean[r] = mu;
            if (invStd != nullptr) invStd[r] = s;
        }
        T *zr = z + r * zv.row;
#pragma unroll
        for (int j = 0; j < PACKS; j++)
            if (lane + j * size < vectors) {
                Pack<T> o;
                if (!HELD && gain != nullptr) g[j] = loadPackAnywhere(gain + at[j]);
                if (!HELD && bias != nullptr) b[j] = loadPackAnywhere(bias + at[j]);
#pragma unroll
                for (int e = 0; e < N; e++) {
                    C h = less(v[j].v[e], mu) * s;
                    if (gain != nullptr) h = fused(h, toCompute(g[j].v[e]), bias != nullptr ? toCompute(b[j].v[e]) : (C)0);
                    else if (bias != nullptr) h += toCompute(b[j].v[e]);
                    o.v[e] = fromCompute<T>(h);
                }
                streamPackAnywhere(zr + at[j], o);
            }
        if (rest < length) zr[rest] = fromCompute<T>(fused((vRest - mu) * s, gRest, bRest));
    }
}

// The backward pass of the same views as layerNormAnyKernel's: dx alone, in two sweeps
template <typename T, bool UNIT, typename F>
__device__ __forceinline__ void sweepTwo(const T *one, Long el1, const T *two, Long el2, Long length, F f) {
    constexpr int N = Pack<T>::N;
    if constexpr (UNIT) {
        const Long whole = length / N * N;
#pragma unroll 2
        for (Long c = (Long)threadIdx.x * N; c < whole; c += kLongThreads * N) {
            const Pack<T> v = loadPackAnywhere(one + c), w = loadPackAnywhere(two + c);
#pragma unroll
            for (int e = 0; e < N; e++) f(c + e, v.v[e], w.v[e]);
        }
        if (whole + threadIdx.x < length) f(whole + threadIdx.x, one[whole + threadIdx.x], two[whole + threadIdx.x]);
    } else {
#pragma unroll 4
        for (Long c = threadIdx.x; c < length; c += kLongThreads) f(c, one[c * el1], two[c * el2]);
    }
}
template <typename T, bool UNIT>
__global__ void __launch_bounds__(kLongThreads) layerNormBpAnyKernel(const T *x, RowView xv, const T *gain,
                                                                     const typename Compute<T>::type *mean,
                                                                     const typename Compute<T>::type *invStd, const T *dz, RowView dzv, T *dx,
                                                                     RowView dxv) {
    typedef typename Compute<T>::type C;
    __shared__ C smem[kLongThreads / kWaveLanes];
    for (Long r = blockIdx.x; r < xv.rows; r += gridDim.x) {
        const T *xr = x + r * xv.row, *dzr = dz + r * dzv.row;
        T *dxr = dx + r * dxv.row;
        const C mu = mean[r], s = invStd[r];
        C sumA = (C)0, sumAH = (C)0;
        sweepTwo<T, UNIT>(xr, xv.el, dzr, dzv.el, xv.length, [&](Long c, T v, T d) {
            C a = toCompute(d);
            if (gain != nullptr) a *= toCompute(gain[c]);
            sumA += a;
            sumAH += a * ((toCompute(v) - mu) * s);
        });
        const C meanA = blockAll<kLongThreads>(sumA, Add(), smem) / (C)xv.length;
        const C meanAH = blockAll<kLongThreads>(sumAH, Add(), smem) / (C)xv.length;
        sweepTwo<T, UNIT>(xr, xv.el, dzr, dzv.el, xv.length, [&](Long c, T v, T d) {
            C a = toCompute(d);
            if (gain != nullptr) a *= toCompute(gain[c]);
            const C h = (toCompute(v) - mu) * s;
            dxr[c * dxv.el] = fromCompute<T>(s * (a - meanA - h * meanAH));
        });
    }
}

// ... and of layerNormAcrossKernel's
template <typename T>
__global__ void __launch_bounds__(kAcrossThreads) layerNormBpAcrossKernel(const T *x, RowView xv, const T *gain,
                                                                          const typename Compute<T>::type *mean,
                                                                          const typename Compute<T>::type *invStd, const T *dz, RowView dzv,
                                                                          T *dx, RowView dxv) {
    typedef typename Compute<T>::type C;
    __shared__ C smem[kAcrossGroups][kWaveLanes];
    const int lane = threadIdx.x % kWaveLanes, group = threadIdx.x / kWaveLanes;
    for (Long r0 = (Long)blockIdx.x * kWaveLanes; r0 < xv.rows; r0 += (Long)gridDim.x * kWaveLanes) {
        const bool live = r0 + lane < xv.rows;
        const Long r = live ? r0 + lane : r0;
        const T *xr = x + r * xv.row, *dzr = dz + r * dzv.row;
        const C mu = mean[r], s = invStd[r];
        C sumA = (C)0, sumAH = (C)0;
#pragma unroll 4
        for (Long c = group; c < xv.length; c += kAcrossGroups) {
            C a = toCompute(dzr[c * dzv.el]);
            if (gain != nullptr) a *= toCompute(gain[c]);
            sumA += a;
            sumAH += a * ((toCompute(xr[c * xv.el]) - mu) * s);
        }
        const C meanA = acrossSum(sumA, smem) / (C)xv.length, meanAH = acrossSum(sumAH, smem) / (C)xv.length;
        if (!live) continue;
#pragma unroll 4
        for (Long c = group; c < xv.length; c += kAcrossGroups) {
            C a = toCompute(dzr[c * dzv.el]);
            if (gain != nullptr) a *= toCompute(gain[c]);
            const C h = (toCompute(xr[c * xv.el]) - mu) * s;
            dx[r * dxv.row + c * dxv.el] = fromCompute<T>(s * (a - meanA - h * meanAH));
        }
    }
}

// The backward pass of rows that a team holds in its registers (as in layerNormRowsKernel): dx, and the row's share of the
// gain's and bias's gradients added onto sums that a lane keeps for its own columns over all rows of its team.  At the end
// the teams of a block add theirs up in LDS, and partial[0 / 1][block][column] receives the block's sums (null: not wanted).
//
// One block of 1024 threads a compute unit (two where a lane holds one vector): every block leaves two rows of partial sums,
// which is why there are no more of them, and 16 waves hide the loads of each other.  (Blocks of a single team, which need not
// wait for others but leave three times the partial sums, took 50 us where these take 35.)
//
// [16384, 1024] floats 39 us, 5.1 TB/s of x, dz and dx: bound by memory.  [4097, 5003] halves 35 us, of which the sums of the
// columns by the kernel below are 5: 28 vector instructions an element, which hold the SIMDs for 14.5 us, six rows for every team
// where 5.3 would be even, and 9 MB of partial sums written and read again.
constexpr int kBpThreads = 1024;
// the elements from one row of partial sums to the next: vectors of any type begin at a multiple of 16 bytes
__host__ __device__ inline Long partialPitch(Long length) { return (length + 7) / 8 * 8; }
template <typename C, int N> struct alignas(16) Aligned {
    C v[N];
};
template <typename T, int LANES, int PACKS>
__global__ void __launch_bounds__(kBpThreads)
    layerNormBpRowsKernel(const T *x, RowView xv, const T *gain, const typename Compute<T>::type *mean, const typename Compute<T>::type *invStd,
                          const T *dz, RowView dzv, T *dx, RowView dxv, typename Compute<T>::type *partial, int teamWaves) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N;
    // Long rows of floats and doubles are read with the streaming policy: [16384, 1024] floats 40.0 us, 41.6 with the ordinary one.
    // (Short ones, [100000, 64] floats, 22.0 and 19.7; [4097, 5003] halves 40.0 and 35.2.)
    constexpr bool STREAM = sizeof(T) > 2 && PACKS > 1;
    constexpr bool LATE = sizeof(T) == 2;  // s multiplied in where it costs least, an instruction an element instead of three
    extern __shared__ __align__(16) char dynamicLds[];
    C *columns = reinterpret_cast<C *>(dynamicLds);  // [half of the teams][columns of a row]
    __shared__ C sums[8 * (kBpThreads / kWaveLanes)];  // (the waves behind the last whole team have places too)
    const int size = LANES < kWaveLanes ? LANES : teamWaves * kWaveLanes, teams = kBpThreads / size;
    const int team = threadIdx.x / size, lane = threadIdx.x - team * size;
    C *smem = sums + 4 * team * teamWaves;
    int turn = 0;
    const int length = (int)xv.length, vectors = length / N, rest = vectors * N + lane;
    int at[PACKS];
    Pack<T> g[PACKS];
    C gainSum[PACKS][N], biasSum[PACKS][N], gainRest = (C)0, biasRest = (C)0, gRest = (C)1;
#pragma unroll
    for (int j = 0; j < PACKS; j++) {
        at[j] = lane + j * size < vectors ? (lane + j * size) * N : 0;
#pragma unroll
        for (int e = 0; e < N; e++) {
            gainSum[j][e] = biasSum[j][e] = (C)0;
            g[j].v[e] = fromCompute<T>((C)1);  // no gain: dz times 1, which is dz
        }
        if (vectors > 0 && gain != nullptr) g[j] = loadPackAnywhere(gain + at[j]);
    }
    if (rest < length && gain != nullptr) gRest = toCompute(gain[rest]);
    // the next row is on its way while this one is worked on (two places that take turns, without the copy below, took 38 us
    // where this takes 35: two more bodies in the loop, and registers to spare for neither)
    Pack<T> v[PACKS], d[PACKS], nextV[PACKS], nextD[PACKS];
    C vRest = (C)0, dRest = (C)0, nextVRest = (C)0, nextDRest = (C)0, mu = (C)0, s = (C)0, nextMu = (C)0, nextS = (C)0;
    const Long step = (Long)gridDim.x * teams;
    auto ask = [&](Long r0) {
        const Long r = team < teams && r0 + team < xv.rows ? r0 + team : r0;
        const T *xr = x + r * xv.row, *dzr = dz + r * dzv.row;
        if (vectors > 0) {
#pragma unroll
            for (int j = 0; j < PACKS; j++) {
                nextV[j] = STREAM ? streamPackAnywhere(xr + at[j]) : loadPackAnywhere(xr + at[j]);
                nextD[j] = STREAM ? streamPackAnywhere(dzr + at[j]) : loadPackAnywhere(dzr + at[j]);
            }
        }
        nextMu = mean[r];
        nextS = invStd[r];
        if (rest < length) {
            nextVRest = toCompute(xr[rest]);
            nextDRest = toCompute(dzr[rest]);
        }
    };
    ask((Long)blockIdx.x * teams);
    for (Long r0 = (Long)blockIdx.x * teams; r0 < xv.rows; r0 += step) {
        const bool live = team < teams && r0 + team < xv.rows;
        const Long r = live ? r0 + team : r0;
#pragma unroll
        for (int j = 0; j < PACKS; j++) {
            v[j] = nextV[j];
            d[j] = nextD[j];
        }
        vRest = nextVRest;
        dRest = nextDRest;
        mu = nextMu;
        s = nextS;
        if (r0 + step < xv.rows) ask(r0 + step);
        C sum[2] = {(C)0, (C)0};  // of a and of a h (halves: of a (x - mean), which cannot leave a float's range, and s behind the row)
        if (live) {
#pragma unroll
            for (int j = 0; j < PACKS; j++)
                if (lane + j * size < vectors) {
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const C dd = toCompute(d[j].v[e]), m = less(v[j].v[e], mu);
                        const C a = times(d[j].v[e], g[j].v[e]);
                        sum[0] += a;
                        if constexpr (LATE) {
                            sum[1] = fused(a, m, sum[1]);
                            gainSum[j][e] = fused(dd * s, m, gainSum[j][e]);
                        } else {
                            sum[1] = fused(a, m * s, sum[1]);
                            gainSum[j][e] = fused(dd, m * s, gainSum[j][e]);
                        }
                        biasSum[j][e] = plus(biasSum[j][e], d[j].v[e]);
                    }
                }
            if (rest < length) {
                const C h = (vRest - mu) * s, a = dRest * gRest;
                sum[0] += a;
                sum[1] = fused(a, LATE ? vRest - mu : h, sum[1]);
                gainRest = fused(dRest, h, gainRest);
                biasRest += dRest;
            }
        }
        if (dx == nullptr) continue;
        teamSums<LANES>(sum, smem, teamWaves, turn);
        if (LATE) sum[1] *= s;
        const C meanA = sum[0] / (C)length, meanAH = sum[1] / (C)length, share = s * meanAH;  // (of x - mean: h meanAH)
        if (!live) continue;
        T *dxr = dx + r * dxv.row;
        auto store = [&](auto convert) {
#pragma unroll
            for (int j = 0; j < PACKS; j++)
                if (lane + j * size < vectors) {
                    Pack<T> o;
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const C m = less(v[j].v[e], mu), a = fused(toCompute(d[j].v[e]), toCompute(g[j].v[e]), -meanA);
                        o.v[e] = convert(s * (LATE ? fused(-m, share, a) : fused(-(m * s), meanAH, a)));
                    }
                    streamPackAnywhere(dxr + at[j], o);
                }
        };
        if constexpr (sizeof(T) == 2) {
            // Finite sums have finite terms, a and x - mean then are finite too, and what an infinite product adds up to is no NaN:
            // so is no element of dx, unless s is 0.  (A NaN's own bits take a compare and a select an element: 39 us where this
            // takes 35, a select for a missing gain among them, which is a gain of 1 now.)
            if (::fabsf(sum[0]) < infinite<C>() && ::fabsf(share) < infinite<C>() && s != (C)0)
                store([](C o) { return fromNumber(o); });
            else
                store([](C o) { return fromCompute<T>(o); });
        } else {
            store([](C o) { return fromCompute<T>(o); });
        }
        if (rest < length) dxr[rest] = fromCompute<T>(s * (dRest * gRest - meanA - (vRest - mu) * s * meanAH));
    }
    if (partial == nullptr) return;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        // the upper half of the teams hands its sums to the lower half, until the first team has them all
        // (an element of a lane's vector lies beside those of its neighbours: next to its own, they would meet in an eighth of
        // LDS's banks, which made this end 6.7 us instead of 3.4)
        for (int have = teams; have > 1; have = (have + 1) / 2) {
            const int half = (have + 1) / 2;
            C *shared = columns + (size_t)(team < half ? team : team - half) * (N * PACKS * size + N) + lane;
            __syncthreads();
            if (team >= half && team < have) {
#pragma unroll
                for (int j = 0; j < PACKS; j++)
#pragma unroll
                    for (int e = 0; e < N; e++) shared[(e * PACKS + j) * size] = which == 0 ? gainSum[j][e] : biasSum[j][e];
                if (lane < N) shared[N * PACKS * size] = which == 0 ? gainRest : biasRest;
            }
            __syncthreads();
            if (team < have - half) {
#pragma unroll
                for (int j = 0; j < PACKS; j++)
#pragma unroll
                    for (int e = 0; e < N; e++) (which == 0 ? gainSum[j][e] : biasSum[j][e]) += shared[(e * PACKS + j) * size];
                if (lane < N) (which == 0 ? gainRest : biasRest) += shared[N * PACKS * size];
            }
        }
        if (team > 0) continue;
        C *out = partial + ((size_t)which * gridDim.x + blockIdx.x) * partialPitch(length);
#pragma unroll
        for (int j = 0; j < PACKS; j++)
            if (lane + j * size < vectors) {
                Aligned<C, N> sums;
#pragma unroll
                for (int e = 0; e < N; e++) sums.v[e] = which == 0 ? gainSum[j][e] : biasSum[j][e];
                *reinterpret_cast<Aligned<C, N> *>(out + at[j]) = sums;
            }
        if (rest < length) out[rest] = which == 0 ? gainRest : biasRest;
    }
}

// The gradients of gain and bias: a wave's lanes take neighbouring columns, its block's row range is `split` of `splits`;
// partial[0 / 1][split][column] receives the range's sums, merged by layerNormBpFinishKernel in the order of the splits.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) layerNormBpColumnsKernel(const T *x, RowView xv, const typename Compute<T>::type *mean,
                                                                        const typename Compute<T>::type *invStd, const T *dz, RowView dzv,
                                                                        typename Compute<T>::type *partial, int splits) {
    typedef typename Compute<T>::type C;
    constexpr int WAVES = kRowThreads / kWaveLanes;
    __shared__ C smem[2][WAVES][kWaveLanes];
    const int lane = threadIdx.x % kWaveLanes, wave = threadIdx.x / kWaveLanes;
    const Long tiles = (xv.length + kWaveLanes - 1) / kWaveLanes;
    for (Long work = blockIdx.x; work < tiles * splits; work += gridDim.x) {
        const Long c = work % tiles * kWaveLanes + lane, split = work / tiles;
        C gainSum = (C)0, biasSum = (C)0;
        if (c < xv.length)
#pragma unroll 4
            for (Long r = split * WAVES + wave; r < xv.rows; r += (Long)splits * WAVES) {
                const C d = toCompute(dz[r * dzv.row + c * dzv.el]);
                gainSum += d * ((toCompute(x[r * xv.row + c * xv.el]) - mean[r]) * invStd[r]);
                biasSum += d;
            }
        __syncthreads();
        smem[0][wave][lane] = gainSum;
        smem[1][wave][lane] = biasSum;
        __syncthreads();
        if (wave < 2 && c < xv.length) {
            C sum = smem[wave][0][lane];
#pragma unroll
            for (int w = 1; w < WAVES; w++) sum += smem[wave][w][lane];
            partial[((Long)wave * splits + split) * partialPitch(xv.length) + c] = sum;
        }
    }
}

// The same for views whose rows are nearer to each other than a row's elements: a wave takes a column, its lanes neighbouring
// rows of its split.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) layerNormBpColumnsAcrossKernel(const T *x, RowView xv, const typename Compute<T>::type *mean,
                                                                              const typename Compute<T>::type *invStd, const T *dz, RowView dzv,
                                                                              typename Compute<T>::type *partial, int splits) {
    typedef typename Compute<T>::type C;
    constexpr int WAVES = kRowThreads / kWaveLanes;
    const int lane = threadIdx.x % kWaveLanes, wave = threadIdx.x / kWaveLanes;
    for (Long work = (Long)blockIdx.x * WAVES + wave; work < xv.length * splits; work += (Long)gridDim.x * WAVES) {
        const Long c = work % xv.length, split = work / xv.length;
        C gainSum = (C)0, biasSum = (C)0;
#pragma unroll 4
        for (Long r = split * kWaveLanes + lane; r < xv.rows; r += (Long)splits * kWaveLanes) {
            const C d = toCompute(dz[r * dzv.row + c * dzv.el]);
            gainSum += d * ((toCompute(x[r * xv.row + c * xv.el]) - mean[r]) * invStd[r]);
            biasSum += d;
        }
        gainSum = waveAll<kWaveLanes>(gainSum, Add());
        biasSum = waveAll<kWaveLanes>(biasSum, Add());
        if (lane < 2) partial[((Long)lane * splits + split) * partialPitch(xv.length) + c] = lane == 0 ? gainSum : biasSum;
    }
}

// A block takes 32 columns: its 32 half waves share the splits, then add up in LDS in a fixed order.
constexpr int kFinishThreads = 1024, kFinishColumns = 32, kFinishGroups = kFinishThreads / kFinishColumns;
template <typename T>
__global__ void __launch_bounds__(kFinishThreads) layerNormBpFinishKernel(const typename Compute<T>::type *partial, int splits, Long length,
                                                                          T *dGain, T *dBias) {
    typedef typename Compute<T>::type C;
    __shared__ C smem[kFinishGroups][kFinishColumns + 1];
    const int column = threadIdx.x % kFinishColumns, group = threadIdx.x / kFinishColumns;
    const int which = blockIdx.y;
    T *out = which == 0 ? dGain : dBias;
    if (out == nullptr) return;
    const Long tiles = (length + kFinishColumns - 1) / kFinishColumns;
    for (Long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const Long c = tile * kFinishColumns + column;
        C sum = (C)0;
        if (c < length) {
            const Long pitch = partialPitch(length);
            const C *from = partial + (size_t)which * splits * pitch + c;
#pragma unroll 8
            for (int s = group; s < splits; s += kFinishGroups) sum += from[(size_t)s * pitch];
        }
        __syncthreads();
        smem[group][column] = sum;
        __syncthreads();
        if (group == 0 && c < length) {
#pragma unroll
            for (int k = 1; k < kFinishGroups; k++) sum += smem[k][column];
            out[c] = fromCompute<T>(sum);
        }
    }
}

// How many row ranges the column sums are split into: enough blocks to fill the chip, at least 32 rows in a range
int columnSplits(Long rows, Long length) {
    const Long tiles = (length + kWaveLanes - 1) / kWaveLanes;
    Long splits = (2048 + tiles - 1) / tiles;
    if (splits > (rows + 31) / 32) splits = (rows + 31) / 32;
    return (int)(splits < 1 ? 1 : splits);
}

// the waves of a team that holds a row in `packs` vectors a lane
int teamWaves(Long vectors, int packs) {
    const Long waves = (vectors + (Long)kWaveLanes * packs - 1) / ((Long)kWaveLanes * packs);
    return (int)(waves < 1 ? 1 : waves);
}
// The blocks of the forward kernel.  Halves, and teams of more than eight waves: as many as the 256 compute units hold at once
// (32 waves a unit at one vector a lane, by registers 20 at two and 16 at four), each going on from row to row: where [16384, 1024]
// halves took 14.4 us, 32 waves a unit throughout took 15.4 and a block for every row 16.4; [4096, 8192] floats 52 and 68.  Smaller
// teams of floats and doubles: three times the 32, which spreads what is left at the end: [16384, 1024] floats 21.0 us, 23.5
// with 32 and 20.8 with a block for every row, [65536, 256] 21.7, 23.4 and 25.5.
int rowBlocks(int packs, int size, int blockWaves, int teamWaves) {
    if (size > 2 && teamWaves <= 8) return 256 * 96 / blockWaves;
    const int held = (packs == 1 ? 32 : (packs == 2 ? 20 : 16)) / blockWaves;
    return 256 * (held < 1 ? 1 : held);
}

unsigned gridOf(Long blocks) { return (unsigned)(blocks < 1 ? 1 : (blocks > (1 << 20) ? (1 << 20) : blocks)); }

}  // namespace

constexpr int kBpBlocks = 256;  // of the register kernel; twice as many where a lane holds one vector
constexpr Long kBpOnePack = 64, kBpTwoPacks = 2048;  // vectors of a row that its lanes hold one and two of; longer rows go elsewhere

// the most blocks of the register kernel for rows of this many vectors (0: they are not its)
static Long mostBpBlocks(Long vectors) { return vectors <= kBpOnePack ? 2 * kBpBlocks : (vectors <= kBpTwoPacks ? kBpBlocks : 0); }
template <typename T> static size_t bpScratch(Long rows, Long length) {
    // (views that are not dense go by columnSplits whatever their length; no kernel has more blocks than rows)
    const Long any = columnSplits(rows, length), most = mostBpBlocks(length / Pack<T>::N), held = rows < most ? rows : most;
    return (size_t)2 * (any > held ? any : held) * partialPitch(length) * sizeof(typename Compute<T>::type);
}
size_t layerNormBpScratch(Long rows, Long length) {
    const size_t half = bpScratch<float16>(rows, length), single = bpScratch<float>(rows, length), twice = bpScratch<double>(rows, length);
    const size_t most = half > single ? half : single;
    return most > twice ? most : twice;
}

// Blocks of about four waves, whole teams: more teams in a block would wait for each other.
template <typename T, int LANES, int PACKS>
void runRows(hipStream_t s, const T *x, const RowView &xv, const T *gain, const T *bias, T *z, const RowView &zv,
             typename Compute<T>::type *mean, typename Compute<T>::type *invStd, double epsilon) {
    typedef typename Compute<T>::type C;
    const int waves = teamWaves(xv.length / Pack<T>::N, PACKS), teams = LANES < kWaveLanes ? 256 / LANES : (waves >= 4 ? 1 : 4 / waves);
    const int threads = LANES < kWaveLanes ? 256 : teams * waves * kWaveLanes;
    const unsigned blocks = (unsigned)gridFor(xv.rows, teams, rowBlocks(PACKS, (int)sizeof(T), threads / kWaveLanes, waves));
    ND4J_LAUNCH((layerNormRowsKernel<T, LANES, PACKS>), dim3(blocks), dim3(threads), 0, s, x, xv, gain, bias, z, zv, mean, invStd, (C)epsilon,
                waves);
}

template <typename T>
void launchLayerNorm(hipStream_t s, const T *x, const RowView &xv, const T *gain, const T *bias, T *z, const RowView &zv,
                     typename Compute<T>::type *mean, typename Compute<T>::type *invStd, double epsilon) {
    typedef typename Compute<T>::type C;
    if (xv.el == 1 && zv.el == 1) {
        const Long vectors = xv.length / Pack<T>::N;
#define ROWS(LANES, PACKS) return runRows<T, LANES, PACKS>(s, x, xv, gain, bias, z, zv, mean, invStd, epsilon)
        if (vectors <= 16) ROWS(16, 1);
        if (vectors <= 32) ROWS(16, 2);
        if (vectors <= 64) ROWS(64, 1);
        if (vectors <= 2048) ROWS(64, 2);
        if constexpr (sizeof(T) > 2)  // (32 halves a lane do not fit its 128 registers as floats)
            if (vectors <= 4096) ROWS(64, 4);
#undef ROWS
    }
    const dim3 grid(gridOf(xv.rows)), block(kLongThreads);
    if (xv.el == 1 && zv.el == 1)
        ND4J_LAUNCH((layerNormAnyKernel<T, true>), grid, block, 0, s, x, xv, gain, bias, z, zv, mean, invStd, (C)epsilon);
    else if (rowsAreNear(xv) && rowsAreNear(zv))
        ND4J_LAUNCH((layerNormAcrossKernel<T>), dim3(gridOf((xv.rows + kWaveLanes - 1) / kWaveLanes)), dim3(kAcrossThreads), 0, s, x, xv, gain,
                    bias, z, zv, mean, invStd, (C)epsilon);
    else
        ND4J_LAUNCH((layerNormAnyKernel<T, false>), grid, block, 0, s, x, xv, gain, bias, z, zv, mean, invStd, (C)epsilon);
}

// runs the register kernel and returns the number of its blocks
template <typename T, int LANES, int PACKS>
int runBpRows(hipStream_t s, const T *x, const RowView &xv, const T *gain, const typename Compute<T>::type *mean,
              const typename Compute<T>::type *invStd, const T *dz, const RowView &dzv, T *dx, const RowView &dxv,
              typename Compute<T>::type *partial) {
    typedef typename Compute<T>::type C;
    const int waves = teamWaves(xv.length / Pack<T>::N, PACKS);
    const int teams = LANES < kWaveLanes ? kBpThreads / LANES : kBpThreads / kWaveLanes / waves;
    // as many turns as the most blocks would take, the rows spread evenly over them
    const Long most = mostBpBlocks(xv.length / Pack<T>::N), turns = (xv.rows + most * teams - 1) / (most * teams);
    const int blocks = gridFor(xv.rows, turns * teams, (int)most);
    const int size = LANES < kWaveLanes ? LANES : waves * kWaveLanes;
    const size_t lds = partial != nullptr ? (size_t)(teams / 2) * (Pack<T>::N * PACKS * size + Pack<T>::N) * sizeof(C) : 0;
    ND4J_LAUNCH((layerNormBpRowsKernel<T, LANES, PACKS>), dim3(blocks), dim3(kBpThreads), lds, s, x, xv, gain, mean, invStd, dz, dzv, dx, dxv,
                partial, waves);
    return blocks;
}

template <typename T>
void launchLayerNormBp(hipStream_t s, const T *x, const RowView &xv, const T *gain, const typename Compute<T>::type *mean,
                       const typename Compute<T>::type *invStd, const T *dz, const RowView &dzv, T *dx, const RowView &dxv, T *dGain,
                       T *dBias, void *scratch) {
    typedef typename Compute<T>::type C;
    const bool columns = dGain != nullptr || dBias != nullptr;
    C *partial = columns ? reinterpret_cast<C *>(scratch) : nullptr;
    int splits = 0;
    if (xv.el == 1 && dzv.el == 1 && dxv.el == 1 && xv.rows > 0) {
        const Long vectors = xv.length / Pack<T>::N;
#define ROWS(LANES, PACKS) splits = runBpRows<T, LANES, PACKS>(s, x, xv, gain, mean, invStd, dz, dzv, dx, dxv, partial)
        if (vectors <= 16) ROWS(16, 1);
        else if (vectors <= kBpOnePack) ROWS(64, 1);
        else if (vectors <= kBpTwoPacks) ROWS(64, 2);
#undef ROWS
    }
    if (splits == 0) {  // any other view: the columns first, since dx may lie where dz or x does
        splits = columnSplits(xv.rows, xv.length);
        const Long tiles = (xv.length + kWaveLanes - 1) / kWaveLanes;
        const bool across = rowsAreNear(xv) && rowsAreNear(dzv);
        if (columns && across)
            ND4J_LAUNCH((layerNormBpColumnsAcrossKernel<T>), dim3(gridOf(xv.length * splits / 4 + 1)), dim3(kRowThreads), 0, s, x, xv, mean, invStd, dz,
                        dzv, partial, splits);
        else if (columns)
            ND4J_LAUNCH((layerNormBpColumnsKernel<T>), dim3(gridOf(tiles * splits)), dim3(kRowThreads), 0, s, x, xv, mean, invStd, dz, dzv, partial,
                        splits);
        if (dx != nullptr && xv.rows > 0) {
            const dim3 grid(gridOf(xv.rows)), block(kLongThreads);
            if (xv.el == 1 && dzv.el == 1 && dxv.el == 1)
                ND4J_LAUNCH((layerNormBpAnyKernel<T, true>), grid, block, 0, s, x, xv, gain, mean, invStd, dz, dzv, dx, dxv);
            else if (across && rowsAreNear(dxv))
                ND4J_LAUNCH((layerNormBpAcrossKernel<T>), dim3(gridOf((xv.rows + kWaveLanes - 1) / kWaveLanes)), dim3(kAcrossThreads), 0, s, x, xv, gain,
                            mean, invStd, dz, dzv, dx, dxv);
            else
                ND4J_LAUNCH((layerNormBpAnyKernel<T, false>), grid, block, 0, s, x, xv, gain, mean, invStd, dz, dzv, dx, dxv);
        }
    }
    if (columns)
        ND4J_LAUNCH((layerNormBpFinishKernel<T>), dim3(gridOf((xv.length + kFinishColumns - 1) / kFinishColumns), 2), dim3(kFinishThreads), 0, s,
                    partial, splits, xv.length, dGain, dBias);
}

#define INST(T)                                                                                                                       \
    template void launchLayerNorm<T>(hipStream_t, const T *, const RowView &, const T *, const T *, T *, const RowView &,              \
                                     Compute<T>::type *, Compute<T>::type *, double);                                                 \
    template void launchLayerNormBp<T>(hipStream_t, const T *, const RowView &, const T *, const Compute<T>::type *,                   \
                                       const Compute<T>::type *, const T *, const RowView &, T *, const RowView &, T *, T *, void *);
INST(float)
INST(float16)
INST(double)
#undef INST

}  // namespace nd4j_amd
