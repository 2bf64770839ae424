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

// Any view: a block per row, element by element.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) layerNormAnyKernel(const T *x, RowView xv, const T *gain, const T *bias, T *z, RowView zv,
                                                                  typename Compute<T>::type *mean, typename Compute<T>::type *invStd,
                                                                  typename Compute<T>::type epsilon) {
    typedef typename Compute<T>::type C;
    __shared__ C smem[kRowThreads / kWaveLanes];
    for (Long r = blockIdx.x; r < xv.rows; r += gridDim.x) {
        const T *xr = x + r * xv.row;
        T *zr = z + r * zv.row;
        C sum = (C)0;
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) sum += toCompute(xr[c * xv.el]);
        const C mu = blockAll<kRowThreads>(sum, Add(), smem) / (C)xv.length;
        C squares = (C)0;
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) {
            const C d = toCompute(xr[c * xv.el]) - mu;
            squares += d * d;
        }
        const C s = (C)1 / sqrtOf(blockAll<kRowThreads>(squares, Add(), smem) / (C)xv.length + epsilon);
        if (threadIdx.x == 0) {
            if (mean != nullptr) mean[r] = mu;
            if (invStd != nullptr) invStd[r] = s;
        }
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) {
            C v = (toCompute(xr[c * xv.el]) - mu) * s;
            if (gain != nullptr) v *= toCompute(gain[c]);
            if (bias != nullptr) v += toCompute(bias[c]);
            zr[c * zv.el] = fromCompute<T>(v);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) layerNormBpAnyKernel(const T *x, RowView xv, const T *gain,
                                                                    const typename Compute<T>::type *mean,
                                                                    const typename Compute<T>::type *invStd, const T *dz, RowView dzv, T *dx,
                                                                    RowView dxv) {
    typedef typename Compute<T>::type C;
    __shared__ C smem[kRowThreads / kWaveLanes];
    for (Long r = blockIdx.x; r < xv.rows; r += gridDim.x) {
        const T *xr = x + r * xv.row, *dzr = dz + r * dzv.row;
        T *dxr = dx + r * dxv.row;
        const C mu = mean[r], s = invStd[r];
        C sumA = (C)0, sumAH = (C)0;
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) {
            C a = toCompute(dzr[c * dzv.el]);
            if (gain != nullptr) a *= toCompute(gain[c]);
            sumA += a;
            sumAH += a * ((toCompute(xr[c * xv.el]) - mu) * s);
        }
        const C meanA = blockAll<kRowThreads>(sumA, Add(), smem) / (C)xv.length;
        const C meanAH = blockAll<kRowThreads>(sumAH, Add(), smem) / (C)xv.length;
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) {
            C a = toCompute(dzr[c * dzv.el]);
            if (gain != nullptr) a *= toCompute(gain[c]);
            const C h = (toCompute(xr[c * xv.el]) - mu) * s;
            dxr[c * dxv.el] = fromCompute<T>(s * (a - meanA - h * meanAH));
        }
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
            partial[((Long)wave * splits + split) * xv.length + c] = sum;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) layerNormBpFinishKernel(const typename Compute<T>::type *partial, int splits, Long length, T *dGain,
                                                                       T *dBias) {
    typedef typename Compute<T>::type C;
    constexpr int WAVES = kRowThreads / kWaveLanes;
    __shared__ C smem[WAVES][kWaveLanes];
    const int lane = threadIdx.x % kWaveLanes, wave = threadIdx.x / kWaveLanes;
    const int which = blockIdx.y;
    T *out = which == 0 ? dGain : dBias;
    if (out == nullptr) return;
    const Long tiles = (length + kWaveLanes - 1) / kWaveLanes;
    for (Long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const Long c = tile * kWaveLanes + lane;
        C sum = (C)0;
        if (c < length)
            for (int s = wave; s < splits; s += WAVES) sum += partial[((Long)which * splits + s) * length + c];
        __syncthreads();
        smem[wave][lane] = sum;
        __syncthreads();
        if (wave == 0 && c < length) {
#pragma unroll
            for (int w = 1; w < WAVES; w++) sum += smem[w][lane];
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

unsigned gridOf(Long blocks) { return (unsigned)(blocks < 1 ? 1 : (blocks > (1 << 20) ? (1 << 20) : blocks)); }

}  // namespace

size_t layerNormBpScratch(Long rows, Long length) { return (size_t)2 * columnSplits(rows, length) * length * sizeof(double); }

template <typename T>
void launchLayerNorm(hipStream_t s, const T *x, const RowView &xv, const T *gain, const T *bias, T *z, const RowView &zv,
                     typename Compute<T>::type *mean, typename Compute<T>::type *invStd, double epsilon) {
    typedef typename Compute<T>::type C;
    ND4J_LAUNCH((layerNormAnyKernel<T>), dim3(gridOf(xv.rows)), dim3(kRowThreads), 0, s, x, xv, gain, bias, z, zv, mean, invStd, (C)epsilon);
}

template <typename T>
void launchLayerNormBp(hipStream_t s, const T *x, const RowView &xv, const T *gain, const typename Compute<T>::type *mean,
                       const typename Compute<T>::type *invStd, const T *dz, const RowView &dzv, T *dx, const RowView &dxv, T *dGain,
                       T *dBias, void *scratch) {
    typedef typename Compute<T>::type C;
    if (dGain != nullptr || dBias != nullptr) {
        // before dx is written, which may lie where dz or x does
        const int splits = columnSplits(xv.rows, xv.length);
        const Long tiles = (xv.length + kWaveLanes - 1) / kWaveLanes;
        C *partial = reinterpret_cast<C *>(scratch);
        ND4J_LAUNCH((layerNormBpColumnsKernel<T>), dim3(gridOf(tiles * splits)), dim3(kRowThreads), 0, s, x, xv, mean, invStd, dz, dzv, partial,
                    splits);
        ND4J_LAUNCH((layerNormBpFinishKernel<T>), dim3(gridOf(tiles), 2), dim3(kRowThreads), 0, s, partial, splits, xv.length, dGain, dBias);
    }
    if (dx != nullptr && xv.rows > 0)
        ND4J_LAUNCH((layerNormBpAnyKernel<T>), dim3(gridOf(xv.rows)), dim3(kRowThreads), 0, s, x, xv, gain, mean, invStd, dz, dzv, dx, dxv);
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
