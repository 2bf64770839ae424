// The norm over all elements of many tensors, and the tensors scaled down to a largest norm.
//
//   norm = sqrt(sum of g^2),  f = maxNorm / norm where maxNorm < norm < infinity, else 1,  out = f g
//
// The tensors' elements count as one range of `total` elements; a block takes the same part of it in both launches.  Squares
// are summed in double: the square of any float is finite there, and the order of the sum does not show in the result's type.
#include "launch.h"
#include "training.cuh"

namespace nd4j_amd {
namespace {

using namespace tr;

constexpr int kNormThreads = 256;
constexpr int kNormBlocks = 1024;

// The elements of the range: what the offsets say, and no more than the host was told.
__device__ __forceinline__ Long wholeLength(const Long *offsets, int n, Long total) {
    if (n == 0) return 0;
    return offsets[n] < total ? offsets[n] : total;
}
// The tensor i with offsets[i] <= at < offsets[i + 1] (at < offsets[n]); 0 where at lies before the first.
__device__ __forceinline__ int tensorAt(const Long *offsets, int n, Long at) {
    int low = 0, high = n;
    while (high - low > 1) {
        const int mid = (low + high) >> 1;
        if (offsets[mid] <= at) low = mid;
        else high = mid;
    }
    return low;
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) squaresKernel(const T *const *in, const Long *offsets, int n, Long total, double *partial) {
    __shared__ double smem[kNormThreads / kWaveLanes];
    double sum = 0.0;
    const Long end = wholeLength(offsets, n, total);
    for (Long i = (Long)blockIdx.x * kNormThreads + threadIdx.x; i < end; i += (Long)gridDim.x * kNormThreads) {
        const int k = tensorAt(offsets, n, i);
        if (i < offsets[k]) continue;
        const double v = (double)toCompute(in[k][i - offsets[k]]);
        sum += v * v;
    }
    sum = blockAll<kNormThreads>(sum, Add(), smem);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <typename T>
__global__ void __launch_bounds__(kNormThreads) clipKernel(const T *const *in, T *const *out, const Long *offsets, int n, Long total,
                                                           double maxNorm, typename Compute<T>::type *norm, const double *partial, int parts) {
    typedef typename Compute<T>::type C;
    __shared__ double smem[kNormThreads / kWaveLanes];
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += kNormThreads) sum += partial[i];
    const double whole = ::sqrt(blockAll<kNormThreads>(sum, Add(), smem));
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (C)whole;
    if (out == nullptr) return;
    // (a NaN norm compares false, so it leaves the factor at 1 like one that is infinite)
    const C factor = whole > maxNorm && whole < infinite<double>() ? (C)(maxNorm / whole) : (C)1;
    const Long end = wholeLength(offsets, n, total);
    for (Long i = (Long)blockIdx.x * kNormThreads + threadIdx.x; i < end; i += (Long)gridDim.x * kNormThreads) {
        const int k = tensorAt(offsets, n, i);
        if (i < offsets[k]) continue;
        out[k][i - offsets[k]] = fromCompute<T>(toCompute(in[k][i - offsets[k]]) * factor);
    }
}

}  // namespace

size_t clipByGlobalNormScratch(Long) { return kNormBlocks * sizeof(double); }

template <typename T>
void launchClipByGlobalNorm(hipStream_t s, const T *const *in, T *const *out, const Long *offsets, int n, Long total, double maxNorm,
                            typename Compute<T>::type *norm, void *scratch) {
    double *partial = reinterpret_cast<double *>(scratch);
    const int blocks = gridFor(total, kNormThreads, kNormBlocks);
    ND4J_LAUNCH((squaresKernel<T>), dim3(blocks), dim3(kNormThreads), 0, s, in, offsets, n, total, partial);
    ND4J_LAUNCH((clipKernel<T>), dim3(out != nullptr ? blocks : 1), dim3(kNormThreads), 0, s, in, out, offsets, n, total, maxNorm, norm, partial,
                blocks);
}

#define INST(T)                                                                                                                    \
    template void launchClipByGlobalNorm<T>(hipStream_t, const T *const *, T *const *, const Long *, int, Long, double,              \
                                            Compute<T>::type *, void *);
INST(float)
INST(float16)
INST(double)
#undef INST

}  // namespace nd4j_amd
