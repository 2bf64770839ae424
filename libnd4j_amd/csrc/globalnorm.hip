// The norm over all elements of many tensors, and the tensors scaled down to a largest norm.
//
//   norm = sqrt(sum of g^2),  f = maxNorm / norm where maxNorm < norm < infinity, else 1,  out = f g
//
// A norm counts as infinite where the type that the caller gets it in does not hold it, so that what the caller reads and what
// was done to the tensors agree.
//
// The tensors' elements count as one range, cut into tiles that the blocks take in turn.  A tile inside one tensor is walked
// in vectors (unaligned ones: tensors may begin anywhere), a tile that holds ends of tensors vector by vector too, every
// thread looking the tensor up for its own (a vector across tensors goes element by element): a thousand tensors of ten
// elements cost no more launches than one of ten thousand.
//
// Bound by memory: the elements are read twice and written once.  The first sweep reads with the ordinary policy, which
// leaves what fits in the last-level cache, the second reads and writes with the streaming one: 60 tensors of 124M floats
// 245 us, 6.1 TB/s of the 1.49 GB (streaming in the first sweep too took a tenth longer; ordinary loads in the second 6 %,
// and ordinary stores 14 %; the second sweep from the end of the range is as fast).  20 tensors of 100003 halves in all
// take 12.6 us, which is two launches.
//
// Squares are summed in double: the square of any float is finite there, and the order of the sum does not show in the
// result's type.  (Squares of halves are exact in float; eight of them are added there first.)  Squares of doubles have three
// sums, of elements around 1 and of those far above and below it, scaled by a power of two, so that any norm that a double holds
// comes out.
#include "launch.h"
#include "training.cuh"

namespace nd4j_amd {
namespace {

using namespace tr;

constexpr int kNormThreads = 512;
constexpr int kNormBlocks = 512;  // of the first sweep, whose sums every block of the second adds up (1024: 250 us where these take 245)

// The elements of the range: what the offsets say, and no more than the host was told.
__device__ __forceinline__ Long wholeLength(const Long *offsets, int n, Long total) {
    if (n == 0) return 0;
    return offsets[n] < total ? offsets[n] : total;
}
// The tensor i with offsets[i] <= at < offsets[i + 1], known to lie in low .. high (low where at lies before the first).
__device__ __forceinline__ int tensorAt(const Long *offsets, int low, int high, Long at) {
    while (high > low) {
        const int mid = (low + high + 1) >> 1;
        if (offsets[mid] <= at) low = mid;
        else high = mid - 1;
    }
    return low;
}

// Searches wait for one offset after the other, and for the tensor's address then, a trip to the cache each: of up to
// kStaged - 1 tensors a block copies both tables into LDS first.
constexpr int kStaged = 1024;
template <typename T> struct Tables {
    const Long *offsets;
    const T *const *in;
};
template <typename T>
__device__ __forceinline__ Tables<T> stagedTables(const T *const *in, const Long *offsets, int n, Long *stagedOffsets, const T **stagedIn) {
    Tables<T> t;
    t.offsets = offsets;
    t.in = in;
    if (n >= kStaged || n == 0) return t;
    for (int i = threadIdx.x; i <= n; i += kNormThreads) {
        stagedOffsets[i] = offsets[i];
        if (i < n) stagedIn[i] = in[i];
    }
    __syncthreads();
    t.offsets = stagedOffsets;
    t.in = stagedIn;
    return t;
}

template <typename C> __device__ __forceinline__ C smallestNormal() { return sizeof(C) == 4 ? (C)0x1p-126 : (C)0x1p-1022; }

// A sum of squares
template <typename T> struct Squares {
    double sum;
    __device__ __forceinline__ void clear() { sum = 0.0; }
    __device__ __forceinline__ void join(const Squares &o) { sum += o.sum; }
    __device__ __forceinline__ void add(T v) {
        const double d = (double)toCompute(v);
        sum += d * d;
    }
    template <int VECTORS> __device__ __forceinline__ void add(const Pack<T> (&v)[VECTORS]) {
#pragma unroll
        for (int j = 0; j < VECTORS; j++) add(v[j]);
    }
    __device__ __forceinline__ void add(const Pack<T> &v) {
        constexpr int N = Pack<T>::N;
        if constexpr (sizeof(T) == 2) {
            float eight = 0.0f;
#pragma unroll
            for (int e = 0; e < N; e++) eight += toCompute(v.v[e]) * toCompute(v.v[e]);
            sum += (double)eight;
        } else {
            double four = 0.0;
#pragma unroll
            for (int e = 0; e < N; e++) four = __builtin_fma((double)toCompute(v.v[e]), (double)toCompute(v.v[e]), four);
            sum += four;
        }
    }
    __device__ __forceinline__ bool sumIsAll() const { return true; }
    __device__ __forceinline__ double root() const { return ::sqrt(sum); }
};
// Elements beyond 2^480 are squared as 2^-600 of themselves (2^56 of the largest squares that are not scaled, 2^960, are a double
// still), those below 2^-400 as 2^600 of themselves (what is not scaled has normal squares).  NaN counts as usual, infinity as large.
template <> struct Squares<double> {
    double sum, large, small;
    __device__ __forceinline__ void clear() { sum = large = small = 0.0; }
    __device__ __forceinline__ void join(const Squares &o) {
        sum += o.sum;
        large += o.large;
        small += o.small;
    }
    __device__ __forceinline__ void add(double v) {
        const double size = ::fabs(v);
        if (size > 0x1p480) large = __builtin_fma(v * 0x1p-600, v * 0x1p-600, large);
        else if (size < 0x1p-400) small = __builtin_fma(v * 0x1p600, v * 0x1p600, small);
        else sum = __builtin_fma(v, v, sum);
    }
    // Several at once: squared as they are, if the sum says that none was large and none small that counts (looked at element by
    // element, 50M doubles took 203 us instead of 195).
    template <int VECTORS> __device__ __forceinline__ void add(const Pack<double> (&v)[VECTORS]) {
        double all = 0.0;
#pragma unroll
        for (int j = 0; j < VECTORS; j++) all = __builtin_fma(v[j].v[0], v[j].v[0], __builtin_fma(v[j].v[1], v[j].v[1], all));
        if (all >= 0x1p-740 && all <= 0x1p960) {
            sum += all;
        } else {
#pragma unroll
            for (int j = 0; j < VECTORS; j++) {
                add(v[j].v[0]);
                add(v[j].v[1]);
            }
        }
    }
    __device__ __forceinline__ bool sumIsAll() const { return large == 0.0 && small == 0.0; }
    __device__ __forceinline__ double root() const {
        if (large != 0.0) return ::sqrt(large + sum * 0x1p-600 * 0x1p-600) * 0x1p600;  // (what is small is lost beside it)
        if (sum != 0.0) return ::sqrt(sum + small * 0x1p-600 * 0x1p-600);
        return ::sqrt(small) * 0x1p-600;
    }
};
// What the blocks of the first sweep leave: their sums, and of doubles all three, NaN as the sum saying that they are needed (to
// read and add up three for every block of the second sweep took 4 % longer over 50M doubles).
template <typename T> struct Partial {
    double sums[kNormBlocks];
    Squares<double> whole[sizeof(T) == 8 ? kNormBlocks : 1];
};
struct JoinSquares {
    template <typename S> __device__ __forceinline__ S operator()(S a, S b) const {
        a.join(b);
        return a;
    }
};

template <typename T, int VECTORS>
__global__ void __launch_bounds__(kNormThreads) squaresKernel(const T *const *givenIn, const Long *givenOffsets, int n, Long total, Partial<T> *partial) {
    constexpr int N = Pack<T>::N;
    constexpr Long tile = (Long)kNormThreads * VECTORS * N;
    __shared__ Squares<T> smem[kNormThreads / kWaveLanes];
    __shared__ Long stagedOffsets[kStaged];
    __shared__ const T *stagedIn[kStaged];
    const Tables<T> tables = stagedTables<T>(givenIn, givenOffsets, n, stagedOffsets, stagedIn);
    const Long *offsets = tables.offsets;
    const T *const *in = tables.in;
    const Long whole = wholeLength(offsets, n, total);
    Squares<T> sum;
    sum.clear();
    int low = 0;  // (the tiles of a block ascend)
    for (Long t = (Long)blockIdx.x * tile; t < whole; t += (Long)gridDim.x * tile) {
        const Long end = t + tile < whole ? t + tile : whole;
        low = tensorAt(offsets, low, n - 1, t);
        const int high = end <= offsets[low + 1] ? low : tensorAt(offsets, low, n - 1, end - 1);
        if (low == high && end - t == tile && t >= offsets[low]) {
            const T *from = in[low] + (t - offsets[low]) + threadIdx.x * N;
            Pack<T> v[VECTORS];
#pragma unroll
            for (int j = 0; j < VECTORS; j++) v[j] = loadPackAnywhere(from + j * (kNormThreads * N));
            sum.add(v);
        } else {
            for (Long i = t + threadIdx.x * N; i < end; i += kNormThreads * N) {
                int k = tensorAt(offsets, low, high, i);
                if (i >= offsets[k] && i + N <= end && i + N <= offsets[k + 1]) {
                    const Pack<T> one[1] = {loadPackAnywhere(in[k] + (i - offsets[k]))};
                    sum.add(one);
                    continue;
                }
                for (Long j = i; j < i + N && j < end; j++) {
                    while (k < high && j >= offsets[k + 1]) k++;
                    if (j < offsets[k]) continue;
                    sum.add(in[k][j - offsets[k]]);
                }
            }
        }
    }
    sum = blockAll<kNormThreads>(sum, JoinSquares(), smem);
    if (threadIdx.x == 0) {
        partial->sums[blockIdx.x] = sum.sumIsAll() ? sum.sum : (double)notANumber<float>();
        if constexpr (sizeof(T) == 8) partial->whole[blockIdx.x] = sum;
    }
}

template <typename T, int VECTORS>
__global__ void __launch_bounds__(kNormThreads) clipKernel(const T *const *givenIn, T *const *out, const Long *givenOffsets, int n, Long total,
                                                           double maxNorm, typename Compute<T>::type *norm, const Partial<T> *partial, int parts) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N;
    constexpr Long tile = (Long)kNormThreads * VECTORS * N;
    __shared__ double smem[kNormThreads / kWaveLanes];
    __shared__ Long stagedOffsets[kStaged];
    __shared__ const T *stagedIn[kStaged];
    const Tables<T> tables = stagedTables<T>(givenIn, givenOffsets, n, stagedOffsets, stagedIn);
    const Long *offsets = tables.offsets;
    const T *const *in = tables.in;
    double sum = 0.0;
    for (int i = threadIdx.x; i < parts; i += kNormThreads) sum += partial->sums[i];
    double value = ::sqrt(blockAll<kNormThreads>(sum, Add(), smem));
    if constexpr (sizeof(T) == 8) {
        if (value != value) {  // (of all threads of the block, which have the same one)
            __shared__ Squares<T> wholes[kNormThreads / kWaveLanes];
            Squares<T> whole;
            whole.clear();
            for (int i = threadIdx.x; i < parts; i += kNormThreads) whole.join(partial->whole[i]);
            value = blockAll<kNormThreads>(whole, JoinSquares(), wholes).root();
        }
    }
    if (norm != nullptr && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (C)value;
    if (out == nullptr) return;
    // (a NaN norm compares false, so it leaves the factor at 1 like one that is infinite)
    const C factor = value > maxNorm && (C)value < infinite<C>() ? (C)(maxNorm / value) : (C)1;
    const Long whole = wholeLength(offsets, n, total);
    auto walk = [&](auto scaled) {
        int low = 0;
        for (Long t = (Long)blockIdx.x * tile; t < whole; t += (Long)gridDim.x * tile) {
            const Long end = t + tile < whole ? t + tile : whole;
            low = tensorAt(offsets, low, n - 1, t);
            const int high = end <= offsets[low + 1] ? low : tensorAt(offsets, low, n - 1, end - 1);
            if (low == high && end - t == tile && t >= offsets[low]) {
                const Long at = (t - offsets[low]) + threadIdx.x * N;
                const T *from = in[low] + at;
                T *to = out[low] + at;
                Pack<T> v[VECTORS];
#pragma unroll
                for (int j = 0; j < VECTORS; j++) v[j] = streamPackAnywhere(from + j * (kNormThreads * N));
#pragma unroll
                for (int j = 0; j < VECTORS; j++) {
#pragma unroll
                    for (int e = 0; e < N; e++) v[j].v[e] = fromCompute<T>(scaled(toCompute(v[j].v[e])));
                    streamPackAnywhere(to + j * (kNormThreads * N), v[j]);
                }
            } else {
                for (Long i = t + threadIdx.x * N; i < end; i += kNormThreads * N) {
                    int k = tensorAt(offsets, low, high, i);
                    if (i >= offsets[k] && i + N <= end && i + N <= offsets[k + 1]) {
                        Pack<T> v = loadPackAnywhere(in[k] + (i - offsets[k]));
#pragma unroll
                        for (int e = 0; e < N; e++) v.v[e] = fromCompute<T>(scaled(toCompute(v.v[e])));
                        storePackAnywhere(out[k] + (i - offsets[k]), v);
                        continue;
                    }
                    for (Long j = i; j < i + N && j < end; j++) {
                        while (k < high && j >= offsets[k + 1]) k++;
                        if (j < offsets[k]) continue;
                        out[k][j - offsets[k]] = fromCompute<T>(scaled(toCompute(in[k][j - offsets[k]])));
                    }
                }
            }
        }
    };
    if constexpr (sizeof(T) > 2) {
        // Of a factor below the type's normal range few bits are left, or none: it goes in two steps then, in double.  (Halves are
        // far below their range with such a factor.)
        if (factor < smallestNormal<C>()) {
            const double down = 0x1p-600, rest = maxNorm / (value * down);
            walk([=](C v) { return (C)((double)v * down * rest); });
            return;
        }
    }
    walk([=](C v) { return v * factor; });
}

}  // namespace

size_t clipByGlobalNormScratch(Long) { return sizeof(Partial<double>); }

template <typename T>
void launchClipByGlobalNorm(hipStream_t s, const T *const *in, T *const *out, const Long *offsets, int n, Long total, double maxNorm,
                            typename Compute<T>::type *norm, void *scratch) {
    Partial<T> *partial = reinterpret_cast<Partial<T> *>(scratch);
    // From 25 MB on the first sweep takes tiles of eight vectors a thread and the second tiles of four, a block each (as many blocks
    // as the first, tile after tile: 270 us where these take 245; eight vectors 250, two 294, since every block adds up the sums
    // first).  Smaller ones go in tiles of one vector, for more blocks: 6M floats 26.3 us, 27.0 in large tiles, but 8M 35.9 and 30.5.
    const Long wide = (Long)kNormThreads * 8 * Pack<T>::N, half = wide / 2, narrow = (Long)kNormThreads * Pack<T>::N;
    const dim3 block(kNormThreads);
    if (total >= wide * (kNormBlocks * 3 / 4)) {
        const int parts = gridFor(total, wide, kNormBlocks);
        ND4J_LAUNCH((squaresKernel<T, 8>), dim3(parts), block, 0, s, in, offsets, n, total, partial);
        ND4J_LAUNCH((clipKernel<T, 4>), dim3(out != nullptr ? gridFor(total, half, 1 << 20) : 1), block, 0, s, in, out, offsets, n, total, maxNorm,
                    norm, partial, parts);
    } else {
        const int parts = gridFor(total, narrow, kNormBlocks);
        ND4J_LAUNCH((squaresKernel<T, 1>), dim3(parts), block, 0, s, in, offsets, n, total, partial);
        ND4J_LAUNCH((clipKernel<T, 1>), dim3(out != nullptr ? parts : 1), block, 0, s, in, out, offsets, n, total, maxNorm, norm, partial, parts);
    }
}

#define INST(T)                                                                                                                    \
    template void launchClipByGlobalNorm<T>(hipStream_t, const T *const *, T *const *, const Long *, int, Long, double,              \
                                            Compute<T>::type *, void *);
INST(float)
INST(float16)
INST(double)
#undef INST

}  // namespace nd4j_amd
