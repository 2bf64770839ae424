// Log probabilities of given tokens, with the distribution's entropy and its likeliest alternatives, and their gradient.
//
//   m = max x,  S = sum exp(x - m),  logSum = m + log S,  logProb = (x[token] - m) - log S
//   entropy = -sum p log p = log S + sum (m - x) exp(x - m) / S     (two sums of terms >= 0: nothing cancels)
//   dx = a (delta(token) - p) - b p (log p + entropy)               for the gradients a of logProb and b of entropy
//
// A row of which every element is -infinity has no distribution: logSum -infinity, entropy 0, gradient 0.  Elements of
// -infinity in other rows have probability 0.  A NaN or +infinity makes the row's results NaN.
#include "launch.h"
#include "training.cuh"

namespace nd4j_amd {
namespace {

using namespace tr;

constexpr int kRowThreads = 256;

template <typename C> struct Entry {
    C value;
    int index;
};
template <typename C> struct Better {  // larger value first, then lower index; an index of -1 is no entry
    __device__ __forceinline__ Entry<C> operator()(Entry<C> a, Entry<C> b) const {
        if (b.index < 0) return a;
        if (a.index < 0) return b;
        return b.value > a.value || (b.value == a.value && b.index < a.index) ? b : a;
    }
};

// Any view: a block per row, element by element, and a sweep of the row for every alternative.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) tokenProbsAnyKernel(const T *x, RowView xv, const Long *tokens, TokenProbsOut<T> out) {
    typedef typename Compute<T>::type C;
    __shared__ C smem[kRowThreads / kWaveLanes];
    __shared__ Entry<C> entries[kRowThreads / kWaveLanes];
    for (Long r = blockIdx.x; r < xv.rows; r += gridDim.x) {
        const T *xr = x + r * xv.row;
        C mx = -infinite<C>();
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) mx = Largest()(mx, toCompute(xr[c * xv.el]));
        mx = blockAll<kRowThreads>(mx, Largest(), smem);
        if (mx == -infinite<C>()) mx = (C)0;
        C sum = (C)0, weighted = (C)0;
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) {
            const C d = toCompute(xr[c * xv.el]) - mx, e = m::expSoft_(d);
            sum += e;
            if (d > -infinite<C>()) weighted -= d * e;
        }
        sum = blockAll<kRowThreads>(sum, Add(), smem);
        weighted = blockAll<kRowThreads>(weighted, Add(), smem);
        const bool none = sum == (C)0;
        const C logSum = m::logSoft_(sum);
        if (threadIdx.x == 0) {
            if (out.logSum != nullptr) out.logSum[r] = mx + logSum;
            if (out.entropy != nullptr) out.entropy[r] = none ? (C)0 : logSum + weighted / sum;
            if (out.logProbs != nullptr) {
                const Long t = tokens[r];
                C lp = (C)0;
                if (t >= xv.length) lp = notANumber<C>();
                else if (t >= 0) lp = none ? -infinite<C>() : (toCompute(xr[t * xv.el]) - mx) - logSum;
                out.logProbs[r] = lp;
            }
        }
        Entry<C> last;
        last.value = infinite<C>();
        last.index = -1;
        for (int k = 0; k < out.k; k++) {
            Entry<C> best;
            best.value = (C)0;
            best.index = -1;
            for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) {
                Entry<C> e;
                e.value = toCompute(xr[c * xv.el]);
                e.index = (int)c;
                if (e.value != e.value) continue;
                if (k > 0 && !(e.value < last.value || (e.value == last.value && e.index > last.index))) continue;
                best = Better<C>()(best, e);
            }
            last = blockAll<kRowThreads>(best, Better<C>(), entries);
            if (threadIdx.x == 0) {
                out.top[r * out.k + k] = last.index;
                if (out.topLogProbs != nullptr)
                    out.topLogProbs[r * out.k + k] =
                        last.index < 0 ? notANumber<C>() : (none ? -infinite<C>() : (last.value - mx) - logSum);
            }
            if (last.index < 0) {  // fewer than k elements are numbers
                for (int j = k + 1 + (int)threadIdx.x; j < out.k; j += kRowThreads) {
                    out.top[r * out.k + j] = -1;
                    if (out.topLogProbs != nullptr) out.topLogProbs[r * out.k + j] = notANumber<C>();
                }
                break;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) tokenProbsBpAnyKernel(const T *x, RowView xv, const Long *tokens,
                                                                     const typename Compute<T>::type *logSum,
                                                                     const typename Compute<T>::type *entropy,
                                                                     const typename Compute<T>::type *dLogProbs,
                                                                     const typename Compute<T>::type *dEntropy, T *dx, RowView dxv) {
    typedef typename Compute<T>::type C;
    for (Long r = blockIdx.x; r < xv.rows; r += gridDim.x) {
        const T *xr = x + r * xv.row;
        T *dxr = dx + r * dxv.row;
        const C ls = logSum[r];
        const Long t = dLogProbs != nullptr ? tokens[r] : -1;
        C a = t < 0 ? (C)0 : dLogProbs[r];
        if (t >= xv.length) a = notANumber<C>();
        const C b = dEntropy != nullptr ? dEntropy[r] : (C)0, h = dEntropy != nullptr ? entropy[r] : (C)0;
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) {
            const C lp = toCompute(xr[c * xv.el]) - ls, p = m::expSoft_(lp);
            C d = (c == t ? a : (C)0) - a * p;
            if (dEntropy != nullptr && p != (C)0) d -= b * p * (lp + h);
            dxr[c * dxv.el] = fromCompute<T>(ls == -infinite<C>() ? (C)0 : d);
        }
    }
}

unsigned gridOf(Long blocks) { return (unsigned)(blocks < 1 ? 1 : (blocks > (1 << 20) ? (1 << 20) : blocks)); }

}  // namespace

size_t tokenLogProbsScratch(Long, Long, int) { return 0; }

template <typename T>
void launchTokenLogProbs(hipStream_t s, const T *x, const RowView &xv, const Long *tokens, const TokenProbsOut<T> &out, void *) {
    ND4J_LAUNCH((tokenProbsAnyKernel<T>), dim3(gridOf(xv.rows)), dim3(kRowThreads), 0, s, x, xv, tokens, out);
}

template <typename T>
void launchTokenLogProbsBp(hipStream_t s, const T *x, const RowView &xv, const Long *tokens, const typename Compute<T>::type *logSum,
                           const typename Compute<T>::type *entropy, const typename Compute<T>::type *dLogProbs,
                           const typename Compute<T>::type *dEntropy, T *dx, const RowView &dxv) {
    ND4J_LAUNCH((tokenProbsBpAnyKernel<T>), dim3(gridOf(xv.rows)), dim3(kRowThreads), 0, s, x, xv, tokens, logSum, entropy, dLogProbs, dEntropy,
                dx, dxv);
}

#define INST(T)                                                                                                                           \
    template void launchTokenLogProbs<T>(hipStream_t, const T *, const RowView &, const Long *, const TokenProbsOut<T> &, void *);         \
    template void launchTokenLogProbsBp<T>(hipStream_t, const T *, const RowView &, const Long *, const Compute<T>::type *,                \
                                           const Compute<T>::type *, const Compute<T>::type *, const Compute<T>::type *, T *,              \
                                           const RowView &);
INST(float)
INST(float16)
INST(double)
#undef INST

}  // namespace nd4j_amd
