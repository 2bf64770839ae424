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

// Views of any other strides: a block per row, element by element, and a sweep of the row for every alternative.
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

// Views whose rows lie nearer to each other than a row's elements (an f-order matrix, as products of matrices often are):
// lanes take neighbouring rows, the waves of a block share the columns; a sweep for every alternative here too.
constexpr int kAcrossThreads = 1024, kAcrossGroups = kAcrossThreads / kWaveLanes;
template <typename T>
__global__ void __launch_bounds__(kAcrossThreads) tokenProbsAcrossKernel(const T *x, RowView xv, const Long *tokens, TokenProbsOut<T> out) {
    typedef typename Compute<T>::type C;
    __shared__ C one[kAcrossGroups][kWaveLanes], two[kAcrossGroups][kWaveLanes];
    __shared__ int indexes[kAcrossGroups][kWaveLanes];
    const int lane = threadIdx.x % kWaveLanes, group = threadIdx.x / kWaveLanes;
    for (Long r0 = (Long)blockIdx.x * kWaveLanes; r0 < xv.rows; r0 += (Long)gridDim.x * kWaveLanes) {
        const bool live = r0 + lane < xv.rows;
        const Long r = live ? r0 + lane : r0;
        const T *xr = x + r * xv.row;
        C mx = -infinite<C>();
#pragma unroll 8
        for (Long c = group; c < xv.length; c += kAcrossGroups) mx = Largest()(mx, toCompute(xr[c * xv.el]));
        __syncthreads();
        one[group][lane] = mx;
        __syncthreads();
        for (int g = 0; g < kAcrossGroups; g++) mx = Largest()(mx, one[g][lane]);
        if (mx == -infinite<C>()) mx = (C)0;
        C sum = (C)0, weighted = (C)0;
#pragma unroll 4
        for (Long c = group; c < xv.length; c += kAcrossGroups) {
            const C d = toCompute(xr[c * xv.el]) - mx, e = m::expSoft_(d);
            sum += e;
            if (d > -infinite<C>()) weighted -= d * e;
        }
        __syncthreads();
        one[group][lane] = sum;
        two[group][lane] = weighted;
        __syncthreads();
        sum = one[0][lane];
        weighted = two[0][lane];
        for (int g = 1; g < kAcrossGroups; g++) {
            sum += one[g][lane];
            weighted += two[g][lane];
        }
        const bool none = sum == (C)0;
        const C logSum = m::logSoft_(sum);
        if (live && group == 0) {
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
        bool more = true;  // (a lane whose row has no more numbers goes on with the others)
        for (int k = 0; k < out.k; k++) {
            Entry<C> best;
            best.value = (C)0;
            best.index = -1;
#pragma unroll 4
            for (Long c = group; c < xv.length; c += kAcrossGroups) {
                Entry<C> e;
                e.value = toCompute(xr[c * xv.el]);
                e.index = (int)c;
                const bool is = more && e.value == e.value && (k == 0 || e.value < last.value || (e.value == last.value && e.index > last.index));
                if (is) best = Better<C>()(best, e);
            }
            __syncthreads();
            one[group][lane] = best.value;
            indexes[group][lane] = best.index;
            __syncthreads();
            for (int g = 0; g < kAcrossGroups; g++) {
                Entry<C> e;
                e.value = one[g][lane];
                e.index = indexes[g][lane];
                best = Better<C>()(best, e);
            }
            last = best;
            more = more && last.index >= 0;
            if (live && group == 0) {
                out.top[r * out.k + k] = more ? last.index : -1;
                if (out.topLogProbs != nullptr)
                    out.topLogProbs[r * out.k + k] = !more ? notANumber<C>() : (none ? -infinite<C>() : (last.value - mx) - logSum);
            }
        }
    }
}

// ---- rows of contiguous elements, forward ------------------------------------------------------------------------------
// One sweep of a row by a block: every thread keeps the maximum of its elements, the sum of exp(x - maximum) and of
// (maximum - x) exp(x - maximum), rescaled where its next elements raise the maximum.  The alternatives cost that sweep
// nothing: if k / 4 threads of each of the block's four waves have a maximum of at least b, the row's k-th largest element
// is no less than b, and only threads whose maximum reaches b hold alternatives - k of them and a few more, where values
// differ.  Only their elements are read again, by all threads together, and those that reach b (a few more than k) find
// their places by counting.  Where rows are few they are cut into slices, whose sums and lists a second launch joins.
//
// (Keeping the best elements during the sweep, as the first form did, took 118 us over [4096, 32000] floats at k = 5, where
// the sweep alone takes 81.  This form takes 86, 6.1 TB/s.  One row of 50257 halves takes 11 us, which is two launches.)
// Short rows pay for the selection, once a row by a whole block: [20000, 5000] halves 115 us at k = 5, 52 without alternatives.

// exp for the sums: the relative error grows with |d| (a rounding of d log2 e), on terms whose share is exp(d)
__device__ __forceinline__ float expOf(float d) { return __builtin_amdgcn_exp2f(d * 1.44269502162933349609375f); }
__device__ __forceinline__ double expOf(double d) { return ::exp(d); }
__device__ __forceinline__ float fma_(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return __builtin_fma(a, b, c); }

// A value of one lane, for all of them (in scalar registers)
template <typename C> __device__ __forceinline__ C laneValue(C v, int lane) {
    constexpr int W = sizeof(C) / 4;
    struct Words { int w[W]; };
    Words in = __builtin_bit_cast(Words, v), out;
#pragma unroll
    for (int i = 0; i < W; i++) out.w[i] = __builtin_amdgcn_readlane(in.w[i], lane);
    return __builtin_bit_cast(C, out);
}
template <typename C> __device__ __forceinline__ C laneBelow(C v) {  // lane l gets lane l - 1's (lane 0 its own)
    return laneDpp<0x138>(v);
}
constexpr int kNoIndex = 0x7fffffff;
// The k best elements a wave has seen, the j-th in lane j: larger values first, lower indexes first among equals.  Places
// not taken yet hold -infinity under kNoIndex, which every element beats, one of -infinity too.
template <typename C> struct BestList {
    C value;
    int index;
    C worstValue;  // of place k - 1, in all lanes
    int worstIndex;
    int k;
    __device__ __forceinline__ void clear(int places) {
        k = places;
        value = worstValue = -infinite<C>();
        index = worstIndex = kNoIndex;
    }
    __device__ __forceinline__ bool beats(C v, int i) const { return v > worstValue || (v == worstValue && i < worstIndex); }
    // v and i are the same in all lanes, and beat the worst entry
    __device__ __forceinline__ void insert(C v, int i) {
        const int lane = threadIdx.x % kWaveLanes;
        const int place = __popcll(__ballot(value > v || (value == v && index < i)));
        const C above = laneBelow(value);
        const int aboveIndex = laneBelow(index);
        value = lane == place ? v : (lane > place ? above : value);
        index = lane == place ? i : (lane > place ? aboveIndex : index);
        worstValue = laneValue(value, k - 1);
        worstIndex = laneValue(index, k - 1);
    }
    // every lane offers an element
    __device__ __forceinline__ void offer(C v, int i, bool live) {
        unsigned long long mask = __ballot(live && beats(v, i));
        while (mask != 0ull) {
            const int from = __ffsll((unsigned long long)mask) - 1;
            insert(laneValue(v, from), laneValue(i, from));
            mask &= mask - 1;
            mask &= __ballot(live && beats(v, i));
        }
    }
};

struct Lowest {
    __device__ __forceinline__ int operator()(int a, int b) const { return a < b ? a : b; }
};

// The k best of several sorted lists, one a lane (list l: `count` places at values + l * count, indexes + l * count): the
// best of the lists' heads k times over.
template <typename C>
__device__ __forceinline__ void mergeLists(BestList<C> &best, int lists, int count, const C *values, const int *indexes) {
    const int lane = threadIdx.x % kWaveLanes;
    best.clear(count);
    int at = 0;
    C head = lane < lists ? values[lane * count] : -infinite<C>();
    int headIndex = lane < lists ? indexes[lane * count] : kNoIndex;
    for (int j = 0; j < count; j++) {
        const C top = waveAll<kWaveLanes>(head, Largest());
        bool first = headIndex != kNoIndex && head == top;
        unsigned long long mask = __ballot(first);
        if (mask == 0ull) return;  // (no list holds more: the places left are not taken)
        if ((mask & (mask - 1)) != 0ull) {
            const int lowest = waveAll<kWaveLanes>(first ? headIndex : kNoIndex, Lowest());
            first = first && headIndex == lowest;
            mask = __ballot(first);
        }
        const int index = laneValue(headIndex, __ffsll(mask) - 1);
        if (lane == j) {
            best.value = top;
            best.index = index;
        }
        if (first) {
            at++;
            head = at < count ? values[lane * count + at] : -infinite<C>();
            headIndex = at < count ? indexes[lane * count + at] : kNoIndex;
        }
    }
}

// whole numbers in the order of the values (none of them NaN)
__device__ __forceinline__ unsigned orderOf(float v) {
    const unsigned b = __builtin_bit_cast(unsigned, v);
    return (b >> 31) != 0u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long orderOf(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    return (b >> 63) != 0ull ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float valueOf(unsigned o) { return __builtin_bit_cast(float, (o >> 31) != 0u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ double valueOf(unsigned long long o) {
    return __builtin_bit_cast(double, (o >> 63) != 0ull ? o & 0x7fffffffffffffffull : ~o);
}
// the k-th largest of a wave's 64 values, by its bits from the highest on
// (down to bit `last`: a bound below it by what the lower bits may hold)
template <typename C> __device__ __forceinline__ C kthLargest(C v, int k, int last) {
    const auto mine = orderOf(v);
    auto found = mine;
    found = 0;
#pragma unroll 4
    for (int bit = (int)sizeof(C) * 8 - 1; bit >= last; bit--) {
        auto with = found;
        with |= (decltype(found))1 << bit;
        if (__popcll(__ballot(mine >= with)) >= k) found = with;
    }
    const C bound = valueOf(found);
    return bound == bound ? bound : -infinite<C>();  // (what lies below minus infinity is written like a NaN)
}

// maximum, sum of exp(x - maximum), sum of (maximum - x) exp(x - maximum)
template <typename C> struct Sums {
    C largest, sum, weighted;
    __device__ __forceinline__ void clear() {
        largest = -infinite<C>();
        sum = weighted = (C)0;
    }
    __device__ __forceinline__ void raiseTo(C to) {  // to >= largest
        if (!(to > largest)) return;
        if (largest > -infinite<C>()) {
            const C d = largest - to, f = expOf(d);
            // (from the type's lowest value d sum may overflow, and nothing of it is left)
            weighted = f > (C)0 ? (weighted - d * sum) * f : (C)0;
            sum *= f;
        }
        largest = to;
    }
    __device__ __forceinline__ void add(Sums o) {
        const C to = Largest()(largest, o.largest);
        raiseTo(to);
        o.raiseTo(to);
        sum += o.sum;
        weighted += o.weighted;
    }
};

template <typename T>
__device__ __forceinline__ void writeRow(Long length, Long r, Long token, typename Compute<T>::type tokenValue, const TokenProbsOut<T> &out,
                                         const Sums<typename Compute<T>::type> &s) {
    typedef typename Compute<T>::type C;
    const bool none = s.sum == (C)0;
    const C from = s.largest > -infinite<C>() ? s.largest : (C)0, logSum = m::logSoft_(s.sum);
    if (threadIdx.x % kWaveLanes == 0) {
        if (out.logSum != nullptr) out.logSum[r] = from + logSum;
        if (out.entropy != nullptr) out.entropy[r] = none ? (C)0 : logSum + s.weighted / s.sum;
        if (out.logProbs != nullptr) {
            C lp = (C)0;
            if (token >= length) lp = notANumber<C>();
            else if (token >= 0) lp = none ? -infinite<C>() : (tokenValue - from) - logSum;
            out.logProbs[r] = lp;
        }
    }
}
template <typename T>
__device__ __forceinline__ void writeBest(Long r, const TokenProbsOut<T> &out, const Sums<typename Compute<T>::type> &s,
                                          const BestList<typename Compute<T>::type> &best) {
    typedef typename Compute<T>::type C;
    const int lane = threadIdx.x % kWaveLanes;
    if (lane >= out.k) return;
    const bool none = s.sum == (C)0, entry = best.index != kNoIndex;
    const C from = s.largest > -infinite<C>() ? s.largest : (C)0, logSum = m::logSoft_(s.sum);
    out.top[r * out.k + lane] = entry ? best.index : -1;
    if (out.topLogProbs != nullptr)
        out.topLogProbs[r * out.k + lane] = !entry ? notANumber<C>() : (none ? -infinite<C>() : (best.value - from) - logSum);
}

// A slice's tiles fall into at most this many spans of equal length, of which every thread keeps its maxima
constexpr int kSpans = 16;

// A slice of a row leaves 3 + 2 k values for the join: its sums, and its list's values and indexes.

template <typename T, int THREADS, int VECTORS, bool ENTROPY, bool TOP>
__global__ void __launch_bounds__(THREADS) tokenProbsRowsKernel(const T *x, RowView xv, const Long *tokens, TokenProbsOut<T> out,
                                                                typename Compute<T>::type *scratch, int slices, int sliceLength) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N, WAVES = THREADS / kWaveLanes, ROUND = THREADS * N, TILE = ROUND * VECTORS;
    __shared__ Sums<C> waveSums[WAVES];
    __shared__ C bounds[WAVES];
    __shared__ C maxima[TOP ? kSpans : 1][THREADS];  // of a thread's elements in each span of tiles
    __shared__ int hotCount, hot[TOP ? THREADS : 1];  // (span, thread) pairs that reach the bound
    __shared__ int found, candidateIndexes[TOP ? THREADS : 1];
    __shared__ C candidates[TOP ? THREADS : 1];
    extern __shared__ __align__(16) char dynamicLds[];
    C *values = reinterpret_cast<C *>(dynamicLds);  // [WAVES][k], and as many indexes behind them
    int *indexes = reinterpret_cast<int *>(values + WAVES * out.k);
    const int lane = threadIdx.x % kWaveLanes, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveLanes);
    for (Long work = blockIdx.x; work < xv.rows * slices; work += gridDim.x) {
        const Long r = work / slices;
        const int slice = (int)(work - r * slices);
        const int begin = slice * sliceLength, end = (int)(begin + (Long)sliceLength < xv.length ? begin + sliceLength : xv.length);
        const T *xr = x + r * xv.row;
        const Long token = slices == 1 && wave == 0 && out.logProbs != nullptr ? tokens[r] : -1;
        const C tokenValue = token >= 0 && token < xv.length ? toCompute(xr[token]) : (C)0;
        Sums<C> s;
        s.clear();
        const int tiles = (end - begin + TILE - 1) / TILE, spanTiles = (tiles + kSpans - 1) / kSpans;
        int span = 0, spanLeft = spanTiles;
        C spanLargest = -infinite<C>();
        int lastShift = 0;  // by which the first vector of the last tile lies in front of its place
        Pack<T> v[VECTORS];
        for (int t = begin; t < end; t += TILE) {
            if (t + TILE <= end) {
#pragma unroll
                for (int j = 0; j < VECTORS; j++) v[j] = streamPackAnywhere(xr + t + (j * THREADS + (int)threadIdx.x) * N);
            } else if (end - begin >= N) {
                // a vector that passes the end is the last whole one: its elements that are another lane's add nothing
                int shift[VECTORS];
#pragma unroll
                for (int j = 0; j < VECTORS; j++) {
                    const int c = t + (j * THREADS + (int)threadIdx.x) * N, at = c < end - N ? c : end - N;
                    shift[j] = c - at;
                    v[j] = loadPackAnywhere(xr + at);
                }
#pragma unroll
                for (int j = 0; j < VECTORS; j++)
                    if (shift[j] > 0) {
#pragma unroll
                        for (int e = 0; e < N; e++)
                            if (e < shift[j]) v[j].v[e] = fromCompute<T>(-infinite<C>());
                    }
                lastShift = shift[0];
            } else {
#pragma unroll
                for (int j = 0; j < VECTORS; j++) {
                    const int c = t + (j * THREADS + (int)threadIdx.x) * N;
#pragma unroll
                    for (int e = 0; e < N; e++) v[j].v[e] = c + e < end ? xr[c + e] : fromCompute<T>(-infinite<C>());
                }
            }
            // the wave's vectors with elements of the row: in a last tile most may have none, which shows where the arithmetic takes as
            // long as the memory ([20000, 5000] halves 70 -> 53 us; floats 2 % longer)
            const int here = end - t - wave * kWaveLanes * N, packs = sizeof(T) == 2 ? (here + ROUND - 1) / ROUND : VECTORS;
            C tileLargest = -infinite<C>();
#pragma unroll
            for (int j = 0; j < VECTORS; j++)
                if (j < packs) {
#pragma unroll
                    for (int e = 0; e < N; e++) tileLargest = Largest()(tileLargest, toCompute(v[j].v[e]));
                }
            if (TOP) {
                spanLargest = Largest()(spanLargest, tileLargest);
                maxima[span][threadIdx.x] = spanLargest;
                if (--spanLeft == 0) {
                    span++;
                    spanLeft = spanTiles;
                    spanLargest = -infinite<C>();
                }
            }
            s.raiseTo(tileLargest);
            const C from = s.largest > -infinite<C>() ? s.largest : (C)0;
#pragma unroll
            for (int j = 0; j < VECTORS; j++)
                if (j < packs) {
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const C d = toCompute(v[j].v[e]) - from, p = expOf(d);
                        s.sum += p;
                        // (0 for an element of -infinity, where d p is not a number)
                        if (ENTROPY) s.weighted = fma_(Largest()(d, (C)-1e30f), -p, s.weighted);
                    }
                }
        }
        const C own = s.largest;
        // the wave's sums: everything relative to the largest maximum first
        s.raiseTo(waveAll<kWaveLanes>(s.largest, Largest()));
        s.sum = waveAll<kWaveLanes>(s.sum, Add());
        if (ENTROPY) s.weighted = waveAll<kWaveLanes>(s.weighted, Add());
        __syncthreads();  // the arrays may still be read from the round before
        if (lane == 0) waveSums[wave] = s;
        BestList<C> best;
        if (TOP) {
            constexpr int LAST = sizeof(T) == 2 ? 13 : 0;  // (a half's bits end there)
            const C waveBound = kthLargest(own, (out.k + WAVES - 1) / WAVES, LAST);
            if (lane == 0) bounds[wave] = waveBound;
            if (threadIdx.x == 0) found = hotCount = 0;
            __syncthreads();
            C bound = bounds[0];
#pragma unroll
            for (int w = 1; w < WAVES; w++) bound = bounds[w] < bound ? bounds[w] : bound;
            if (WAVES > 1 && bound == -infinite<C>()) {
                // A wave without as many elements, as at a row's end: the waves that have one in every lane share k, and the k-th
                // largest of any one wave will do too.  (The second alone lets half of a short slice pass at k = 64.)
                const bool full = __ballot(own > -infinite<C>()) == ~0ull;
                const C alone = kthLargest(own, out.k, LAST);
                __syncthreads();
                if (lane == 0) bounds[wave] = full ? (C)1 : (C)0;
                __syncthreads();
                int fulls = 0;
#pragma unroll
                for (int w = 0; w < WAVES; w++) fulls += bounds[w] > (C)0 ? 1 : 0;
                const C shared = full ? kthLargest(own, (out.k + fulls - 1) / fulls, LAST) : infinite<C>();
                __syncthreads();
                if (lane == 0) bounds[wave] = shared;
                __syncthreads();
                C least = bounds[0];
#pragma unroll
                for (int w = 1; w < WAVES; w++) least = bounds[w] < least ? bounds[w] : least;
                __syncthreads();
                if (lane == 0) bounds[wave] = alone;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WAVES; w++) bound = Largest()(bound, bounds[w]);
                if (fulls > 0) bound = Largest()(bound, least);
            }
            const bool held = VECTORS == 1 && tiles == 1;  // every thread's elements are in its registers still
            if (!held) {
                if (own >= bound) {
                    for (int k = 0; k * spanTiles < tiles; k++)
                        if (maxima[k][threadIdx.x] >= bound) {
                            const int place = atomicAdd(&hotCount, 1);
                            if (place < THREADS) hot[place] = k * THREADS + (int)threadIdx.x;
                        }
                }
                __syncthreads();
            }
            // The vectors of the hot pairs - where there are too many of them, all vectors - are the items.  The elements that
            // reach the bound are gathered, and each counts those that come before it, which is its place.
            const int hots = hotCount, perPair = spanTiles * VECTORS;
            const bool few = !held && hots <= THREADS;
            const Long items = few ? (Long)hots * perPair : ((Long)end - begin + N - 1) / N;
            auto itemAt = [&](Long item, int &c, Pack<T> &v) {
                c = end;
                if (item < items) {
                    Long at = item;
                    if (few) {
                        const int h = (int)item / perPair, q = (int)item - h * perPair, pair = hot[h], k = pair / THREADS;
                        at = (Long)(k * perPair + q) * THREADS + pair % THREADS;
                    }
                    if (at * N < end - begin) c = begin + (int)at * N;
                }
                if (c + N <= end) {
                    v = loadPackAnywhere(xr + c);
                } else {
#pragma unroll
                    for (int e = 0; e < N; e++) v.v[e] = c + e < end ? xr[c + e] : fromCompute<T>((C)0);
                }
            };
            auto gather = [&](int c, int first, const Pack<T> &from) {
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const C value = toCompute(from.v[e]);
                    const bool is = e >= first && c + e < end && value >= bound;
                    const unsigned long long which = __ballot(is);
                    if (which == 0ull) continue;
                    int place = 0;
                    if (lane == 0) place = atomicAdd(&found, __popcll(which));
                    place = __builtin_amdgcn_readfirstlane(place) + __popcll(which & ((1ull << lane) - 1));
                    if (is && place < THREADS) {
                        candidates[place] = value;
                        candidateIndexes[place] = c + e;
                    }
                }
            };
            if (held) {
                gather(begin + (int)threadIdx.x * N - lastShift, lastShift, v[0]);
            } else {
                for (Long i = wave * kWaveLanes; i < items; i += THREADS) {
                    int c;
                    Pack<T> item;
                    itemAt(i + lane, c, item);
                    gather(c, 0, item);
                    if (*(volatile int *)&found > THREADS) break;
                }
            }
            __syncthreads();
            const int count = found;
            if (count <= THREADS) {
                C value = -infinite<C>();
                int index = kNoIndex, place = threadIdx.x;
                if ((int)threadIdx.x < count) {
                    value = candidates[threadIdx.x];
                    index = candidateIndexes[threadIdx.x];
                    place = 0;
#pragma unroll 4
                    for (int j = 0; j < count; j++) {
                        const C other = candidates[j];
                        const int otherIndex = candidateIndexes[j];
                        place += (int)(other > value) | ((int)(other == value) & (int)(otherIndex < index));
                    }
                }
                if (place < out.k) {
                    values[place] = value;
                    indexes[place] = index;
                }
                __syncthreads();
                best.value = lane < out.k ? values[lane] : -infinite<C>();
                best.index = lane < out.k ? indexes[lane] : kNoIndex;
            } else {
                // More than that are as large as the bound - rows of few different values: every wave keeps a list of its items,
                // and the lists are merged.
                best.clear(out.k);
                for (Long i = wave * kWaveLanes; i < items; i += THREADS) {
                    int c;
                    Pack<T> item;
                    itemAt(i + lane, c, item);
                    unsigned offers = 0;  // a bit per element
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const C value = toCompute(item.v[e]);
                        if (c + e < end && value >= bound && best.beats(value, c + e)) offers |= 1u << e;
                    }
                    while (__ballot(offers != 0u) != 0ull) {
                        const int which = __ffs((int)offers) - 1;
                        C value = -infinite<C>();
#pragma unroll
                        for (int e = 0; e < N; e++)
                            if (e == which) value = toCompute(item.v[e]);
                        best.offer(value, c + which, offers != 0u);
                        offers &= offers - 1;
                    }
                }
                if (WAVES > 1) {
                    if (lane < out.k) {
                        values[wave * out.k + lane] = best.value;
                        indexes[wave * out.k + lane] = best.index;
                    }
                    __syncthreads();
                    if (wave == 0) mergeLists<C>(best, WAVES, out.k, values, indexes);
                }
            }
        } else if (WAVES > 1) {
            __syncthreads();
        }
        if (wave != 0) continue;
#pragma unroll
        for (int w = 1; w < WAVES; w++) s.add(waveSums[w]);
        if (slices == 1) {
            writeRow<T>(xv.length, r, token, tokenValue, out, s);
            if (TOP) writeBest<T>(r, out, s, best);
        } else {
            C *to = scratch + (size_t)work * (3 + 2 * out.k);
            if (lane < 3) to[lane] = lane == 0 ? s.largest : (lane == 1 ? s.sum : s.weighted);
            if (TOP && lane < out.k) {
                to[3 + lane] = best.value;
                reinterpret_cast<int *>(to + 3 + out.k)[lane] = best.index;
            }
        }
    }
}

// A wave takes a row and joins its slices, of which there are at most kMostSlices: one a lane.  (Of 200 list entries the best
// eight by merging take 2.4 us; counting, as above, took 10.)
constexpr int kMostSlices = kWaveLanes;
template <typename T, bool TOP>
__global__ void __launch_bounds__(kWaveLanes) tokenProbsJoinKernel(const T *x, RowView xv, const Long *tokens, TokenProbsOut<T> out,
                                                                   const typename Compute<T>::type *scratch, int slices) {
    typedef typename Compute<T>::type C;
    extern __shared__ __align__(16) char dynamicLds[];
    const int lane = threadIdx.x, entries = slices * out.k, each = 3 + 2 * out.k;
    C *values = reinterpret_cast<C *>(dynamicLds);  // [slices][k], and as many indexes behind them
    int *indexes = reinterpret_cast<int *>(values + entries);
    for (Long r = blockIdx.x; r < xv.rows; r += gridDim.x) {
        const C *from = scratch + (size_t)r * slices * each;
        // (everything that has to come from memory is asked for before anything waits)
        const Long token = out.logProbs != nullptr ? tokens[r] : -1;
        const C tokenValue = token >= 0 && token < xv.length ? toCompute(x[r * xv.row + token]) : (C)0;
        Sums<C> s;
        s.clear();
        if (lane < slices) {
            s.largest = from[lane * each];
            s.sum = from[lane * each + 1];
            s.weighted = from[lane * each + 2];
        }
        if (TOP) {
            __syncthreads();
#pragma unroll 4
            for (int i = lane; i < entries; i += kWaveLanes) {
                const int slice = i / out.k, place = i - slice * out.k;
                values[i] = from[slice * each + 3 + place];
                indexes[i] = reinterpret_cast<const int *>(from + slice * each + 3 + out.k)[place];
            }
            __syncthreads();
        }
        s.raiseTo(waveAll<kWaveLanes>(s.largest, Largest()));
        s.sum = waveAll<kWaveLanes>(s.sum, Add());
        s.weighted = waveAll<kWaveLanes>(s.weighted, Add());
        writeRow<T>(xv.length, r, token, tokenValue, out, s);
        if (TOP) {
            BestList<C> best;
            mergeLists<C>(best, slices, out.k, values, indexes);
            writeBest<T>(r, out, s, best);
        }
    }
}

// ---- backward ----------------------------------------------------------------------------------------------------------
// A row is zero if it has no distribution, or if its token is padding and no entropy is differentiated: padded places may hold
// anything, NaN too, which 0 times p would let through.
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
        const bool zero = ls == -infinite<C>() || (t < 0 && dEntropy == nullptr);
        for (Long c = threadIdx.x; c < xv.length; c += kRowThreads) {
            const C lp = toCompute(xr[c * xv.el]) - ls, p = m::expSoft_(lp);
            C d = (c == t ? a : (C)0) - a * p;
            if (dEntropy != nullptr && p != (C)0) d -= b * p * (lp + h);
            dxr[c * dxv.el] = fromCompute<T>(zero ? (C)0 : d);
        }
    }
}

// Views whose rows lie nearer to each other than a row's elements: lanes take neighbouring rows, a wave a stretch of columns.
constexpr int kAcrossColumns = 64;
template <typename T>
__global__ void __launch_bounds__(kRowThreads) tokenProbsBpAcrossKernel(const T *x, RowView xv, const Long *tokens,
                                                                        const typename Compute<T>::type *logSum,
                                                                        const typename Compute<T>::type *entropy,
                                                                        const typename Compute<T>::type *dLogProbs,
                                                                        const typename Compute<T>::type *dEntropy, T *dx, RowView dxv,
                                                                        Long rowTiles) {
    typedef typename Compute<T>::type C;
    constexpr int WAVES = kRowThreads / kWaveLanes;
    const int lane = threadIdx.x % kWaveLanes, wave = threadIdx.x / kWaveLanes;
    const Long stretches = (xv.length + kAcrossColumns - 1) / kAcrossColumns;
    for (Long work = (Long)blockIdx.x * WAVES + wave; work < rowTiles * stretches; work += (Long)gridDim.x * WAVES) {
        const Long r = work % rowTiles * kWaveLanes + lane, begin = work / rowTiles * kAcrossColumns;
        const Long end = begin + kAcrossColumns < xv.length ? begin + kAcrossColumns : xv.length;
        if (r >= xv.rows) continue;
        const C ls = logSum[r];
        const Long t = dLogProbs != nullptr ? tokens[r] : -1;
        C a = t < 0 ? (C)0 : dLogProbs[r];
        if (t >= xv.length) a = notANumber<C>();
        const C b = dEntropy != nullptr ? dEntropy[r] : (C)0, h = dEntropy != nullptr ? entropy[r] : (C)0;
        const bool zero = ls == -infinite<C>() || (t < 0 && dEntropy == nullptr);
#pragma unroll 4
        for (Long c = begin; c < end; c++) {
            const C lp = toCompute(x[r * xv.row + c * xv.el]) - ls, p = m::expSoft_(lp);
            C d = (c == t ? a : (C)0) - a * p;
            if (dEntropy != nullptr && p != (C)0) d -= b * p * (lp + h);
            dx[r * dxv.row + c * dxv.el] = fromCompute<T>(zero ? (C)0 : d);
        }
    }
}

// Rows of contiguous elements: a team of a wave or a block takes a stretch of a row, kBpVectors vectors a lane.  Bound by
// memory: [4096, 50257] halves, whose rows begin anywhere, 140 us, 5.9 TB/s (with four vectors a lane 148).
constexpr int kBpVectors = 2;
template <typename T, int TEAM, bool ENTROPY>
__global__ void __launch_bounds__(kRowThreads) tokenProbsBpRowsKernel(const T *x, RowView xv, const Long *tokens,
                                                                      const typename Compute<T>::type *logSum,
                                                                      const typename Compute<T>::type *entropy,
                                                                      const typename Compute<T>::type *dLogProbs,
                                                                      const typename Compute<T>::type *dEntropy, T *dx, RowView dxv,
                                                                      int stretches, int stretch) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N, VECTORS = kBpVectors, TEAMS = kRowThreads / TEAM, ROUND = TEAM * N * VECTORS;
    const int lane = threadIdx.x % TEAM, team = TEAM == kRowThreads ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM);
    for (Long work = (Long)blockIdx.x * TEAMS + team; work < xv.rows * stretches; work += (Long)gridDim.x * TEAMS) {
        const Long r = work / stretches;
        const int begin = (int)(work - r * stretches) * stretch, end = (int)(begin + (Long)stretch < xv.length ? begin + stretch : xv.length);
        const T *xr = x + r * xv.row;
        T *dxr = dx + r * dxv.row;
        const C ls = logSum[r];
        const Long t = dLogProbs != nullptr ? tokens[r] : -1;
        C a = t < 0 ? (C)0 : dLogProbs[r];
        if (t >= xv.length) a = notANumber<C>();
        const C b = ENTROPY ? dEntropy[r] : (C)0, h = ENTROPY ? entropy[r] : (C)0;
        const bool zero = ls == -infinite<C>() || (t < 0 && !ENTROPY);
        auto gradient = [&](C v) {
            // (a half keeps 2^-11 of it; of what is stored in more bits, expOf would be 15 x 2^-24 off at a log probability of -20, and
            // 0 where p is subnormal: [4096,32000] floats 168 us with the exact one, 165 with expOf)
            const C lp = v - ls, p = sizeof(T) == 2 ? expOf(lp) : m::expSoft_(lp);
            C d = -a * p;
            if (ENTROPY) d -= p != (C)0 ? b * p * (lp + h) : (C)0;
            return zero ? (C)0 : d;
        };
        for (int c0 = begin; c0 < end; c0 += ROUND) {
            const bool hasToken = t >= c0 && t < (Long)c0 + ROUND && !zero;
            if (c0 + (Long)ROUND <= end) {
                Pack<T> v[VECTORS];
#pragma unroll
                for (int j = 0; j < VECTORS; j++) v[j] = streamPackAnywhere(xr + c0 + (j * TEAM + lane) * N);
#pragma unroll
                for (int j = 0; j < VECTORS; j++) {
                    const int c = c0 + (j * TEAM + lane) * N;
                    C d[N];
#pragma unroll
                    for (int e = 0; e < N; e++) d[e] = gradient(toCompute(v[j].v[e]));
                    if (hasToken) {
#pragma unroll
                        for (int e = 0; e < N; e++) d[e] += c + e == t ? a : (C)0;
                    }
#pragma unroll
                    for (int e = 0; e < N; e++) v[j].v[e] = fromCompute<T>(d[e]);
                    streamPackAnywhere(dxr + c, v[j]);
                }
            } else {
                for (int c = c0 + lane * N; c < end; c += TEAM * N) {
                    if (c + N <= end) {
                        Pack<T> v = streamPackAnywhere(xr + c);
#pragma unroll
                        for (int e = 0; e < N; e++) v.v[e] = fromCompute<T>(gradient(toCompute(v.v[e])) + (hasToken && c + e == t ? a : (C)0));
                        streamPackAnywhere(dxr + c, v);
                    } else {
                        for (int i = c; i < end; i++)
                            dxr[i] = fromCompute<T>(gradient(toCompute(xr[i])) + (hasToken && i == t ? a : (C)0));
                    }
                }
            }
        }
    }
}

unsigned gridOf(Long blocks) { return (unsigned)(blocks < 1 ? 1 : (blocks > (1 << 20) ? (1 << 20) : blocks)); }

}  // namespace

namespace {

// The slices of a row: rows alone fill the chip from kEnoughBlocks on; fewer are cut into equal slices of whole rounds of a
// block.  `vectors`: 16-byte vectors a thread and round, four for the most in flight, one where that leaves too few blocks.
// Rows of up to eight vectors a lane of one wave are a wave's, when there are enough of them.
constexpr Long kEnoughBlocks = 1024;
struct Cut {
    int threads, vectors, slices, sliceLength;
};
Cut cutOf(Long rows, Long length, int perVector) {
    Cut c;
    c.threads = rows >= kEnoughBlocks && length <= (Long)kWaveLanes * perVector * 8 ? kWaveLanes : kRowThreads;
    const Long wide = (Long)c.threads * perVector * 4;
    c.vectors = rows * ((length + wide - 1) / wide) >= kEnoughBlocks ? 4 : 1;
    const Long round = (Long)c.threads * perVector * c.vectors, most = (length + round - 1) / round;
    Long slices = (kEnoughBlocks + rows - 1) / rows;
    if (slices > kMostSlices) slices = kMostSlices;
    if (slices > most) slices = most;
    const Long rounds = (most + slices - 1) / slices;
    c.slices = (int)((most + rounds - 1) / rounds);
    c.sliceLength = c.slices == 1 ? (int)length : (int)(rounds * round);
    return c;
}

template <typename T, int THREADS, int VECTORS>
void runTokenProbs(hipStream_t s, const T *x, const RowView &xv, const Long *tokens, const TokenProbsOut<T> &out,
                   typename Compute<T>::type *scratch, const Cut &cut) {
    typedef typename Compute<T>::type C;
    const dim3 grid(gridOf(xv.rows * cut.slices)), block(THREADS);
    const size_t lds = (size_t)(THREADS / kWaveLanes) * out.k * (sizeof(C) + sizeof(int));
#define RUN(ENTROPY, TOP)                                                                                                              \
    ND4J_LAUNCH((tokenProbsRowsKernel<T, THREADS, VECTORS, ENTROPY, TOP>), grid, block, lds, s, x, xv, tokens, out, scratch, cut.slices, \
                cut.sliceLength)
    if (out.entropy != nullptr) {
        if (out.k > 0) RUN(true, true);
        else RUN(true, false);
    } else {
        if (out.k > 0) RUN(false, true);
        else RUN(false, false);
    }
#undef RUN
}

}  // namespace

// (Bounded over the types: a double's rounds are the shortest, so its rows are cut into the most slices.)
size_t tokenLogProbsScratch(Long rows, Long length, int k) {
    if (rows <= 0 || rows >= kEnoughBlocks) return 0;
    const Long round = (Long)kRowThreads * 2, most = (length + round - 1) / round;
    Long slices = (kEnoughBlocks + rows - 1) / rows;
    if (slices > kMostSlices) slices = kMostSlices;
    if (slices > most) slices = most;
    return slices <= 1 ? 0 : (size_t)rows * slices * (3 + 2 * k) * sizeof(double);
}

template <typename T>
void launchTokenLogProbs(hipStream_t s, const T *x, const RowView &xv, const Long *tokens, const TokenProbsOut<T> &out, void *scratch) {
    typedef typename Compute<T>::type C;
    if (xv.el == 1) {
        const Cut cut = cutOf(xv.rows, xv.length, Pack<T>::N);
        C *work = reinterpret_cast<C *>(scratch);
        if (cut.threads == kWaveLanes) runTokenProbs<T, kWaveLanes, 4>(s, x, xv, tokens, out, work, cut);
        else if (cut.vectors == 4) runTokenProbs<T, kRowThreads, 4>(s, x, xv, tokens, out, work, cut);
        else runTokenProbs<T, kRowThreads, 1>(s, x, xv, tokens, out, work, cut);
        if (cut.slices > 1) {
            const dim3 grid(gridOf(xv.rows)), block(kWaveLanes);
            const size_t lds = (size_t)cut.slices * out.k * (sizeof(C) + sizeof(int));
            if (out.k > 0) ND4J_LAUNCH((tokenProbsJoinKernel<T, true>), grid, block, lds, s, x, xv, tokens, out, work, cut.slices);
            else ND4J_LAUNCH((tokenProbsJoinKernel<T, false>), grid, block, 0, s, x, xv, tokens, out, work, cut.slices);
        }
        return;
    }
    if (rowsAreNear(xv)) {
        ND4J_LAUNCH((tokenProbsAcrossKernel<T>), dim3(gridOf((xv.rows + kWaveLanes - 1) / kWaveLanes)), dim3(kAcrossThreads), 0, s, x, xv, tokens, out);
        return;
    }
    ND4J_LAUNCH((tokenProbsAnyKernel<T>), dim3(gridOf(xv.rows)), dim3(kRowThreads), 0, s, x, xv, tokens, out);
}

template <typename T>
void launchTokenLogProbsBp(hipStream_t s, const T *x, const RowView &xv, const Long *tokens, const typename Compute<T>::type *logSum,
                           const typename Compute<T>::type *entropy, const typename Compute<T>::type *dLogProbs,
                           const typename Compute<T>::type *dEntropy, T *dx, const RowView &dxv) {
    if (xv.el == 1 && dxv.el == 1) {
        // a wave for rows of up to one round of a wave, else a block for every round of a block
        const bool waves = xv.length <= (Long)kWaveLanes * Pack<T>::N * kBpVectors;
        const int stretch = waves ? (int)xv.length : kRowThreads * Pack<T>::N * kBpVectors, stretches = (int)((xv.length + stretch - 1) / stretch);
        const Long teams = xv.rows * stretches;
        const dim3 grid(gridOf(waves ? (teams + 3) / 4 : teams)), block(kRowThreads);
#define RUN(TEAM, ENTROPY)                                                                                                                 \
    ND4J_LAUNCH((tokenProbsBpRowsKernel<T, TEAM, ENTROPY>), grid, block, 0, s, x, xv, tokens, logSum, entropy, dLogProbs, dEntropy, dx, dxv, \
                stretches, stretch)
        if (waves) {
            if (dEntropy != nullptr) RUN(kWaveLanes, true);
            else RUN(kWaveLanes, false);
        } else {
            if (dEntropy != nullptr) RUN(kRowThreads, true);
            else RUN(kRowThreads, false);
        }
#undef RUN
        return;
    }
    if (rowsAreNear(xv) && rowsAreNear(dxv)) {
        const Long rowTiles = (xv.rows + kWaveLanes - 1) / kWaveLanes, work = rowTiles * ((xv.length + kAcrossColumns - 1) / kAcrossColumns);
        ND4J_LAUNCH((tokenProbsBpAcrossKernel<T>), dim3(gridOf((work + 3) / 4)), dim3(kRowThreads), 0, s, x, xv, tokens, logSum, entropy, dLogProbs,
                    dEntropy, dx, dxv, rowTiles);
        return;
    }
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
