// Rows of a table looked up by token and scaled, and the table's gradient.
//
//   z[i] = scale * table[tokens[i]],   dTable[v] = scale * sum of dz[i] over the i with tokens[i] == v
//
// The gradient sorts the tokens (stably, so that equal tokens stay in the order of their positions), cuts the sorted list
// into chunks of equal length, sums every run of equal tokens inside a chunk in a wave's registers, and joins the runs that
// cross chunks in the chunks' order: no atomics on values, the same bits from every run, and a token that comes a hundred
// thousand times is shared by many waves.  Sums are held in the compute type and rounded to the storage type once.
//
// The sort's launches are a few small blocks that wait for memory; unless the gradient is added onto what the table holds,
// the rest of the chip clears the table meanwhile, the rows that get sums later among them (they are few where clearing
// takes long: clearing only the others, behind the sort, made [16384 of 32000, 768] floats 65 us).  Those take 40 us: the sort's
// four launches 23, of which clearing 98 MB needs 15, the sums 14, the join 4, all with a launch's latency in them.  Up to 4096
// tokens it is three launches, 14 us for 257 tokens.
#include "launch.h"
#include "training.cuh"

namespace nd4j_amd {
namespace {

using namespace tr;

constexpr int kThreads = 256;

// Any view: a thread per element, neighbouring threads along the dimension in which z's elements are nearer to each other.
template <typename T>
__global__ void __launch_bounds__(kThreads) embeddingAnyKernel(const T *table, RowView tv, const Long *tokens, T *z, RowView zv,
                                                               typename Compute<T>::type scale, bool rowsFirst) {
    typedef typename Compute<T>::type C;
    const Long total = zv.rows * zv.length;
    for (Long i = (Long)blockIdx.x * kThreads + threadIdx.x; i < total; i += (Long)gridDim.x * kThreads) {
        const Long r = rowsFirst ? i % zv.rows : i / zv.length, c = rowsFirst ? i / zv.rows : i - r * zv.length, t = tokens[r];
        C v = t < 0 ? (C)0 : notANumber<C>();
        if (t >= 0 && t < tv.rows) v = toCompute(table[t * tv.row + c * tv.el]) * scale;
        z[r * zv.row + c * zv.el] = fromCompute<T>(v);
    }
}

// Rows of contiguous elements: a thread takes vectors of 16 bytes of the rows as they lie behind each other, kInFlight of
// them at a time, since each waits for its token first and for the table then.  Bound by memory: 32768 rows of 1024 halves
// 16.3 us, 8.2 TB/s of what it reads and writes, of which the frequent rows come from the caches (eight at a time: 19.1 us).
constexpr int kInFlight = 2;
constexpr int kRowBlocks = 1 << 22;  // (as many as there are turns: with at most 8192 blocks 65536 rows of 4096 floats took 319 us, now 284)
template <typename T>
__global__ void __launch_bounds__(kThreads) embeddingRowsKernel(const T *table, RowView tv, const Long *tokens, T *z, RowView zv,
                                                                typename Compute<T>::type scale, FastDiv perRow, unsigned units) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N;
    const int length = (int)zv.length;
    const unsigned step = gridDim.x * kThreads;
    for (unsigned long long first = (unsigned long long)blockIdx.x * kThreads + threadIdx.x; first < units; first += (unsigned long long)step * kInFlight) {
        unsigned row[kInFlight];
        int c[kInFlight];
        Long t[kInFlight];
        Pack<T> v[kInFlight];
#pragma unroll
        for (int k = 0; k < kInFlight; k++) {
            const unsigned long long u = first + (unsigned long long)k * step;
            unsigned vec;
            row[k] = perRow.divmod(u < units ? (unsigned)u : (unsigned)first, vec);  // (behind the end: the first one again)
            c[k] = (int)vec * N;
            t[k] = tokens[row[k]];
        }
#pragma unroll
        for (int k = 0; k < kInFlight; k++) {
            const T *from = table + (t[k] >= 0 && t[k] < tv.rows ? t[k] : 0) * tv.row + c[k];
            if (c[k] + N <= length) {
                v[k] = loadPackAnywhere(from);
            } else {
#pragma unroll
                for (int e = 0; e < N; e++) v[k].v[e] = c[k] + e < length ? from[e] : fromCompute<T>((C)0);
            }
        }
#pragma unroll
        for (int k = 0; k < kInFlight; k++) {
            if (first + (unsigned long long)k * step >= units) break;
            const C other = t[k] < 0 ? (C)0 : notANumber<C>();
            const bool has = t[k] >= 0 && t[k] < tv.rows;
#pragma unroll
            for (int e = 0; e < N; e++) v[k].v[e] = fromCompute<T>(has ? toCompute(v[k].v[e]) * scale : other);
            T *to = z + (Long)row[k] * zv.row + c[k];
            if (c[k] + N <= length) {
                streamPackAnywhere(to, v[k]);
            } else {
#pragma unroll
                for (int e = 0; e < N; e++)
                    if (c[k] + e < length) to[e] = v[k].v[e];
            }
        }
    }
}

// ---- sorting the tokens ----------------------------------------------------------------------------------------------
// Least significant digit first, 8 bits a pass.  A block counts the digits of its tile (a multiple of kSortThreads tokens); a
// second launch places the tile's tokens behind those of lower digits and of the blocks before it.  (Counting the next
// pass's digits while placing, by atomics where the tokens come to lie, took longer than the launch that it saved: frequent
// tokens meet in one counter.)  At most kSortBlocks tiles, so that the placing block can add up the counts of all blocks
// itself.
constexpr int kSortBits = 8, kDigits = 1 << kSortBits;
constexpr int kSortThreads = 1024;
constexpr int kSortBlocks = 256;

// the sort key of token t: tokens outside the table come last, under the key `vocabulary`
__device__ __forceinline__ unsigned keyOf(Long t, unsigned vocabulary) { return t >= 0 && t < (Long)vocabulary ? (unsigned)t : vocabulary; }

// A share of a table to be cleared, by the blocks of a launch from `firstBlock` on: `rows` rows of `bytes` bytes a `pitch` apart,
// or, where elements are `apart` bytes from each other, of bytes / size elements
struct Clearing {
    char *base = nullptr;
    Long rows = 0, bytes = 0, pitch = 0, apart = 0;
    Long lastBytes = 0;  // of the last row
    int size = 0;
    unsigned firstBlock = 0;
};
typedef U32x4 U32x4Any __attribute__((aligned(2)));  // (the least that an element is aligned to)
__device__ __forceinline__ void clearShare(const Clearing &c) {
    const int lane = threadIdx.x % kWaveLanes, waves = blockDim.x / kWaveLanes;
    const Long each = (Long)(gridDim.x - c.firstBlock) * waves;
    for (Long r = (Long)(blockIdx.x - c.firstBlock) * waves + threadIdx.x / kWaveLanes; r < c.rows; r += each) {
        char *row = c.base + r * c.pitch;
        if (c.apart == c.size) {
            const U32x4 zero = {0u, 0u, 0u, 0u};
            const Long bytes = r + 1 < c.rows ? c.bytes : c.lastBytes;
            for (Long at = (Long)lane * 16; at < bytes; at += kWaveLanes * 16) {
                if (at + 16 <= bytes) {
                    __builtin_nontemporal_store(zero, reinterpret_cast<U32x4Any *>(row + at));
                } else {
                    for (Long b = at; b < bytes; b += 2) *reinterpret_cast<unsigned short *>(row + b) = 0;
                }
            }
        } else {
            for (Long e = lane; e < c.bytes / c.size; e += kWaveLanes)
                for (int b = 0; b < c.size; b += 2) *reinterpret_cast<unsigned short *>(row + e * c.apart + b) = 0;
        }
    }
}
__global__ void __launch_bounds__(kThreads) clearKernel(Clearing clearing) { clearShare(clearing); }

__global__ void __launch_bounds__(kSortThreads) sortCountKernel(const Long *tokens, const unsigned *keys, unsigned n, unsigned vocabulary,
                                                                unsigned tile, int shift, unsigned *counts, Clearing clearing) {
    __shared__ unsigned local[kDigits];
    if (blockIdx.x >= clearing.firstBlock) return clearShare(clearing);
    if (threadIdx.x < kDigits) local[threadIdx.x] = 0;
    __syncthreads();
    const unsigned long long first = (unsigned long long)blockIdx.x * tile;
    const unsigned end = (unsigned)(first + tile < n ? first + tile : n);
    for (unsigned i = (unsigned)first + threadIdx.x; i < end; i += kSortThreads) {
        const unsigned key = keys != nullptr ? keys[i] : keyOf(tokens[i], vocabulary);
        atomicAdd(&local[(key >> shift) & (kDigits - 1)], 1u);
    }
    __syncthreads();
    if (threadIdx.x < kDigits) counts[(size_t)blockIdx.x * kDigits + threadIdx.x] = local[threadIdx.x];
}

// How many of the wave's live lanes below this one have the same digit; whole: how many lanes have it in all
__device__ __forceinline__ unsigned equalBelow(unsigned digit, bool live, unsigned &whole) {
    unsigned long long equal = __ballot(live);
#pragma unroll
    for (int bit = 0; bit < kSortBits; bit++) {
        const unsigned long long set = __ballot((digit >> bit) & 1);
        equal &= (digit >> bit) & 1 ? set : ~set;
    }
    whole = (unsigned)__popcll(equal);
    return (unsigned)__popcll(equal & ((1ull << (threadIdx.x % kWaveLanes)) - 1));
}
// where a digit's tokens begin, for the thread of that digit: the sum over lower digits (threads 0 .. 255; all threads of the
// block call it)
__device__ __forceinline__ unsigned digitStart(unsigned mine, unsigned *waveTotals) {
    const int lane = threadIdx.x % kWaveLanes, wave = threadIdx.x / kWaveLanes;
    unsigned sum = mine;
#pragma unroll
    for (int step = 1; step < kWaveLanes; step <<= 1) {
        const unsigned v = __shfl_up(sum, step);
        if (lane >= step) sum += v;
    }
    if (lane == kWaveLanes - 1 && wave < kDigits / kWaveLanes) waveTotals[wave] = sum;
    __syncthreads();
    sum -= mine;
    for (int w = 0; w < wave && w < kDigits / kWaveLanes; w++) sum += waveTotals[w];
    return sum;
}

__global__ void __launch_bounds__(kSortThreads) sortPlaceKernel(const Long *tokens, const unsigned *keys, const unsigned *positions, unsigned n,
                                                                unsigned vocabulary, unsigned tile, int shift, const unsigned *counts,
                                                                unsigned *keysOut, unsigned *positionsOut, Clearing clearing) {
    constexpr int WAVES = kSortThreads / kWaveLanes;
    __shared__ unsigned starts[kDigits], waveTotals[WAVES];
    __shared__ unsigned waveCounts[WAVES][kDigits];
    const int d = threadIdx.x, wave = threadIdx.x / kWaveLanes;
    const unsigned blocks = clearing.firstBlock;
    if (blockIdx.x >= blocks) return clearShare(clearing);
    const unsigned long long first = (unsigned long long)blockIdx.x * tile;
    const unsigned long long end = first + tile < n ? first + tile : n;
    unsigned key = 0, position = 0;
    auto load = [&](unsigned long long i) {
        if (i < end) {
            key = keys != nullptr ? keys[i] : keyOf(tokens[i], vocabulary);
            position = positions != nullptr ? positions[i] : (unsigned)i;
        }
    };
    load(first + threadIdx.x);  // (on its way while the counts are added up)
    // where this block's tokens of digit d begin: all tokens of lower digits, then those of digit d in the blocks before
    unsigned before = 0, all = 0;
    if (d < kDigits) {
#pragma unroll 8
        for (unsigned b = 0; b < blocks; b++) {
            const unsigned c = counts[(size_t)b * kDigits + d];
            all += c;
            if (b < blockIdx.x) before += c;
        }
    }
    const unsigned start = digitStart(all, waveTotals) + before;
    if (d < kDigits) starts[d] = start;
    for (unsigned long long at = first; at < end; at += kSortThreads) {
        for (int i = threadIdx.x; i < WAVES * kDigits; i += kSortThreads) (&waveCounts[0][0])[i] = 0;
        __syncthreads();
        const unsigned long long i = at + threadIdx.x;
        const bool live = i < end;
        const unsigned digit = (key >> shift) & (kDigits - 1);
        unsigned whole;
        const unsigned lower = equalBelow(digit, live, whole);
        if (live && lower == 0) waveCounts[wave][digit] = whole;
        __syncthreads();
        if (d < kDigits) {
            unsigned running = starts[d];
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const unsigned c = waveCounts[w][d];
                waveCounts[w][d] = running;
                running += c;
            }
            starts[d] = running;
        }
        __syncthreads();
        if (live) {
            const unsigned to = waveCounts[wave][digit] + lower;
            keysOut[to] = key;
            positionsOut[to] = position;
        }
        load(i + kSortThreads);
        __syncthreads();
    }
}

// Up to kSmallSort tokens of a vocabulary below 2^(32 - kSmallBits): one block does all passes in LDS, in one launch instead of
// two a pass, each token as one word of its key (the key `vocabulary` among them) and, below it, its position.  (A round of 1024 tokens takes about 1 us a pass: 16384 tokens took
// 35 us this way.)
constexpr int kSmallThreads = 1024, kSmallBits = 12, kSmallSort = 1 << kSmallBits, kSmallRounds = kSmallSort / kSmallThreads;
__global__ void __launch_bounds__(kSmallThreads) sortSmallKernel(const Long *tokens, unsigned n, unsigned vocabulary, int passes, unsigned *keysOut,
                                                                 unsigned *positionsOut, Clearing clearing) {
    constexpr int WAVES = kSmallThreads / kWaveLanes;
    __shared__ unsigned sorted[kSmallSort];
    __shared__ unsigned short waveCounts[WAVES][kDigits];
    __shared__ unsigned waveTotals[WAVES];
    if (blockIdx.x >= clearing.firstBlock) return clearShare(clearing);
    const int d = threadIdx.x, lane = threadIdx.x % kWaveLanes, wave = threadIdx.x / kWaveLanes;
    const int rounds = (int)((n + kSmallThreads - 1) / kSmallThreads);  // a wave's tokens: rounds x 64 consecutive ones
    const unsigned mine = (unsigned)(wave * rounds) * kWaveLanes + lane;
    unsigned word[kSmallRounds], rank[kSmallRounds];
#pragma unroll
    for (int k = 0; k < kSmallRounds; k++) {
        const unsigned i = mine + k * kWaveLanes;
        word[k] = k < rounds && i < n ? keyOf(tokens[i], vocabulary) << kSmallBits | i : 0u;
    }
    for (int pass = 0; pass < passes; pass++) {
        const int shift = kSmallBits + pass * kSortBits;
        for (int i = threadIdx.x; i < WAVES * kDigits; i += kSmallThreads) (&waveCounts[0][0])[i] = 0;
        __syncthreads();
        volatile unsigned short *mineCounts = waveCounts[wave];
#pragma unroll
        for (int k = 0; k < kSmallRounds; k++) {
            if (k >= rounds) break;
            const bool live = mine + k * kWaveLanes < n;
            const unsigned digit = (word[k] >> shift) & (kDigits - 1);
            unsigned whole;
            const unsigned lower = equalBelow(digit, live, whole);
            if (live) {
                const unsigned seen = mineCounts[digit];
                rank[k] = seen + lower;
                if (lower == 0) mineCounts[digit] = (unsigned short)(seen + whole);
            }
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
        unsigned whole = 0;
        if (d < kDigits) {
#pragma unroll
            for (int w = 0; w < WAVES; w++) whole += waveCounts[w][d];
        }
        unsigned running = digitStart(whole, waveTotals);
        if (d < kDigits) {
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const unsigned c = waveCounts[w][d];
                waveCounts[w][d] = (unsigned short)running;
                running += c;
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSmallRounds; k++)
            if (k < rounds && mine + k * kWaveLanes < n) sorted[waveCounts[wave][(word[k] >> shift) & (kDigits - 1)] + rank[k]] = word[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSmallRounds; k++)
            if (k < rounds && mine + k * kWaveLanes < n) word[k] = sorted[mine + k * kWaveLanes];
    }
#pragma unroll
    for (int k = 0; k < kSmallRounds; k++) {
        const unsigned i = mine + k * kWaveLanes;
        if (k < rounds && i < n) {
            keysOut[i] = word[k] >> kSmallBits;
            positionsOut[i] = word[k] & (kSmallSort - 1);
        }
    }
}

// ---- summing ---------------------------------------------------------------------------------------------------------
constexpr int kMostChunk = 64;   // a wave holds its chunk's keys and positions one a lane
constexpr int kRowsInFlight = 8;

// How the sorted list is cut, and where the columns are
struct SumPlan {
    unsigned n, vocabulary;
    int chunk;
    unsigned chunks;
    Long length;
    Long vectors;    // of columns
    unsigned tiles;  // tiles of 64 vectors
};

// A lane's columns: N of them from c0 on.  With UNIT (elements next to each other, rows of N elements or more) a lane whose
// vector would pass the row's end takes the row's last N columns instead, so that every load is one vector without a
// branch, and stores those from `first` on, which are its own.  Otherwise element by element.
template <typename T> struct Columns {
    Long c0;
    int first, count;  // own: [first, count) of the N from c0 on
};
template <typename T, bool UNIT> __device__ __forceinline__ Columns<T> columnsOf(Long vector, Long length) {
    constexpr int N = Pack<T>::N;
    Columns<T> c;
    const Long c0 = vector * N;
    if (UNIT) {
        c.c0 = c0 + N <= length ? c0 : length - N;
        c.first = (int)(c0 - c.c0 < N ? c0 - c.c0 : N);
        c.count = N;
    } else {
        c.c0 = c0;
        c.first = 0;
        c.count = (int)(c0 >= length ? 0 : (length - c0 < N ? length - c0 : N));
    }
    return c;
}
template <typename T, bool UNIT> __device__ __forceinline__ void loadColumns(const T *row, Long el, const Columns<T> &c, Pack<T> &v) {
    constexpr int N = Pack<T>::N;
    if (UNIT) {
        v = loadPackAnywhere(row + c.c0);
    } else {
#pragma unroll
        for (int e = 0; e < N; e++) v.v[e] = e < c.count ? row[(c.c0 + e) * el] : fromCompute<T>((typename Compute<T>::type)0);
    }
}
template <typename T, bool UNIT>
__device__ __forceinline__ void storeSum(T *row, Long el, const Columns<T> &c, const typename Compute<T>::type *acc,
                                         typename Compute<T>::type scale, bool accumulate) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N;
    if (UNIT && c.first == 0) {
        Pack<T> o;
        if (accumulate) o = loadPackAnywhere(row + c.c0);
#pragma unroll
        for (int e = 0; e < N; e++) o.v[e] = fromCompute<T>(acc[e] * scale + (accumulate ? toCompute(o.v[e]) : (C)0));
        streamPackAnywhere(row + c.c0, o);
        return;
    }
#pragma unroll
    for (int e = 0; e < N; e++)
        if (e >= c.first && e < c.count) {
            T *p = row + (c.c0 + e) * el;
            *p = fromCompute<T>(acc[e] * scale + (accumulate ? toCompute(*p) : (C)0));
        }
}

// the partial sums of a chunk, a vector of columns next to the other: which = 0 for a run that began in an earlier chunk, 1
// for one that goes on behind it
template <typename C> __device__ __forceinline__ C *partialRow(C *partial, unsigned chunk, int which, Long vectors, int perVector) {
    return partial + ((size_t)chunk * 2 + which) * vectors * perVector;
}
template <typename C, int N> struct alignas(16) Partial {
    C v[N];
};

// A wave takes one chunk and one tile of columns.
template <typename T, bool UNIT>
__global__ void __launch_bounds__(kThreads) embeddingBpSumKernel(const T *dz, RowView dzv, const unsigned *keys, const unsigned *positions,
                                                                 SumPlan plan, T *dTable, RowView tv, typename Compute<T>::type scale,
                                                                 int accumulate, typename Compute<T>::type *partial) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N, WAVES = kThreads / kWaveLanes;
    const int lane = threadIdx.x % kWaveLanes, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWaveLanes);
    const unsigned long long work = (unsigned long long)blockIdx.x * WAVES + wave;
    if (work >= (unsigned long long)plan.chunks * plan.tiles) return;
    const unsigned chunk = (unsigned)(work / plan.tiles), tile = (unsigned)(work % plan.tiles);
    const Long vector = (Long)tile * kWaveLanes + lane;
    const Columns<T> columns = columnsOf<T, UNIT>(vector, plan.length);
    const unsigned long long first = (unsigned long long)chunk * plan.chunk;
    const int count = (int)(first + plan.chunk <= plan.n ? plan.chunk : plan.n - first);
    const int mineAt = lane < count ? lane : count - 1;
    const unsigned myKey = keys[first + mineAt], myPosition = positions[first + mineAt];
    const unsigned keyBefore = first > 0 ? keys[first - 1] : 0xffffffffu;
    const unsigned keyBehind = first + count < plan.n ? keys[first + count] : 0xffffffffu;
    C acc[N];
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = (C)0;
    unsigned current = __builtin_amdgcn_readlane(myKey, 0);
    bool fromBefore = current == keyBefore;
    auto finish = [&](bool goesOn) {
        if (current < plan.vocabulary && vector < plan.vectors) {
            if (fromBefore || goesOn) {
                Partial<C, N> sums;
#pragma unroll
                for (int e = 0; e < N; e++) sums.v[e] = acc[e];
                reinterpret_cast<Partial<C, N> *>(partialRow(partial, chunk, fromBefore ? 0 : 1, plan.vectors, N))[vector] = sums;
            } else {
                storeSum<T, UNIT>(dTable + (Long)current * tv.row, tv.el, columns, acc, scale, accumulate != 0);
            }
        }
#pragma unroll
        for (int e = 0; e < N; e++) acc[e] = (C)0;
        fromBefore = false;
    };
    for (int i = 0; i < count; i += kRowsInFlight) {
        Pack<T> v[kRowsInFlight];
#pragma unroll
        for (int u = 0; u < kRowsInFlight; u++) {
            const int at = i + u < count ? i + u : count - 1;
            const unsigned p = __builtin_amdgcn_readlane(myPosition, at);
            loadColumns<T, UNIT>(dz + (Long)p * dzv.row, dzv.el, columns, v[u]);
        }
#pragma unroll
        for (int u = 0; u < kRowsInFlight; u++) {
            if (i + u < count) {
                const unsigned key = __builtin_amdgcn_readlane(myKey, i + u);
                if (key != current) {
                    finish(false);
                    current = key;
                }
#pragma unroll
                for (int e = 0; e < N; e++) acc[e] += toCompute(v[u].v[e]);
            }
        }
    }
    finish(current == keyBehind);
}

// A block takes one chunk and one tile: where a run begins in the chunk and goes on behind it, the run's partial sums are
// added up in the order of the chunks (each wave every eighth of them, then the waves in order).  With four waves of four
// rows in flight the most frequent of 32000 tokens, 7 % of 16384, took 8 us, with eight of eight 6.6 us.
constexpr int kJoinThreads = 512;
template <typename T, bool UNIT>
__global__ void __launch_bounds__(kJoinThreads) embeddingBpJoinKernel(const unsigned *keys, SumPlan plan, T *dTable, RowView tv,
                                                                      typename Compute<T>::type scale, int accumulate,
                                                                      const typename Compute<T>::type *partial) {
    typedef typename Compute<T>::type C;
    constexpr int N = Pack<T>::N, WAVES = kJoinThreads / kWaveLanes;
    __shared__ C smem[WAVES][N][kWaveLanes];
    const int lane = threadIdx.x % kWaveLanes, wave = threadIdx.x / kWaveLanes;
    const unsigned chunk = (unsigned)(blockIdx.x / plan.tiles), tile = (unsigned)(blockIdx.x % plan.tiles);
    const unsigned long long first = (unsigned long long)chunk * plan.chunk, behind = first + plan.chunk;
    if (behind >= plan.n) return;
    // (all of these are asked for before any is waited for)
    const unsigned key = keys[behind - 1], keyBehind = keys[behind], keyFirst = keys[first], keyBefore = first > 0 ? keys[first - 1] : 0xffffffffu;
    // the run reaches into every chunk that begins with its key, as far as these follow each other: 64 looked at a time
    unsigned lastChunk = chunk + 1;
    auto beginOf = [&](unsigned c) {
        const unsigned long long at = ((unsigned long long)c + lane) * plan.chunk;
        return at < plan.n ? keys[at] : 0xffffffffu;
    };
    unsigned begins = beginOf(lastChunk + 1);
    if (key >= plan.vocabulary || keyBehind != key) return;
    if (keyFirst == key && keyBefore == key) return;  // the run began in an earlier chunk, whose block joins it
    for (;;) {
        const unsigned long long other = __ballot(begins != key);
        if (other != 0ull) {
            lastChunk += (unsigned)__ffsll(other) - 1;
            break;
        }
        lastChunk += kWaveLanes;
        begins = beginOf(lastChunk + 1);
    }
    const Long vector = (Long)tile * kWaveLanes + lane;
    C acc[N];
#pragma unroll
    for (int e = 0; e < N; e++) acc[e] = (C)0;
    if (vector < plan.vectors) {
#pragma unroll 8
        for (unsigned c = chunk + wave; c <= lastChunk; c += WAVES) {
            const Partial<C, N> sums =
                reinterpret_cast<const Partial<C, N> *>(partialRow(const_cast<C *>(partial), c, c == chunk ? 1 : 0, plan.vectors, N))[vector];
#pragma unroll
            for (int e = 0; e < N; e++) acc[e] += sums.v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < N; e++) smem[wave][e][lane] = acc[e];
    __syncthreads();
    if (wave != 0 || vector >= plan.vectors) return;
#pragma unroll
    for (int w = 1; w < WAVES; w++)
#pragma unroll
        for (int e = 0; e < N; e++) acc[e] += smem[w][e][lane];
    storeSum<T, UNIT>(dTable + (Long)key * tv.row, tv.el, columnsOf<T, UNIT>(vector, plan.length), acc, scale, accumulate != 0);
}

constexpr Long kClearPiece = 16384;

// the chunk's length: long enough that few runs cross chunks, short enough that a few thousand waves share a small batch
int chunkOf(Long n) { return n >= (1 << 18) ? kMostChunk : (n >= (1 << 12) ? 32 : 8); }

size_t aligned(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

// the scratch's parts, in bytes from its start
struct Layout {
    size_t keys[2], positions[2], counts, partial, bytes;
};
Layout layoutOf(Long n, Long length) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += aligned(bytes); return here; };
    for (int i = 0; i < 2; i++) {
        l.keys[i] = take((size_t)n * 4);
        l.positions[i] = take((size_t)n * 4);
    }
    l.counts = take((size_t)kSortBlocks * kDigits * 4);
    const Long chunk = chunkOf(n), chunks = (n + chunk - 1) / chunk;
    l.partial = take((size_t)chunks * 2 * ((length + 7) / 8 * 8) * sizeof(double));  // (a half's vectors are 8 columns)
    l.bytes = at;
    return l;
}

}  // namespace

// (a launch holds fewer than 2^32 threads)
bool embeddingBpFits(Long n, Long length) {
    const Long chunk = chunkOf(n), tiles = length / (kWaveLanes * Pack<double>::N) + 1;
    return n / chunk + 1 < ((Long)1 << 22) / tiles;
}
size_t embeddingBpScratch(Long n, Long length) { return layoutOf(n, length).bytes; }

template <typename T>
void launchEmbedding(hipStream_t s, const T *table, const RowView &tv, const Long *tokens, T *z, const RowView &zv, double scale) {
    typedef typename Compute<T>::type C;
    if (tv.el == 1 && zv.el == 1 && tv.rows > 0) {
        // (FastDiv takes units below 2^31: more are several launches of whole rows)
        const Long perRow = (zv.length + Pack<T>::N - 1) / Pack<T>::N, most = (((Long)1 << 31) - 1) / perRow;
        for (Long r = 0; r < zv.rows; r += most) {
            const Long rows = zv.rows - r < most ? zv.rows - r : most;
            const unsigned units = (unsigned)(rows * perRow);
            ND4J_LAUNCH((embeddingRowsKernel<T>), dim3(gridFor(units, (Long)kThreads * kInFlight, kRowBlocks)), dim3(kThreads), 0, s, table, tv,
                        tokens + r, z + r * zv.row, zv, (C)scale, FastDiv((unsigned)perRow), units);
        }
        return;
    }
    ND4J_LAUNCH((embeddingAnyKernel<T>), dim3(gridFor(zv.rows * zv.length, kThreads, kGridCap)), dim3(kThreads), 0, s, table, tv, tokens, z, zv,
                (C)scale, rowsAreNear(zv));
}

template <typename T>
void launchEmbeddingBp(hipStream_t s, const T *dz, const RowView &dzv, const Long *tokens, T *dTable, const RowView &tv, double scale,
                       bool accumulate, void *scratch) {
    typedef typename Compute<T>::type C;
    const unsigned n = (unsigned)dzv.rows, vocabulary = (unsigned)tv.rows;
    int bits = 1;
    while (bits < 32 && ((unsigned long long)1 << bits) <= vocabulary) bits++;  // the key `vocabulary` occurs too
    const int passes = (bits + kSortBits - 1) / kSortBits;

    // The table to be cleared, in equal shares for the sort's launches.  Rows that follow each other without gaps are one
    // stretch, cut into pieces of kClearPiece bytes.
    Clearing all;
    if (!accumulate) {
        all.base = reinterpret_cast<char *>(dTable);
        all.size = (int)sizeof(T);
        all.rows = tv.rows;
        all.bytes = all.lastBytes = tv.length * sizeof(T);
        all.pitch = tv.row * sizeof(T);
        all.apart = tv.el * sizeof(T);
        if (tv.el == 1 && (tv.row == tv.length || tv.rows == 1)) {
            const Long bytes = tv.rows * all.bytes;
            all.rows = (bytes + kClearPiece - 1) / kClearPiece;
            all.lastBytes = bytes - (all.rows - 1) * kClearPiece;
            all.bytes = all.pitch = kClearPiece;
        }
    }
    const bool small = n <= (unsigned)kSmallSort && vocabulary < 1u << (32 - kSmallBits);
    int sharesLeft = small ? 1 : 2 * passes;
    auto nextShare = [&](unsigned blocks) {
        Clearing share = all;
        share.firstBlock = blocks;
        share.rows = (all.rows + sharesLeft - 1) / sharesLeft;
        if (share.rows < all.rows) share.lastBytes = all.bytes;
        all.base += share.rows * all.pitch;
        all.rows -= share.rows;
        sharesLeft--;
        return share;
    };
    auto gridWith = [&](const Clearing &share, int threads) {
        return dim3(share.firstBlock + (share.rows > 0 ? (unsigned)gridFor(share.rows, threads / kWaveLanes, 4096) : 0u));
    };
    if (n == 0) {
        const Clearing share = nextShare(0);
        if (share.rows > 0) ND4J_LAUNCH(clearKernel, gridWith(share, kThreads), dim3(kThreads), 0, s, share);
        return;
    }

    const Layout l = layoutOf(n, tv.length);
    char *base = reinterpret_cast<char *>(scratch);
    unsigned *keys[2], *positions[2];
    for (int i = 0; i < 2; i++) {
        keys[i] = reinterpret_cast<unsigned *>(base + l.keys[i]);
        positions[i] = reinterpret_cast<unsigned *>(base + l.positions[i]);
    }
    unsigned *counts = reinterpret_cast<unsigned *>(base + l.counts);
    C *partial = reinterpret_cast<C *>(base + l.partial);
    constexpr unsigned long long most = (unsigned long long)kSortBlocks * kSortThreads;
    const unsigned tile = (unsigned)((n + most - 1) / most * kSortThreads);
    const unsigned blocks = (unsigned)(((unsigned long long)n + tile - 1) / tile);
    const unsigned *from = nullptr, *fromPositions = nullptr;
    int to = 0;
    if (small) {
        const Clearing share = nextShare(1);
        ND4J_LAUNCH(sortSmallKernel, gridWith(share, kSmallThreads), dim3(kSmallThreads), 0, s, tokens, n, vocabulary, passes, keys[0], positions[0],
                    share);
        from = keys[0];
        fromPositions = positions[0];
    }
    for (int pass = 0; pass < passes && !small; pass++) {
        const int shift = pass * kSortBits;
        Clearing share = nextShare(blocks);
        ND4J_LAUNCH(sortCountKernel, gridWith(share, kSortThreads), dim3(kSortThreads), 0, s, tokens, from, n, vocabulary, tile, shift, counts,
                    share);
        share = nextShare(blocks);
        ND4J_LAUNCH(sortPlaceKernel, gridWith(share, kSortThreads), dim3(kSortThreads), 0, s, tokens, from, fromPositions, n, vocabulary, tile,
                    shift, counts, keys[to], positions[to], share);
        from = keys[to];
        fromPositions = positions[to];
        to ^= 1;
    }
    SumPlan plan;
    plan.n = n;
    plan.vocabulary = vocabulary;
    plan.chunk = chunkOf(n);
    plan.chunks = (unsigned)(((unsigned long long)n + plan.chunk - 1) / plan.chunk);
    plan.length = tv.length;
    plan.vectors = (tv.length + Pack<T>::N - 1) / Pack<T>::N;
    plan.tiles = (unsigned)((plan.vectors + kWaveLanes - 1) / kWaveLanes);
    constexpr int WAVES = kThreads / kWaveLanes;
    const unsigned sumBlocks = (unsigned)(((unsigned long long)plan.chunks * plan.tiles + WAVES - 1) / WAVES);
    const bool unit = dzv.el == 1 && tv.el == 1 && tv.length >= Pack<T>::N;
    if (unit)
        ND4J_LAUNCH((embeddingBpSumKernel<T, true>), dim3(sumBlocks), dim3(kThreads), 0, s, dz, dzv, from, fromPositions, plan, dTable, tv,
                    (C)scale, accumulate ? 1 : 0, partial);
    else
        ND4J_LAUNCH((embeddingBpSumKernel<T, false>), dim3(sumBlocks), dim3(kThreads), 0, s, dz, dzv, from, fromPositions, plan, dTable, tv,
                    (C)scale, accumulate ? 1 : 0, partial);
    if (plan.chunks > 1) {
        const unsigned joinBlocks = (plan.chunks - 1) * plan.tiles;
        if (unit)
            ND4J_LAUNCH((embeddingBpJoinKernel<T, true>), dim3(joinBlocks), dim3(kJoinThreads), 0, s, from, plan, dTable, tv, (C)scale,
                        accumulate ? 1 : 0, partial);
        else
            ND4J_LAUNCH((embeddingBpJoinKernel<T, false>), dim3(joinBlocks), dim3(kJoinThreads), 0, s, from, plan, dTable, tv, (C)scale,
                        accumulate ? 1 : 0, partial);
    }
}

#define INST(T)                                                                                                                    \
    template void launchEmbedding<T>(hipStream_t, const T *, const RowView &, const Long *, T *, const RowView &, double);           \
    template void launchEmbeddingBp<T>(hipStream_t, const T *, const RowView &, const Long *, T *, const RowView &, double, bool, void *);
INST(float)
INST(float16)
INST(double)
#undef INST

}  // namespace nd4j_amd
