// Host side of the operators around a language model's matrix products (training.h): layer norm, embedding, log
// probabilities of tokens, clipping by the global norm.  They have no counterpart in the reference's NativeOps and are
// reached through the C ABI (include/nd4j_native_c.h), which documents them.  Everything a kernel takes for granted is
// checked here, before anything is enqueued; what cannot be checked on the host (token values, offsets) the kernels bound.
#include <cmath>
#include <numeric>
#include <stdexcept>
#include <string>

#include "native_training.h"
#include "runtime.h"
#include "training.h"

namespace nd4j_amd {

namespace {

[[noreturn]] void refuse(const char *op, const std::string &why) { throw std::invalid_argument(std::string(op) + ": " + why); }

const Long kMostRows = (Long)1 << 40;
const Long kMostLength = ((Long)1 << 31) - ((Long)1 << 20);  // columns fit an int with any block's round to spare

// The rows of a view: its last dimension, at every position of the others, which have to lie a common distance apart.
RowView rowsOf(const char *op, const char *name, Nd4jPointer *extra, int slot, const Long *arg, std::vector<Long> &storage, hipStream_t s) {
    // (a read-back synchronises the stream, which would end its capture)
    const Long *info = nullptr;
    if (slotOf(extra, slot) == nullptr && arg != nullptr && isDeviceMemory(arg)) {
        if (streamIsCapturing(s)) refuse(op, std::string("the stream is being captured, which needs a host copy of the shapeInfo of ") + name);
        const OutsideCaptures outside;
        info = hostShapeInfo(extra, slot, arg, storage, s);
    } else {
        info = hostShapeInfo(extra, slot, arg, storage, s);
    }
    if (info == nullptr) refuse(op, std::string("no shapeInfo of ") + name);
    const int rank = siRank(info);
    if (rank < 1 || rank > kMaxRank) refuse(op, std::string(name) + " needs a rank between 1 and 32");
    const Long *shape = siShape(info), *stride = siStride(info);
    RowView v;
    v.length = shape[rank - 1];
    v.el = stride[rank - 1];
    v.rows = 1;
    v.row = 0;
    bool first = true;
    for (int d = rank - 2; d >= 0; d--) {
        if (shape[d] < 0) refuse(op, std::string(name) + " has a negative extent");
        if (shape[d] == 0) { v.rows = 0; break; }
        if (shape[d] == 1) continue;
        if (first) {
            v.row = stride[d];
            first = false;
        } else if (stride[d] != v.row * v.rows) {
            refuse(op, std::string("the leading dimensions of ") + name + " do not merge into rows a common distance apart");
        }
        if (shape[d] > kMostRows / v.rows) refuse(op, std::string(name) + " has too many rows");
        v.rows *= shape[d];
    }
    if (v.length < 1) refuse(op, std::string(name) + " has rows without elements");
    if (v.length > kMostLength) refuse(op, std::string(name) + " has rows of more than 2^31 - 2^20 elements");
    return v;
}

// A result's elements have places of their own: d rows further and e elements on is the same place where d row = e el.
void apart(const char *op, const char *name, const RowView &v) {
    const Long row = v.row < 0 ? -v.row : v.row, el = v.el < 0 ? -v.el : v.el, common = std::gcd(row, el);
    const bool meet = common == 0 ? v.rows > 1 || v.length > 1 : el / common < v.rows && row / common < v.length;
    if (v.rows > 0 && meet) refuse(op, std::string("elements of ") + name + " share places");
}

template <typename P> void need(const char *op, const char *name, const P *p, size_t alignment) {
    if (p == nullptr) refuse(op, std::string(name) + " is null");
    if (reinterpret_cast<uintptr_t>(p) % alignment != 0) refuse(op, std::string(name) + " is not aligned to its elements");
}
template <typename P> void mayBe(const char *op, const char *name, const P *p) {
    if (p != nullptr) need(op, name, p, sizeof(P));
}
template <typename P> void must(const char *op, const char *name, const P *p) { need(op, name, p, sizeof(P)); }

void sameShape(const char *op, const char *a, const RowView &x, const char *b, const RowView &z) {
    if (x.rows != z.rows || x.length != z.length) refuse(op, std::string(a) + " and " + b + " differ in shape");
}

// The caller's scratch when it is given one, else the stream's, kept until the call's launches are enqueued.  A stream under
// capture gets none of the library's: two graphs captured on it would share the block, and releasing the stream would free it
// under them.
OperatorScratch scratchFor(const char *op, hipStream_t s, void *given, Long givenBytes, size_t bytes) {
    OperatorScratch scratch;
    if (bytes == 0) return scratch;
    if (given != nullptr) {
        if (givenBytes < 0 || (size_t)givenBytes < bytes)
            refuse(op, "the scratch holds " + std::to_string(givenBytes) + " bytes, " + std::to_string(bytes) + " are needed");
        if (reinterpret_cast<uintptr_t>(given) % 16 != 0) refuse(op, "the scratch is not aligned to 16 bytes");
        scratch.ptr = given;
        return scratch;
    }
    if (streamIsCapturing(s))
        throw std::runtime_error(std::string(op) + ": the stream is being captured, which needs scratch of the graph's own (" +
                                 std::to_string(bytes) + " bytes)");
    return operatorScratchFor(s, bytes);
}

}  // namespace

template <typename T>
void layerNorm(Nd4jPointer *extra, T *x, Long *xInfo, T *gain, T *bias, T *z, Long *zInfo, typename Compute<T>::type *mean,
               typename Compute<T>::type *invStd, double epsilon) {
    const char *op = "layerNorm";
    hipStream_t s = streamOf(extra);
    std::vector<Long> sx, sz;
    const RowView xv = rowsOf(op, "x", extra, X_HOST_X_SHAPE, xInfo, sx, s), zv = rowsOf(op, "z", extra, X_HOST_Z_SHAPE, zInfo, sz, s);
    sameShape(op, "x", xv, "z", zv);
    apart(op, "z", zv);
    if (!(epsilon >= 0.0)) refuse(op, "epsilon is negative or not a number");
    if (xv.rows == 0) return;
    must(op, "x", x);
    must(op, "z", z);
    mayBe(op, "gain", gain);
    mayBe(op, "bias", bias);
    mayBe(op, "mean", mean);
    mayBe(op, "invStd", invStd);
    launchLayerNorm<T>(s, x, xv, gain, bias, z, zv, mean, invStd, epsilon);
    checkLaunch(op, s);
}

template <typename T>
void layerNormBp(Nd4jPointer *extra, T *x, Long *xInfo, T *gain, typename Compute<T>::type *mean, typename Compute<T>::type *invStd, T *dz,
                 Long *dzInfo, T *dx, Long *dxInfo, T *dGain, T *dBias, void *scratch, Long scratchBytes) {
    const char *op = "layerNormBp";
    hipStream_t s = streamOf(extra);
    std::vector<Long> sx, sy, sz;
    const RowView xv = rowsOf(op, "x", extra, X_HOST_X_SHAPE, xInfo, sx, s), dzv = rowsOf(op, "dz", extra, X_HOST_Y_SHAPE, dzInfo, sy, s);
    sameShape(op, "x", xv, "dz", dzv);
    RowView dxv = xv;
    if (dx != nullptr) {
        dxv = rowsOf(op, "dx", extra, X_HOST_Z_SHAPE, dxInfo, sz, s);
        sameShape(op, "x", xv, "dx", dxv);
        apart(op, "dx", dxv);
    }
    mayBe(op, "dx", dx);
    mayBe(op, "dGain", dGain);
    mayBe(op, "dBias", dBias);
    mayBe(op, "gain", gain);
    if (dx == nullptr && dGain == nullptr && dBias == nullptr) refuse(op, "no gradient is asked for");
    if (xv.rows > 0) {
        must(op, "x", x);
        must(op, "dz", dz);
        must(op, "mean", mean);
        must(op, "invStd", invStd);
    } else if (dGain == nullptr && dBias == nullptr) {
        return;
    }
    const bool columns = dGain != nullptr || dBias != nullptr;
    const OperatorScratch work = scratchFor(op, s, scratch, scratchBytes, columns ? layerNormBpScratch(xv.rows, xv.length) : 0);
    launchLayerNormBp<T>(s, x, xv, gain, mean, invStd, dz, dzv, dx, dxv, dGain, dBias, work.ptr);
    checkLaunch(op, s);
}

template <typename T>
void embedding(Nd4jPointer *extra, T *table, Long *tableInfo, Long *tokens, Long n, T *z, Long *zInfo, double scale) {
    const char *op = "embedding";
    hipStream_t s = streamOf(extra);
    std::vector<Long> sx, sz;
    const RowView tv = rowsOf(op, "the table", extra, X_HOST_X_SHAPE, tableInfo, sx, s);
    if (n < 0) refuse(op, "a negative number of tokens");
    if (n == 0) return;
    const RowView zv = rowsOf(op, "z", extra, X_HOST_Z_SHAPE, zInfo, sz, s);
    if (zv.rows != n || zv.length != tv.length) refuse(op, "z is not a row of the table's length for every token");
    apart(op, "z", zv);
    if (n > ((Long)1 << 56) / tv.length) refuse(op, "too many elements");
    must(op, "the table", table);
    must(op, "tokens", tokens);
    must(op, "z", z);
    launchEmbedding<T>(s, table, tv, tokens, z, zv, scale);
    checkLaunch(op, s);
}

template <typename T>
void embeddingBp(Nd4jPointer *extra, T *dz, Long *dzInfo, Long *tokens, Long n, T *dTable, Long *tableInfo, double scale, int accumulate,
                 void *scratch, Long scratchBytes) {
    const char *op = "embeddingBp";
    hipStream_t s = streamOf(extra);
    std::vector<Long> sx, sz;
    const RowView tv = rowsOf(op, "dTable", extra, X_HOST_Z_SHAPE, tableInfo, sz, s);
    if (n < 0) refuse(op, "a negative number of tokens");
    RowView dzv;
    dzv.length = tv.length;
    if (n > 0) dzv = rowsOf(op, "dz", extra, X_HOST_X_SHAPE, dzInfo, sx, s);
    if (dzv.rows != n || dzv.length != tv.length) refuse(op, "dz is not a row of the table's length for every token");
    if (tv.rows == 0 || (n == 0 && accumulate != 0)) return;
    apart(op, "dTable", tv);
    // (tokens are sorted as 32-bit keys with 32-bit positions)
    if (n > kMostLength || tv.rows > kMostLength) refuse(op, "more than 2^31 - 2^20 tokens or rows of the table are not supported");
    if (!embeddingBpFits(n, tv.length)) refuse(op, "too many elements");
    must(op, "dTable", dTable);
    if (n > 0) {
        must(op, "dz", dz);
        must(op, "tokens", tokens);
    }
    const OperatorScratch work = scratchFor(op, s, scratch, scratchBytes, n > 0 ? embeddingBpScratch(n, tv.length) : 0);
    launchEmbeddingBp<T>(s, dz, dzv, tokens, dTable, tv, scale, accumulate != 0, work.ptr);
    checkLaunch(op, s);
}

template <typename T>
void tokenLogProbs(Nd4jPointer *extra, T *x, Long *xInfo, Long *tokens, typename Compute<T>::type *logProbs, typename Compute<T>::type *logSum,
                   typename Compute<T>::type *entropy, int k, Long *top, typename Compute<T>::type *topLogProbs, void *scratch,
                   Long scratchBytes) {
    const char *op = "tokenLogProbs";
    hipStream_t s = streamOf(extra);
    std::vector<Long> sx;
    const RowView xv = rowsOf(op, "x", extra, X_HOST_X_SHAPE, xInfo, sx, s);
    if (k < 0 || k > kMostAlternatives) refuse(op, "the number of alternatives has to be between 0 and 64");
    if (k > xv.length) refuse(op, "more alternatives than the rows have elements");
    if (xv.rows == 0) return;
    must(op, "x", x);
    if (logProbs != nullptr) must(op, "tokens", tokens);
    if (k > 0) must(op, "topTokens", top);
    mayBe(op, "logProbs", logProbs);
    mayBe(op, "logSum", logSum);
    mayBe(op, "entropy", entropy);
    mayBe(op, "topLogProbs", topLogProbs);
    if (logProbs == nullptr && logSum == nullptr && entropy == nullptr && k == 0) refuse(op, "no result is asked for");
    TokenProbsOut<T> out;
    out.logProbs = logProbs;
    out.logSum = logSum;
    out.entropy = entropy;
    out.k = k;
    out.top = top;
    out.topLogProbs = k > 0 ? topLogProbs : nullptr;
    const OperatorScratch work = scratchFor(op, s, scratch, scratchBytes, tokenLogProbsScratch(xv.rows, xv.length, k));
    launchTokenLogProbs<T>(s, x, xv, tokens, out, work.ptr);
    checkLaunch(op, s);
}

template <typename T>
void tokenLogProbsBp(Nd4jPointer *extra, T *x, Long *xInfo, Long *tokens, typename Compute<T>::type *logSum, typename Compute<T>::type *entropy,
                     typename Compute<T>::type *dLogProbs, typename Compute<T>::type *dEntropy, T *dx, Long *dxInfo) {
    const char *op = "tokenLogProbsBp";
    hipStream_t s = streamOf(extra);
    std::vector<Long> sx, sz;
    const RowView xv = rowsOf(op, "x", extra, X_HOST_X_SHAPE, xInfo, sx, s), dxv = rowsOf(op, "dx", extra, X_HOST_Z_SHAPE, dxInfo, sz, s);
    sameShape(op, "x", xv, "dx", dxv);
    apart(op, "dx", dxv);
    if (dLogProbs == nullptr && dEntropy == nullptr) refuse(op, "neither the log probabilities' gradient nor the entropies' is given");
    if (xv.rows == 0) return;
    must(op, "x", x);
    must(op, "logSum", logSum);
    must(op, "dx", dx);
    if (dLogProbs != nullptr) {
        must(op, "dLogProbs", dLogProbs);
        must(op, "tokens", tokens);
    }
    if (dEntropy != nullptr) {
        must(op, "dEntropy", dEntropy);
        must(op, "entropy", entropy);
    }
    launchTokenLogProbsBp<T>(s, x, xv, tokens, logSum, entropy, dLogProbs, dEntropy, dx, dxv);
    checkLaunch(op, s);
}

template <typename T>
void clipByGlobalNorm(Nd4jPointer *extra, Nd4jPointer *dx, Nd4jPointer *dz, Long *offsets, int n, Long total, double maxNorm,
                      typename Compute<T>::type *norm, void *scratch, Long scratchBytes) {
    const char *op = "clipByGlobalNorm";
    hipStream_t s = streamOf(extra);
    if (n < 0 || total < 0) refuse(op, "a negative number of tensors or elements");
    if (total > ((Long)1 << 56)) refuse(op, "too many elements");
    if (dz != nullptr && !(maxNorm > 0.0)) refuse(op, "the largest norm has to be greater than 0");
    if (dz == nullptr && norm == nullptr) refuse(op, "no result is asked for");
    if (n == 0 && total > 0) refuse(op, "elements without a tensor");
    mayBe(op, "norm", norm);
    if (n > 0) {
        must(op, "the table of tensors", dx);
        must(op, "offsets", offsets);
        mayBe(op, "the table of results", dz);
    }
    const OperatorScratch work = scratchFor(op, s, scratch, scratchBytes, clipByGlobalNormScratch(total));
    launchClipByGlobalNorm<T>(s, reinterpret_cast<const T *const *>(dx), reinterpret_cast<T *const *>(dz), offsets, n, total, maxNorm, norm,
                              work.ptr);
    checkLaunch(op, s);
}

Long layerNormBpScratchBytes(Long rows, Long length) {
    const char *op = "scratchLayerNormBp";
    if (rows < 0 || length < 1 || rows > kMostRows || length > kMostLength) refuse(op, "rows or length out of range");
    return (Long)layerNormBpScratch(rows, length);
}
Long embeddingBpScratchBytes(Long n, Long vocabulary, Long length) {
    const char *op = "scratchEmbeddingBp";
    if (n < 0 || vocabulary < 0 || length < 1 || n > kMostLength || vocabulary > kMostLength || length > kMostLength)
        refuse(op, "the number of tokens, the vocabulary or the length is out of range");
    if (!embeddingBpFits(n, length)) refuse(op, "too many elements");
    return (Long)embeddingBpScratch(n, length);
}
Long tokenLogProbsScratchBytes(Long rows, Long length, int k) {
    const char *op = "scratchTokenLogProbs";
    if (rows < 0 || length < 1 || rows > kMostRows || length > kMostLength || k < 0 || k > kMostAlternatives)
        refuse(op, "rows, length or the number of alternatives out of range");
    return (Long)tokenLogProbsScratch(rows, length, k);
}
Long clipByGlobalNormScratchBytes(Long total) {
    if (total < 0) refuse("scratchClipByGlobalNorm", "a negative number of elements");
    return (Long)clipByGlobalNormScratch(total);
}

#define INST(T)                                                                                                                            \
    template void layerNorm<T>(Nd4jPointer *, T *, Long *, T *, T *, T *, Long *, Compute<T>::type *, Compute<T>::type *, double);          \
    template void layerNormBp<T>(Nd4jPointer *, T *, Long *, T *, Compute<T>::type *, Compute<T>::type *, T *, Long *, T *, Long *, T *,    \
                                 T *, void *, Long);                                                                                       \
    template void embedding<T>(Nd4jPointer *, T *, Long *, Long *, Long, T *, Long *, double);                                             \
    template void embeddingBp<T>(Nd4jPointer *, T *, Long *, Long *, Long, T *, Long *, double, int, void *, Long);                        \
    template void tokenLogProbs<T>(Nd4jPointer *, T *, Long *, Long *, Compute<T>::type *, Compute<T>::type *, Compute<T>::type *, int,     \
                                   Long *, Compute<T>::type *, void *, Long);                                                              \
    template void tokenLogProbsBp<T>(Nd4jPointer *, T *, Long *, Long *, Compute<T>::type *, Compute<T>::type *, Compute<T>::type *,        \
                                     Compute<T>::type *, T *, Long *);                                                                     \
    template void clipByGlobalNorm<T>(Nd4jPointer *, Nd4jPointer *, Nd4jPointer *, Long *, int, Long, double, Compute<T>::type *, void *,   \
                                      Long);
INST(float)
INST(float16)
INST(double)
#undef INST

}  // namespace nd4j_amd
