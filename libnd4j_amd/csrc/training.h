// Interface between the host boundary (native_training.cpp) and the kernels of the operators around a language model's
// matrix products: layer norm, embedding, log probabilities of tokens, and clipping by the global norm.  As in launch.h,
// every launcher enqueues on `stream` and returns; the host side has checked the arguments.
#pragma once

#include <hip/hip_runtime.h>

#include "types.h"
#include "view.h"

namespace nd4j_amd {

// A view as rows: element (r, c) lies r * row + c * el elements behind the view's start.
struct RowView {
    Long rows = 0, length = 0;
    Long row = 0, el = 1;
};

// whether a view's rows lie nearer to each other than a row's elements (an f-order matrix): lanes then take rows
inline bool rowsAreNear(const RowView &v) {
    const Long row = v.row < 0 ? -v.row : v.row, el = v.el < 0 ? -v.el : v.el;
    return v.rows > 1 && row < el;
}

// ---- layer norm (layernorm.hip) ----------------------------------------------------------------------------------------
// z = (x - mean) / sqrt(variance + epsilon) * gain + bias over the rows; gain, bias, mean, invStd may be null
template <typename T>
void launchLayerNorm(hipStream_t stream, const T *x, const RowView &xv, const T *gain, const T *bias, T *z, const RowView &zv,
                     typename Compute<T>::type *mean, typename Compute<T>::type *invStd, double epsilon);
// the gradients of x, gain and bias (each may be null) for the gradient dz of z; scratch: layerNormBpScratch bytes
template <typename T>
void launchLayerNormBp(hipStream_t stream, const T *x, const RowView &xv, const T *gain, const typename Compute<T>::type *mean,
                       const typename Compute<T>::type *invStd, const T *dz, const RowView &dzv, T *dx, const RowView &dxv, T *dGain,
                       T *dBias, void *scratch);
// scratch of launchLayerNormBp in bytes, for the widest compute type; the launcher's split of the rows follows the same rule
size_t layerNormBpScratch(Long rows, Long length);

// ---- embedding (embedding.hip) -----------------------------------------------------------------------------------------
// row i of z = scale * row tokens[i] of the table; a negative token gives zeros, one beyond the table NaN
template <typename T>
void launchEmbedding(hipStream_t stream, const T *table, const RowView &tv, const Long *tokens, T *z, const RowView &zv, double scale);
// row v of dTable = (accumulate: what it held, else 0) + scale * the sum of the rows i of dz with tokens[i] == v, in the order of i
template <typename T>
void launchEmbeddingBp(hipStream_t stream, const T *dz, const RowView &dzv, const Long *tokens, T *dTable, const RowView &tv, double scale,
                       bool accumulate, void *scratch);
size_t embeddingBpScratch(Long n, Long length);
bool embeddingBpFits(Long n, Long length);  // whether its grids hold n tokens of rows of this length

// ---- log probabilities of tokens (tokenprobs.hip) ------------------------------------------------------------------------
static const int kMostAlternatives = 64;
template <typename T> struct TokenProbsOut {
    typedef typename Compute<T>::type C;
    C *logProbs;   // per row: the log probability of the row's token; null: not wanted (as the others)
    C *logSum;     // per row: log(sum of exp(x))
    C *entropy;    // per row
    int k;         // alternatives per row, 0 .. kMostAlternatives
    Long *top;     // [rows, k]
    C *topLogProbs;  // [rows, k] or null
};
template <typename T>
void launchTokenLogProbs(hipStream_t stream, const T *x, const RowView &xv, const Long *tokens, const TokenProbsOut<T> &out, void *scratch);
size_t tokenLogProbsScratch(Long rows, Long length, int k);
template <typename T>
void launchTokenLogProbsBp(hipStream_t stream, const T *x, const RowView &xv, const Long *tokens, const typename Compute<T>::type *logSum,
                           const typename Compute<T>::type *entropy, const typename Compute<T>::type *dLogProbs,
                           const typename Compute<T>::type *dEntropy, T *dx, const RowView &dxv);

// ---- clipping by the global norm (globalnorm.hip) -------------------------------------------------------------------------
// norm[0] = sqrt(sum of the squares of all elements); tensors of out = those of in, times maxNorm / norm where the norm is
// finite and greater than maxNorm.  in / out: device tables of n device pointers (out null: the norm alone); tensor i has
// offsets[i + 1] - offsets[i] elements.
template <typename T>
void launchClipByGlobalNorm(hipStream_t stream, const T *const *in, T *const *out, const Long *offsets, int n, Long total, double maxNorm,
                            typename Compute<T>::type *norm, void *scratch);
size_t clipByGlobalNormScratch(Long total);

}  // namespace nd4j_amd
