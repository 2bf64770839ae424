// Host entry points of the operators around a language model's matrix products (native_training.cpp), which c_api.cpp
// forwards to; include/nd4j_native_c.h documents them.
#pragma once

#include "runtime.h"

namespace nd4j_amd {

template <typename T>
void layerNorm(Nd4jPointer *extra, T *x, Long *xInfo, T *gain, T *bias, T *z, Long *zInfo, typename Compute<T>::type *mean,
               typename Compute<T>::type *invStd, double epsilon);
template <typename T>
void layerNormBp(Nd4jPointer *extra, T *x, Long *xInfo, T *gain, typename Compute<T>::type *mean, typename Compute<T>::type *invStd, T *dz,
                 Long *dzInfo, T *dx, Long *dxInfo, T *dGain, T *dBias, void *scratch, Long scratchBytes);
template <typename T>
void embedding(Nd4jPointer *extra, T *table, Long *tableInfo, Long *tokens, Long n, T *z, Long *zInfo, double scale);
template <typename T>
void embeddingBp(Nd4jPointer *extra, T *dz, Long *dzInfo, Long *tokens, Long n, T *dTable, Long *tableInfo, double scale, int accumulate,
                 void *scratch, Long scratchBytes);
template <typename T>
void tokenLogProbs(Nd4jPointer *extra, T *x, Long *xInfo, Long *tokens, typename Compute<T>::type *logProbs, typename Compute<T>::type *logSum,
                   typename Compute<T>::type *entropy, int k, Long *top, typename Compute<T>::type *topLogProbs, void *scratch,
                   Long scratchBytes);
template <typename T>
void tokenLogProbsBp(Nd4jPointer *extra, T *x, Long *xInfo, Long *tokens, typename Compute<T>::type *logSum, typename Compute<T>::type *entropy,
                     typename Compute<T>::type *dLogProbs, typename Compute<T>::type *dEntropy, T *dx, Long *dxInfo);
template <typename T>
void clipByGlobalNorm(Nd4jPointer *extra, Nd4jPointer *dx, Nd4jPointer *dz, Long *offsets, int n, Long total, double maxNorm,
                      typename Compute<T>::type *norm, void *scratch, Long scratchBytes);

// bytes of scratch for any of the types; std::invalid_argument for sizes that the operators refuse
Long layerNormBpScratchBytes(Long rows, Long length);
Long embeddingBpScratchBytes(Long n, Long vocabulary, Long length);
Long tokenLogProbsScratchBytes(Long rows, Long length, int k);
Long clipByGlobalNormScratchBytes(Long total);

}  // namespace nd4j_amd
