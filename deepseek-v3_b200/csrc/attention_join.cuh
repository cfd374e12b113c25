// Joining the parts of an attention's result.
#pragma once

#include "common.cuh"

namespace dsv3 {

constexpr int kMaxJoinParts = 32;

// Parts in fp32, one behind the other: partial [n, rows, dim], partial_lse [n, rows]; a row is a head of a token.  With cu (device memory, [n_seqs + 1]) only the tokens of
// [cu[0], cu[n_seqs]) are joined.
int join_partials(const float* partial, const float* partial_lse, int n, int64_t rows, int dim, const int32_t* cu, int n_seqs, int heads, void* out, float* lse,
                  cudaStream_t stream);

}  // namespace dsv3
