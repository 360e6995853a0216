// The front end's kernels as capi.cu launches them, after the argument checks.
#pragma once
#include <cuda.h>
#include "defs.h"

namespace dsa {

constexpr int kDIndex = DSA_V32_D_INDEX;

// TMEM columns of a query row's heads
inline int index_score_cols(int H) { return H <= 16 ? 16 : H <= 32 ? 32 : 64; }

cudaError_t launch_norm_rotate(const dsa_v32_norm_rotate_args& a, cudaStream_t stream);
cudaError_t launch_append(const dsa_v32_append_args& a, cudaStream_t stream);
// tk, tq: tensor maps of the keys and of the query rows (index_score_cols heads in a box)
cudaError_t launch_index_scores(const dsa_v32_index_scores_args& a, const CUtensorMap& tk, const CUtensorMap& tq, cudaStream_t stream);
cudaError_t launch_block_select(const float* scores, int64_t stride_row, const int32_t* valid_len, int total_q, int num_blocks, int block, int num_selected,
                                int first, int local, int32_t* indices_out, cudaStream_t stream);

}  // namespace dsa
