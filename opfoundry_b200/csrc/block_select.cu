// Selection of the best blocks of positions for every query row, written as the lists of positions that the attention takes (sm_100a).
//
// One CTA a row.  A block's score becomes a 32-bit key of the same order, the largest key for the blocks that are always selected;
// the threshold is found bit by bit, its ties go to the lowest blocks, and the selected blocks are expanded in ascending order.
#include "front.h"

namespace dsa {
namespace {

constexpr int kSelThreads = 256;

// float -> key with the same order as the values, at least 1; NaN lowest, -0.0 ties with +0.0 (as in topk_select.cu)
__device__ __forceinline__ uint32_t block_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return x != x ? 1u : k;
}

__device__ __forceinline__ int block_sum(int x, int* tmp) {
    x = __reduce_add_sync(0xffffffffu, x);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) tmp[threadIdx.x >> 5] = x;
    __syncthreads();
    int s = 0;
    for (int i = 0; i < kSelThreads / 32; ++i) s += tmp[i];
    return s;
}

__global__ void __launch_bounds__(kSelThreads) block_select_kernel(const float* __restrict__ scores, int64_t stride_row, const int32_t* __restrict__ valid_len,
                                                                   int num_blocks, int block, int num_selected, int first, int local, int32_t* __restrict__ indices_out) {
    __shared__ int tmp[kSelThreads / 32];
    const int q = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t most = (int64_t)num_blocks * block;
    const int valid = (int)min(most, (int64_t)max(0, valid_len != nullptr ? valid_len[q] : (int)most));
    const int live = (valid + block - 1) / block;
    const int64_t topk = (int64_t)num_selected * block;
    const float* row = scores + q * stride_row;
    int32_t* out = indices_out + q * topk;
    if (live <= num_selected) {
        for (int64_t i = tid; i < topk; i += kSelThreads) out[i] = i < valid ? (int)i : -1;
        return;
    }
    auto key = [&](int b) { return b < first || b >= live - local ? 0xFFFFFFFFu : block_key(row[b]); };
    // the largest threshold that at least num_selected keys reach
    uint32_t threshold = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t trial = threshold | (1u << bit);
        int n = 0;
        for (int b = tid; b < live; b += kSelThreads) n += key(b) >= trial;
        if (block_sum(n, tmp) >= num_selected) threshold = trial;
    }
    int n = 0;
    for (int b = tid; b < live; b += kSelThreads) n += key(b) > threshold;
    const int ties = num_selected - block_sum(n, tmp);   // blocks at the threshold that are taken
    int done = 0, equal = 0;                              // selected, and at the threshold, before this round of blocks
    for (int b0 = 0; b0 < live; b0 += kSelThreads) {
        const int b = b0 + tid;
        const uint32_t k = b < live ? key(b) : 0u;
        const bool eq = b < live && k == threshold;
        const uint32_t eq_vote = __ballot_sync(0xffffffffu, eq);
        __syncthreads();
        if (lane == 0) tmp[warp] = __popc(eq_vote);
        __syncthreads();
        int eq_before = equal + __popc(eq_vote & ((1u << lane) - 1u));
        for (int i = 0; i < kSelThreads / 32; ++i) {
            if (i < warp) eq_before += tmp[i];
            equal += tmp[i];
        }
        const bool take = b < live && (k > threshold || (eq && eq_before < ties));
        const uint32_t vote = __ballot_sync(0xffffffffu, take);
        __syncthreads();
        if (lane == 0) tmp[warp] = __popc(vote);
        __syncthreads();
        int at = done + __popc(vote & ((1u << lane) - 1u));
        for (int i = 0; i < kSelThreads / 32; ++i) {
            if (i < warp) at += tmp[i];
            done += tmp[i];
        }
        if (take)
            for (int i = 0; i < block; ++i) out[(int64_t)at * block + i] = b * block + i < valid ? b * block + i : -1;
    }
}

}  // namespace

cudaError_t launch_block_select(const float* scores, int64_t stride_row, const int32_t* valid_len, int total_q, int num_blocks, int block, int num_selected,
                                int first, int local, int32_t* indices_out, cudaStream_t stream) {
    if (total_q == 0) return cudaSuccess;
    block_select_kernel<<<(unsigned)total_q, kSelThreads, 0, stream>>>(scores, stride_row, valid_len, num_blocks, block, num_selected, first, local, indices_out);
    return cudaGetLastError();
}

}  // namespace dsa
