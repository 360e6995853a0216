// Index scores of blocks of positions (sm_100a): s[q, p] = ks[p] * sum_h w[q, h] max(0, q_h . k_p), and the largest of a block.
//
// The plain form of the kernel: a thread holds one key in registers, the heads of a few query rows pass by in shared memory.
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include "front.h"
#include "ptx.cuh"

namespace dsa {
namespace {

constexpr int kTile = 128;   // positions of a CTA
constexpr int kRows = 4;     // query rows of a CTA, of one sequence

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

template <bool kFp8>
__global__ void __launch_bounds__(kTile) index_scores_kernel(const __grid_constant__ dsa_v32_index_scores_args p, int tiles, int groups) {
    __shared__ float qs[64][kDIndex];
    __shared__ float ws[64];
    __shared__ float best[4];
    const int tile = blockIdx.x % tiles;
    const int64_t unit = blockIdx.x / tiles;
    const int seq = (int)(unit / groups), r0 = (int)(unit % groups) * kRows;
    const int pos = tile * kTile + threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the row of the position
    int64_t row = -1;
    if (pos < p.kv_len) {
        if (p.block_table != nullptr) {
            const int blk = pos / p.page_block_size;
            if (blk < p.block_table_stride) {
                const int page = __ldg(p.block_table + (int64_t)seq * p.block_table_stride + blk);
                if (page >= 0) row = (int64_t)page * p.page_block_size + pos % p.page_block_size;
            }
        } else {
            if (p.kv_batch_stride_rows == 0 || pos < p.kv_batch_stride_rows) row = (int64_t)seq * p.kv_batch_stride_rows + pos;
        }
        if (row >= p.num_index_rows) row = -1;
    }
    float k[kDIndex], ks = 1.0f;
#pragma unroll
    for (int i = 0; i < kDIndex; ++i) k[i] = 0.0f;
    if (row >= 0) {
        if constexpr (kFp8) {
            const int64_t page = row / p.page_block_size, at = row % p.page_block_size;
            const uint8_t* base = reinterpret_cast<const uint8_t*>(p.index_cache) + page * p.page_block_size * (kDIndex + 4);
            ks = __ldg(reinterpret_cast<const float*>(base + (int64_t)p.page_block_size * kDIndex) + at);
            const __nv_fp8_e4m3* key = reinterpret_cast<const __nv_fp8_e4m3*>(base + at * kDIndex);
#pragma unroll
            for (int i = 0; i < kDIndex; ++i) k[i] = static_cast<float>(key[i]);
        } else {
            const __nv_bfloat16* key = reinterpret_cast<const __nv_bfloat16*>(p.index_cache) + row * kDIndex;
#pragma unroll
            for (int i = 0; i < kDIndex; ++i) k[i] = __bfloat162float(key[i]);
        }
    }
    for (int r = r0; r < min(r0 + kRows, p.s_q); ++r) {
        const int64_t q = (int64_t)seq * p.s_q + r;
        __syncthreads();
        for (int i = threadIdx.x; i < p.H * kDIndex; i += kTile) {
            const int64_t at = q * p.stride_q_row + (i / kDIndex) * p.stride_q_head + i % kDIndex;
            qs[i / kDIndex][i % kDIndex] = kFp8 ? static_cast<float>(reinterpret_cast<const __nv_fp8_e4m3*>(p.q)[at]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.q)[at]);
        }
        if (threadIdx.x < p.H) ws[threadIdx.x] = p.weights[q * p.stride_w_row + threadIdx.x];
        __syncthreads();
        float s = 0.0f;
        for (int h = 0; h < p.H; ++h) {
            float d = 0.0f;
#pragma unroll
            for (int i = 0; i < kDIndex; ++i) d = fmaf(qs[h][i], k[i], d);
            s = fmaf(ws[h], max_nan(d, 0.0f), s);
        }
        const int valid = min(p.kv_len, p.valid_len != nullptr ? p.valid_len[q] : p.kv_len);
        s = row >= 0 && pos < valid ? s * ks : -INFINITY;
        float* out = p.out + q * p.stride_o_row;
        const int cols = (p.kv_len + p.block - 1) / p.block;
        if (p.block > 1) {
            for (int off = 1; off < min(p.block, 32); off <<= 1) s = max_nan(s, __shfl_xor_sync(0xffffffffu, s, off));
            if (p.block >= 64) {
                __syncthreads();
                if (lane == 0) best[warp] = s;
                __syncthreads();
                s = max_nan(s, best[warp ^ 1]);
                if (p.block == 128) s = max_nan(max_nan(best[0], best[1]), max_nan(best[2], best[3]));
            }
        }
        if (threadIdx.x % p.block == 0 && pos / p.block < cols) out[pos / p.block] = s;
    }
}

}  // namespace

cudaError_t launch_index_scores(const dsa_v32_index_scores_args& a, cudaStream_t stream) {
    if (a.total_q == 0) return cudaSuccess;
    const int tiles = (a.kv_len + kTile - 1) / kTile, groups = (a.s_q + kRows - 1) / kRows;
    const int64_t blocks = (int64_t)tiles * groups * (a.total_q / a.s_q);
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    if (a.cache_dtype == DSA_V32_KV_FP8) index_scores_kernel<true><<<(unsigned)blocks, kTile, 0, stream>>>(a, tiles, groups);
    else index_scores_kernel<false><<<(unsigned)blocks, kTile, 0, stream>>>(a, tiles, groups);
    return cudaGetLastError();
}

}  // namespace dsa
