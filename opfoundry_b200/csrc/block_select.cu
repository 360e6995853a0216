// Selection of the best blocks of positions for every query row, written as the lists of positions that the attention takes (sm_100a).
//
// A block's score becomes a 32-bit key of the same order, the largest key for the blocks that are always selected.  The threshold is the
// largest number that num_selected keys reach: it is found bit by bit from the top on keys that stay in registers, until exactly num_selected
// keys reach the trial or at most 32 are left to decide between, which are ranked against each other at once (equal scores would take all 32
// trials: 64 rows of 2048 blocks, a tenth of the scores rounded, 6.5 instead of 4.7 us, of 7813 blocks 13.7 instead of 10.7; one row without equal
// scores 3.9 instead of 4.3).  Ties at the threshold go to the lowest blocks by one prefix sum, which also gives
// every selected block its place; then the whole team writes the positions, 16 bytes at a time.
//
// A team of one warp takes a row of up to 512 blocks, of a CTA a longer one: up to 8 warps x 32 lanes x 32 keys, or 32 x 32 x 16; rows of
// more blocks are read again for every trial.  Bounds: the chain of trials (about 13, one exchange each), for many rows of up to 512 blocks beside the
// bytes (scores once, lists once).  In a graph, inputs past L2, lists of 2048 positions: 64 rows of 2048 blocks 4.8 us, of 40000 80; 4096 rows of 256
// blocks 10.4 (57 % of a copy's rate), of 512 15.5, of 1024 45, of 2048 47 (floor 9.1): every trial compares all keys of the row, 88 % of the issue slots.
// A CTA a row that read the scores for each of 32 trials and wrote from the selecting threads took 105 us for 4096 rows of 256 blocks and 31 for 64 of 2048.
#include "front.h"
#include "ptx.cuh"

namespace dsa {
namespace {

constexpr int kListed = 4096;   // selected blocks that a team's list in shared memory holds; longer lists are written by the selecting threads

// float -> key with the same order as the values, at least 1; NaN lowest, -0.0 ties with +0.0 (as in topk_select.cu)
__device__ __forceinline__ uint32_t block_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
    return x != x ? 1u : k;
}

struct SelectParams {
    const float* scores;
    const int32_t* valid_len;
    int32_t* out;
    int64_t stride_row;
    int total_q, num_blocks, block, block_shift, num_selected, first, local;   // block_shift: log2(block), or -1
    int wide;      // lists may be written 16 bytes at a time
    int aligned;   // scores may be read 16 bytes at a time
};

// kWarps warps with kPer keys a lane; kReload: of rows of any length, read again whenever they are looked at.
template <int kWarps, int kPer, bool kReload>
__global__ void __launch_bounds__(kWarps == 1 ? 256 : 32 * kWarps) block_select_kernel(const __grid_constant__ SelectParams p) {
    constexpr int kTeam = 32 * kWarps, kTeams = kWarps == 1 ? 8 : 1;
    constexpr int kList = !kReload && kTeam * kPer < kListed ? kTeam * kPer : kListed;
    __shared__ int list[kTeams][kList];
    __shared__ uint32_t parts[3][kWarps == 1 ? 1 : kWarps];
    __shared__ __align__(16) uint32_t left[kTeams][32];   // the keys that are left
    __shared__ uint32_t left_count[kTeams];
    const int tid = kWarps == 1 ? (threadIdx.x & 31) : threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int team = kWarps == 1 ? warp : 0;
    const int q = (int)blockIdx.x * kTeams + team;
    grid_dependency_wait();
    if (kWarps == 1 && q >= p.total_q) return;
    auto team_sync = [] {
        if constexpr (kWarps == 1) __syncwarp();
        else __syncthreads();
    };
    int round = 0;
    // Sums over the team; the third exchange after one may reuse its words
    auto team_sum = [&](uint32_t x) -> uint32_t {
        x = __reduce_add_sync(0xffffffffu, x);
        if constexpr (kWarps > 1) {
            uint32_t* w = parts[round];
            round = round == 2 ? 0 : round + 1;
            if (lane == 0) w[warp] = x;
            __syncthreads();
            x = __reduce_add_sync(0xffffffffu, lane < kWarps ? w[lane] : 0u);
        }
        return x;
    };

    const int most = p.num_blocks * p.block;   // below 2^31
    const int valid = min(most, max(0, p.valid_len != nullptr ? __ldg(p.valid_len + q) : most));
    const int live = p.block_shift >= 0 ? (int)(((int64_t)valid + p.block - 1) >> p.block_shift) : (int)(((int64_t)valid + p.block - 1) / p.block);
    const float* row = p.scores + q * p.stride_row;
    int32_t* out = p.out + (int64_t)q * p.num_selected * p.block;
    const bool listed = p.num_selected <= kList;
    auto key_of = [&](int b, float x) -> uint32_t { return b >= live ? 0u : b < p.first || b >= live - p.local ? 0xFFFFFFFFu : block_key(x); };
    // the positions of the block that stands at place r of the list
    auto write_one = [&](int r, int b) {
        for (int i = 0; i < p.block; ++i) {
            const int pos = b * p.block + i;
            out[(int64_t)r * p.block + i] = pos < valid ? pos : -1;
        }
    };
    const int n = p.num_selected;
    if (live > n) {
        uint32_t key[kReload ? 1 : kPer];
        // thread tid has blocks kPer tid .. of a chunk of kTeam * kPer
        auto load = [&](int chunk, uint32_t (&k)[kPer]) {
            const int b0 = chunk * kTeam * kPer + tid * kPer;
            if (p.aligned && b0 + kPer <= p.num_blocks) {
#pragma unroll
                for (int j = 0; j < kPer; j += 4) {
                    const float4 v = *reinterpret_cast<const float4*>(row + b0 + j);
                    k[j] = key_of(b0 + j, v.x);
                    k[j + 1] = key_of(b0 + j + 1, v.y);
                    k[j + 2] = key_of(b0 + j + 2, v.z);
                    k[j + 3] = key_of(b0 + j + 3, v.w);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kPer; ++j) k[j] = b0 + j < live ? key_of(b0 + j, row[b0 + j]) : 0u;
            }
        };
        const int chunks = kReload ? (live + kTeam * kPer - 1) / (kTeam * kPer) : 1;
        if constexpr (!kReload) load(0, key);
        auto each_chunk = [&](auto f) {
            if constexpr (kReload) {
                uint32_t k[kPer];
                for (int c = 0; c < chunks; ++c) {
                    load(c, k);
                    f(c, k);
                }
            } else {
                f(0, key);
            }
        };
        // floor_key: the largest found number that at least n keys reach, `reach` do; fewer than n, `above`, reach `over` (0: 2^32)
        uint32_t floor_key = 0, reach = 0xFFFFFFFFu, over = 0, above = 0;
        uint32_t ties = 0xFFFFFFFFu;   // of the keys equal to floor_key the lowest so many are taken
        if (tid < 32) left[team][tid] = 0u;
        if (tid == 0) left_count[team] = 0u;
        for (uint32_t bit = 0x80000000u;; bit >>= 1) {
            if (bit == 0) {
                ties = (uint32_t)n - above;
                break;
            }
            const uint32_t trial = floor_key | bit;
            uint32_t c = 0;
            each_chunk([&](int, const uint32_t* k) {
#pragma unroll
                for (int j = 0; j < kPer; ++j) c += k[j] >= trial;
            });
            c = team_sum(c);
            if (c >= (uint32_t)n) floor_key = trial, reach = c;
            else over = trial, above = c;
            if (reach == (uint32_t)n) break;
            if (reach - above <= 32) {
                team_sync();   // (a team of one warp: left is zeros)
                each_chunk([&](int, const uint32_t* k) {
                    uint32_t m = 0;
#pragma unroll
                    for (int j = 0; j < kPer; ++j) m += k[j] - floor_key < over - floor_key;
                    if (m != 0) {
                        uint32_t at = atomicAdd(&left_count[team], m);   // (their order does not matter)
#pragma unroll
                        for (int j = 0; j < kPer; ++j)
                            if (k[j] - floor_key < over - floor_key) left[team][at++] = k[j];
                    }
                });
                team_sync();
                const uint32_t mine = left[team][lane], need = (uint32_t)n - above;
                uint32_t greater = 0, equal = 0;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const uint4 x = *reinterpret_cast<const uint4*>(&left[team][i]);
                    greater += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
                    equal += (x.x == mine) + (x.y == mine) + (x.z == mine) + (x.w == mine);
                }
                // the key that is the need-th largest (a live block's, so not 0): some lane has it
                const int at = __ffs(__ballot_sync(0xffffffffu, greater < need && need <= greater + equal)) - 1;
                floor_key = __shfl_sync(0xffffffffu, mine, at);
                ties = need - __shfl_sync(0xffffffffu, greater, at);
                break;
            }
        }
        uint32_t gt0 = 0, eq0 = 0;   // before the chunk
        each_chunk([&](int chunk, const uint32_t* k) {
            uint32_t gt = 0, eq = 0;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                gt += k[j] > floor_key;
                eq += k[j] == floor_key;
            }
            uint32_t x = gt | (eq << 16), incl = x;   // at most 32768 of a chunk
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const uint32_t o = __shfl_up_sync(0xffffffffu, incl, off);
                if (lane >= off) incl += o;
            }
            uint32_t before = incl - x, all = __shfl_sync(0xffffffffu, incl, 31);
            uint32_t all_gt = all & 0xFFFFu, all_eq = all >> 16, before_gt = before & 0xFFFFu, before_eq = before >> 16;
            if constexpr (kWarps > 1) {
                uint32_t* w = parts[round];
                round = round == 2 ? 0 : round + 1;
                if (lane == 31) w[warp] = incl;
                __syncthreads();
                const uint32_t v = lane < kWarps ? w[lane] : 0u;
                all_gt = __reduce_add_sync(0xffffffffu, v & 0xFFFFu);
                all_eq = __reduce_add_sync(0xffffffffu, v >> 16);
                before_gt += __reduce_add_sync(0xffffffffu, lane < warp ? v & 0xFFFFu : 0u);
                before_eq += __reduce_add_sync(0xffffffffu, lane < warp ? v >> 16 : 0u);
            }
            uint32_t g = gt0 + before_gt, e = eq0 + before_eq;
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                const bool above = k[j] > floor_key, equal = k[j] == floor_key;
                if (above || (equal && e < ties)) {
                    const int r = (int)(g + min(e, ties)), b = chunk * kTeam * kPer + tid * kPer + j;
                    if (listed) list[team][r] = b;
                    else write_one(r, b);
                }
                g += above;
                e += equal;
            }
            gt0 += all_gt;
            eq0 += all_eq;
        });
        if (!listed) return;
        team_sync();
    } else if (!listed) {   // everything that is valid, and padding
        for (int64_t i = tid; i < (int64_t)n * p.block; i += kTeam) out[i] = i < valid ? (int)i : -1;
        return;
    }
    // A place's first position from i on and how many from there on are valid; with every live block selected its place is its number.
    struct Run {
        int pos, left;
    };
    auto run_at = [&](uint32_t at) {
        const int r = (int)(p.block_shift >= 0 ? at >> p.block_shift : at / (uint32_t)p.block);
        const int b = live > n ? list[team][r] : r, pos = b < live ? b * p.block + (int)(at - (uint32_t)r * p.block) : 0;
        return Run{pos, b < live ? valid - pos : 0};
    };
    const uint32_t total = (uint32_t)n * p.block;   // below 2^31
    if (p.wide) {
        for (uint32_t i = 4 * tid; i < total; i += 4 * kTeam) {
            const Run x = run_at(i);
            *reinterpret_cast<int4*>(out + i) = make_int4(x.left > 0 ? x.pos : -1, x.left > 1 ? x.pos + 1 : -1, x.left > 2 ? x.pos + 2 : -1, x.left > 3 ? x.pos + 3 : -1);
        }
    } else {
        for (uint32_t i = tid; i < total; i += kTeam) {
            const Run x = run_at(i);
            out[i] = x.left > 0 ? x.pos : -1;
        }
    }
}

}  // namespace

cudaError_t launch_block_select(const float* scores, int64_t stride_row, const int32_t* valid_len, int total_q, int num_blocks, int block, int num_selected,
                                int first, int local, int32_t* indices_out, cudaStream_t stream) {
    if (total_q == 0) return cudaSuccess;
    SelectParams p{scores, valid_len, indices_out, stride_row, total_q, num_blocks, block, -1, num_selected, first, local, 0, 0};
    for (int sh = 0; sh < 31; ++sh)
        if (block == (1 << sh)) p.block_shift = sh;
    p.wide = block % 4 == 0 && (reinterpret_cast<uintptr_t>(indices_out) & 15u) == 0;
    p.aligned = stride_row % 4 == 0 && (reinterpret_cast<uintptr_t>(scores) & 15u) == 0;
    auto go = [&](auto kernel, int threads, int rows) {
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute attr[1];
        cfg.gridDim = dim3((unsigned)(((int64_t)total_q + rows - 1) / rows), 1, 1);
        cfg.blockDim = dim3(threads, 1, 1);
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, kernel, p);
    };
    if (num_blocks <= 256) return go(block_select_kernel<1, 8, false>, 256, 8);
    if (num_blocks <= 512) return go(block_select_kernel<1, 16, false>, 256, 8);
    if (num_blocks <= 2048) return go(block_select_kernel<8, 8, false>, 256, 1);
    if (num_blocks <= 8192) return go(block_select_kernel<8, 32, false>, 256, 1);
    if (num_blocks <= 16384) return go(block_select_kernel<32, 16, false>, 1024, 1);
    return go(block_select_kernel<32, 16, true>, 1024, 1);
}

}  // namespace dsa
