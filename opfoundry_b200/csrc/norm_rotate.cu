// Norm and rotation of queries and keys, and the append of new tokens to the paged caches (sm_100a).
//
// A vector x of one head (or one latent): with mu its mean (0 unless centred), y = (x - mu) / sqrt(mean((x - mu)^2) + eps) * w + b, then
// pairs of its rotated values turned by the angle of the token's position, then one rounding to bf16, or to e4m3 with scale = amax / 448.
// Everything between the load and that rounding is fp32.  Bound by HBM: every value is read and written once.
#include <cuda_bf16.h>
#include "front.h"
#include "ptx.cuh"

namespace dsa {
namespace {

// ------------------------------------------------------------------ values
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
    v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xFFFF0000u);
    v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xFFFF0000u);
}
__device__ __forceinline__ void load2(const float* p, float (&v)[2]) {
    const float2 a = __ldg(reinterpret_cast<const float2*>(p));
    v[0] = a.x, v[1] = a.y;
}
__device__ __forceinline__ void load2(const __nv_bfloat16* p, float (&v)[2]) {
    const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(p));
    v[0] = __uint_as_float(u << 16), v[1] = __uint_as_float(u & 0xFFFF0000u);
}

template <int kLanes> __device__ __forceinline__ float sum_over(float x) {
#pragma unroll
    for (int off = kLanes / 2; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
    return x;
}
template <int kLanes> __device__ __forceinline__ float max_over(float x) {
#pragma unroll
    for (int off = kLanes / 2; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
    return x;
}

// Quotients by one scale, each the rounded quotient (the steps of pack_fp8_rows_kernel in merge_pack.cu).
struct Divider {
    float scale, recip;
    bool plain;
    __device__ explicit Divider(float amax) {
        scale = amax > 0.0f ? __fdiv_rn(amax, 448.0f) : 1.0f;
        recip = __frcp_rn(scale);
        plain = scale >= 0x1p-80f && scale <= 0x1p80f;
    }
    __device__ float operator()(float a) const {
        if (!plain) return __fdiv_rn(a, scale);
        const float q = __fmul_rn(a, recip);
        return copysignf(__fmaf_rn(__fmaf_rn(-q, scale, a), recip, q), a);
    }
};
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)lo | ((uint32_t)hi << 16);
}

// ------------------------------------------------------------------ heads of queries and keys
struct RotateSide {
    const void* x;
    void* out;
    float* scale;
    const float* weight;
    const float* bias;
    const float* gate;
    int64_t x_row, x_head, o_row, o_head;
};
struct RotateParams {
    RotateSide side[2];
    const float* cos_sin;
    const int32_t* positions;
    int64_t rows;          // tokens x (heads of queries + of keys)
    int q_heads, heads, head_dim, rope_begin, rope_dim, max_positions, interleaved, center;
    float eps;
};

// kLanes lanes take a row; a lane holds kVecs times eight consecutive values.
template <typename In, bool kE4m3, int kLanes, int kVecs>
__global__ void __launch_bounds__(256) norm_rotate_kernel(const __grid_constant__ RotateParams p) {
    const int lane = threadIdx.x % kLanes;
    const int64_t row = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    bool live = row < p.rows;
    const int64_t token = live ? row / p.heads : 0;
    int head = live ? (int)(row - token * p.heads) : 0;
    const RotateSide& s = p.side[head >= p.q_heads ? 1 : 0];
    const bool is_q = head < p.q_heads;
    if (!is_q) head -= p.q_heads;
    int pos = 0;
    if (live && p.positions != nullptr) {
        pos = __ldg(p.positions + token);
        live = pos >= 0 && pos < p.max_positions;
    }
    const In* x = reinterpret_cast<const In*>(s.x) + token * s.x_row + head * s.x_head;
    float v[kVecs][8];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int c = 8 * (lane + k * kLanes);
        if (live && c < p.head_dim) {
            load8(x + c, v[k]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = 0.0f;
        }
    }
    float mean = 0.0f, rstd = 1.0f;
    const bool norm = s.weight != nullptr;
    if (p.side[0].weight != nullptr || p.side[1].weight != nullptr) {   // (the whole warp, whichever side its rows are of)
        if (p.center) {
            float t = 0.0f;
#pragma unroll
            for (int k = 0; k < kVecs; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) t += v[k][i];
            mean = sum_over<kLanes>(t) / (float)p.head_dim;
        }
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < kVecs; ++k)
            if (8 * (lane + k * kLanes) < p.head_dim)
#pragma unroll
                for (int i = 0; i < 8; ++i) t = fmaf(v[k][i] - mean, v[k][i] - mean, t);
        rstd = 1.0f / sqrtf(sum_over<kLanes>(t) / (float)p.head_dim + p.eps);
    }
    auto normed = [&](float (&u)[8], int c) {
        if (!norm) return;
        float w[8], b[8];
        load8(s.weight + c, w);
        if (s.bias != nullptr) load8(s.bias + c, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = (u[i] - mean) * rstd * w[i] + (s.bias != nullptr ? b[i] : 0.0f);
    };
    const float* table = p.cos_sin + (int64_t)pos * p.rope_dim;
    const int half = p.rope_dim / 2;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int c = 8 * (lane + k * kLanes);
        if (!live || c >= p.head_dim) continue;
        normed(v[k], c);
        const int r = c - p.rope_begin;
        if (r < 0 || r >= p.rope_dim) continue;
        if (p.interleaved) {
            float co[4], si[4];
            load4(table + r / 2, co);
            load4(table + half + r / 2, si);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = v[k][2 * i], b = v[k][2 * i + 1];
                v[k][2 * i] = a * co[i] - b * si[i];
                v[k][2 * i + 1] = a * si[i] + b * co[i];
            }
        } else {
            const bool upper = r >= half;
            float o[8], co[8], si[8];
            load8(x + c + (upper ? -half : half), o);
            normed(o, c + (upper ? -half : half));
            load8(table + r - (upper ? half : 0), co);
            load8(table + half + r - (upper ? half : 0), si);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = upper ? o[i] * si[i] + v[k][i] * co[i] : v[k][i] * co[i] - o[i] * si[i];
        }
    }
    if constexpr (kE4m3) {
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < kVecs; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[k][i]));
        const Divider d(max_over<kLanes>(amax));
        if (!live) return;
        uint8_t* out = reinterpret_cast<uint8_t*>(s.out) + token * s.o_row + head * s.o_head;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const int c = 8 * (lane + k * kLanes);
            if (c < p.head_dim)
                *reinterpret_cast<uint2*>(out + c) = make_uint2(e4m3x4(d(v[k][0]), d(v[k][1]), d(v[k][2]), d(v[k][3])), e4m3x4(d(v[k][4]), d(v[k][5]), d(v[k][6]), d(v[k][7])));
        }
        if (lane == 0) {
            const int64_t at = token * (is_q ? p.q_heads : p.heads - p.q_heads) + head;
            s.scale[at] = s.gate != nullptr ? d.scale * __ldg(s.gate + at) : d.scale;
        }
    } else {
        __syncwarp();   // in place: a lane's values may still be another's partners
        if (!live) return;
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(s.out) + token * s.o_row + head * s.o_head;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const int c = 8 * (lane + k * kLanes);
            if (c < p.head_dim)
                *reinterpret_cast<uint4*>(out + c) = make_uint4(pack_bf16x2(v[k][0], v[k][1]), pack_bf16x2(v[k][2], v[k][3]), pack_bf16x2(v[k][4], v[k][5]), pack_bf16x2(v[k][6], v[k][7]));
        }
    }
}

template <typename In, bool kE4m3> cudaError_t launch_rotate(const RotateParams& p, cudaStream_t stream) {
    auto go = [&](auto kernel, int lanes) {
        const int64_t blocks = (p.rows * lanes + 255) / 256;
        if (blocks > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
        kernel<<<(unsigned)blocks, 256, 0, stream>>>(p);
        return cudaGetLastError();
    };
    if (p.head_dim <= 64) return go(norm_rotate_kernel<In, kE4m3, 8, 1>, 8);
    if (p.head_dim <= 128) return go(norm_rotate_kernel<In, kE4m3, 16, 1>, 16);
    if (p.head_dim <= 256) return go(norm_rotate_kernel<In, kE4m3, 32, 1>, 32);
    if (p.head_dim <= 512) return go(norm_rotate_kernel<In, kE4m3, 32, 2>, 32);
    if (p.head_dim <= 768) return go(norm_rotate_kernel<In, kE4m3, 32, 3>, 32);
    return go(norm_rotate_kernel<In, kE4m3, 32, 4>, 32);
}

// ------------------------------------------------------------------ append to the paged caches
struct AppendParams {
    dsa_v32_append_args a;
    int page_shift;      // log2(page_block_size), or -1
};

// The physical row of a token, or -1: padding, or outside the table or the cache.
__device__ __forceinline__ int64_t append_row(const AppendParams& p, int t, int pos) {
    if (pos < 0 || pos >= p.a.max_positions) return -1;
    const int seq = p.a.seq_ids != nullptr ? __ldg(p.a.seq_ids + t) : t / p.a.s_q;
    if (seq < 0) return -1;
    int64_t row;
    if (p.a.block_table != nullptr) {
        const int blk = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.a.page_block_size;
        if (seq >= p.a.num_seqs || blk >= p.a.block_table_stride) return -1;
        const int page = __ldg(p.a.block_table + (int64_t)seq * p.a.block_table_stride + blk);
        if (page < 0) return -1;
        row = (int64_t)page * p.a.page_block_size + (pos - blk * p.a.page_block_size);
    } else {
        if (p.a.num_seqs > 0 && seq >= p.a.num_seqs) return -1;
        if (p.a.kv_batch_stride_rows > 0 && pos >= p.a.kv_batch_stride_rows) return -1;   // the next sequence's rows
        row = (int64_t)seq * p.a.kv_batch_stride_rows + pos;
    }
    return row < p.a.num_kv_rows ? row : -1;
}

// One warp a row.  Units 0 .. tokens - 1 are rows of the attention's cache (when it is given), then those of the index cache.
template <typename In, bool kFp8>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int n = p.a.num_tokens, n_kv = p.a.kv != nullptr ? n : 0;
    if (unit >= (int64_t)n_kv + (p.a.index_cache != nullptr ? n : 0)) return;
    const bool index = unit >= n_kv;
    const int t = (int)(index ? unit - n_kv : unit);
    const int pos = __ldg(p.a.positions + t);
    const int64_t row = append_row(p, t, pos);
    if (row < 0) return;
    const float* table = p.a.cos_sin + (int64_t)pos * kDRope;

    if (!index) {
        // lane = eight of them a group of 128 values: 16 values each, and two of the rope key
        const In* x = reinterpret_cast<const In*>(p.a.latent) + t * p.a.stride_latent + 16 * lane;
        float v[2][8];
        load8(x, v[0]);
        load8(x + 8, v[1]);
        const In* r = reinterpret_cast<const In*>(p.a.rope) + t * p.a.stride_rope;
        uint32_t rope;
        if (p.a.interleaved) {
            float u[2];
            load2(r + 2 * lane, u);
            const float co = __ldg(table + lane), si = __ldg(table + 32 + lane);
            rope = pack_bf16x2(u[0] * co - u[1] * si, u[0] * si + u[1] * co);
        } else {
            const bool upper = lane >= 16;
            float u[2], o[2], co[2], si[2];
            load2(r + 2 * lane, u);
            load2(r + 2 * (lane ^ 16), o);
            load2(table + 2 * (lane & 15), co);
            load2(table + 32 + 2 * (lane & 15), si);
            rope = upper ? pack_bf16x2(o[0] * si[0] + u[0] * co[0], o[1] * si[1] + u[1] * co[1]) : pack_bf16x2(u[0] * co[0] - o[0] * si[0], u[1] * co[1] - o[1] * si[1]);
        }
        if (p.a.latent_weight != nullptr) {
            float t2 = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) t2 = fmaf(v[k][i], v[k][i], t2);
            const float rstd = 1.0f / sqrtf(sum_over<32>(t2) / (float)kDV + p.a.eps);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float w[8];
                load8(p.a.latent_weight + 16 * lane + 8 * k, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[k][i] = v[k][i] * rstd * w[i];
            }
        }
        if constexpr (kFp8) {
            float amax = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[k][i]));
            const Divider d(max_over<8>(amax));
            uint8_t* out = reinterpret_cast<uint8_t*>(p.a.kv) + row * kFp8RowBytes;
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = e4m3x4(d(v[k >> 1][4 * (k & 1)]), d(v[k >> 1][4 * (k & 1) + 1]), d(v[k >> 1][4 * (k & 1) + 2]), d(v[k >> 1][4 * (k & 1) + 3]));
            reinterpret_cast<uint4*>(out)[lane] = make_uint4(w[0], w[1], w[2], w[3]);
            if ((lane & 7) == 0) reinterpret_cast<float*>(out + kDV)[lane >> 3] = d.scale;
            reinterpret_cast<uint32_t*>(out + kDV + 16)[lane] = rope;
        } else {
            uint8_t* out = reinterpret_cast<uint8_t*>(p.a.kv) + row * (2 * kDQK);
#pragma unroll
            for (int k = 0; k < 2; ++k)
                reinterpret_cast<uint4*>(out)[2 * lane + k] = make_uint4(pack_bf16x2(v[k][0], v[k][1]), pack_bf16x2(v[k][2], v[k][3]), pack_bf16x2(v[k][4], v[k][5]), pack_bf16x2(v[k][6], v[k][7]));
            reinterpret_cast<uint32_t*>(out + 2 * kDV)[lane] = rope;
        }
    } else {
        // lane = values 4 lane .. 4 lane + 3; the first 16 lanes hold the rotated half
        float v[4];
        load4(reinterpret_cast<const In*>(p.a.index_key) + t * p.a.stride_index_key + 4 * lane, v);
        if (p.a.index_weight != nullptr) {
            float mean = 0.0f;
            if (p.a.index_center) mean = sum_over<32>((v[0] + v[1]) + (v[2] + v[3])) / (float)kDIndex;
            float t2 = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) t2 = fmaf(v[i] - mean, v[i] - mean, t2);
            const float rstd = 1.0f / sqrtf(sum_over<32>(t2) / (float)kDIndex + p.a.eps);
            float w[4], b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            load4(p.a.index_weight + 4 * lane, w);
            if (p.a.index_bias != nullptr) load4(p.a.index_bias + 4 * lane, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = (v[i] - mean) * rstd * w[i] + b[i];
        }
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = __shfl_xor_sync(0xffffffffu, v[i], 8);   // 32 values on: the other half of the rotated ones
        if (lane < 16) {
            if (p.a.index_interleaved) {
                float co[2], si[2];
                load2(table + 2 * lane, co);
                load2(table + 32 + 2 * lane, si);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float a = v[2 * i], b = v[2 * i + 1];
                    v[2 * i] = a * co[i] - b * si[i];
                    v[2 * i + 1] = a * si[i] + b * co[i];
                }
            } else {
                float co[4], si[4];
                load4(table + 4 * (lane & 7), co);
                load4(table + 32 + 4 * (lane & 7), si);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = lane >= 8 ? o[i] * si[i] + v[i] * co[i] : v[i] * co[i] - o[i] * si[i];
            }
        }
        if constexpr (kFp8) {
            const Divider d(max_over<32>(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])))));
            const int64_t page = row / p.a.page_block_size, at = row - page * p.a.page_block_size;
            uint8_t* base = reinterpret_cast<uint8_t*>(p.a.index_cache) + page * p.a.page_block_size * (kDIndex + 4);
            reinterpret_cast<uint32_t*>(base + at * kDIndex)[lane] = e4m3x4(d(v[0]), d(v[1]), d(v[2]), d(v[3]));
            if (lane == 0) reinterpret_cast<float*>(base + (int64_t)p.a.page_block_size * kDIndex)[at] = d.scale;
        } else {
            reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(p.a.index_cache) + row * (2 * kDIndex))[lane] = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
        }
    }
}

}  // namespace

cudaError_t launch_norm_rotate(const dsa_v32_norm_rotate_args& a, cudaStream_t stream) {
    RotateParams p = {};
    p.side[0] = RotateSide{a.q, a.q_out, a.q_scale, a.q_weight, a.q_bias, a.head_weight, a.stride_q_row, a.stride_q_head, a.stride_qo_row, a.stride_qo_head};
    p.side[1] = RotateSide{a.k, a.k_out, a.k_scale, a.k_weight, a.k_bias, nullptr, a.stride_k_row, a.stride_k_head, a.stride_ko_row, a.stride_ko_head};
    p.cos_sin = a.cos_sin;
    p.positions = a.positions;
    p.q_heads = a.q_heads;
    p.heads = a.q_heads + a.k_heads;
    p.rows = (int64_t)a.num_tokens * p.heads;
    p.head_dim = a.head_dim;
    p.rope_begin = a.rope_begin;
    p.rope_dim = a.rope_dim;
    p.max_positions = a.max_positions;
    p.interleaved = a.interleaved;
    p.center = a.center;
    p.eps = a.eps;
    if (p.rows == 0) return cudaSuccess;
    // In place and without a norm only the rotated values change: they are taken as the whole vectors.
    bool same = a.in_dtype == DSA_V32_DTYPE_BF16 && a.out_dtype == DSA_V32_DTYPE_BF16;
    for (int i = 0; i < 2; ++i) {
        const RotateSide& s = p.side[i];
        if (i == 0 || a.k_heads > 0) same = same && s.weight == nullptr && s.x == s.out && s.x_row == s.o_row && s.x_head == s.o_head;
    }
    if (same) {
        if (a.rope_dim == 0) return cudaSuccess;
        for (int i = 0; i < 2; ++i) {
            p.side[i].x = reinterpret_cast<const __nv_bfloat16*>(p.side[i].x) + a.rope_begin;
            p.side[i].out = reinterpret_cast<__nv_bfloat16*>(p.side[i].out) + a.rope_begin;
        }
        p.head_dim = a.rope_dim;
        p.rope_begin = 0;
    }
    const bool e4m3 = a.out_dtype == DSA_V32_DTYPE_E4M3;
    if (a.in_dtype == DSA_V32_DTYPE_FP32) return e4m3 ? launch_rotate<float, true>(p, stream) : launch_rotate<float, false>(p, stream);
    return e4m3 ? launch_rotate<__nv_bfloat16, true>(p, stream) : launch_rotate<__nv_bfloat16, false>(p, stream);
}

cudaError_t launch_append(const dsa_v32_append_args& a, cudaStream_t stream) {
    AppendParams p{a, -1};
    for (int sh = 0; sh < 31; ++sh)
        if (a.page_block_size == (1 << sh)) p.page_shift = sh;
    const int64_t units = (int64_t)a.num_tokens * ((a.kv != nullptr) + (a.index_cache != nullptr));
    if (units == 0) return cudaSuccess;
    const unsigned blocks = (unsigned)((units + 7) / 8);
    const bool fp8 = a.kv_dtype == DSA_V32_KV_FP8;
    auto kernel = a.in_dtype == DSA_V32_DTYPE_FP32 ? (fp8 ? append_kernel<float, true> : append_kernel<float, false>)
                                                   : (fp8 ? append_kernel<__nv_bfloat16, true> : append_kernel<__nv_bfloat16, false>);
    kernel<<<blocks, 256, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace dsa
