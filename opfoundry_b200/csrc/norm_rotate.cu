// Norm and rotation of queries and keys, and the append of new tokens to the paged caches (sm_100a).
//
// A vector x of one head (or one latent): with mu its mean (0 unless centred), y = (x - mu) / sqrt(mean((x - mu)^2) + eps) * w + b, then
// pairs of its rotated values turned by the angle of the token's position, then one rounding to bf16, or to e4m3 with scale = amax / 448.
// Everything between the load and that rounding is fp32.  Bound by HBM: every value is read and written once.
#include <cuda_bf16.h>
#include <type_traits>
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
    int64_t units;         // tokens x chunks of heads
    int q_chunks, chunks;  // of a token: those of queries, all
    int q_heads, heads, head_dim, rope_begin, rope_dim, max_positions, interleaved, center;
    float eps, inv_dim;
};

// What a group of lanes works on: kHeads heads of one token's queries or keys.
struct RotateUnit {
    int64_t token;
    int head, count, pos;
    bool is_q, live;
};
template <int kHeads> __device__ __forceinline__ RotateUnit unit_of(const RotateParams& p, int64_t unit) {
    RotateUnit u;
    u.live = unit < p.units;
    if (!u.live) unit = 0;
    if (p.units <= 0x7FFFFFFF) u.token = (uint32_t)unit / (uint32_t)p.chunks;   // (a 64-bit division is a hundred instructions)
    else u.token = unit / p.chunks;
    int chunk = (int)(unit - u.token * p.chunks);
    u.is_q = chunk < p.q_chunks;
    if (!u.is_q) chunk -= p.q_chunks;
    u.head = chunk * kHeads;
    u.count = min(kHeads, (u.is_q ? p.q_heads : p.heads - p.q_heads) - u.head);
    u.pos = 0;
    if (u.live && p.positions != nullptr) {
        u.pos = __ldg(p.positions + u.token);
        u.live = u.pos >= 0 && u.pos < p.max_positions;
    }
    if (!u.live) u.count = 0;
    return u;
}
// Subtracts the mean (center) and returns 1 / sqrt(mean of the squares + eps) (rsqrtf: two units in the last place).  Values behind the vector
// stay zeros.
template <int kLanes> __device__ __forceinline__ float centred_rstd(float (&v)[8], bool inside, float inv_dim, bool center, float eps) {
    if (center) {
        const float mean = sum_over<kLanes>(((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]))) * inv_dim;
        if (inside)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] -= mean;
    }
    float t = 0.0f, u = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        t = fmaf(v[i], v[i], t);
        u = fmaf(v[i + 1], v[i + 1], u);
    }
    return rsqrtf(fmaf(sum_over<kLanes>(t + u), inv_dim, eps));
}
__device__ __forceinline__ void store8(__nv_bfloat16* out, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
// The scale of a vector, and its values over it: eight products with a reciprocal (within a unit in the last place of 1 / scale) where the scale
// is an ordinary number, else quotients.
__device__ __forceinline__ float scale_of(float amax) {
    if (!(amax >= 0x1p-90f && amax <= 0x1p90f)) return amax > 0.0f ? __fdiv_rn(amax, 448.0f) : 1.0f;
    constexpr float r = 1.0f / 448.0f;
    const float q = amax * r;
    return __fmaf_rn(__fmaf_rn(-q, 448.0f, amax), r, q);   // the rounded quotient (Markstein, as in merge_pack.cu)
}
__device__ __noinline__ uint2 divide8(float a, float b, float c, float d, float e, float f, float g, float h, float scale) {
    return make_uint2(e4m3x4(__fdiv_rn(a, scale), __fdiv_rn(b, scale), __fdiv_rn(c, scale), __fdiv_rn(d, scale)),
                      e4m3x4(__fdiv_rn(e, scale), __fdiv_rn(f, scale), __fdiv_rn(g, scale), __fdiv_rn(h, scale)));
}
__device__ __forceinline__ uint2 pack8(const float (&v)[8], float scale) {
    if (!(scale >= 0x1p-100f && scale <= 0x1p100f)) return divide8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], scale);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
    r = fmaf(fmaf(-scale, r, 1.0f), r, r);
    return make_uint2(e4m3x4(v[0] * r, v[1] * r, v[2] * r, v[3] * r), e4m3x4(v[4] * r, v[5] * r, v[6] * r, v[7] * r));
}
__device__ __forceinline__ void put_scale(const RotateSide& s, int64_t at, float scale) { s.scale[at] = s.gate != nullptr ? scale * __ldg(s.gate + at) : scale; }

// Eight values as they come: one 16-byte load of bf16, or two loads, the second `apart` values further on.
template <typename In, bool kPairs> struct Raw;
template <> struct Raw<__nv_bfloat16, true> {
    uint4 u;
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int64_t, bool there) {
        u = make_uint4(0u, 0u, 0u, 0u);
        if (there) u = __ldg(reinterpret_cast<const uint4*>(p));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
template <> struct Raw<__nv_bfloat16, false> {
    uint2 a, b;
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int64_t apart, bool there) {
        a = b = make_uint2(0u, 0u);
        if (there) {
            a = __ldg(reinterpret_cast<const uint2*>(p));
            b = __ldg(reinterpret_cast<const uint2*>(p + apart));
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {a.x, a.y, b.x, b.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
template <bool kPairs> struct Raw<float, kPairs> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p, int64_t apart, bool there) {
        a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (there) {
            a = __ldg(reinterpret_cast<const float4*>(p));
            b = __ldg(reinterpret_cast<const float4*>(p + apart));
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w; }
};

// Vectors of up to 256 values: kLanes lanes a head, eight values a lane, kHeads heads of a token one after the other, all loaded first.  A lane's
// values are consecutive ones where pairs of neighbours are turned (kPairs), else a lane of the rotated part has four of one half and the four
// that they are turned against, so no value is exchanged.  Weights and angles of a lane's values stay in registers over the heads.
template <typename In, bool kE4m3, int kLanes, int kHeads, bool kPairs, bool kNorm>
__global__ void __launch_bounds__(256, kHeads == 1 ? 4 : 3) norm_rotate_kernel(const __grid_constant__ RotateParams p) {
    grid_dependency_wait();
    const int lane = threadIdx.x % kLanes;
    const RotateUnit u = unit_of<kHeads>(p, (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes);
    const RotateSide& s = p.side[u.is_q ? 0 : 1];
    const bool inside = 8 * lane < p.head_dim;
    const int count = inside ? u.count : 0;       // heads that this lane has values of
    // the lane's values: four from c0 on, four from c1 on
    const int half = p.rope_dim / 2;
    int c0 = 8 * lane, c1 = c0 + 4, angle = -1;   // angle: its first pair of the table, -1: not turned
    if (kPairs) {
        if (c0 >= p.rope_begin && c0 < p.rope_begin + p.rope_dim) angle = (c0 - p.rope_begin) / 2;
    } else if (c0 < p.rope_dim) {                 // the first lanes take the rotated part
        angle = 4 * lane;
        c0 = p.rope_begin + angle;
        c1 = c0 + half;
    } else if (c0 - p.rope_dim < p.rope_begin) {  // then what lies before it
        c0 -= p.rope_dim;
        c1 = c0 + 4;
    }
    const bool turns = angle >= 0 && count > 0;
    const int64_t x_head = s.x_head, o_head = s.o_head;
    const int64_t apart = kPairs ? 4 : c1 - c0;
    const In* x = reinterpret_cast<const In*>(s.x) + u.token * s.x_row + u.head * x_head + c0;
    Raw<In, kPairs> raw[kHeads];
#pragma unroll
    for (int k = 0; k < kHeads; ++k, x += x_head) raw[k].load(x, apart, k < count);
    const bool norm = kNorm && s.weight != nullptr, center = kNorm && norm && p.center, shifted = norm && s.bias != nullptr;
    float w[8], co[4], si[4];
    if (norm) {
        Raw<float, kPairs> t;
        t.load(s.weight + c0, apart, inside);         // (lanes behind the vector stay zero)
        t.get(w);
    }
    if (turns) {
        const float* table = p.cos_sin + (int64_t)u.pos * p.rope_dim + angle;
        load4(table, co);
        load4(table + half, si);
    }
    using Out = typename std::conditional<kE4m3, uint8_t, __nv_bfloat16>::type;
    Out* out = reinterpret_cast<Out*>(s.out) + u.token * s.o_row + u.head * o_head + c0;
#pragma unroll
    for (int k = 0; k < kHeads; ++k, out += o_head) {
        float y[8];
        raw[k].get(y);
        if (kNorm) {
            const float rstd = centred_rstd<kLanes>(y, inside, p.inv_dim, center, p.eps);   // (the whole warp, whichever side its heads are of)
            if (norm) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = y[i] * rstd * w[i];
                if (shifted) {
                    float b[8];
                    Raw<float, kPairs> t;
                    t.load(s.bias + c0, apart, inside);
                    t.get(b);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] += b[i];
                }
            }
        }
        if (turns)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int i0 = kPairs ? 2 * i : i, i1 = kPairs ? 2 * i + 1 : i + 4;
                const float a = y[i0], e = y[i1];
                y[i0] = a * co[i] - e * si[i];
                y[i1] = a * si[i] + e * co[i];
            }
        if constexpr (kE4m3) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(y[i]));
            const float scale = scale_of(max_over<kLanes>(amax));
            const uint2 codes = pack8(y, scale);
            if (k < count) {
                if constexpr (kPairs) {
                    *reinterpret_cast<uint2*>(out) = codes;
                } else {
                    *reinterpret_cast<uint32_t*>(out) = codes.x;
                    *reinterpret_cast<uint32_t*>(out + apart) = codes.y;
                }
                if (lane == 0) put_scale(s, u.token * (u.is_q ? p.q_heads : p.heads - p.q_heads) + u.head + k, scale);
            }
        } else if (k < count) {
            if constexpr (kPairs) {
                store8(out, y);
            } else {
                *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
                *reinterpret_cast<uint2*>(out + apart) = make_uint2(pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
            }
        }
    }
}

// Longer vectors: a warp a head, kVecs times eight values a lane.
template <typename In, bool kE4m3, int kVecs>
__global__ void __launch_bounds__(256) norm_rotate_long_kernel(const __grid_constant__ RotateParams p) {
    grid_dependency_wait();
    const int lane = threadIdx.x & 31;
    const RotateUnit u = unit_of<1>(p, (int64_t)blockIdx.x * 8 + threadIdx.x / 32);
    const RotateSide& s = p.side[u.is_q ? 0 : 1];
    const In* x = reinterpret_cast<const In*>(s.x) + u.token * s.x_row + u.head * s.x_head;
    if (!u.live) return;   // (a whole warp)
    float v[kVecs][8];
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int c = 8 * (lane + k * 32);
        if (c < p.head_dim) {
            load8(x + c, v[k]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = 0.0f;
        }
    }
    float mean = 0.0f, rstd = 1.0f;
    const bool norm = s.weight != nullptr;
    if (norm) {
        if (p.center) {
            float t = 0.0f;
#pragma unroll
            for (int k = 0; k < kVecs; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) t += v[k][i];
            mean = sum_over<32>(t) * p.inv_dim;
        }
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < kVecs; ++k)
            if (8 * (lane + k * 32) < p.head_dim)
#pragma unroll
                for (int i = 0; i < 8; ++i) t = fmaf(v[k][i] - mean, v[k][i] - mean, t);
        rstd = rsqrtf(fmaf(sum_over<32>(t), p.inv_dim, p.eps));
    }
    auto normed = [&](float (&y)[8], int c) {
        if (!norm) return;
        float w[8], b[8];
        load8(s.weight + c, w);
        if (s.bias != nullptr) load8(s.bias + c, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (y[i] - mean) * rstd * w[i] + (s.bias != nullptr ? b[i] : 0.0f);
    };
    const float* table = p.cos_sin + (int64_t)u.pos * p.rope_dim;
    const int half = p.rope_dim / 2;
#pragma unroll
    for (int k = 0; k < kVecs; ++k) {
        const int c = 8 * (lane + k * 32);
        if (c >= p.head_dim) continue;
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
        const float scale = scale_of(max_over<32>(amax));
        uint8_t* out = reinterpret_cast<uint8_t*>(s.out) + u.token * s.o_row + u.head * s.o_head;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const int c = 8 * (lane + k * 32);
            if (c < p.head_dim) *reinterpret_cast<uint2*>(out + c) = pack8(v[k], scale);
        }
        if (lane == 0) put_scale(s, u.token * (u.is_q ? p.q_heads : p.heads - p.q_heads) + u.head, scale);
    } else {
        __syncwarp();   // in place: a lane's values may still be another's partners
        __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(s.out) + u.token * s.o_row + u.head * s.o_head;
#pragma unroll
        for (int k = 0; k < kVecs; ++k) {
            const int c = 8 * (lane + k * 32);
            if (c < p.head_dim) store8(out + c, v[k]);
        }
    }
}

// A launch that may begin while the one before it in the stream ends; the kernels wait for it before they read anything.
template <typename P> cudaError_t launch_after(void (*kernel)(P), int64_t blocks, int threads, const P& p, cudaStream_t stream) {
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename In, bool kE4m3> cudaError_t launch_rotate(RotateParams& p, int64_t tokens, cudaStream_t stream) {
    int sms = 0;
    cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    // Four heads a unit once there are threads enough for the device without (2048 an SM).
    auto go = [&](auto one, auto four, int lanes) {
        const bool many = four != nullptr && tokens * p.heads * lanes >= (int64_t)sms * 2048;
        const int each = many ? 4 : 1;
        p.q_chunks = (p.q_heads + each - 1) / each;
        p.chunks = p.q_chunks + (p.heads - p.q_heads + each - 1) / each;
        p.units = tokens * p.chunks;
        return launch_after(many ? four : one, (p.units * lanes + 255) / 256, 256, p, stream);
    };
    using Kernel = void (*)(RotateParams);
    if (p.head_dim <= 256) {
        auto of = [&](auto pairs, auto normed) {
            constexpr bool kPairs = decltype(pairs)::value, kNorm = decltype(normed)::value;
            if (p.head_dim <= 64) return go(Kernel(norm_rotate_kernel<In, kE4m3, 8, 1, kPairs, kNorm>), Kernel(norm_rotate_kernel<In, kE4m3, 8, 4, kPairs, kNorm>), 8);
            if (p.head_dim <= 128) return go(Kernel(norm_rotate_kernel<In, kE4m3, 16, 1, kPairs, kNorm>), Kernel(norm_rotate_kernel<In, kE4m3, 16, 4, kPairs, kNorm>), 16);
            return go(Kernel(norm_rotate_kernel<In, kE4m3, 32, 1, kPairs, kNorm>), Kernel(norm_rotate_kernel<In, kE4m3, 32, 4, kPairs, kNorm>), 32);
        };
        const bool pairs = p.interleaved || p.rope_dim == 0;
        if (p.side[0].weight != nullptr || p.side[1].weight != nullptr) return pairs ? of(std::true_type(), std::true_type()) : of(std::false_type(), std::true_type());
        return pairs ? of(std::true_type(), std::false_type()) : of(std::false_type(), std::false_type());
    }
    if (p.head_dim <= 512) return go(Kernel(norm_rotate_long_kernel<In, kE4m3, 2>), Kernel(nullptr), 32);
    if (p.head_dim <= 768) return go(Kernel(norm_rotate_long_kernel<In, kE4m3, 3>), Kernel(nullptr), 32);
    return go(Kernel(norm_rotate_long_kernel<In, kE4m3, 4>), Kernel(nullptr), 32);
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
    grid_dependency_wait();
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
            const float rstd = rsqrtf(fmaf(sum_over<32>(t2), 1.0f / kDV, p.a.eps));
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
            if (p.a.index_center) mean = sum_over<32>((v[0] + v[1]) + (v[2] + v[3])) * (1.0f / kDIndex);
            float t2 = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) t2 = fmaf(v[i] - mean, v[i] - mean, t2);
            const float rstd = rsqrtf(fmaf(sum_over<32>(t2), 1.0f / kDIndex, p.a.eps));
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
    p.head_dim = a.head_dim;
    p.rope_begin = a.rope_begin;
    p.rope_dim = a.rope_dim;
    p.max_positions = a.max_positions;
    p.interleaved = a.interleaved;
    p.center = a.center;
    p.eps = a.eps;
    p.inv_dim = 1.0f / (float)a.head_dim;
    if (a.num_tokens == 0) return cudaSuccess;
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
    if (a.in_dtype == DSA_V32_DTYPE_FP32) return e4m3 ? launch_rotate<float, true>(p, a.num_tokens, stream) : launch_rotate<float, false>(p, a.num_tokens, stream);
    return e4m3 ? launch_rotate<__nv_bfloat16, true>(p, a.num_tokens, stream) : launch_rotate<__nv_bfloat16, false>(p, a.num_tokens, stream);
}

cudaError_t launch_append(const dsa_v32_append_args& a, cudaStream_t stream) {
    AppendParams p{a, -1};
    for (int sh = 0; sh < 31; ++sh)
        if (a.page_block_size == (1 << sh)) p.page_shift = sh;
    const int64_t units = (int64_t)a.num_tokens * ((a.kv != nullptr) + (a.index_cache != nullptr));
    if (units == 0) return cudaSuccess;
    const bool fp8 = a.kv_dtype == DSA_V32_KV_FP8;
    const auto kernel = a.in_dtype == DSA_V32_DTYPE_FP32 ? (fp8 ? append_kernel<float, true> : append_kernel<float, false>)
                                                   : (fp8 ? append_kernel<__nv_bfloat16, true> : append_kernel<__nv_bfloat16, false>);
    return launch_after(kernel, (units + 7) / 8, 256, p, stream);
}

}  // namespace dsa
