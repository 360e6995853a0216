// Norm and rotation of queries and keys, and the append of new tokens to the paged caches (sm_100a).
//
// A vector x of one head (or one latent): with mu its mean (0 unless centred), y = (x - mu) / sqrt(mean((x - mu)^2) + eps) * w + b, then
// pairs of its rotated values turned by the angle of the token's position, then one rounding to bf16, or to e4m3 with scale = amax / 448.
// Everything between the load and that rounding is fp32.  Every value is read and written once.  Times in a graph, inputs of many tokens past L2:
// 4091 tokens of 64 + 8 heads of 128, bf16 to bf16, 30 us (5.0 TB/s, 78 % of a copy), bound by HBM; 4096 x 64 heads to e4m3 30 us (3.3 TB/s), bound by
// loads and the chain of largest value, scale and quotients behind them (62 % of the issue slots); 4096 x 8 heads of 576 37 us (2.1 TB/s), by loads that
// 16 warps an SM have in flight (93 registers).  A few tokens are bound by the launch (1.7 us), appends by their chain position -> page -> row (64 tokens 2.4 us, 16380 into the fp8 caches
// 16.4, 12.6 with inputs in L2).
#include <cuda_bf16.h>
#include <type_traits>
#include "front.h"
#include "ptx.cuh"

namespace dsa {
namespace {

// ------------------------------------------------------------------ values
// Loads through the read-only path (kReadOnly) may be moved across barriers, so vectors that may be turned in place are read without it.
template <bool kReadOnly, typename T> __device__ __forceinline__ T load_as(const void* p) {
    if constexpr (kReadOnly) return __ldg(reinterpret_cast<const T*>(p));
    else return *reinterpret_cast<const T*>(p);
}
template <bool kReadOnly> __device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 u = load_as<kReadOnly, uint4>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}
template <bool kReadOnly> __device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = load_as<kReadOnly, float4>(p), b = load_as<kReadOnly, float4>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
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
// Subtracts the mean (center) and returns 1 / sqrt(mean of the squares + eps) (rsqrtf: two units in the last place).  The whole warp takes part in
// the sums, so `center` is the same for all of it; a lane whose vector has no norm, or that is behind its vector, keeps its values (`subtract`).
template <int kLanes> __device__ __forceinline__ float centred_rstd(float (&v)[8], bool subtract, float inv_dim, bool center, float eps) {
    if (center) {
        const float mean = __fmul_rn(sum_over<kLanes>(((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]))), inv_dim);
        if (subtract)
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
// A pair turned.  Products and sums of rotation, norm and shift are written out, so that a token's bytes are the same in every variant (left to the
// compiler, each variant fuses another product).
__device__ __forceinline__ float turned0(float a, float e, float co, float si) { return __fmaf_rn(-e, si, __fmul_rn(a, co)); }
__device__ __forceinline__ float turned1(float a, float e, float co, float si) { return __fmaf_rn(e, co, __fmul_rn(a, si)); }
__device__ __forceinline__ float scaled(float y, float rstd, float w) { return __fmul_rn(__fmul_rn(y, rstd), w); }
__device__ __forceinline__ void store8(__nv_bfloat16* out, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(out) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
// The scale of a vector.
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
// Eight values over their scale as e4m3, each the rounded quotient (one step of Markstein, as in merge_pack.cu), two at a time.
// n: the values negated, so that a zero keeps its sign: q = n (-1/s), then q - (q s + n) / s.  (Products with 1 / s alone give another
// code at some ties, in 5 % less time for 4096 x 64 heads of 128.)
__device__ __forceinline__ uint2 quotients8(const uint64_t (&n)[4], float scale) {
    if (!(scale >= 0x1p-80f && scale <= 0x1p80f)) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) unpack2(n[i], v[2 * i], v[2 * i + 1]);
        return divide8(-v[0], -v[1], -v[2], -v[3], -v[4], -v[5], -v[6], -v[7], scale);
    }
    const float r = -__frcp_rn(scale);
    const uint64_t r2 = pack2(r, r), s2 = pack2(scale, scale);
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint64_t q = mul2(n[2 * i + j], r2);
            unpack2(fma2(fma2(q, s2, n[2 * i + j]), r2, q), v[2 * j], v[2 * j + 1]);
        }
        w[i] = e4m3x4(v[0], v[1], v[2], v[3]);
    }
    return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ float amax2(uint64_t v, float m) {
    float a, b;
    unpack2(v, a, b);
    return max3(m, fabsf(a), fabsf(b));
}
__device__ __forceinline__ uint2 quotients8(const float (&v)[8], float scale) {
    const uint64_t n[4] = {pack2(-v[0], -v[1]), pack2(-v[2], -v[3]), pack2(-v[4], -v[5]), pack2(-v[6], -v[7])};
    return quotients8(n, scale);
}
__device__ __forceinline__ void put_scale(const RotateSide& s, int64_t at, float scale) { s.scale[at] = s.gate != nullptr ? scale * __ldg(s.gate + at) : scale; }

// Eight values as they come: one 16-byte load of bf16, or two loads, the second `apart` values further on.
template <typename In, bool kPairs, bool kReadOnly> struct Raw;
template <bool kReadOnly> struct Raw<__nv_bfloat16, true, kReadOnly> {
    uint4 u;
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int64_t, bool there) {
        u = make_uint4(0u, 0u, 0u, 0u);
        if (there) u = load_as<kReadOnly, uint4>(p);
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
template <bool kReadOnly> struct Raw<__nv_bfloat16, false, kReadOnly> {
    uint2 a, b;
    __device__ __forceinline__ void load(const __nv_bfloat16* p, int64_t apart, bool there) {
        a = b = make_uint2(0u, 0u);
        if (there) {
            a = load_as<kReadOnly, uint2>(p);
            b = load_as<kReadOnly, uint2>(p + apart);
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
template <bool kPairs, bool kReadOnly> struct Raw<float, kPairs, kReadOnly> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p, int64_t apart, bool there) {
        a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (there) {
            a = load_as<kReadOnly, float4>(p);
            b = load_as<kReadOnly, float4>(p + apart);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const { v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w; }
};

// Vectors of up to 256 values: kLanes lanes a head, eight values a lane, kHeads heads of a token one after the other, all loaded first.  A lane's
// values are consecutive ones where pairs of neighbours are turned (kPairs), else a lane of the rotated part has four of one half and the four
// that they are turned against, so no value is exchanged.  Weights and angles of a lane's values stay in registers over the heads.
// Small blocks, and 32 warps an SM (28 with fp32 inputs, whose loads take the registers): with blocks of 256 threads and 24 warps 4091 tokens of
// 64 + 8 heads take 36.3 instead of 31.3 us (fp32 45.5 instead of 41.7; 43.1 with 32 warps).
constexpr int kRotateThreads = 128;
template <typename In, bool kE4m3, int kLanes, int kHeads, bool kPairs, bool kNorm>
__global__ void __launch_bounds__(kRotateThreads, kHeads == 1 || sizeof(In) == 2 ? 8 : 7) norm_rotate_kernel(const __grid_constant__ RotateParams p) {
    grid_dependency_wait();
    const int lane = threadIdx.x % kLanes;
    const RotateUnit u = unit_of<kHeads>(p, (int64_t)blockIdx.x * (kRotateThreads / kLanes) + threadIdx.x / kLanes);
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
    constexpr bool kApart = kE4m3 || sizeof(In) != 2;   // the output's type is another one, so it is not the input
    Raw<In, kPairs, kApart> raw[kHeads];
#pragma unroll
    for (int k = 0; k < kHeads; ++k, x += x_head) raw[k].load(x, apart, k < count);
    const bool norm = kNorm && s.weight != nullptr, shifted = norm && s.bias != nullptr;
    float w[8], co[4], si[4];
    if (norm) {
        Raw<float, kPairs, true> t;
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
            const float rstd = centred_rstd<kLanes>(y, inside && norm, p.inv_dim, p.center, p.eps);   // (the whole warp, whichever side its heads are of)
            if (norm) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = scaled(y[i], rstd, w[i]);
                if (shifted) {
                    float b[8];
                    Raw<float, kPairs, true> t;
                    t.load(s.bias + c0, apart, inside);
                    t.get(b);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = __fadd_rn(y[i], b[i]);
                }
            }
        }
        if (turns)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int i0 = kPairs ? 2 * i : i, i1 = kPairs ? 2 * i + 1 : i + 4;
                const float a = y[i0], e = y[i1];
                y[i0] = turned0(a, e, co[i], si[i]);
                y[i1] = turned1(a, e, co[i], si[i]);
            }
        if constexpr (kE4m3) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(y[i]));
            const float scale = scale_of(max_over<kLanes>(amax));
            const uint2 codes = quotients8(y, scale);
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
    constexpr bool kApart = kE4m3 || sizeof(In) != 2;   // the output's type is another one, so it is not the input
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
            load8<kApart>(x + c, v[k]);
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
            mean = __fmul_rn(sum_over<32>(t), p.inv_dim);
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
        load8<true>(s.weight + c, w);
        if (s.bias != nullptr) load8<true>(s.bias + c, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = scaled(__fsub_rn(y[i], mean), rstd, w[i]);
        if (s.bias != nullptr)
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __fadd_rn(y[i], b[i]);
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
                v[k][2 * i] = turned0(a, b, co[i], si[i]);
                v[k][2 * i + 1] = turned1(a, b, co[i], si[i]);
            }
        } else {
            const bool upper = r >= half;
            float o[8], co[8], si[8];
            load8<kApart>(x + c + (upper ? -half : half), o);
            normed(o, c + (upper ? -half : half));
            load8<true>(table + r - (upper ? half : 0), co);
            load8<true>(table + half + r - (upper ? half : 0), si);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[k][i] = upper ? turned1(o[i], v[k][i], co[i], si[i]) : turned0(v[k][i], o[i], co[i], si[i]);
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
            if (c < p.head_dim) *reinterpret_cast<uint2*>(out + c) = quotients8(v[k], scale);
        }
        if (lane == 0) put_scale(s, u.token * (u.is_q ? p.q_heads : p.heads - p.q_heads) + u.head, scale);
    } else {
        if constexpr (!kApart) __syncwarp();   // in place: a lane's values may still be another's partners
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
    // Four heads a unit once there are threads enough for the device without (2048 an SM) and more than half of the units' places have a head.
    // us with four and with one, normed heads of 128 in halves: 300 tokens x 17 heads (82 thousand threads) 3.5 and 2.8, 1000 x 17 (272 thousand) 4.4
    // and 4.6, 4096 x 17 10.1 and 13.1, 4091 x 72 30.3 and 51.6; 40000 tokens of one head 14.0 and 8.0, of two 14.6 and 14.4, of three 15.9 and 21.2.
    auto go = [&](auto one, auto four, int lanes, int threads) {
        const int of_four = (p.q_heads + 3) / 4 + (p.heads - p.q_heads + 3) / 4;
        const bool many = four != nullptr && tokens * p.heads * lanes >= (int64_t)sms * 2048 && p.heads > 2 * of_four;
        const int each = many ? 4 : 1;
        p.q_chunks = (p.q_heads + each - 1) / each;
        p.chunks = p.q_chunks + (p.heads - p.q_heads + each - 1) / each;
        p.units = tokens * p.chunks;
        return launch_after(many ? four : one, (p.units * lanes + threads - 1) / threads, threads, p, stream);
    };
    using Kernel = void (*)(RotateParams);
    if (p.head_dim <= 256) {
        auto of = [&](auto pairs, auto normed) {
            constexpr bool kPairs = decltype(pairs)::value, kNorm = decltype(normed)::value;
            if (p.head_dim <= 64) return go(Kernel(norm_rotate_kernel<In, kE4m3, 8, 1, kPairs, kNorm>), Kernel(norm_rotate_kernel<In, kE4m3, 8, 4, kPairs, kNorm>), 8, kRotateThreads);
            if (p.head_dim <= 128) return go(Kernel(norm_rotate_kernel<In, kE4m3, 16, 1, kPairs, kNorm>), Kernel(norm_rotate_kernel<In, kE4m3, 16, 4, kPairs, kNorm>), 16, kRotateThreads);
            return go(Kernel(norm_rotate_kernel<In, kE4m3, 32, 1, kPairs, kNorm>), Kernel(norm_rotate_kernel<In, kE4m3, 32, 4, kPairs, kNorm>), 32, kRotateThreads);
        };
        const bool pairs = p.interleaved || p.rope_dim == 0;
        if (p.side[0].weight != nullptr || p.side[1].weight != nullptr) return pairs ? of(std::true_type(), std::true_type()) : of(std::false_type(), std::true_type());
        return pairs ? of(std::true_type(), std::false_type()) : of(std::false_type(), std::false_type());
    }
    if (p.head_dim <= 512) return go(Kernel(norm_rotate_long_kernel<In, kE4m3, 2>), Kernel(nullptr), 32, 256);
    if (p.head_dim <= 768) return go(Kernel(norm_rotate_long_kernel<In, kE4m3, 3>), Kernel(nullptr), 32, 256);
    return go(Kernel(norm_rotate_long_kernel<In, kE4m3, 4>), Kernel(nullptr), 32, 256);
}

// ------------------------------------------------------------------ append to the paged caches
struct AppendParams {
    dsa_v32_append_args a;
    int page_shift;      // log2(page_block_size), or -1
    int latent_warps;
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

// The tokens of a warp: lane k resolves token first + k, and holds its position and row (-1: not written).
struct Placed {
    int pos, row;
};
template <int kTokens> __device__ __forceinline__ Placed place(const AppendParams& p, int first, int lane) {
    Placed r{0, -1};
    if (lane < kTokens && first + lane < p.a.num_tokens) {
        r.pos = __ldg(p.a.positions + first + lane);
        r.row = (int)append_row(p, first + lane, r.pos);
    }
    return r;
}

// Rows of the attention's cache: a warp a token, 16 values a lane (eight lanes a group of 128) and two of the rope key.  All inputs of the warp's
// kTokens tokens are loaded before their places are known.
template <typename In, bool kFp8, int kTokens> __device__ __forceinline__ void append_latents(const AppendParams& p, int first, int lane) {
    const int n = p.a.num_tokens;
    Raw<In, true, true> raw[kTokens][2];
    float pe[kTokens][2];
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
        const int t = min(first + k, n - 1);
        const In* x = reinterpret_cast<const In*>(p.a.latent) + t * p.a.stride_latent + 16 * lane;
        raw[k][0].load(x, 4, true);
        raw[k][1].load(x + 8, 4, true);
        load2(reinterpret_cast<const In*>(p.a.rope) + t * p.a.stride_rope + 2 * lane, pe[k]);
    }
    const Placed at = place<kTokens>(p, first, lane);
    const bool norm = p.a.latent_weight != nullptr;
    uint64_t w[8];
    if (norm) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float f[4];
            load4(p.a.latent_weight + 16 * lane + 4 * i, f);
            w[2 * i] = pack2(f[0], f[1]);
            w[2 * i + 1] = pack2(f[2], f[3]);
        }
    }
    int row[kTokens];
    float co[kTokens][2], si[kTokens][2];      // neighbours: one angle; halves: two
    const bool pairs = p.a.interleaved;
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
        row[k] = __shfl_sync(0xffffffffu, at.row, k);
        const int pos = __shfl_sync(0xffffffffu, at.pos, k);
        if (row[k] < 0) continue;
        const float* table = p.a.cos_sin + (int64_t)pos * kDRope;
        if (pairs) {
            co[k][0] = __ldg(table + lane), si[k][0] = __ldg(table + 32 + lane);
        } else {
            load2(table + 2 * (lane & 15), co[k]);
            load2(table + 32 + 2 * (lane & 15), si[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < kTokens; ++k) {
        if (row[k] < 0) continue;
        uint32_t rope;
        if (pairs) {
            rope = pack_bf16x2(turned0(pe[k][0], pe[k][1], co[k][0], si[k][0]), turned1(pe[k][0], pe[k][1], co[k][0], si[k][0]));
        } else {
            const float o0 = __shfl_xor_sync(0xffffffffu, pe[k][0], 16), o1 = __shfl_xor_sync(0xffffffffu, pe[k][1], 16);
            rope = lane >= 16 ? pack_bf16x2(turned1(o0, pe[k][0], co[k][0], si[k][0]), turned1(o1, pe[k][1], co[k][1], si[k][1]))
                              : pack_bf16x2(turned0(pe[k][0], o0, co[k][0], si[k][0]), turned0(pe[k][1], o1, co[k][1], si[k][1]));
        }
        uint64_t v[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            float f[8];
            raw[k][j].get(f);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * j + i] = pack2(f[2 * i], f[2 * i + 1]);
        }
        float factor = kFp8 ? -1.0f : 1.0f;        // (quotients8 takes them negated)
        if (norm) {
            uint64_t t0 = 0, t1 = 0;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                t0 = fma2(v[i], v[i], t0);
                t1 = fma2(v[i + 1], v[i + 1], t1);
            }
            float a, b;
            unpack2(add2(t0, t1), a, b);
            factor *= rsqrtf(fmaf(sum_over<32>(a + b), 1.0f / kDV, p.a.eps));
        }
        if (kFp8 || norm) {
            const uint64_t f2 = pack2(factor, factor);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = mul2(v[i], f2);
        }
        if (norm) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = mul2(v[i], w[i]);
        }
        if constexpr (kFp8) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = amax2(v[i], amax);
            const float scale = scale_of(max_over<8>(amax));
            const uint64_t lo[4] = {v[0], v[1], v[2], v[3]}, hi[4] = {v[4], v[5], v[6], v[7]};
            const uint2 a = quotients8(lo, scale), b = quotients8(hi, scale);
            uint8_t* out = reinterpret_cast<uint8_t*>(p.a.kv) + (int64_t)row[k] * kFp8RowBytes;
            reinterpret_cast<uint4*>(out)[lane] = make_uint4(a.x, a.y, b.x, b.y);
            if ((lane & 7) == 0) reinterpret_cast<float*>(out + kDV)[lane >> 3] = scale;
            reinterpret_cast<uint32_t*>(out + kDV + 16)[lane] = rope;
        } else {
            uint8_t* out = reinterpret_cast<uint8_t*>(p.a.kv) + (int64_t)row[k] * (2 * kDQK);
#pragma unroll
            for (int j = 0; j < 2; ++j)
                reinterpret_cast<uint4*>(out)[2 * lane + j] =
                    make_uint4(pack_bf16x2_from2(v[4 * j]), pack_bf16x2_from2(v[4 * j + 1]), pack_bf16x2_from2(v[4 * j + 2]), pack_bf16x2_from2(v[4 * j + 3]));
            reinterpret_cast<uint32_t*>(out + 2 * kDV)[lane] = rope;
        }
    }
}

// Rows of the index cache: sixteen lanes a token, four values from c0 and four from c1 a lane (as in norm_rotate_kernel), kTokens tokens a warp.
template <typename In, bool kFp8, int kTokens> __device__ __forceinline__ void append_index_keys(const AppendParams& p, int first, int lane) {
    constexpr int kEach = kTokens / 2;
    const int n = p.a.num_tokens, l = lane & 15, mine = lane >> 4;
    const bool pairs = p.a.index_interleaved, turns = l < 8;
    const int c0 = pairs || !turns ? 8 * l : 4 * l, apart = pairs || !turns ? 4 : 32;
    Raw<In, false, true> raw[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k)
        raw[k].load(reinterpret_cast<const In*>(p.a.index_key) + min(first + 2 * k + mine, n - 1) * p.a.stride_index_key + c0, apart, true);
    const Placed at = place<kTokens>(p, first, lane);
    const bool norm = p.a.index_weight != nullptr, shifted = p.a.index_bias != nullptr;
    float w[8], b[8];
    if (norm) {
        Raw<float, false, true> t;
        t.load(p.a.index_weight + c0, apart, true);
        t.get(w);
        if (shifted) {
            t.load(p.a.index_bias + c0, apart, true);
            t.get(b);
        }
    }
    int row[kEach];
    float co[kEach][4], si[kEach][4];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        row[k] = __shfl_sync(0xffffffffu, at.row, 2 * k + mine);
        const int pos = __shfl_sync(0xffffffffu, at.pos, 2 * k + mine);
        if (row[k] < 0 || !turns) continue;
        const float* table = p.a.cos_sin + (int64_t)pos * kDRope + 4 * l;
        load4(table, co[k]);
        load4(table + 32, si[k]);
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        float y[8];
        raw[k].get(y);
        if (norm) {
            const float rstd = centred_rstd<16>(y, true, 1.0f / kDIndex, p.a.index_center, p.a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = scaled(y[i], rstd, w[i]);
            if (shifted)
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = __fadd_rn(y[i], b[i]);
        }
        if (turns && row[k] >= 0) {
            auto turn = [&](float& a, float& e, int i) {
                const float x = a;
                a = turned0(x, e, co[k][i], si[k][i]);
                e = turned1(x, e, co[k][i], si[k][i]);
            };
            if (pairs) {
#pragma unroll
                for (int i = 0; i < 4; ++i) turn(y[2 * i], y[2 * i + 1], i);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) turn(y[i], y[4 + i], i);
            }
        }
        if constexpr (kFp8) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(y[i]));
            const float scale = scale_of(max_over<16>(amax));
            const uint2 codes = quotients8(y, scale);
            if (row[k] < 0) continue;
            const int64_t page = row[k] >> p.page_shift;
            const int in_page = row[k] & (p.a.page_block_size - 1);          // (a power of two: the index cache's pages are)
            uint8_t* base = reinterpret_cast<uint8_t*>(p.a.index_cache) + ((page * (kDIndex + 4)) << p.page_shift);
            uint8_t* out = base + in_page * kDIndex + c0;
            *reinterpret_cast<uint32_t*>(out) = codes.x;
            *reinterpret_cast<uint32_t*>(out + apart) = codes.y;
            if (l == 0) reinterpret_cast<float*>(base + ((int64_t)kDIndex << p.page_shift))[in_page] = scale;
        } else {
            if (row[k] < 0) continue;
            __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.a.index_cache) + (int64_t)row[k] * kDIndex + c0;
            *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
            *reinterpret_cast<uint2*>(out + apart) = make_uint2(pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
        }
    }
}

// (Blocks of 256 threads: 14.8 instead of 12.5 us for 16384 tokens into the fp8 caches, inputs in L2: the last ones leave SMs half empty.)
constexpr int kAppendThreads = 128;
// Warps 0 .. latent_warps - 1 take kTokens tokens' rows of the attention's cache each, the others twice as many (at least two) of the index cache.
template <typename In, bool kFp8, int kTokens>
__global__ void __launch_bounds__(kAppendThreads, 8) append_kernel(const __grid_constant__ AppendParams p) {
    grid_dependency_wait();
    constexpr int kKeys = 2 * kTokens;
    const int lane = threadIdx.x & 31, n = p.a.num_tokens;
    const int64_t warp = (int64_t)blockIdx.x * (kAppendThreads / 32) + (threadIdx.x >> 5);
    if (warp < p.latent_warps) {
        append_latents<In, kFp8, kTokens>(p, (int)warp * kTokens, lane);
    } else if (p.a.index_cache != nullptr && (warp - p.latent_warps) * kKeys < n) {
        append_index_keys<In, kFp8, kKeys>(p, (int)(warp - p.latent_warps) * kKeys, lane);
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
    AppendParams p{a, -1, 0};
    for (int sh = 0; sh < 31; ++sh)
        if (a.page_block_size == (1 << sh)) p.page_shift = sh;
    if (a.num_tokens == 0) return cudaSuccess;
    int sms = 0;
    cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    const bool fp8 = a.kv_dtype == DSA_V32_KV_FP8, wide = a.in_dtype == DSA_V32_DTYPE_FP32;
    auto go = [&](auto kernel, int tokens) {
        p.latent_warps = a.kv != nullptr ? (a.num_tokens + tokens - 1) / tokens : 0;
        const int64_t warps = p.latent_warps + (a.index_cache != nullptr ? ((int64_t)a.num_tokens + 2 * tokens - 1) / (2 * tokens) : 0);
        return launch_after(kernel, (warps + kAppendThreads / 32 - 1) / (kAppendThreads / 32), kAppendThreads, p, stream);
    };
    // Two tokens a warp (their loads in flight together, the weights read once) where warps of one token each are more than the device holds with
    // their CTAs' ends: inputs in L2, 4096 tokens 4.8 instead of 5.6 us, 1024 tokens 3.4 instead of 2.9.  (Four: 14.2 instead of 12.5 us for 16384 tokens.)
    if (a.num_tokens < 16 * sms) {
        if (wide) return fp8 ? go(append_kernel<float, true, 1>, 1) : go(append_kernel<float, false, 1>, 1);
        return fp8 ? go(append_kernel<__nv_bfloat16, true, 1>, 1) : go(append_kernel<__nv_bfloat16, false, 1>, 1);
    }
    if (wide) return fp8 ? go(append_kernel<float, true, 2>, 2) : go(append_kernel<float, false, 2>, 2);
    return fp8 ? go(append_kernel<__nv_bfloat16, true, 2>, 2) : go(append_kernel<__nv_bfloat16, false, 2>, 2);
}

}  // namespace dsa
