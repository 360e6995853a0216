// Index scores of blocks of positions (sm_100a): s[q, p] = ks[p] * sum_h w[q, h] max(0, q_h . k_p), and the largest of a block.
//
// The products run on the tensor cores with the positions on the wide side of the tile: D[128 positions][heads of up to 8 query rows] =
// K Q^T, both operands K-major in shared memory as they lie in global memory (the cache's bytes are never converted).  A TMEM lane is a
// position, so the sum over heads stays inside a thread, a query row's scores of 32 positions are one 128-byte store, a block's largest
// one is a few exchanges, and nothing of a NaN or infinite key reaches another position.
//
// Roles of a CTA (one an SM): warps 0-15 take the scores out of TMEM (four warpgroups, a query row at a time each), warp 16 brings tiles
// of 128 keys page by page (TMA; an fp8 cache's scales by bulk copies), warp 17 the query rows, their weights and lengths, warp 18
// issues the MMAs.  A work item is a group of query rows of one sequence and a chunk of tiles; the CTAs take items in turn, so the
// ends of short rows (whose columns are only filled) are spread over them.
#include <cuda_bf16.h>
#include <mutex>
#include "front.h"
#include "ptx.cuh"

namespace dsa {
namespace scores {

constexpr int kTile = 128;            // positions of a tile: M
constexpr int kMmaCols = 256;         // most N of an MMA
constexpr int kTmemCols = 512;
constexpr int kEpiWarps = 16;
constexpr int kWarps = kEpiWarps + 3;
constexpr int kMaxRows = 32;          // query rows of a group
constexpr int kMaxStages = 12;
constexpr int kMaxSlots = 8;
constexpr int kSmemBytes = 227 * 1024;
constexpr int kScaleBytes = kTile * 4;

struct Control {
    uint64_t k_full[kMaxStages], k_empty[kMaxStages];
    uint64_t acc_full[kMaxSlots], acc_empty[kMaxSlots];
    uint64_t q_full[2], q_empty[2], w_full[2], w_empty[2];
    uint64_t exchange[4];             // per warpgroup, the warps' exchange for blocks of 64 and 128
    uint32_t tmem_base;
    int abort_flag;
    uint32_t page_ok[kMaxStages];     // per stage, a bit per page of the tile
    int valid[2][kMaxRows];
    float best[4][2][4];              // what is exchanged: per warpgroup, twice, the warps' own largest
};
constexpr int kControlBytes = 1024;
static_assert(sizeof(Control) <= kControlBytes, "control block");

struct Params {
    const float* weights;
    const int32_t* valid_len;
    const int32_t* block_table;
    const uint8_t* cache;
    float* out;
    int32_t* status;
    int64_t stride_w_row, stride_o_row, num_pages, seq_stride_pages;
    int H, s_q, kv_len, limit, block, cols, block_table_stride, page_shift;
    int per, groups_per_seq, groups;      // query rows of a group, groups of a sequence and of all
    int tiles, chunk, items;
    int rows_per_acc, acc_cols, slots;    // query rows of an accumulator, its TMEM columns, accumulators in TMEM
    int stages, q_bufs;
    uint32_t off_k, off_s, off_w, q_bytes;   // shared memory: Q buffers | keys | their scales | weights | control
};

// keys of a stage: bf16 two blocks of 64 columns, fp8 one of 128
template <bool kFp8> constexpr int kKeyBytes = kFp8 ? kTile * 128 : kTile * 256;

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// four K = 32 steps of 128 e4m3 columns
__device__ __forceinline__ void umma_f8_ss_x4_el(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t elected) {
    asm volatile(
        "{\n\t.reg .pred q, pt, pf;\n\t.reg .b32 la, lb;\n\t.reg .b64 ad, bd;\n\t"
        "setp.ne.b32 q, %6, 0;\n\t"
        "setp.ne.b32 pf, %6, %6;\n\t"
        "setp.eq.b32 pt, %6, %6;\n\t"
        "mov.b64 ad, {%1, %2};\n\tmov.b64 bd, {%3, %4};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], ad, bd, %5, pf;\n\t"
        "add.u32 la, %1, 2;\n\tadd.u32 lb, %3, 2;\n\tmov.b64 ad, {la, %2};\n\tmov.b64 bd, {lb, %4};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], ad, bd, %5, pt;\n\t"
        "add.u32 la, %1, 4;\n\tadd.u32 lb, %3, 4;\n\tmov.b64 ad, {la, %2};\n\tmov.b64 bd, {lb, %4};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], ad, bd, %5, pt;\n\t"
        "add.u32 la, %1, 6;\n\tadd.u32 lb, %3, 6;\n\tmov.b64 ad, {la, %2};\n\tmov.b64 bd, {lb, %4};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], ad, bd, %5, pt;\n\t}"
        :
        : "r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(elected)
        : "memory");
}

// A work item.  Every role derives it by itself.
struct Item {
    int seq, q0, rows, tile0, tiles;   // tiles: those that hold a position of some row
};
__device__ __forceinline__ int row_limit(const Params& p, int q) { return p.valid_len != nullptr ? max(0, min(p.limit, __ldg(p.valid_len + q))) : p.limit; }
__device__ __forceinline__ Item item_of(const Params& p, int u, int lane) {
    Item it;
    const int c = u / p.groups, g = u - c * p.groups;
    it.seq = g / p.groups_per_seq;
    const int r0 = (g - it.seq * p.groups_per_seq) * p.per;
    it.q0 = it.seq * p.s_q + r0;
    it.rows = min(p.per, p.s_q - r0);
    it.tile0 = c * p.chunk;
    const int n = __reduce_max_sync(0xffffffffu, lane < it.rows ? row_limit(p, it.q0 + lane) : 0);
    it.tiles = max(0, min((n + kTile - 1) / kTile - it.tile0, min(p.chunk, p.tiles - it.tile0)));
    return it;
}

struct Ring {
    int s = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next(int n) {
        if (++s == n) {
            s = 0;
            ph ^= 1u;
        }
    }
};

// kCols: TMEM columns of a query row, its heads padded to 16, 32 or 64; kAll: there are exactly so many.
template <bool kFp8, int kCols, bool kAll>
__global__ void __launch_bounds__(32 * kWarps, 1) index_scores_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tq, const __grid_constant__ Params p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Control* ctl = reinterpret_cast<Control*>(smem + kSmemBytes - kControlBytes);
    float* const w_smem = reinterpret_cast<float*>(smem + p.off_w);
    uint8_t* const k_smem = smem + p.off_k;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    volatile int* abort_flag = &ctl->abort_flag;

    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(smem_u32(&ctl->k_full[i]), 1);
            mbar_init(smem_u32(&ctl->k_empty[i]), 1 + kEpiWarps);
        }
        for (int i = 0; i < p.slots; ++i) {
            mbar_init(smem_u32(&ctl->acc_full[i]), 1);
            mbar_init(smem_u32(&ctl->acc_empty[i]), kEpiWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&ctl->q_full[i]), 1);
            mbar_init(smem_u32(&ctl->q_empty[i]), 1);
            mbar_init(smem_u32(&ctl->w_full[i]), 32);
            mbar_init(smem_u32(&ctl->w_empty[i]), kEpiWarps);
        }
        for (int i = 0; i < 4; ++i) mbar_init(smem_u32(&ctl->exchange[i]), 4);
        ctl->abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 16 && lane == 0) {
        prefetch_tensormap(&tk);
        prefetch_tensormap(&tq);
    }
    if (warp == 18) {
        tmem_alloc(smem_u32(&ctl->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;
    grid_dependency_wait();

    if (warp < kEpiWarps) {
        // ------------------------------------------------ scores out
        const int wg = warp >> 2, sub = warp & 3;
        Ring k, slot, wb;
        uint32_t exchanges = 0;
        bool ok = true;
        int u = blockIdx.x;
        for (; u < p.items && ok; u += gridDim.x) {
            const Item it = item_of(p, u, lane);
            if (it.tiles > 0) {
                ok = warp_wait_short(smem_u32(&ctl->w_full[wb.s]), wb.ph, abort_flag);
                const float* w = w_smem + wb.s * p.per * kCols;
                int job = 0;   // (tile, query row) pairs so far: a warpgroup takes every fourth
                for (int i = 0; i < it.tiles && ok; ++i) {
                    const int pos = (it.tile0 + i) * kTile + 32 * sub + lane;
                    float ks = 1.0f;
                    bool here = false;
                    for (int r0 = 0; r0 < it.rows; r0 += p.rows_per_acc) {
                        if (!warp_wait_short(smem_u32(&ctl->acc_full[slot.s]), slot.ph, abort_flag)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        if (r0 == 0) {
                            if (!warp_wait_short(smem_u32(&ctl->k_full[k.s]), k.ph, abort_flag)) {
                                ok = false;
                                break;
                            }
                            const uint32_t pages = ctl->page_ok[k.s];
                            here = (pages >> ((32 * sub + lane) >> min(p.page_shift, 7))) & 1u;
                            if (kFp8) ks = reinterpret_cast<const float*>(smem + p.off_s + k.s * kScaleBytes)[32 * sub + lane];
                            __syncwarp();
                            if (lane == 0) mbar_arrive(smem_u32(&ctl->k_empty[k.s]));
                            k.next(p.stages);
                        }
                        const int r1 = min(it.rows, r0 + p.rows_per_acc);
                        int mine = r0 + ((wg - job) & 3);
                        const uint32_t acc = tmem + slot.s * p.acc_cols + (static_cast<uint32_t>(32 * sub) << 16);
                        const uint32_t free_bar = smem_u32(&ctl->acc_empty[slot.s]);
                        job += r1 - r0;
                        if (mine >= r1) {   // nothing of this accumulator is this warpgroup's
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(free_bar);
                        }
                        for (; mine < r1; mine += 4) {
                            uint32_t d[kCols];
                            const uint32_t at = acc + (mine - r0) * kCols;
                            if constexpr (kCols == 16) {
                                tmem_ld16(at, d);
                            } else {
#pragma unroll
                                for (int c = 0; c < kCols; c += 32) tmem_ld32(at + c, reinterpret_cast<uint32_t(&)[32]>(d[c]));
                            }
                            tmem_wait_ld();
                            if (mine + 4 >= r1) {
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(free_bar);
                            }
                            const float* wr = w + mine * kCols;
                            uint64_t s0 = 0, s1 = 0;
#pragma unroll
                            for (int h = 0; h < kCols; h += 4) {
                                const ulonglong2 w2 = *reinterpret_cast<const ulonglong2*>(wr + h);
                                float v[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    v[j] = max_nan(__uint_as_float(d[h + j]), 0.0f);
                                    if (!kAll) v[j] = h + j < p.H ? v[j] : 0.0f;   // (zeros times an infinite key)
                                }
                                s0 = fma2(pack2(v[0], v[1]), w2.x, s0);
                                s1 = fma2(pack2(v[2], v[3]), w2.y, s1);
                            }
                            float a, b, e, f;
                            unpack2(s0, a, b);
                            unpack2(s1, e, f);
                            float s = ((a + b) + (e + f)) * ks;
                            s = here && pos < ctl->valid[wb.s][mine] ? s : -INFINITY;
                            float* out = p.out + (int64_t)(it.q0 + mine) * p.stride_o_row;
                            if (p.block == 1) {
                                if (pos < p.kv_len) out[pos] = s;
                            } else {
                                for (int off = 1; off < min(p.block, 32); off <<= 1) s = max_nan(s, __shfl_xor_sync(0xffffffffu, s, off));
                                if (p.block >= 64) {
                                    const int buf = exchanges & 1;   // (a third job's value is written after the exchange of the second)
                                    const uint32_t bar = smem_u32(&ctl->exchange[wg]);
                                    __syncwarp();
                                    if (lane == 0) {
                                        ctl->best[wg][buf][sub] = s;
                                        mbar_arrive(bar);
                                    }
                                    ok = ok && warp_wait_short(bar, buf, abort_flag);
                                    ++exchanges;
                                    s = max_nan(s, ctl->best[wg][buf][sub ^ 1]);
                                    if (p.block == 128) s = max_nan(s, max_nan(ctl->best[wg][buf][sub ^ 2], ctl->best[wg][buf][sub ^ 3]));
                                }
                                const int col = pos / p.block;
                                if ((pos & (p.block - 1)) == 0 && col < p.cols) out[col] = s;
                            }
                        }
                        slot.next(p.slots);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&ctl->w_empty[wb.s]));
                wb.next(p.q_bufs);
            }
            if (!ok) break;
        }
        // The columns behind the last position that a row of an item sees, once nothing waits for this warp any more.  After a wait that
        // gave up: all of the items that were not finished.
        for (int v = blockIdx.x; v < p.items; v += gridDim.x) {
            const Item it = item_of(p, v, lane);
            const bool lost = !ok && v >= u;
            const int from = it.tile0 + (lost ? 0 : it.tiles), to = min(it.tile0 + p.chunk, p.tiles);
            const int c0 = (int)((int64_t)from * kTile / p.block), c1 = (int)min((int64_t)p.cols, (int64_t)to * kTile / p.block);
            for (int r = 0; r < it.rows; ++r)
                for (int c = c0 + (lost ? lane : tid); c < c1; c += lost ? 32 : 32 * kEpiWarps)
                    p.out[(int64_t)(it.q0 + r) * p.stride_o_row + c] = lost ? __int_as_float(0x7FFFFFFF) : -INFINITY;
        }
    } else if (warp == 16) {
        // ------------------------------------------------ keys in
        Ring k;
        const int page_rows = 1 << min(p.page_shift, 7), pages = kTile / page_rows;   // of a tile
        bool ok = true;
        for (int u = blockIdx.x; u < p.items && ok; u += gridDim.x) {
            const Item it = item_of(p, u, lane);
            for (int i = 0; i < it.tiles; ++i, k.next(p.stages)) {
                const int pos = (it.tile0 + i) * kTile;
                int64_t page = -1;
                if (lane < pages) {
                    const int blk = (pos >> p.page_shift) + lane;
                    if (p.block_table == nullptr) page = (int64_t)it.seq * p.seq_stride_pages + blk;
                    else if (blk < p.block_table_stride) page = __ldg(p.block_table + (int64_t)it.seq * p.block_table_stride + blk);
                    if (page < 0 || page >= p.num_pages) page = -1;
                }
                const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
                if (!(ok = warp_wait(smem_u32(&ctl->k_empty[k.s]), k.ph ^ 1u, abort_flag))) break;
                const uint32_t bar = smem_u32(&ctl->k_full[k.s]), dst = smem_u32(k_smem + k.s * kKeyBytes<kFp8>);
                if (lane == 0) {
                    ctl->page_ok[k.s] = there;
                    mbar_arrive_expect_tx(bar, kKeyBytes<kFp8> + (kFp8 ? __popc(there) * page_rows * 4 : 0));
                }
                __syncwarp();
                if (lane < pages) {
                    const int y = pos & ((1 << p.page_shift) - 1) & ~(page_rows - 1);   // first row inside a page of more than a tile
                    const int z = page >= 0 ? (int)page : (int)p.num_pages;             // outside the cache: zeros
                    const uint32_t to = dst + lane * page_rows * 128;
                    tma_load_3d(to, &tk, bar, 0, y, z);
                    if (!kFp8) tma_load_3d(to + kTile * 128, &tk, bar, 64, y, z);
                    if (kFp8 && page >= 0)
                        bulk_load(smem_u32(smem + p.off_s + k.s * kScaleBytes) + lane * page_rows * 4, p.cache + ((page << p.page_shift) * (kDIndex + 4) + ((int64_t)kDIndex << p.page_shift) + 4 * y), page_rows * 4, bar);
                }
            }
        }
    } else if (warp == 17) {
        // ------------------------------------------------ query rows, weights, lengths in
        Ring b;
        bool ok = true;
        for (int u = blockIdx.x; u < p.items && ok; u += gridDim.x) {
            const Item it = item_of(p, u, lane);
            if (it.tiles == 0) continue;
            if (!(ok = warp_wait(smem_u32(&ctl->q_empty[b.s]), b.ph ^ 1u, abort_flag))) break;
            const uint32_t bar = smem_u32(&ctl->q_full[b.s]), dst = smem_u32(smem) + b.s * p.q_bytes;
            if (lane == 0) mbar_arrive_expect_tx(bar, it.rows * kCols * (kFp8 ? 128 : 256));
            __syncwarp();
            if (lane < it.rows) {
                tma_load_3d(dst + lane * kCols * 128, &tq, bar, 0, 0, it.q0 + lane);
                if (!kFp8) tma_load_3d(dst + p.q_bytes / 2 + lane * kCols * 128, &tq, bar, 64, 0, it.q0 + lane);
            }
            if (!(ok = warp_wait(smem_u32(&ctl->w_empty[b.s]), b.ph ^ 1u, abort_flag))) break;
            float* w = w_smem + b.s * p.per * kCols;
            for (int i = lane; i < it.rows * kCols; i += 32) {
                const int r = i / kCols, h = i % kCols;
                w[i] = h < p.H ? __ldg(p.weights + (int64_t)(it.q0 + r) * p.stride_w_row + h) : 0.0f;
            }
            if (lane < it.rows) ctl->valid[b.s][lane] = row_limit(p, it.q0 + lane);
            mbar_arrive(smem_u32(&ctl->w_full[b.s]));
            b.next(p.q_bufs);
        }
    } else {
        // ------------------------------------------------ MMAs
        Ring k, slot, b;
        bool ok = true;
        const uint32_t el = elect_one() ? 1u : 0u;
        const uint64_t k_desc = make_smem_desc_sw128(smem_u32(k_smem), 0, 1024), q_desc = make_smem_desc_sw128(smem_u32(smem), 0, 1024);
        const uint32_t k_lo = (uint32_t)k_desc, q_lo = (uint32_t)q_desc, hi = (uint32_t)(k_desc >> 32);
        for (int u = blockIdx.x; u < p.items && ok; u += gridDim.x) {
            const Item it = item_of(p, u, lane);
            if (it.tiles == 0) continue;
            if (!(ok = warp_wait(smem_u32(&ctl->q_full[b.s]), b.ph, abort_flag))) break;
            for (int i = 0; i < it.tiles && ok; ++i, k.next(p.stages)) {
                if (!(ok = warp_wait(smem_u32(&ctl->k_full[k.s]), k.ph, abort_flag))) break;
                for (int r0 = 0; r0 < it.rows; r0 += p.rows_per_acc, slot.next(p.slots)) {
                    if (!(ok = warp_wait(smem_u32(&ctl->acc_empty[slot.s]), slot.ph ^ 1u, abort_flag))) break;
                    tc_fence_after();
                    const int n = min(p.rows_per_acc, it.rows - r0) * kCols;
                    const uint32_t a = k_lo + ((k.s * kKeyBytes<kFp8>) >> 4), q = q_lo + ((b.s * p.q_bytes + r0 * kCols * 128) >> 4), acc = tmem + slot.s * p.acc_cols;
                    if constexpr (kFp8) {
                        umma_f8_ss_x4_el(acc, a, hi, q, hi, make_idesc_e4m3(kTile, n), el);
                    } else {
                        const uint32_t idesc = make_idesc_bf16(kTile, n, false);
                        umma_ss_x4_el(acc, a, hi, q, hi, idesc, 0u, el);
                        umma_ss_x4_el(acc, a + ((kTile * 128) >> 4), hi, q + ((p.q_bytes / 2) >> 4), hi, idesc, 1u, el);
                    }
                    tc_commit_el(smem_u32(&ctl->acc_full[slot.s]), el);
                }
                if (ok) tc_commit_el(smem_u32(&ctl->k_empty[k.s]), el);
            }
            if (!ok) break;
            tc_commit_el(smem_u32(&ctl->q_empty[b.s]), el);
            b.next(p.q_bufs);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (ctl->abort_flag) {
        if (tid == 0 && p.status != nullptr) atomicExch(p.status, DSA_V32_ERR_DEVICE_WAIT);
        settle_in_flight();
        __syncthreads();
    }
    if (warp == 18) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <bool kFp8, int kCols, bool kAll>
cudaError_t launch(const CUtensorMap& tk, const CUtensorMap& tq, const Params& p, int grid, cudaStream_t stream) {
    static std::mutex mu;
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> guard(mu);
        if (dev < 0 || dev >= 64 || !done[dev]) {
            e = cudaFuncSetAttribute(index_scores_kernel<kFp8, kCols, kAll>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < 64) done[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3(32 * kWarps, 1, 1);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = stream;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, index_scores_kernel<kFp8, kCols, kAll>, tk, tq, p);
}

}  // namespace scores

cudaError_t launch_index_scores(const dsa_v32_index_scores_args& a, const CUtensorMap& tk, const CUtensorMap& tq, cudaStream_t stream) {
    using namespace scores;
    if (a.total_q == 0) return cudaSuccess;
    int sms = 0;
    cudaError_t e = sm_count(&sms);
    if (e != cudaSuccess) return e;
    const bool fp8 = a.cache_dtype == DSA_V32_KV_FP8;
    const int cols = index_score_cols(a.H);
    Params p = {};
    p.weights = a.weights;
    p.valid_len = a.valid_len;
    p.block_table = a.block_table;
    p.cache = reinterpret_cast<const uint8_t*>(a.index_cache);
    p.out = a.out;
    p.status = a.status;
    p.stride_w_row = a.stride_w_row;
    p.stride_o_row = a.stride_o_row;
    while ((1 << p.page_shift) < a.page_block_size) ++p.page_shift;
    p.num_pages = a.num_index_rows >> p.page_shift;
    p.seq_stride_pages = a.kv_batch_stride_rows >> p.page_shift;
    p.H = a.H;
    p.s_q = a.s_q;
    p.kv_len = a.kv_len;
    p.limit = a.kv_len;
    const int64_t reach = a.block_table ? (int64_t)a.block_table_stride << p.page_shift : a.kv_batch_stride_rows;
    if (reach > 0 && reach < p.limit) p.limit = (int)reach;
    p.block = a.block;
    p.cols = (a.kv_len + a.block - 1) / a.block;
    p.block_table_stride = a.block_table_stride;
    // query rows of a group: as many as TMEM has columns for, in groups of equal size
    const int most = kTmemCols / cols;
    p.groups_per_seq = (a.s_q + most - 1) / most;
    p.per = (a.s_q + p.groups_per_seq - 1) / p.groups_per_seq;
    p.groups_per_seq = (a.s_q + p.per - 1) / p.per;
    const int64_t groups = (int64_t)p.groups_per_seq * (a.total_q / a.s_q);
    const int accs = (p.per * cols + kMmaCols - 1) / kMmaCols;
    p.rows_per_acc = (p.per + accs - 1) / accs;
    p.acc_cols = (p.rows_per_acc * cols + 31) & ~31;
    p.slots = kTmemCols / p.acc_cols < kMaxSlots ? kTmemCols / p.acc_cols : kMaxSlots;
    // shared memory: two buffers of query rows where that leaves four stages of keys
    const int stage = fp8 ? kKeyBytes<true> + kScaleBytes : kKeyBytes<false>;
    p.q_bytes = p.per * cols * (fp8 ? 128 : 256);
    auto stages = [&](int bufs) { return (kSmemBytes - kControlBytes - bufs * (int)(p.q_bytes + p.per * cols * 4)) / stage; };
    p.q_bufs = stages(2) >= 4 ? 2 : 1;
    p.stages = stages(p.q_bufs) < kMaxStages ? stages(p.q_bufs) : kMaxStages;
    p.off_k = p.q_bufs * p.q_bytes;
    p.off_s = p.off_k + p.stages * (fp8 ? kKeyBytes<true> : kKeyBytes<false>);
    p.off_w = p.off_k + p.stages * stage;
    // tiles of an item: the least for the busiest CTA, an item counted as two tiles more
    p.tiles = (a.kv_len + kTile - 1) / kTile;
    int64_t best = 0, items = 0;
    for (int c = 1; c <= p.tiles; c = c < 8 ? c + 1 : c + c / 4) {
        const int64_t n = groups * ((p.tiles + c - 1) / c), cost = (n + sms - 1) / sms * (c + 2);
        if (n > 0x7FFFFFFF - 4096) continue;
        if (items == 0 || cost < best) {
            best = cost;
            items = n;
            p.chunk = c;
        }
    }
    if (items == 0) return cudaErrorInvalidConfiguration;
    p.groups = (int)groups;
    p.items = (int)items;
    const int grid = (int)(items < sms ? items : sms);
    const bool all = a.H == cols;
    auto go = [&](auto kernel) { return kernel(tk, tq, p, grid, stream); };
    if (fp8) {
        if (cols == 16) return go(all ? launch<true, 16, true> : launch<true, 16, false>);
        if (cols == 32) return go(all ? launch<true, 32, true> : launch<true, 32, false>);
        return go(all ? launch<true, 64, true> : launch<true, 64, false>);
    }
    if (cols == 16) return go(all ? launch<false, 16, true> : launch<false, 16, false>);
    if (cols == 32) return go(all ? launch<false, 32, true> : launch<false, 32, false>);
    return go(all ? launch<false, 64, true> : launch<false, 64, false>);
}

}  // namespace dsa
