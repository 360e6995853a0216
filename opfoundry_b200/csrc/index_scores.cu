// Index scores of blocks of positions (sm_100a): s[q, p] = ks[p] * sum_h w[q, h] max(0, q_h . k_p), and the largest of a block.
//
// The products run on the tensor cores with the positions on the wide side of the tile: D[128 positions][heads of up to 8 query rows] =
// K Q^T, both operands K-major in shared memory as they lie in global memory (the cache's bytes are never converted).  A TMEM lane is a
// position, so the sum over heads stays inside a quad of threads, a query row's scores of 32 positions are one 128-byte store, a block's
// largest one is a few exchanges, and nothing of a NaN or infinite key reaches another position.
//
// Roles of a CTA (one an SM): warps 0-15 take the scores out of TMEM (four warpgroups, a query row at a time each), warp 16 brings tiles
// of 128 keys page by page (TMA; an fp8 cache's scales by bulk copies), warp 17 the query rows, their weights and lengths, warp 18
// issues the MMAs.  A work item is tiles of a group of query rows of one sequence.  The tiles that the rows see are dealt out evenly over the CTAs
// (up to kDealt groups; more take chunks in turn), and columns that no row sees are filled by warps that have nothing else to do.
//
// Bounds (64 heads; times in a graph, inputs past L2): decode HBM and about 6 us that are fixed (fp8: 64 x 2 rows of 16384 to 32768 positions, 208 MB,
// 48 us; 56 as a call among others; bf16: 73).  Chunks: the drain of the accumulators.  4096 rows over 16384 positions take 515 us in bursts of 40 ms
// (1.965 GHz) and 591 back to back for seconds, where the power cap holds 1.717 GHz: 1.01 million cycles either way, of which the fp8 MMAs use two
// fifths and the sums over heads two thirds of the issue slots, so neither is full; a warpgroup loads, waits for and sums its rows one after the
// other.  In bf16 the MMAs are the larger part: 656 and 747 us (at 1.425 GHz).
#include <cuda_bf16.h>
#include <cstddef>
#include <mutex>
#include "front.h"
#include "ptx.cuh"

namespace dsa {
namespace scores {

constexpr int kTile = 128;            // positions of a tile: M
constexpr int kMmaCols = 256;         // most N of an MMA
constexpr int kTmemCols = 512;
constexpr int kEpiWarps = 16;          // four warpgroups
constexpr int kWarps = kEpiWarps + 3;
constexpr int kMaxRows = 32;          // query rows of a group
constexpr int kMaxStages = 12;
constexpr int kMaxSlots = 8;
constexpr int kSmemBytes = 227 * 1024;
constexpr int kScaleBytes = kTile * 4;
// Most groups whose tiles are dealt out evenly.  us dealt and in turn, 64 heads, fp8, ragged lengths from a half of the longest on: 64 x 2 rows to
// 32768 positions 48 and 56, 256 sequences to 8192 44 and 50, 1000 to 4096 84 and 93, 4096 rows over 16384 516 and 545.  It costs every CTA a pass
// over the lengths: one sequence 7.1 and 5.6 (but the lengths are not known here, and one far shorter than kv_len would keep a few CTAs busy only),
// 1100 sequences to 200 positions 24 and 19, 2000 to 512 39 and 37, 10000 to 1000 253 and 230.  Between 1024 and 4096 groups of many tiles it would
// still gain (2500 to 4096: 199 and 222).
constexpr int kDealt = 1024;

struct Control {
    uint64_t k_full[kMaxStages], k_empty[kMaxStages];
    uint64_t acc_full[kMaxSlots], acc_empty[kMaxSlots];
    uint64_t q_full[2], q_empty[2], w_full[2], w_empty[2];
    uint64_t exchange[4];             // per warpgroup, the warps' exchange for blocks of 64 and 128
    uint32_t tmem_base;
    int abort_flag;
    uint32_t page_ok[kMaxStages];     // per stage, a bit per page of the tile
    int valid[2][kMaxRows];
    int sums[kWarps];                 // dealing the tiles out
    int share, first_group, first_tile;   // this CTA's tiles, and where they begin
    int filled;                       // items whose unseen columns some warp has taken
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
    int H, s_q, kv_len, limit, block, block_shift, cols, block_table_stride, page_shift;
    int per, groups_per_seq, groups;      // query rows of a group, groups of a sequence and of all
    int tiles, chunk, items;              // items: groups x chunks of tiles
    int even;                             // the tiles of all groups are dealt out evenly
    int acc_cols, slots;                  // narrow: TMEM columns of an accumulator, accumulators in TMEM
    int fulls;                            // barriers that say an accumulator is full
    int stages, q_bufs;
    uint32_t off_k, off_s, off_w, q_bytes;   // shared memory: Q buffers | keys | their scales | weights | control
};

// keys of a stage: bf16 two blocks of 64 columns, fp8 one of 128
template <bool kFp8> constexpr int kKeyBytes = kFp8 ? kTile * 128 : kTile * 256;

// A warp's wait, bounded: in plain try_waits, whose first usually finds the phase complete, and no sleep in between (with a suspend-time
// hint a failed try sleeps, and every hand-over in this kernel took some hundred cycles more).  Gives up by time or when another warp has.
__device__ __forceinline__ bool try_all(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)); }
__device__ __noinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    const uint64_t t0 = global_ns();
#pragma unroll 1
    for (uint32_t n = 1;; ++n) {
        if (try_all(bar, parity)) return true;
        if (*abort_flag) return false;
        if ((n & 63u) == 0 && __any_sync(0xffffffffu, global_ns() - t0 > DSA_WAIT_BUDGET_NS)) {
            *abort_flag = 1;
            return false;
        }
    }
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) { return try_all(bar, parity) || wait_on(bar, parity, abort_flag); }

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN where either is
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float warp_max_nan(float a) {   // (volatile: the whole warp executes it, also where one lane uses the result)
    float d;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(d) : "f"(a));
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

// A work item: tiles of one group.
struct Item {
    int seq, q0, rows, tile0, tiles;   // tiles: those that hold a position of some row
};
__device__ __forceinline__ int row_limit(const Params& p, int q) { return p.valid_len != nullptr ? max(0, min(p.limit, __ldg(p.valid_len + q))) : p.limit; }
__device__ __forceinline__ void group_of(const Params& p, int g, Item& it) {
    it.seq = g / p.groups_per_seq;
    const int r0 = (g - it.seq * p.groups_per_seq) * p.per;
    it.q0 = it.seq * p.s_q + r0;
    it.rows = min(p.per, p.s_q - r0);
}
// tiles of the group that hold a position of some row: one warp
__device__ __forceinline__ int live_tiles(const Params& p, const Item& it, int lane) {
    return (__reduce_max_sync(0xffffffffu, lane < it.rows ? row_limit(p, it.q0 + lane) : 0) + kTile - 1) / kTile;
}
// item u of the groups x chunks
__device__ __forceinline__ Item item_of(const Params& p, int u, int lane) {
    Item it;
    const int c = u / p.groups;
    group_of(p, u - c * p.groups, it);
    it.tile0 = c * p.chunk;
    it.tiles = max(0, min(live_tiles(p, it, lane) - it.tile0, min(p.chunk, p.tiles - it.tile0)));
    return it;
}
// The items of a CTA, walked by every role for itself.  Few groups (a decode batch of ragged lengths): the CTA's share of all tiles, counted
// through the groups.  Many: every gridDim-th of groups x chunks.
struct Walk {
    const Params& p;
    int left, g, t, u, lane;
    __device__ __forceinline__ Walk(const Params& p_, const Control* ctl, int lane_)
        : p(p_), left(ctl->share), g(ctl->first_group), t(ctl->first_tile), u(blockIdx.x), lane(lane_) {}
    __device__ __forceinline__ bool next(Item& it) {   // false: no more
        if (p.even) {
            while (left > 0) {
                group_of(p, g++, it);
                it.tile0 = t;
                it.tiles = min(live_tiles(p, it, lane) - t, left);
                t = 0;
                if (it.tiles <= 0) continue;
                left -= it.tiles;
                return true;
            }
            return false;
        }
        while (u < p.items) {
            it = item_of(p, u, lane);
            u += gridDim.x;
            if (it.tiles > 0) return true;
        }
        return false;
    }
};
// All threads of the CTA: its share.
__device__ void deal_out(const Params& p, Control* ctl) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = (p.groups + 32 * kWarps - 1) / (32 * kWarps);
    const int g0 = min(tid * each, p.groups), g1 = min(g0 + each, p.groups);
    auto tiles_of = [&](int g) {
        Item it;
        group_of(p, g, it);
        int n = 0;
        for (int r = 0; r < it.rows; ++r) n = max(n, row_limit(p, it.q0 + r));
        return (n + kTile - 1) / kTile;
    };
    int sum = 0;
    for (int g = g0; g < g1; ++g) sum += tiles_of(g);
    int incl = sum;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += o;
    }
    if (lane == 31) ctl->sums[warp] = incl;
    __syncthreads();
    int before = incl - sum, all = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += ctl->sums[w];
        all += ctl->sums[w];
    }
    const int lo = (int)((int64_t)all * blockIdx.x / gridDim.x), hi = (int)((int64_t)all * (blockIdx.x + 1) / gridDim.x);
    if (tid == 0) ctl->share = hi - lo;
    if (lo >= before && lo < before + sum) {   // one thread, when there is a tile at all
        int g = g0, n = 0;
        for (; before + (n = tiles_of(g)) <= lo; ++g) before += n;
        ctl->first_group = g;
        ctl->first_tile = lo - before;
    }
    __syncthreads();
}
// One warp: value into columns of tiles [tile0, tile1) of the item's rows.
__device__ __forceinline__ void fill(const Params& p, const Item& it, int tile0, int tile1, float value, int lane) {
    const int c0 = (int)((int64_t)tile0 * kTile / p.block), c1 = (int)min((int64_t)p.cols, (int64_t)tile1 * kTile / p.block);
    for (int r = 0; r < it.rows; ++r)
        for (int c = c0 + lane; c < c1; c += 32) p.out[(int64_t)(it.q0 + r) * p.stride_o_row + c] = value;
}
// The columns behind the last position that a row of an item sees; whichever warp has nothing else to do takes the next item of the CTA's.
__device__ __forceinline__ void fill_unseen(const Params& p, Control* ctl, int lane) {
    while (true) {
        int n = 0;
        if (lane == 0) n = atomicAdd(&ctl->filled, 1);
        n = __shfl_sync(0xffffffffu, n, 0);
        const int64_t u = blockIdx.x + (int64_t)n * gridDim.x;
        if (u >= p.items) return;
        const Item it = item_of(p, (int)u, lane);
        fill(p, it, it.tile0 + it.tiles, min(it.tile0 + p.chunk, p.tiles), -INFINITY, lane);
    }
}

// ------------------------------------------------ sums over heads
// Twice 16 lanes x kCols columns of an accumulator: of either half thread t gets, for i < kCols / 8, columns 8 i + 2 (t % 4) and the next of lane t / 4 in
// d[4 i], d[4 i + 1] and of lane t / 4 + 8 in d[4 i + 2], d[4 i + 3].  So a thread needs the weights of a quarter of the heads only (all of
// them for every position, read from shared memory for every accumulator, were as many wavefronts as the MMAs' own operands and kept the
// kernel at 1 800 cycles an accumulator), and the four threads of a quad add up their parts for four positions.
// The loads and their wait are one statement, as the sums read nothing but registers: with a wait of its own nothing would keep them behind it.
// (Apart, with the scores of the row before on their way out in between, some sums were wrong.)
template <int kCols> __device__ __forceinline__ void load_row(uint32_t taddr, uint32_t (&lo)[kCols / 2], uint32_t (&hi)[kCols / 2]) {
    if constexpr (kCols == 64) {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
            "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
            "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
            "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(lo[0]), "=r"(lo[1]), "=r"(lo[2]), "=r"(lo[3]), "=r"(lo[4]), "=r"(lo[5]), "=r"(lo[6]), "=r"(lo[7]),
              "=r"(lo[8]), "=r"(lo[9]), "=r"(lo[10]), "=r"(lo[11]), "=r"(lo[12]), "=r"(lo[13]), "=r"(lo[14]), "=r"(lo[15]),
              "=r"(lo[16]), "=r"(lo[17]), "=r"(lo[18]), "=r"(lo[19]), "=r"(lo[20]), "=r"(lo[21]), "=r"(lo[22]), "=r"(lo[23]),
              "=r"(lo[24]), "=r"(lo[25]), "=r"(lo[26]), "=r"(lo[27]), "=r"(lo[28]), "=r"(lo[29]), "=r"(lo[30]), "=r"(lo[31]),
              "=r"(hi[0]), "=r"(hi[1]), "=r"(hi[2]), "=r"(hi[3]), "=r"(hi[4]), "=r"(hi[5]), "=r"(hi[6]), "=r"(hi[7]),
              "=r"(hi[8]), "=r"(hi[9]), "=r"(hi[10]), "=r"(hi[11]), "=r"(hi[12]), "=r"(hi[13]), "=r"(hi[14]), "=r"(hi[15]),
              "=r"(hi[16]), "=r"(hi[17]), "=r"(hi[18]), "=r"(hi[19]), "=r"(hi[20]), "=r"(hi[21]), "=r"(hi[22]), "=r"(hi[23]),
              "=r"(hi[24]), "=r"(hi[25]), "=r"(hi[26]), "=r"(hi[27]), "=r"(hi[28]), "=r"(hi[29]), "=r"(hi[30]), "=r"(hi[31])
            : "r"(taddr), "r"(taddr + (16u << 16))
            : "memory");
    } else if constexpr (kCols == 32) {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n\t"
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(lo[0]), "=r"(lo[1]), "=r"(lo[2]), "=r"(lo[3]), "=r"(lo[4]), "=r"(lo[5]), "=r"(lo[6]), "=r"(lo[7]),
              "=r"(lo[8]), "=r"(lo[9]), "=r"(lo[10]), "=r"(lo[11]), "=r"(lo[12]), "=r"(lo[13]), "=r"(lo[14]), "=r"(lo[15]),
              "=r"(hi[0]), "=r"(hi[1]), "=r"(hi[2]), "=r"(hi[3]), "=r"(hi[4]), "=r"(hi[5]), "=r"(hi[6]), "=r"(hi[7]),
              "=r"(hi[8]), "=r"(hi[9]), "=r"(hi[10]), "=r"(hi[11]), "=r"(hi[12]), "=r"(hi[13]), "=r"(hi[14]), "=r"(hi[15])
            : "r"(taddr), "r"(taddr + (16u << 16))
            : "memory");
    } else {
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%16];\n\t"
            "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%8, %9, %10, %11, %12, %13, %14, %15}, [%17];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(lo[0]), "=r"(lo[1]), "=r"(lo[2]), "=r"(lo[3]), "=r"(lo[4]), "=r"(lo[5]), "=r"(lo[6]), "=r"(lo[7]),
              "=r"(hi[0]), "=r"(hi[1]), "=r"(hi[2]), "=r"(hi[3]), "=r"(hi[4]), "=r"(hi[5]), "=r"(hi[6]), "=r"(hi[7])
            : "r"(taddr), "r"(taddr + (16u << 16))
            : "memory");
    }
}
// where head h's weight stands in its row, so that a thread's are 16 bytes at a time: 16 j + 4 (t % 4) + ..
__device__ __forceinline__ int weight_at(int h) { return (h & ~15) + 4 * ((h & 7) >> 1) + 2 * ((h >> 3) & 1) + (h & 1); }
// the position inside the warp's 32 whose sum a thread ends up with
__device__ __forceinline__ int lane_position(int lane) { return (lane >> 2) + 8 * (lane & 1) + 16 * ((lane >> 1) & 1); }
// the lane whose position is `off` further on, off a power of two
__device__ __forceinline__ int lane_of_offset(int off) { return off < 8 ? 4 * off : off >> 3; }

// The sum of w_h max(0, d_h) over a pair of heads is two maxima (half rate) and two multiply-adds.  With max(0, d) taken as (d + |d|) / 2 it is a
// two-wide multiply-add and two with |d|, three instructions: when it was tried, within 1 % for 4096 rows over 16384 positions and 4 % slower for 64 x 2
// rows over 32768, so it stays out.
struct Sum {
    float a = 0.0f, b = 0.0f;
    __device__ __forceinline__ void add(uint32_t d0, uint32_t d1, float u, float v) {
        a = fmaf(max_nan(__uint_as_float(d0), 0.0f), u, a);
        b = fmaf(max_nan(__uint_as_float(d1), 0.0f), v, b);
    }
    __device__ __forceinline__ float total() const { return a + b; }
};
// The row's sum of the thread's position (lane_position).  w: shared-memory address of the thread's first four weights; heads: how many there
// are, when not all columns are one.
template <bool kFp8, int kCols, bool kAll>
__device__ __forceinline__ float sum_heads(const uint32_t (&lo)[kCols / 2], const uint32_t (&hi)[kCols / 2], uint32_t w, int heads, int lane) {
    Sum s[4];
#pragma unroll
    for (int j = 0; j < kCols / 16; ++j) {
        float w4[4];
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(w4[0]), "=f"(w4[1]), "=f"(w4[2]), "=f"(w4[3]) : "r"(w + 64 * j));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int i = 2 * j + e;
            uint32_t v[8] = {lo[4 * i], lo[4 * i + 1], lo[4 * i + 2], lo[4 * i + 3], hi[4 * i], hi[4 * i + 1], hi[4 * i + 2], hi[4 * i + 3]};
            if (!kFp8 && !kAll) {   // columns behind the heads: zeros times an infinite key (e4m3 has none) are NaN
                const int h = 8 * i + 2 * (lane & 3);
#pragma unroll
                for (int c = 0; c < 8; ++c) v[c] = h + (c & 1) < heads ? v[c] : 0u;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) s[c].add(v[2 * c], v[2 * c + 1], w4[2 * e], w4[2 * e + 1]);
        }
    }
    // the quad's parts: after the first exchange a thread has two positions, after the second its own
    const bool b0 = lane & 1, b1 = lane & 2;
    const float t0 = s[0].total(), t1 = s[1].total(), t2 = s[2].total(), t3 = s[3].total();
    const float x = (b0 ? t1 : t0) + __shfl_xor_sync(0xffffffffu, b0 ? t0 : t1, 1), y = (b0 ? t3 : t2) + __shfl_xor_sync(0xffffffffu, b0 ? t2 : t3, 1);
    return (b1 ? y : x) + __shfl_xor_sync(0xffffffffu, b1 ? x : y, 2);
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
    __device__ __forceinline__ void skip(int by, int n) {
        for (s += by; s >= n; s -= n) ph ^= 1u;
    }
};

// kCols: TMEM columns of a query row, its heads padded to 16, 32 or 64; kAll: there are exactly so many.
// kWide: groups of 512 columns.  A tile has two accumulators of 256, and every warpgroup takes its half of one.  Otherwise groups of at most 256 columns, one accumulator a tile, and the warpgroups take tiles in turn.
template <bool kFp8, int kCols, bool kAll, bool kWide>
__global__ void __launch_bounds__(32 * kWarps, 1) index_scores_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tq, const __grid_constant__ Params p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Control* ctl = reinterpret_cast<Control*>(smem + kSmemBytes - kControlBytes);
    float* const w_smem = reinterpret_cast<float*>(smem + p.off_w);
    uint8_t* const k_smem = smem + p.off_k;
    const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    volatile int* abort_flag = &ctl->abort_flag;
    const uint32_t base = smem_u32(smem);
    auto bar_at = [&](size_t offset, int i) { return base + (uint32_t)(kSmemBytes - kControlBytes + offset) + 8u * i; };

    if (tid == 0) {
        for (int i = 0; i < p.stages; ++i) {
            mbar_init(bar_at(offsetof(Control, k_full), i), 1);
            mbar_init(bar_at(offsetof(Control, k_empty), i), 1 + (kWide ? kEpiWarps : 4));
        }
        for (int i = 0; i < p.fulls; ++i) mbar_init(bar_at(offsetof(Control, acc_full), i), 2);
        for (int i = 0; i < p.slots; ++i) {
            mbar_init(bar_at(offsetof(Control, acc_empty), i), kWide ? kEpiWarps / 2 : 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_at(offsetof(Control, q_full), i), 1);
            mbar_init(bar_at(offsetof(Control, q_empty), i), 1);
            mbar_init(bar_at(offsetof(Control, w_full), i), 32);
            mbar_init(bar_at(offsetof(Control, w_empty), i), kEpiWarps);
        }
        for (int i = 0; i < 4; ++i) mbar_init(bar_at(offsetof(Control, exchange), i), 4);
        ctl->abort_flag = 0;
        ctl->share = ctl->first_group = ctl->first_tile = ctl->filled = 0;
        fence_mbar_init();
    }
    if (warp == kEpiWarps && lane == 0) {
        prefetch_tensormap(&tk);
        prefetch_tensormap(&tq);
    }
    if (warp == kWarps - 1) {
        tmem_alloc(smem_u32(&ctl->tmem_base), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;
    grid_dependency_wait();
    if (p.even) deal_out(p, ctl);
    Walk walk(p, ctl, lane);
    Item it;

    if (warp < kEpiWarps) {
        // ------------------------------------------------ scores out
        const int wg = warp >> 2, sub = warp & 3;
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * sub) << 16);
        const int mine = 32 * sub + lane_position(lane);   // of a tile's positions
        const int page_bit = mine >> min(p.page_shift, 7), block = p.block, kv_len = p.kv_len;
        Ring k, acc, fl, wb;
        uint32_t exchanges = 0;
        bool ok = true;
        int done = 0;      // items
        // A score to its place: s of position pos, -inf unless it counts; `stored`: the row is one.  Blocks of more than a warp's positions are joined
        // over the warpgroup when the next row's scores are there (or the item ends), by when the other warps' parts have long come (joined
        // at once, 1500 rows of 32 heads in blocks of 64 took 103 instead of 83 us).
        bool pending = false, pending_stored = false;
        float pending_s = 0.0f;
        float* pending_at = nullptr;
        auto join = [&]() {
            if (!pending) return;
            pending = false;
            const int buf = (exchanges - 1) & 1;   // (a third job's value is written after the exchange of the second)
            ok = ok && wait(bar_at(offsetof(Control, exchange), wg), buf, abort_flag);
            float s = max_nan(pending_s, ctl->best[wg][buf][sub ^ 1]);
            if (block == 128) s = max_nan(s, max_nan(ctl->best[wg][buf][sub ^ 2], ctl->best[wg][buf][sub ^ 3]));
            if (pending_stored) *pending_at = s;
        };
        auto put = [&](float s, bool counts, int pos, float* at, bool stored) {
            s = counts ? s : -INFINITY;
            stored = stored && pos < kv_len;
            if (block == 1) {
                if (stored) *at = s;
                return;
            }
            stored = stored && (pos & (block - 1)) == 0;
            if (block < 32) {
                for (int off = 1; off < block; off <<= 1) s = max_nan(s, __shfl_xor_sync(0xffffffffu, s, lane_of_offset(off)));
            } else {
                s = warp_max_nan(s);
            }
            if (block < 64) {
                if (stored) *at = s;
                return;
            }
            join();
            __syncwarp();
            if (lane == 0) {
                ctl->best[wg][exchanges & 1][sub] = s;
                mbar_arrive(bar_at(offsetof(Control, exchange), wg));
            }
            ++exchanges;
            pending = true, pending_stored = stored, pending_s = s, pending_at = at;
        };
        // (acc_full has an arrival of the MMA warp's own besides the MMAs': what that warp saw in the tile's barrier is visible here)
        auto tile_facts = [&](float& ks, bool& here) {
            here = (ctl->page_ok[k.s] >> page_bit) & 1u;
            ks = kFp8 ? reinterpret_cast<const float*>(smem + p.off_s + k.s * kScaleBytes)[mine] : 1.0f;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_at(offsetof(Control, k_empty), k.s));
        };
        uint32_t lo[kCols / 2], hi[kCols / 2];
        auto give_back = [&](uint32_t bar) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        if constexpr (kWide) {
            constexpr int kRows = 128 / kCols;                         // of a warpgroup: half of an accumulator
            const int half = wg >> 1, row0 = wg * kRows;
            const uint32_t at = lanes + row0 * kCols, full = bar_at(offsetof(Control, acc_full), half), empty = bar_at(offsetof(Control, acc_empty), half);
            for (; ok && walk.next(it); ++done) {
                if (!(ok = wait(bar_at(offsetof(Control, w_full), wb.s), wb.ph, abort_flag))) break;
                int pos = it.tile0 * kTile + mine, end[kRows];
                const uint32_t w = base + p.off_w + wb.s * p.per * kCols * 4 + 16 * (lane & 3) + row0 * kCols * 4;
#pragma unroll
                for (int j = 0; j < kRows; ++j) end[j] = row0 + j < it.rows ? ctl->valid[wb.s][row0 + j] : -1;   // -1: there is no such row
                float* out = p.out + (int64_t)(it.q0 + row0) * p.stride_o_row + (pos >> p.block_shift);
                const int64_t stride = p.stride_o_row;
                const int step = kTile >> p.block_shift;
                for (int i = 0; i < it.tiles; ++i, pos += kTile, out += step) {
                    if (!(ok = ok && wait(full, acc.ph, abort_flag))) break;
                    tc_fence_after();
                    load_row<kCols>(at, lo, hi);
                    float ks;
                    bool here;
                    tile_facts(ks, here);
                    float* o = out;
#pragma unroll
                    for (int j = 0; j < kRows; ++j, o += stride) {
                        if (j == kRows - 1) give_back(empty);
                        const float s = sum_heads<kFp8, kCols, kAll>(lo, hi, w + j * kCols * 4, p.H, lane) * ks;
                        if (j + 1 < kRows) load_row<kCols>(at + (j + 1) * kCols, lo, hi);
                        put(s, here && pos < end[j], pos, o, end[j] >= 0);
                    }
                    acc.ph ^= 1u;
                    k.next(p.stages);
                }
                join();
                if (!ok) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_at(offsetof(Control, w_empty), wb.s));
                wb.next(p.q_bufs);
            }
        } else {
            int turn = wg;                     // tiles until this warpgroup's next one
            k.skip(wg, p.stages);
            acc.skip(wg, p.slots);
            fl.skip(wg, p.fulls);
            for (; ok && walk.next(it); ++done) {
                if (!(ok = wait(bar_at(offsetof(Control, w_full), wb.s), wb.ph, abort_flag))) break;
                int i = turn;
                for (; i < it.tiles && ok; i += 4, k.skip(4, p.stages), acc.skip(4, p.slots), fl.skip(4, p.fulls)) {
                    const int pos = (it.tile0 + i) * kTile + mine;
                    if (!(ok = wait(bar_at(offsetof(Control, acc_full), fl.s), fl.ph, abort_flag))) break;
                    tc_fence_after();
                    uint32_t at = lanes + acc.s * p.acc_cols, w = base + p.off_w + wb.s * p.per * kCols * 4 + 16 * (lane & 3);
                    load_row<kCols>(at, lo, hi);
                    float ks;
                    bool here;
                    tile_facts(ks, here);
                    float* out = p.out + (int64_t)it.q0 * p.stride_o_row + (pos >> p.block_shift);
                    for (int r = 0; r < it.rows; ++r, w += kCols * 4, out += p.stride_o_row) {
                        if (r == it.rows - 1) give_back(bar_at(offsetof(Control, acc_empty), acc.s));
                        const float s = sum_heads<kFp8, kCols, kAll>(lo, hi, w, p.H, lane) * ks;
                        if (r + 1 < it.rows) load_row<kCols>(at += kCols, lo, hi);
                        put(s, here && pos < ctl->valid[wb.s][r], pos, out, true);
                    }
                }
                join();
                if (!ok) break;
                turn = i - it.tiles;
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_at(offsetof(Control, w_empty), wb.s));
                wb.next(p.q_bufs);
            }
        }
        if (!ok) {   // a wait gave up: every warp that saw it marks all of the items that were not finished
            Walk again(p, ctl, lane);
            for (int n = 0; again.next(it); ++n)
                if (n >= done) fill(p, it, it.tile0, it.tile0 + it.tiles, __int_as_float(0x7FFFFFFF), lane);
        }
    } else if (warp == kEpiWarps) {
        // ------------------------------------------------ keys in
        Ring k;
        const int page_rows = 1 << min(p.page_shift, 7), pages = kTile / page_rows;   // of a tile
        bool ok = true;
        while (ok && walk.next(it)) {
            // Page numbers come 32 at a time, a batch ahead of their use (a load of them per tile was 700 clocks of every tile).
            const int per_batch = 32 / pages;   // tiles of a batch
            auto batch = [&](int first) {
                const int pos = (it.tile0 + first) * kTile + lane * page_rows;
                int64_t page = -1;
                if (first < it.tiles) {
                    const int blk = pos >> p.page_shift;
                    if (p.block_table == nullptr) page = (int64_t)it.seq * p.seq_stride_pages + blk;
                    else if (blk < p.block_table_stride) page = __ldg(p.block_table + (int64_t)it.seq * p.block_table_stride + blk);
                }
                return page >= 0 && page < p.num_pages ? (int)page : -1;
            };
            int now = -1, ahead = batch(0);
            for (int i = 0; i < it.tiles; ++i, k.next(p.stages)) {
                const int pos = (it.tile0 + i) * kTile, in_batch = i & (per_batch - 1);
                if (in_batch == 0) {
                    now = ahead;
                    ahead = batch(i + per_batch);
                }
                const int got = __shfl_sync(0xffffffffu, now, (in_batch * pages + lane) & 31);
                const int64_t page = lane < pages ? got : -1;
                const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
                if (!(ok = wait(bar_at(offsetof(Control, k_empty), k.s), k.ph ^ 1u, abort_flag))) break;
                const uint32_t bar = bar_at(offsetof(Control, k_full), k.s), dst = smem_u32(k_smem + k.s * kKeyBytes<kFp8>);
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
    } else if (warp == kEpiWarps + 1) {
        // ------------------------------------------------ query rows, weights, lengths in
        Ring b;
        bool ok = true;
        while (ok && walk.next(it)) {
            if (!(ok = wait(bar_at(offsetof(Control, q_empty), b.s), b.ph ^ 1u, abort_flag))) break;
            const uint32_t bar = bar_at(offsetof(Control, q_full), b.s), dst = smem_u32(smem) + b.s * p.q_bytes;
            if (lane == 0) mbar_arrive_expect_tx(bar, it.rows * kCols * (kFp8 ? 128 : 256));
            __syncwarp();
            if (lane < it.rows) {
                tma_load_3d(dst + lane * kCols * 128, &tq, bar, 0, 0, it.q0 + lane);
                if (!kFp8) tma_load_3d(dst + p.q_bytes / 2 + lane * kCols * 128, &tq, bar, 64, 0, it.q0 + lane);
            }
            if (!(ok = wait(bar_at(offsetof(Control, w_empty), b.s), b.ph ^ 1u, abort_flag))) break;
            float* w = w_smem + b.s * p.per * kCols;
            for (int i = lane; i < it.rows * kCols; i += 32) {
                const int r = i / kCols, h = i % kCols;
                w[r * kCols + weight_at(h)] = h < p.H ? __ldg(p.weights + (int64_t)(it.q0 + r) * p.stride_w_row + h) : 0.0f;
            }
            if (lane < it.rows) ctl->valid[b.s][lane] = row_limit(p, it.q0 + lane);
            mbar_arrive(bar_at(offsetof(Control, w_full), b.s));
            b.next(p.q_bufs);
        }
    } else {
        // ------------------------------------------------ MMAs
        Ring k, acc, fl, b;
        bool ok = true;
        const uint32_t el = elect_one() ? 1u : 0u;
        const uint64_t k_desc = make_smem_desc_sw128(smem_u32(k_smem), 0, 1024), q_desc = make_smem_desc_sw128(smem_u32(smem), 0, 1024);
        const uint32_t k_lo = (uint32_t)k_desc, q_lo = (uint32_t)q_desc, hi = (uint32_t)(k_desc >> 32);
        while (ok && walk.next(it)) {
            if (!(ok = wait(bar_at(offsetof(Control, q_full), b.s), b.ph, abort_flag))) break;
            for (int i = 0; i < it.tiles && ok; ++i, k.next(p.stages)) {
                if (!(ok = wait(bar_at(offsetof(Control, k_full), k.s), k.ph, abort_flag))) break;
#pragma unroll
                for (int part = 0; part < (kWide ? 2 : 1); ++part) {
                    if (!(ok = ok && wait(bar_at(offsetof(Control, acc_empty), acc.s), acc.ph ^ 1u, abort_flag))) break;
                    tc_fence_after();
                    const int n = kWide ? kMmaCols : it.rows * kCols;   // (wide: rows that there are not are never read back)
                    const uint32_t a = k_lo + ((k.s * kKeyBytes<kFp8>) >> 4), q = q_lo + ((b.s * p.q_bytes + part * kMmaCols * 128) >> 4);
                    const uint32_t d = tmem + acc.s * (kWide ? kMmaCols : p.acc_cols), full = bar_at(offsetof(Control, acc_full), fl.s);
                    if constexpr (kFp8) {
                        umma_f8_ss_x4_el(d, a, hi, q, hi, make_idesc_e4m3(kTile, n), el);
                    } else {
                        const uint32_t idesc = make_idesc_bf16(kTile, n, false);
                        umma_ss_x4_el(d, a, hi, q, hi, idesc, 0u, el);
                        umma_ss_x4_el(d, a + ((kTile * 128) >> 4), hi, q + ((p.q_bytes / 2) >> 4), hi, idesc, 1u, el);
                    }
                    tc_commit_el(full, el);
                    if (el) mbar_arrive(full);
                    acc.next(p.slots);
                    fl.next(p.fulls);
                }
                if (ok) tc_commit_el(bar_at(offsetof(Control, k_empty), k.s), el);
            }
            if (!ok) break;
            tc_commit_el(bar_at(offsetof(Control, q_empty), b.s), el);
            b.next(p.q_bufs);
        }
    }
    __syncwarp();
    if (warp != kWarps - 1) fill_unseen(p, ctl, lane);
    tc_fence_before();
    __syncthreads();
    if (ctl->abort_flag) {
        if (tid == 0 && p.status != nullptr) atomicExch(p.status, DSA_V32_ERR_DEVICE_WAIT);
        settle_in_flight();
        __syncthreads();
    }
    if (warp == kWarps - 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <bool kFp8, int kCols, bool kAll, bool kWide>
cudaError_t launch(const CUtensorMap& tk, const CUtensorMap& tq, const Params& p, int grid, cudaStream_t stream) {
    static std::mutex mu;
    static bool done[64] = {};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> guard(mu);
        if (dev < 0 || dev >= 64 || !done[dev]) {
            e = cudaFuncSetAttribute(index_scores_kernel<kFp8, kCols, kAll, kWide>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
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
    return cudaLaunchKernelEx(&cfg, index_scores_kernel<kFp8, kCols, kAll, kWide>, tk, tq, p);
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
    while ((1 << p.block_shift) < a.block) ++p.block_shift;
    p.cols = (a.kv_len + a.block - 1) / a.block;
    p.block_table_stride = a.block_table_stride;
    // Query rows of a group: 512 columns' worth, or up to 256 in groups of equal size.  A group of 512 reads the keys half as often, but takes two
    // full accumulators of every tile however many rows there are: its time is that of about 0.6 of its rows in groups of 256, so wide groups it is
    // where all narrow ones' rows are more than 0.6 of all wide ones' places.
    // us wide and narrow, fp8, 16384 positions, 64 heads: 64 sequences of 3 rows 80 and 59, 4 82 and 76, 5 83 and 106, 6 84 and 107, 7 85 and 136, 8 86
    // and 138; 16 sequences of 9 rows 49 and 44, 10 49 and 56, 16 50 and 72 (bf16 9 rows 53 and 46, 10 53 and 59).  32 heads: 64 sequences of 8 rows 85
    // and 75, 9 86 and 93; 16 of 18 rows 50 and 47, 19 50 and 53.  16 heads: 16 of 18 rows 38 and 37, 19 39 and 40, 36 67 and 64, 40 67 and 73.
    const int most = kTmemCols / cols, wide_groups = (int)(((int64_t)a.s_q + most - 1) / most), narrow_groups = (int)(((int64_t)a.s_q + most / 2 - 1) / (most / 2));
    const int narrow_per = (int)(((int64_t)a.s_q + narrow_groups - 1) / narrow_groups);
    const bool wide = 5 * (int64_t)narrow_groups * narrow_per > 3 * (int64_t)wide_groups * most;
    p.per = wide ? most : narrow_per;
    p.groups_per_seq = (a.s_q + p.per - 1) / p.per;
    const int64_t groups = (int64_t)p.groups_per_seq * (a.total_q / a.s_q);
    p.acc_cols = 64;
    while (p.acc_cols < p.per * cols) p.acc_cols *= 2;
    p.slots = wide ? 2 : kTmemCols / p.acc_cols;
    // Tiles go to four warpgroups in turn.  With two accumulators two of them share one, and a wait by parity must not be two phases ahead of its
    // barrier, so every warpgroup has a full barrier of its own.
    p.fulls = wide || p.slots > 4 ? p.slots : 4;
    // shared memory: two buffers of query rows where that leaves four stages of keys
    const int stage = fp8 ? kKeyBytes<true> + kScaleBytes : kKeyBytes<false>;
    p.q_bytes = p.per * cols * (fp8 ? 128 : 256);
    auto stages = [&](int bufs) { return (kSmemBytes - kControlBytes - bufs * (int)(p.q_bytes + p.per * cols * 4)) / stage; };
    p.q_bufs = stages(2) >= 4 ? 2 : 1;
    p.stages = stages(p.q_bufs) < kMaxStages ? stages(p.q_bufs) : kMaxStages;
    p.off_k = p.q_bufs * p.q_bytes;
    p.off_s = p.off_k + p.stages * (fp8 ? kKeyBytes<true> : kKeyBytes<false>);
    p.off_w = p.off_k + p.stages * stage;
    // tiles of an item: the least for the busiest CTA, an item counted as two tiles more (for few groups the items are only what is filled)
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
    const int64_t most_tiles = groups * p.tiles;
    p.even = groups <= kDealt && most_tiles <= 0x7FFFFFFF;
    const int grid = (int)(p.even ? (most_tiles < sms ? most_tiles : sms) : (items < sms ? items : sms));
    const bool all = a.H == cols;
    auto go = [&](auto kernel) { return kernel(tk, tq, p, grid, stream); };
#define DSA_SCORES_OF(fp8_, cols_)                                                                                       \
    if (fp8 == fp8_ && cols == cols_) {                                                                                  \
        if (wide) return go(all ? launch<fp8_, cols_, true, true> : launch<fp8_, cols_, false, true>);                   \
        return go(all ? launch<fp8_, cols_, true, false> : launch<fp8_, cols_, false, false>);                           \
    }
    DSA_SCORES_OF(true, 16)
    DSA_SCORES_OF(true, 32)
    DSA_SCORES_OF(true, 64)
    DSA_SCORES_OF(false, 16)
    DSA_SCORES_OF(false, 32)
    DSA_SCORES_OF(false, 64)
#undef DSA_SCORES_OF
    return cudaErrorInvalidValue;
}

}  // namespace dsa
