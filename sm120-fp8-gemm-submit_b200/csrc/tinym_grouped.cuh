// tinym_grouped.cuh -- products with the weight chosen per row group, in E4M3
// and in MXFP4 (E2M1 elements, one E8M0 scale per 32 of them).
//
//   Y[r, n] = bf16( alpha[e] * sum_k X[r, k] * W[e, n, k] )
//                                      for offsets[e] <= r < offsets[e + 1]
//
// X holds the rows of every group one after the other ([rows, K]), W one
// matrix per group ([experts, N, K]).  A single matrix is one group over all
// rows.  As in tinym_kernels.cuh the W rows are the MMA's M side (128 TMEM
// lanes) and X rows its N side, which here is a run-time value in steps of 16
// up to TN: a group of one row costs an MMA of N = 16, not a padded 128-row
// tile, and ragged groups waste at most 15 columns of the last tile.
//
// The group sizes are read on the device, so nothing about them has to reach
// the host: a persistent grid of one CTA per SM builds the prefix sum of the
// groups' row tiles in shared memory and every role of the CTA walks the same
// list of pieces (group, row tile, W rows).
//
//  * Stream pieces (TILE = false), for few rows per group, where the time is
//    W's bytes: the W rows of all non-empty groups are laid end to end in
//    units of 8 rows and each CTA takes an equal, contiguous share of them,
//    walked in pieces of at most 128 rows with the whole of K.  The shares
//    differ by at most one unit, so every SM streams the same number of bytes
//    whatever the groups are, with no split of K, no workspace and one fixed
//    order of every sum.  A stage is 512 bytes of K, fetched by one
//    {128 B, 8 rows, 4 chunks} box per unit.
//  * Tile pieces (TILE = true), for many rows per group, where the time is
//    the tensor core's: 128 W rows x up to TN X rows, 128 bytes of K a stage.
//
// Rows of a piece past its W or X rows hold whatever the ring held before:
// the MMA computes lanes and columns for them that nobody reads.
#pragma once

#include <algorithm>

#include "tinym_kernels.cuh"

namespace tinym {

constexpr int kGrpThreads = 256;     // warp 0 TMA, 1 MMA, 2-3 scale factors, 4-7 epilogue
constexpr int kGrpMaxExperts = 1024;
constexpr int kGrpBand = 8;          // row tiles walked together for each W tile (L2 reuse)
constexpr int kScaleBlock = 512;     // scale bytes of 128 rows x 4 scales
constexpr int kSfSlotCols = 32;      // TMEM columns of one chunk's scales (8 for W, 16 for X)

struct GroupedParams {
    __nv_bfloat16* y;
    const int32_t* offsets;   // null: one group over all rows
    const float* alpha;       // null: 1
    const uint8_t* x_scales;  // MXFP4 only
    const uint8_t* w_scales;
    int64_t ldy;
    int64_t w_scale_stride;   // scale bytes per expert
    int32_t rows, experts, n;
    int32_t k_bytes;          // bytes of one operand row
    int32_t alpha_stride;     // 0: one alpha for all groups
    int32_t tn;               // X rows per tile, at most
    int32_t units;            // stream: units of 8 W rows; tile: tiles of 128 W rows
    int32_t piece_units;      // stream: units per piece, at most
    int32_t stages;
    int32_t chunked;          // stream: one box per unit covers the whole stage
    int32_t w_stage, x_stage, sf_stage;  // bytes
    uint32_t bar_off, sf_off, tab_off;   // shared-memory offsets
    uint32_t tmem_cols, acc_cols, sf_col;
    uint32_t flags;
    uint32_t* err_host;
    uint64_t timeout_ns;
};
constexpr uint32_t kGrpZeroRest = 1u;  // rows of no group are written as zeros

// 128-row scale blocks of the X rows of a tile: stream tiles have at most 128 rows.
__host__ __device__ constexpr int grouped_x_scale_blocks(bool tile) { return tile ? 2 : 1; }

struct GroupedPiece {
    int e, row0, rows, w0, h;
};

// The pieces of one CTA, in the order in which every role walks them.
template <bool TILE>
struct GroupedWalk {
    const int32_t* off;     // [experts + 1] group starts
    const int32_t* prefix;  // [experts + 1] row tiles before each group
    int experts, units, piece_units, tn;
    int cur, end, step;
    int e;

    __host__ __device__ GroupedWalk(const GroupedParams& p, const int32_t* o, const int32_t* pre,
                                    int block, int blocks)
        : off(o), prefix(pre), experts(p.experts), units(p.units), piece_units(p.piece_units),
          tn(p.tn), e(-1) {
        const int64_t total = static_cast<int64_t>(pre[p.experts]) * p.units;
        if constexpr (TILE) {
            cur = block;
            end = static_cast<int>(total);
            step = blocks;
        } else {
            cur = static_cast<int>(total * block / blocks);
            end = static_cast<int>(total * (block + 1) / blocks);
            step = 0;
        }
    }

    __host__ __device__ static int least(int a, int b) { return a < b ? a : b; }

    __host__ __device__ bool next(GroupedPiece* w) {
        if (cur >= end) return false;
        const int seg = cur / units;
        if (e < 0 || seg >= prefix[e + 1]) {
            int lo = e < 0 ? 0 : e, hi = experts - 1;  // the group whose tiles hold seg
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (prefix[mid + 1] <= seg) lo = mid + 1;
                else hi = mid;
            }
            e = lo;
        }
        const int tiles = prefix[e + 1] - prefix[e];
        const int count = off[e + 1] - off[e];
        int t;
        if constexpr (TILE) {
            const int local = cur - prefix[e] * units;
            const int band = local / (kGrpBand * units);
            const int width = least(kGrpBand, tiles - band * kGrpBand);
            const int rem = local - band * kGrpBand * units;
            const int wt = rem / width;
            t = band * kGrpBand + rem - wt * width;
            w->w0 = wt * kTileRows;
            w->h = kTileRows;
            cur += step;
        } else {
            t = seg - prefix[e];
            const int u = cur - seg * units;
            const int left = least(end - cur, units - u);
            const int pieces = (left + piece_units - 1) / piece_units;
            const int take = (left + pieces - 1) / pieces;
            w->w0 = u * 8;
            w->h = take * 8;
            cur += take;
        }
        // Equal tiles in whole MMA columns of 16: 300 rows are 160 + 140, not
        // 256 + 44.  (tiles - 1) * wide < count, since wide <= tn.
        const int wide = ((count + tiles - 1) / tiles + 15) & ~15;
        w->e = e;
        w->row0 = off[e] + t * wide;
        w->rows = least(wide, count - t * wide);
        return true;
    }
};

// How a call is cut.
struct GroupedPlan {
    bool tile;
    int grid;
    uint32_t smem;
    GroupedParams prm;  // the shape and layout fields
};

// Host only.  Group sizes live on the device, so the plan goes by the rows per
// group that the shapes allow (at most min(experts, rows) groups have any); it
// is right for every distribution of the rows.  Returns null, or why the
// shape is not supported.
inline const char* grouped_plan(bool fp4, int64_t rows, int64_t experts, int64_t n, int64_t k_bytes,
                                int sm_count, uint32_t smem_limit, GroupedPlan* out) {
    GroupedPlan g{};
    GroupedParams& p = g.prm;
    const int64_t groups = std::min(experts, rows);
    const int64_t avg = (rows + groups - 1) / groups;
    g.tile = avg > 64;
    p.rows = static_cast<int32_t>(rows);
    p.experts = static_cast<int32_t>(experts);
    p.n = static_cast<int32_t>(n);
    p.k_bytes = static_cast<int32_t>(k_bytes);
    const int64_t k_chunks = (k_bytes + kBlockK - 1) / kBlockK;
    int64_t nkb;
    if (g.tile) {
        p.tn = fp4 ? 192 : 256;
        p.units = static_cast<int32_t>((n + kTileRows - 1) / kTileRows);
        p.piece_units = 1;
        p.w_stage = kTileRows * kBlockK;
        p.x_stage = p.tn * kBlockK;
        nkb = k_chunks;
    } else {
        p.tn = static_cast<int32_t>(std::min<int64_t>(64, (3 * avg + 15) / 16 * 16));
        p.units = static_cast<int32_t>((n + 7) / 8);
        const int64_t share = (groups * p.units + sm_count - 1) / sm_count;
        p.piece_units = static_cast<int32_t>(std::min<int64_t>(16, share));
        p.w_stage = p.piece_units * 8 * 4 * kBlockK;
        p.x_stage = p.tn * 4 * kBlockK;
        p.chunked = k_bytes % kBlockK == 0;
        nkb = (k_chunks + 3) / 4;
    }
    if (fp4)
        p.sf_stage = (g.tile ? 1 : 4) * 2 * (1 + grouped_x_scale_blocks(g.tile)) * kScaleBlock;
    const int64_t max_tiles = groups + rows / p.tn;
    if (max_tiles * p.units > (int64_t(1) << 31) - (int64_t(1) << 20)) return "too many tiles";
    g.grid = static_cast<int>(std::min<int64_t>(sm_count, max_tiles * p.units));
    p.acc_cols = static_cast<uint32_t>(p.tn);
    p.sf_col = 2 * p.acc_cols;
    p.tmem_cols = 32;
    while (p.tmem_cols < 2 * p.acc_cols + (fp4 ? 2 * kSfSlotCols : 0)) p.tmem_cols *= 2;

    const uint32_t tables = 8u * static_cast<uint32_t>(experts + 1);
    auto bytes_for = [&](int stages) -> uint32_t {
        p.stages = stages;
        p.sf_off = static_cast<uint32_t>(stages * (p.w_stage + p.x_stage));
        p.bar_off = p.sf_off + static_cast<uint32_t>(stages * p.sf_stage);
        p.tab_off = p.bar_off + 8u * (3 * stages + 5) + 8u;
        // The MMA reads 128 W rows whatever the piece holds: the last stage's
        // read has to end inside the allocation.
        const uint32_t read_end = static_cast<uint32_t>((stages - 1) * p.w_stage) +
                                  kTileRows * kBlockK * (g.tile ? 1u : 4u);
        return std::max(p.tab_off + tables, read_end) + 1024u;
    };
    int stages = static_cast<int>(std::max<int64_t>(2, std::min<int64_t>(12, 2 * nkb)));
    while (stages >= 2 && bytes_for(stages) > smem_limit) --stages;
    if (stages < 2) return "no two stages fit";
    g.smem = bytes_for(stages);
    *out = g;
    return nullptr;
}

// K-major SW128 operand whose 8-row groups lie `sbo` bytes apart.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t smem_addr, uint32_t sbo) {
    return (sw128_kmajor_desc(smem_addr) & ~(0x3FFFull << 32)) |
           (static_cast<uint64_t>(sbo >> 4) << 32);
}

// Unswizzled 32 rows x 16 bytes (a scale block): 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
    return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) |
           (static_cast<uint64_t>(128u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46);
}

// One 512-byte scale block to 4 TMEM columns, repeated in the four 32-lane
// subpartitions: lane i, column j gets the four scales of row 32 j + i.
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc)
                 : "memory");
}

// Instruction descriptor of kind::mxf4: A = B = E2M1 (1) at [7,10) and
// [10,13), N >> 3 at [17,23), E8M0 scales (1) at 23, M >> 7 at [27,29).
// The scale ids (byte pair of the 32-bit scale word: 0 or 2) go to [4,6) for
// B and [29,31) for A.
__host__ __device__ constexpr uint32_t idesc_mxf4(int mma_m, int mma_n) {
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(mma_n >> 3) << 17) | (1u << 23) |
           (static_cast<uint32_t>(mma_m >> 7) << 27);
}
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                          uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                          uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], "
        "[%5], p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int32_t c0, int32_t c1, int32_t c2, int32_t c3,
                                            uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3),
        "l"(policy)
        : "memory");
}

__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void tmem_ld_x16_nowait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Group starts (made non-decreasing and inside the rows, so that no offsets
// can lead out of X or Y) and the prefix sum of the groups' row tiles, by one
// warp.
__device__ __forceinline__ void grouped_tables(const GroupedParams& p, int32_t* off,
                                               int32_t* prefix, int lane) {
    int start = 0, tiles = 0;  // running maximum of the offsets, running tile count
    if (!p.offsets) {
        if (lane == 0) {
            off[0] = 0;
            off[1] = p.rows;
            prefix[0] = 0;
            prefix[1] = (p.rows + p.tn - 1) / p.tn;
        }
        return;
    }
    for (int base = 0; base <= p.experts; base += 32) {
        const int i = base + lane;
        int v = i <= p.experts ? min(max(__ldg(p.offsets + i), 0), p.rows) : 0;
        v = max(v, start);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, v, d);
            if (lane >= d) v = max(v, o);
        }
        int before = __shfl_up_sync(0xFFFFFFFFu, v, 1);
        if (lane == 0) before = start;
        // tiles of group i - 1, whose end is offset i
        int t = i == 0 || i > p.experts ? 0 : (v - before + p.tn - 1) / p.tn;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, t, d);
            if (lane >= d) t += o;
        }
        if (i <= p.experts) {
            off[i] = v;
            prefix[i] = tiles + t;
        }
        start = __shfl_sync(0xFFFFFFFFu, v, 31);
        tiles += __shfl_sync(0xFFFFFFFFu, t, 31);
    }
}

template <bool FP4, bool TILE>
__global__ void __launch_bounds__(kGrpThreads, 1)
    tinym_grouped_kernel(const __grid_constant__ CUtensorMap tm_w,
                         const __grid_constant__ CUtensorMap tm_x, const GroupedParams p) {
    // Bytes of K per stage in 128-byte chunks; rows of one W and one X box.
    constexpr int kChunks = TILE ? 1 : 4;
    constexpr int kXBox = TILE ? 32 : 8;
    // Operand layout of a stage: 8-row swizzle atoms of 1024 bytes; the four
    // chunks of a unit are consecutive in a stream stage.
    constexpr uint32_t kSbo = kChunks * 1024;
    constexpr int kMmaK = 32;        // bytes of K per MMA (32 E4M3 or 64 E2M1 elements)
    constexpr int kSfPerChunk = 2;   // MXFP4: scale blocks (128 elements) per chunk
    constexpr int kXsBlocks = grouped_x_scale_blocks(TILE);

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align1024(smem_raw);
    const uint32_t s_base = smem_u32(smem);
    const int stages = p.stages;
    const uint32_t w_ring = s_base;
    const uint32_t x_ring = s_base + stages * p.w_stage;
    const uint32_t sf_ring = s_base + p.sf_off;
    const uint32_t bars = s_base + p.bar_off;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (stages + s); };
    auto sf_bar = [&](int s) { return bars + 8u * (2 * stages + s); };
    auto acc_full = [&](int b) { return bars + 8u * (3 * stages + b); };
    auto acc_empty = [&](int b) { return bars + 8u * (3 * stages + 2 + b); };
    const uint32_t drain_bar = bars + 8u * (3 * stages + 4);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + p.bar_off + 8u * (3 * stages + 5));
    volatile uint32_t* abort_flag = tmem_slot + 1;
    int32_t* off = reinterpret_cast<int32_t*>(smem + p.tab_off);
    int32_t* prefix = off + p.experts + 1;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const WaitGuard guard{abort_flag, &g_err_word, p.timeout_ns, p.err_host};
    const int k_chunks = (p.k_bytes + kBlockK - 1) / kBlockK;
    const int nkb = (k_chunks + kChunks - 1) / kChunks;

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
            mbar_init(sf_bar(s), 2);  // one arrival per scale warp
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), 1);
            mbar_init(acc_empty(b), 4);  // one arrival per epilogue warp
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0u;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), p.tmem_cols);
        tmem_relinquish();
    }
    // Everything above overlaps the previous kernel's tail (programmatic
    // dependent launch); no global memory is read before it has completed.
    grid_dependency_wait();
    grid_launch_dependents();
    if (warp == 2) grouped_tables(p, off, prefix, lane);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    GroupedWalk<TILE> walk(p, off, prefix, blockIdx.x, gridDim.x);
    GroupedPiece w;
    if (warp == 0) {
        // ---------------- TMA producer
        if (lane == 0) {
            const uint64_t pol_w = TILE ? l2_policy_evict_normal() : l2_policy_w();
            const uint64_t pol_x = l2_policy_evict_last();
            int s = 0, issued = 0;
            uint32_t ph = 1u;  // the first pass over the ring does not wait
            bool ok = true;
            while (ok && walk.next(&w)) {
                const int w_units = TILE ? 1 : w.h / 8;
                const int x_boxes = (w.rows + kXBox - 1) / kXBox;
                for (int i = 0; i < nkb; ++i) {
                    if (!(ok = mbar_wait_inline(empty_bar(s), ph, guard, kErrProducerWait, true)))
                        break;
                    const uint32_t wd = w_ring + s * p.w_stage, xd = x_ring + s * p.x_stage;
                    const uint32_t bar = full_bar(s);
                    const int c0 = i * kChunks;
                    if constexpr (TILE) {
                        mbar_expect_tx(bar, kTileRows * kBlockK + x_boxes * kXBox * kBlockK);
                        tma_load_3d(wd, &tm_w, bar, c0 * kBlockK, w.w0, w.e, pol_w);
                        for (int b = 0; b < x_boxes; ++b)
                            tma_load_3d(xd + b * kXBox * kBlockK, &tm_x, bar, c0 * kBlockK,
                                        w.row0 + b * kXBox, 0, pol_x);
                    } else if (p.chunked) {
                        mbar_expect_tx(bar, (w_units + x_boxes) * kChunks * 1024);
                        for (int b = 0; b < x_boxes; ++b)
                            tma_load_4d(xd + b * kChunks * 1024, &tm_x, bar, 0, w.row0 + b * 8, c0,
                                        0, pol_x);
                        for (int b = 0; b < w_units; ++b)
                            tma_load_4d(wd + b * kChunks * 1024, &tm_w, bar, 0, w.w0 + b * 8, c0,
                                        w.e, pol_w);
                    } else {
                        const int nc = min(kChunks, k_chunks - c0);
                        mbar_expect_tx(bar, (w_units + x_boxes) * nc * 1024);
                        for (int b = 0; b < x_boxes; ++b)
                            for (int c = 0; c < nc; ++c)
                                tma_load_3d(xd + (b * kChunks + c) * 1024, &tm_x, bar,
                                            (c0 + c) * kBlockK, w.row0 + b * 8, 0, pol_x);
                        for (int b = 0; b < w_units; ++b)
                            for (int c = 0; c < nc; ++c)
                                tma_load_3d(wd + (b * kChunks + c) * 1024, &tm_w, bar,
                                            (c0 + c) * kBlockK, w.w0 + b * 8, w.e, pol_w);
                    }
                    ++issued;
                    if (++s == stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            if (*abort_flag) {
                // Drain the copies still in flight before shared memory is released.
                for (int j = max(0, issued - stages); j < issued; ++j)
                    mbar_drain(full_bar(j % stages), (j / stages) & 1, guard, kErrDrain);
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (the whole warp walks, one lane issues)
        const uint32_t tmem_u = __shfl_sync(0xFFFFFFFFu, tmem, 0);
        const uint64_t da0 = sw128_desc(w_ring, kSbo);
        const uint64_t db0 = sw128_desc(x_ring, kSbo);
        int s = 0, piece = 0, slot = 0;
        uint32_t ph = 0u;
        bool ok = true;
        while (ok && walk.next(&w)) {
            const int b = piece & 1;
            const uint32_t mma_n = (w.rows + 15) & ~15;
            const uint32_t idesc = FP4 ? idesc_mxf4(128, mma_n) : idesc_e4m3_f32(128, mma_n);
            const uint32_t acc = tmem_u + b * p.acc_cols;
            const bool two = mma_n > 128;  // X scale blocks of the tile
            if (lane == 0)
                ok = mbar_wait_inline(acc_empty(b), ((piece >> 1) & 1) ^ 1u, guard, kErrMmaWait, true);
            if (!(ok = __shfl_sync(0xFFFFFFFFu, ok, 0))) break;
            tc_fence_after_sync();
            for (int i = 0; i < nkb; ++i) {
                if (lane == 0) {
                    ok = mbar_wait_inline(full_bar(s), ph, guard, kErrMmaWait, true);
                    if (FP4 && ok)
                        ok = mbar_wait_inline(sf_bar(s), ph, guard, kErrMmaWait, true);
                }
                if (!(ok = __shfl_sync(0xFFFFFFFFu, ok, 0))) break;
                tc_fence_after_sync();
                const uint64_t da = da0 + static_cast<uint64_t>((s * p.w_stage) >> 4);
                const uint64_t db = db0 + static_cast<uint64_t>((s * p.x_stage) >> 4);
                const uint32_t sf = sf_ring + s * p.sf_stage;
                const int nc = min(kChunks, k_chunks - i * kChunks);
                if (elect_one()) {
#pragma unroll
                    for (int c = 0; c < kChunks; ++c) {
                        if (c >= nc) break;
                        uint32_t sfa = 0, sfb = 0;
                        if constexpr (FP4) {
                            // this chunk's scales: 2 blocks of W, 2 or 4 of X
                            sfa = tmem_u + p.sf_col + ((slot + c) & 1) * kSfSlotCols;
                            sfb = sfa + 4 * kSfPerChunk;
                            const uint32_t xs = sf + kChunks * kSfPerChunk * kScaleBlock;
#pragma unroll
                            for (int q = 0; q < kSfPerChunk; ++q) {
                                tmem_cp_scales(sfa + 4 * q,
                                               scale_desc(sf + (c * kSfPerChunk + q) * kScaleBlock));
                                tmem_cp_scales(sfb + 8 * q,
                                               scale_desc(xs + (c * kSfPerChunk + q) * kXsBlocks * kScaleBlock));
                                if (TILE && two)
                                    tmem_cp_scales(
                                        sfb + 8 * q + 4,
                                        scale_desc(xs + ((c * kSfPerChunk + q) * kXsBlocks + 1) * kScaleBlock));
                            }
                        }
#pragma unroll
                        for (int kk = 0; kk < kBlockK / kMmaK; ++kk) {
                            const uint64_t step = static_cast<uint64_t>((c * 1024 + kk * kMmaK) >> 4);
                            const uint32_t accumulate = (i | c | kk) ? 1u : 0u;
                            if constexpr (FP4) {
                                // 64 elements: scales 2 (kk % 2), +1 of block kk / 2
                                const uint32_t id = (kk & 1) * 2;
                                umma_mxf4(acc, da + step, db + step, idesc | (id << 4) | (id << 29),
                                          sfa + 4 * (kk >> 1), sfb + 8 * (kk >> 1), accumulate);
                            } else {
                                umma_e4m3(acc, da + step, db + step, idesc, accumulate);
                            }
                        }
                    }
                    umma_commit(empty_bar(s));
                    if (i == nkb - 1) umma_commit(acc_full(b));
                }
                __syncwarp();
                slot += kChunks;
                if (++s == stages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
            ++piece;
        }
        if (!ok) {
            // An abort: wait for every MMA issued so far.
            if (elect_one()) umma_commit(drain_bar);
            __syncwarp();
            if (lane == 0) mbar_drain(drain_bar, 0, guard, kErrDrain);
            __syncwarp();
        }
    } else if (warp < 4) {
        // ---------------- MXFP4 scales: 4-byte words (128 elements of a row)
        // gathered into the 128-row block order that tcgen05.cp takes, since a
        // piece may start at any row.  Warp 2 and 3 take alternate blocks of K.
        if constexpr (FP4) {
            const int blocks = (p.k_bytes * 2 + 127) / 128;     // scale blocks along K
            const int tail = (p.k_bytes * 2 % 128) / 32;        // scales in the last one, 0: all
            int s = 0, pending = 0, ps = 0;
            uint32_t ph = 1u;
            bool ok = true;
            auto arrive = [&](int slot_) {
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(sf_bar(slot_));
            };
            auto flush = [&]() {
                cp_async_wait<0>();
                for (; pending > 0; --pending) {
                    arrive(ps);
                    if (++ps == stages) ps = 0;
                }
            };
            while (ok && walk.next(&w)) {
                const uint8_t* ws = p.w_scales + w.e * p.w_scale_stride;
                const int w_groups = (min(w.h, p.n - w.w0) + 31) / 32;
                const int x_groups = (w.rows + 31) / 32;
                for (int i = 0; i < nkb; ++i) {
                    if (!__all_sync(0xFFFFFFFFu, mbar_try_wait(empty_bar(s), ph))) {
                        flush();  // before blocking: the MMA may need what is pending
                        ok = __all_sync(0xFFFFFFFFu, mbar_wait(empty_bar(s), ph, guard, kErrProducerWait));
                        if (!ok) break;
                    }
                    const uint32_t sf = sf_ring + s * p.sf_stage;
                    const uint32_t xs = sf + kChunks * kSfPerChunk * kScaleBlock;
                    const int b0 = i * kChunks * kSfPerChunk;
                    const int nb = min(kChunks * kSfPerChunk, blocks - b0);
                    for (int q = warp - 2; q < kChunks * kSfPerChunk; q += 2) {
                        const bool in = q < nb;
                        const bool cut = in && tail && b0 + q == blocks - 1;
                        auto word = [&](uint32_t dst, const uint8_t* base, int row) {
                            const uint8_t* src = base +
                                (static_cast<int64_t>(row >> 7) * blocks + b0 + q) * kScaleBlock +
                                (row & 31) * 16 + ((row >> 5) & 3) * 4;
                            if (in && !cut) {
                                cp_async_4(dst, src);
                            } else {
                                // past K: the data are zeros, the scales 2^-127
                                uint32_t v = in ? __ldg(reinterpret_cast<const uint32_t*>(src)) : 0u;
                                v &= (1u << (8 * tail)) - 1u;
                                asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst), "r"(v) : "memory");
                            }
                        };
                        for (int g = 0; g < w_groups; ++g) {
                            const int r = w.w0 + g * 32 + lane;
                            if (r < p.n)
                                word(sf + q * kScaleBlock + lane * 16 + g * 4, ws, r);
                        }
                        for (int g = 0; g < x_groups; ++g) {
                            const int r = g * 32 + lane;
                            if (r < w.rows)
                                word(xs + (q * kXsBlocks + (g >> 2)) * kScaleBlock + lane * 16 + (g & 3) * 4,
                                     p.x_scales, w.row0 + r);
                        }
                    }
                    cp_async_commit();
                    if (++pending == 3) {
                        cp_async_wait<2>();
                        arrive(ps);
                        if (++ps == stages) ps = 0;
                        --pending;
                    }
                    if (++s == stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
            }
            flush();
        }
    } else {
        // ---------------- epilogue: warp w reads TMEM lanes 32 (w % 4) ..
        const int q = warp & 3;
        int piece = 0;
        while (walk.next(&w)) {
            const int b = piece & 1;
            const bool ready =
                mbar_wait_inline(acc_full(b), (piece >> 1) & 1, guard, kErrEpilogueWait, true) &&
                !*abort_flag;
            if (!__all_sync(0xFFFFFFFFu, ready)) break;
            tc_fence_after_sync();
            const float alpha = p.alpha ? __ldg(p.alpha + w.e * p.alpha_stride) : 1.0f;
            const int r = q * 32 + lane;
            const int n = w.w0 + r;
            const bool mine = r < w.h && n < p.n;
            __nv_bfloat16* dst = p.y + static_cast<int64_t>(w.row0) * p.ldy + n;
            const uint32_t taddr = tmem + b * p.acc_cols + (static_cast<uint32_t>(q * 32) << 16);
            for (int c = 0; c < w.rows; c += 16) {
                uint32_t v[16];
                tmem_ld_x16_nowait(taddr + c, v);
                tmem_ld_wait();
                if (mine) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        if (c + j < w.rows)
                            dst[(c + j) * p.ldy] = __float2bfloat16_rn(__uint_as_float(v[j]) * alpha);
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty(b));
            ++piece;
        }
        if (p.flags & kGrpZeroRest) {
            // rows before the first group and behind the last
            const int lo = off[0], hi = off[p.experts];
            const int rest = lo + p.rows - hi;
            for (int i = blockIdx.x; i < rest; i += gridDim.x) {
                __nv_bfloat16* dst = p.y + static_cast<int64_t>(i < lo ? i : hi + i - lo) * p.ldy;
                for (int n = threadIdx.x - 128; n < p.n; n += 128) dst[n] = __float2bfloat16_rn(0.0f);
            }
        }
    }
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc(tmem, p.tmem_cols);
}

}  // namespace tinym
