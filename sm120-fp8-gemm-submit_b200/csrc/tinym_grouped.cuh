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
// tile, and ragged groups waste at most 15 columns of a tile (31 for a pair).
//
// The group sizes are read on the device, so nothing about them has to reach
// the host: a persistent grid of one CTA per SM builds the prefix sum of the
// groups' row tiles in shared memory and every role of the CTA walks the same
// list of pieces (group, row tile, W rows).
//
//  * Stream pieces, for few rows per group, where the time is W's bytes: the W
//    rows of all non-empty groups are laid end to end in units of 8 rows and
//    each CTA takes an equal, contiguous share of them, walked in pieces of at
//    most 128 rows with the whole of K.  The shares differ by at most one
//    unit, so every SM streams the same number of bytes whatever the groups
//    are, with no split of K over CTAs, no workspace and one fixed order of
//    every sum.  28 experts of 2048 x 5120 E4M3 with 128 rows: 52.5 us, 5.6 TB/s
//    (86 % of the measured copy); 60 of 2000 x 4096 MXFP4 with 256 rows: 46 us,
//    5.7 TB/s.
//  * Folded stream pieces, for so little work that a CTA's share is at most 64
//    W rows and a tile at most 16 X rows.  An MMA costs ~45 cycles to
//    issue whether 30 or 128 of its rows are used, and a share takes K / 32
//    bytes of them.  So K is cut into S segments that stand side by side in
//    one MMA: A row a h + r is W row r in segment a, B column b x + t is X row
//    t in segment b, the S diagonal blocks of the product are the segments'
//    sums, and the epilogue adds them in order: an S-th of the instructions
//    (1 x 5120 x 6144: E4M3 11.2 -> 9.2 us, MXFP4 8.4 -> 7.2 us when it came in).
//  * Pair pieces, for many rows per group, where the time is the
//    tensor core's: two CTAs (cta_group::2) compute 256 W rows x up to 256 X
//    rows, 128 bytes of K a stage.  Each loads its 128 W rows and half of the
//    X rows, so a CTA moves 256 rows of K for 128 x 256 sums where one CTA
//    alone would move 384: the L2 feeds the SMs at ~42 bytes/clk/SM here,
//    which held single-CTA 128 x 256 tiles at 1.77 PFLOP/s of E4M3.  Measured:
//    E4M3 3.0 PFLOP/s in a burst and 2.4 under the power cap (one matrix, 8192 x
//    5120 x 6144; the same rows in 8 groups: 2.5 and 2.15), MXFP4 4.9 and 4.2
//    (4096 x 16384 x 5120); both sit at 1,000 W with the SM clock at 1.1 - 1.4
//    GHz.
//    CTA 0 issues the MMAs.  The copies of both CTAs complete on its barriers
//    and its commits arrive at both CTAs, so no thread passes on what it has
//    waited for; CTA 1's scales, which threads store, are released to CTA 0 at
//    cluster scope.
//
// MXFP4 scales reach TMEM by tcgen05.cp in blocks of 128 rows x 4 scales
// (lane i, column j = row 32 j + i), the order in which they lie in memory.
// W row r is therefore always MMA row r % 128 (but in folded pieces): a stream
// piece never crosses a multiple of 128 rows, and its block is copied as it
// is.  X tiles start at any row; their scale words are gathered into the block
// order.
//
// A stage's W and X are one box each, [chunks of 128 B][rows][128 B]: a bulk
// copy costs its issuing thread ~90 cycles whatever its size (measured), so
// there is a tensor map for every height that a piece can have.  The MMA reads
// 128 W rows and whole columns of 16 whatever the piece holds: the lanes and
// columns of rows that are not the piece's come from whatever lies there and
// nobody reads them.
#pragma once

#include <algorithm>

#include "tinym_kernels.cuh"

namespace tinym {

constexpr int kGrpThreads = 256;     // warp 0 TMA, 1 MMA, 2-3 scales, 4-7 epilogue
constexpr int kGrpMaxExperts = 1024;
constexpr int kGrpBand = 8;          // row tiles walked together for each W tile (L2 reuse)
constexpr int kScaleBlock = 512;     // scale bytes of 128 rows x 4 scales
constexpr int kGrpBars = 5;          // barriers beside the two per stage
constexpr int kFoldOutBytes = kTileRows * 17 * 4;  // folded: FP32 sums of 128 MMA rows x 16 X rows
constexpr int kOutBytes = 32 * 64;   // an epilogue warp's output buffer: 32 X rows x 32 W rows
constexpr int kSfSlotCols = 32;      // TMEM columns of one chunk's scales (8 for W, 16 for X)

// Loads that stay behind the grid dependency wait: volatile, since the compiler
// may move others ahead of it.  Not .nc: the kernel before may still write
// what they read while this one already runs, which .nc does not allow.
__device__ __forceinline__ uint32_t ld_after_wait(const uint32_t* p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_after_wait(const uint8_t* p) {
    uint32_t v;
    asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint4 ld_after_wait(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}

// n / d for 0 <= n < 2^31: multiply by ceil(2^(31 + s) / d), 2^s >= d, and shift.
struct FastDiv {
    uint32_t mul, shift, d;
    __host__ static FastDiv make(uint32_t d) {
        uint32_t s = 0;
        while ((1ull << s) < d) ++s;
        return {static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d), 31 + s, d};
    }
    __host__ __device__ uint32_t div(uint32_t n) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift);
    }
};

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
    int32_t units;            // per X tile; stream: units of 8 W rows, or parts; pair: 256-row tiles
    int32_t part_units;       // stream: if non-zero, a block of 16 units is cut into parts of so many
    int32_t piece_units;      // stream: units per piece, at most
    int32_t blocked;          // stream: pieces stay inside 128-row blocks (MXFP4)
    int32_t stages;
    int32_t chunked;          // stream: one box covers a whole stage (K a multiple of 128 bytes)
    int32_t fold, fold_x;     // folded: segments of K, X rows of a segment's columns (8 or 16)
    int32_t w_stage, x_stage, sf_stage;  // bytes
    uint32_t w_off, sf_off, out_off, bar_off, tab_off;  // shared-memory offsets (X ring at 0)
    int32_t wide_y;           // Y takes 16-byte stores
    uint32_t tmem_cols, acc_cols, sf_col;
    FastDiv by_grid, by_units, by_band, by_parts, by_width[kGrpBand];  // walk: CTAs, units, 8 units, parts of a block, 1 .. 8
    int32_t cut_parts[kGrpBand], cut_units[kGrpBand];  // stream: CTAs, units per matrix of 1 .. 8
    uint32_t flags;
    uint32_t* err_host;
    uint64_t timeout_ns;
};
// Tensor maps: W in boxes of 8 (i + 1) rows, X in boxes of four heights.
struct GroupedMaps {
    CUtensorMap w[kTileRows / 8];
    CUtensorMap x[4];
    // stream, K no multiple of 128 bytes: boxes of one chunk for the last stage
    CUtensorMap w_tail[kTileRows / 8];
    CUtensorMap x_tail[4];
};
__host__ __device__ constexpr int grouped_x_box(bool pair, int i) { return (pair ? 16 : 8) << i; }
constexpr uint32_t kGrpZeroRest = 1u;  // rows of no group are written as zeros
// Self-test, so that the waits behind run out: copies or MMAs are not issued,
// or accumulators wait for one commit more than there is (a branch where the
// commits are issued cost MXFP4 pairs 1 %).
constexpr uint32_t kGrpNoLoads = 2u, kGrpNoMma = 4u, kGrpNoCommit = 8u;

constexpr int kBlockUnits = kTileRows / 8;  // 8-row units of a 128-row block

enum GroupedMode { kStream, kFold, kPair };
// 128-byte chunks of K in a stage: one for a pair's 512 cycles of MMAs, four
// where the bytes of W bind (two took 4-6 % longer on decode batches), two for
// the smallest calls, whose first MMA waits for a whole stage (four took 5 %
// longer at 1 x 5120 x 6144).
__host__ __device__ constexpr int grouped_chunks(GroupedMode m) {
    return m == kPair ? 1 : m == kFold ? 2 : 4;
}

// 128-row scale blocks of the X rows of a tile: stream tiles have at most 128 rows.
__host__ __device__ constexpr int grouped_x_scale_blocks(bool pair) { return pair ? 2 : 1; }

struct GroupedPiece {
    int e, row0, rows, w0, h;  // group, X rows, W rows (pair: of both CTAs)
};

// The pieces of one CTA, in the order in which every role walks them.
template <bool PAIR>
struct GroupedWalk {
    const GroupedParams& p;
    const int32_t* off;     // [experts + 1] group starts
    const int32_t* prefix;  // [experts + 1] X tiles before each group
    int cur, end, step;
    int e, tiles, wide;  // group, its X tiles, rows of each

    __host__ __device__ GroupedWalk(const GroupedParams& prm, const int32_t* o, const int32_t* pre,
                                    int block, int blocks)
        : p(prm), off(o), prefix(pre), e(-1), tiles(0), wide(0) {
        const int total = pre[p.experts] * p.units;  // below 2^31 (grouped_plan)
        if constexpr (PAIR) {
            cur = block;
            end = total;
            step = blocks;
        } else {
            // shares of total / blocks units, the first ones one more
            const int share = static_cast<int>(p.by_grid.div(total));
            const int more = total - share * blocks;
            cur = block * share + least(block, more);
            end = cur + share + (block < more ? 1 : 0);
            step = 0;
            // A share that crosses from one matrix to the next takes two passes
            // over K, and with shares below a piece those CTAs are the last to
            // finish: then every matrix is cut into the same number of parts,
            // a CTA each, unless that makes them half as large again (8
            // experts of 2048 x 4096 E4M3: 18.8 -> 14.9 us, the one shape that
            // the limit of a half was measured on).
            const int all = pre[p.experts];
            if (!p.blocked && !p.part_units && all > 1 && all <= blocks && share < p.piece_units) {
                const bool few = all <= kGrpBand;  // worked out by the host: divisions take a while
                const int parts = few ? p.cut_parts[all - 1] : blocks / all;
                const int least_units = few ? p.cut_units[all - 1] : p.units / parts;
                const int rest = p.units - least_units * parts;
                const int most = least_units + (rest ? 1 : 0);
                if (most <= p.piece_units && 2 * most <= 3 * (share + 1)) {
                    int m = 0;
                    if (few)
                        for (int j = 1; j <= kGrpBand; ++j) m += block >= j * parts ? 1 : 0;
                    else
                        m = block / parts;
                    const int i = block - m * parts;
                    cur = m < all ? m * p.units + i * least_units + least(i, rest) : 0;
                    end = m < all ? cur + least_units + (i < rest ? 1 : 0) : 0;
                }
            }
        }
    }

    __host__ __device__ static int least(int a, int b) { return a < b ? a : b; }

    // First unit of part i of a matrix.
    __host__ __device__ int part_unit(int i) const {
        const int block = static_cast<int>(p.by_parts.div(i));
        return block * kBlockUnits + (i - block * static_cast<int>(p.by_parts.d)) * p.part_units;
    }

    __host__ __device__ bool next(GroupedPiece* w) {
        if constexpr (!PAIR) {
            // parts past N in a matrix's last block
            while (p.part_units && cur < end &&
                   part_unit(cur - static_cast<int>(p.by_units.div(cur)) * p.units) * 8 >= p.n)
                ++cur;
        }
        if (cur >= end) return false;
        const int seg = static_cast<int>(p.by_units.div(cur));
        if (e < 0 || seg >= prefix[e + 1]) {
            int lo = e + 1, hi = p.experts - 1;  // the group whose tiles hold seg
            for (int i = 0; i < 2 && lo < hi && prefix[lo + 1] <= seg; ++i) ++lo;  // often the next
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (prefix[mid + 1] <= seg) lo = mid + 1;
                else hi = mid;
            }
            e = lo;
            // Equal tiles in whole steps of the MMA's columns: 300 rows are
            // 160 + 140, not 256 + 44.  (tiles - 1) * wide < count, since
            // wide <= tn.
            constexpr int kStep = PAIR ? 32 : 16;
            tiles = prefix[e + 1] - prefix[e];
            int count = off[e + 1] - off[e];
            if (tiles > 1) count = (count + tiles - 1) / tiles;
            wide = (count + kStep - 1) & ~(kStep - 1);
        }
        int t;
        if constexpr (PAIR) {
            const int local = cur - prefix[e] * p.units;
            const int band = static_cast<int>(p.by_band.div(local));
            const int width = least(kGrpBand, tiles - band * kGrpBand);
            const int rem = local - band * kGrpBand * p.units;
            const int wt = static_cast<int>(p.by_width[width - 1].div(rem));
            t = band * kGrpBand + rem - wt * width;
            w->w0 = wt * 2 * kTileRows;
            w->h = 2 * kTileRows;
            cur += step;
        } else {
            t = seg - prefix[e];
            int u = cur - seg * p.units, take;
            if (p.part_units) {
                u = part_unit(u);
                take = least(least(p.part_units, kBlockUnits - u % kBlockUnits), (p.n + 7) / 8 - u);
                ++cur;
            } else {
                int left = least(end - cur, p.units - u);
                if (p.blocked) left = least(left, kBlockUnits - u % kBlockUnits);
                take = left <= p.piece_units ? left
                       : left < 2 * p.piece_units ? (left + 1) / 2 : p.piece_units;
                cur += take;
            }
            w->w0 = u * 8;
            w->h = take * 8;
        }
        w->e = e;
        w->row0 = off[e] + t * wide;
        w->rows = least(wide, off[e + 1] - w->row0);
        return true;
    }
};

// A walk that works out the next piece ahead of time (a few
// hundred cycles of dependent steps), while a role has nothing urgent to do.
template <bool PAIR>
struct GroupedAhead {
    GroupedWalk<PAIR> walk;
    GroupedPiece nx;
    bool have, more;

    __device__ __forceinline__ GroupedAhead(const GroupedParams& p, const int32_t* o,
                                            const int32_t* pre, int block, int blocks)
        : walk(p, o, pre, block, blocks), have(false), more(false) {}
    __device__ __forceinline__ void ahead() {
        if (!have) more = walk.next(&nx);
        have = true;
    }
    __device__ __forceinline__ bool next(GroupedPiece* w) {
        ahead();
        have = false;
        *w = nx;
        return more;
    }
};

// How a call is cut.
struct GroupedPlan {
    GroupedMode mode;
    bool pair;  // mode == kPair
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
    // A pair takes 2 - 4 us longer (fewer CTAs, start and end), a stream plan reads
    // W once more for every 64 rows.  us in a graph, stream at 64 rows, then pair and
    // stream at 65 and at 256 (K = 6144): E4M3, N = 1024: 11.9, 16.2 and 18.5,
    // 20.1 and 34.6; N = 5120: 13.2, 16.9 and 24.7, 20.9 and 42.4; MXFP4, N =
    // 1024: 9.3, 11.5 and 13.8, 11.9 and 23.8; N = 5120: 10.1, 12.3 and 14.1,
    // 13.8 and 23.9.
    g.pair = avg > 64;
    g.mode = g.pair ? kPair : kStream;
    p.rows = static_cast<int32_t>(rows);
    p.experts = static_cast<int32_t>(experts);
    p.n = static_cast<int32_t>(n);
    p.k_bytes = static_cast<int32_t>(k_bytes);
    const int64_t k_chunks = (k_bytes + kBlockK - 1) / kBlockK;
    // Bytes in front of the W ring that an MMA may read: a piece that starts
    // inside a scale block stands that many rows into the MMA's rows.
    const uint32_t front = fp4 && !g.pair ? kTileRows * kBlockK : 0;
    if (g.pair) {
        p.units = static_cast<int32_t>((n + 2 * kTileRows - 1) / (2 * kTileRows));
        p.piece_units = kBlockUnits;
        // Two accumulators, so that a tile is stored while the next one is
        // computed; the scales take 64 of the 512 columns.  (Two of 256 that
        // share 64 columns cost ~2,600 cycles a tile until those are free.)
        p.tn = fp4 ? 224 : 256;
        p.acc_cols = static_cast<uint32_t>(p.tn);
        p.x_stage = kTileRows * kBlockK;
        p.sf_col = 448;
        p.tmem_cols = 512;
    } else {
        // Room for a group of three times the average; a single group is known.
        p.tn = static_cast<int32_t>(std::min<int64_t>(64, ((experts == 1 ? 1 : 3) * avg + 15) / 16 * 16));
        const int64_t n_units = (n + 7) / 8, blocks = (n_units + kBlockUnits - 1) / kBlockUnits;
        p.units = static_cast<int32_t>(n_units);
        p.blocked = fp4 ? 1 : 0;
        p.chunked = k_bytes % kBlockK == 0;
        // Units of a CTA: a share of them all, or of one of equal parts of a matrix.
        const int64_t parts = std::max<int64_t>(1, sm_count / groups);
        const int64_t share = std::max((groups * n_units + sm_count - 1) / sm_count,
                                       std::min<int64_t>(kBlockUnits, (n_units + parts - 1) / parts));
        if (p.tn == 16 && p.chunked && share <= kBlockUnits / 2) {
            // The most segments that divide K's chunks, fit 128 MMA rows and
            // keep the MMA at 64 columns (where its time starts to grow).
            p.fold_x = rows <= 8 ? 8 : 16;
            for (int s = 2; s * share <= kBlockUnits && s * p.fold_x <= 64; ++s)
                if (k_chunks % s == 0) p.fold = s;
        }
        if (p.fold) {
            g.mode = kFold;
            p.blocked = 0;
            p.piece_units = static_cast<int32_t>(share);
        } else if (fp4 && groups * blocks < sm_count) {
            // Less than a block per SM: equal parts of a block, one piece each
            // (a share that crosses a block would take two passes over K).
            const int per = static_cast<int>(std::min<int64_t>(kBlockUnits, sm_count / (groups * blocks)));
            p.part_units = (kBlockUnits + per - 1) / per;
            p.units = static_cast<int32_t>(blocks * ((kBlockUnits + p.part_units - 1) / p.part_units));
            p.piece_units = p.part_units;
        } else {
            p.piece_units = static_cast<int32_t>(fp4 ? kBlockUnits : std::min<int64_t>(kBlockUnits, share));
        }
        int x_rows = 8;
        while (x_rows < p.tn) x_rows *= 2;
        p.acc_cols = static_cast<uint32_t>(p.tn);
        if (p.fold) {
            x_rows = p.fold * p.fold_x;
            p.acc_cols = static_cast<uint32_t>((x_rows + 15) / 16 * 16);
        }
        p.x_stage = x_rows * grouped_chunks(g.mode) * kBlockK;
        p.sf_col = 2 * p.acc_cols;
        p.tmem_cols = 32;
        while (p.tmem_cols < 2 * p.acc_cols + (fp4 ? 2 * kSfSlotCols : 0)) p.tmem_cols *= 2;
    }
    p.by_units = FastDiv::make(static_cast<uint32_t>(p.units));
    p.by_band = FastDiv::make(static_cast<uint32_t>(kGrpBand * p.units));
    p.by_parts = FastDiv::make(static_cast<uint32_t>(
        p.part_units ? (kBlockUnits + p.part_units - 1) / p.part_units : 1));
    for (int i = 0; i < kGrpBand; ++i) p.by_width[i] = FastDiv::make(static_cast<uint32_t>(i + 1));
    const int chunks = grouped_chunks(g.mode);
    p.w_stage = std::max(1, p.fold) * p.piece_units * chunks * 1024;
    if (fp4) p.sf_stage = chunks * 2 * (1 + grouped_x_scale_blocks(g.pair)) * kScaleBlock;
    const int64_t max_items = (groups + rows / p.tn) * p.units;
    if (max_items > (int64_t(1) << 31) - (int64_t(1) << 20)) return "too many tiles";
    g.grid = static_cast<int>(g.pair ? 2 * std::min<int64_t>(sm_count / 2, max_items)
                                     : std::min<int64_t>(sm_count, max_items));

    p.by_grid = FastDiv::make(static_cast<uint32_t>(g.grid));
    for (int i = 0; i < kGrpBand; ++i) {
        p.cut_parts[i] = std::max(1, g.grid / (i + 1));
        p.cut_units[i] = p.units / p.cut_parts[i];
    }
    const uint32_t tables = 8u * static_cast<uint32_t>(experts + 1);
    auto bytes_for = [&](int stages) -> uint32_t {
        p.stages = stages;
        p.sf_off = static_cast<uint32_t>(stages * p.x_stage);
        p.w_off = p.sf_off + static_cast<uint32_t>(stages * p.sf_stage);
        p.w_off = (std::max(p.w_off, front) + 1023u) & ~1023u;
        p.out_off = p.w_off + static_cast<uint32_t>(stages * p.w_stage);
        p.bar_off = p.out_off + (p.fold ? kFoldOutBytes : 4 * kOutBytes);
        p.tab_off = p.bar_off + 8u * (2 * stages + kGrpBars) + 16u;
        // The MMA's 128 W rows of the last chunk end inside the allocation.
        const uint32_t read_end = p.w_off + static_cast<uint32_t>(stages * p.w_stage) + kTileRows * kBlockK;
        return std::max(p.tab_off + tables, g.pair ? 0u : read_end) + 1024u;
    };
    const int64_t seg_chunks = k_chunks / std::max(1, p.fold);
    const int64_t nkb = (seg_chunks + chunks - 1) / chunks;
    int stages = static_cast<int>(std::max<int64_t>(2, std::min<int64_t>(12, 2 * nkb)));
    while (stages >= 2 && bytes_for(stages) > smem_limit) --stages;
    if (stages < 2) return "no two stages fit";
    g.smem = bytes_for(stages);
    // A pair wants 512 columns of tensor memory in two SMs at once.  Its CTAs
    // take all shared memory and so are alone on their SMs: nothing else holds
    // columns there, where two kernels with one SM each would wait for good.
    if (g.pair) g.smem = smem_limit;
    *out = g;
    return nullptr;
}

// Unswizzled 32 rows x 16 bytes (a scale block): 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
    return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) |
           (static_cast<uint64_t>(128u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46);
}

// tcgen05 operations of one CTA, or of both CTAs of a pair.
template <int CTAS>
struct Tc;
#define TINYM_TC_OPS(G)                                                                            \
    template <>                                                                                    \
    struct Tc<G> {                                                                                 \
        /* 512-byte scale block to 4 TMEM columns, repeated in the four 32-lane subpartitions: */  \
        /* lane i, column j gets the four scales of row 32 j + i. */                               \
        __device__ __forceinline__ static void cp_scales(uint32_t taddr, uint64_t desc) {          \
            asm volatile("tcgen05.cp.cta_group::" #G ".32x128b.warpx4 [%0], %1;" ::"r"(taddr),     \
                         "l"(desc)                                                                 \
                         : "memory");                                                              \
        }                                                                                          \
        __device__ __forceinline__ static void mma_e4m3(uint32_t d, uint64_t a, uint64_t b,        \
                                                        uint32_t idesc, uint32_t accumulate) {     \
            asm volatile(                                                                          \
                "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                                 \
                "tcgen05.mma.cta_group::" #G ".kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), \
                "l"(a), "l"(b), "r"(idesc), "r"(accumulate)                                        \
                : "memory");                                                                       \
        }                                                                                          \
        __device__ __forceinline__ static void mma_mxf4(uint32_t d, uint64_t a, uint64_t b,        \
                                                        uint32_t idesc, uint32_t sfa, uint32_t sfb, \
                                                        uint32_t accumulate) {                     \
            asm volatile(                                                                          \
                "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                 \
                "tcgen05.mma.cta_group::" #G                                                       \
                ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::  \
                    "r"(d),                                                                        \
                "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                    \
                : "memory");                                                                       \
        }                                                                                          \
        __device__ __forceinline__ static void commit(uint32_t bar) {                              \
            asm volatile("tcgen05.commit.cta_group::" #G                                           \
                         ".mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)             \
                         : "memory");                                                              \
        }                                                                                          \
        __device__ __forceinline__ static void alloc(uint32_t dst, uint32_t ncols) {               \
            asm volatile("tcgen05.alloc.cta_group::" #G                                            \
                         ".sync.aligned.shared::cta.b32 [%0], %1;\n\t"                             \
                         "tcgen05.relinquish_alloc_permit.cta_group::" #G ".sync.aligned;" ::"r"(dst), \
                         "r"(ncols)                                                                \
                         : "memory");                                                              \
        }                                                                                          \
        __device__ __forceinline__ static void dealloc(uint32_t taddr, uint32_t ncols) {           \
            asm volatile("tcgen05.dealloc.cta_group::" #G ".sync.aligned.b32 %0, %1;" ::"r"(taddr), \
                         "r"(ncols)                                                                \
                         : "memory");                                                              \
        }                                                                                          \
    };
TINYM_TC_OPS(1)
TINYM_TC_OPS(2)
#undef TINYM_TC_OPS

// Instruction descriptor of kind::mxf4: A = B = E2M1 (1) at [7,10) and
// [10,13), N >> 3 at [17,23), E8M0 scales (1) at 23, M >> 7 at [27,29).
// The scale ids (byte pair of the 32-bit scale word: 0 or 2) go to [4,6) for
// B and [29,31) for A.
__host__ __device__ constexpr uint32_t idesc_mxf4(int mma_m, int mma_n) {
    return (1u << 7) | (1u << 10) | (static_cast<uint32_t>(mma_n >> 3) << 17) | (1u << 23) |
           (static_cast<uint32_t>(mma_m >> 7) << 27);
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

// Arrive on a barrier of another CTA of the cluster (a cluster address): what
// this CTA's threads stored in its shared memory, up to here, is ordered at
// cluster scope before what the other CTA does behind its wait.  Nothing else
// is announced this way, so the release is restricted to shared memory: one of
// all memory takes more than two stages' MMAs (MXFP4, 4096 x 16384 x 5120:
// 253 us).
__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_bar) {
    asm volatile(
        "fence.release.sync_restrict::shared::cta.cluster;\n\t"
        "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar)
        : "memory");
}

// 3-D tiled copy of one CTA of a pair to its own shared memory; its bytes are
// completed on `bar`, a barrier of either CTA (a cluster address).
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                                 int32_t c0, int32_t c1, int32_t c2, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
        ".L2::cache_hint [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
        : "memory");
}

// Bounded wait of a whole warp: no lane diverges and the outcome is uniform.
// CLUSTER: other CTAs of the cluster arrive on the barrier.  The clock that
// bounds it is first read after many tries: a read of %globaltimer costs
// several hundred cycles even where its value is not used.
template <bool CLUSTER>
__device__ __forceinline__ bool warp_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    if constexpr (CLUSTER) {
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}\n"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
    } else {
        ok = mbar_try_wait(bar, parity) ? 1u : 0u;
    }
    return __all_sync(0xFFFFFFFFu, ok);
}
// Called now and then while a wait lasts; false: give up.
__device__ __noinline__ bool warp_wait_tick(uint64_t* t0, const WaitGuard& g, uint32_t code) {
    if (__any_sync(0xFFFFFFFFu, *g.abort)) return false;
    const uint64_t t = __shfl_sync(0xFFFFFFFFu, globaltimer_ns(), 0);
    if (*t0 == 0) *t0 = t;
    if (t - *t0 <= g.timeout_ns) return true;
    *g.abort = 1u;
    if ((threadIdx.x & 31) == 0) report_timeout(g.err_word, g.err_host, code);
    return false;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const WaitGuard& g,
                                          uint32_t code) {
    uint64_t t0 = 0;
    for (uint32_t it = 1; !warp_try<CLUSTER>(bar, parity); ++it)
        if ((it & 255u) == 0 && !warp_wait_tick(&t0, g, code)) return false;
    return true;
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int32_t c0, int32_t c1, int32_t c2, int32_t c3, int32_t c4,
                                            uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4, %5, %6, %7}], [%2], %8;" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4),
        "l"(policy)
        : "memory");
}

// Whether `ok` holds in all 128 epilogue threads (named barrier 1).
__device__ __forceinline__ bool epilogue_all(bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}\n"
        : "=r"(all)
        : "r"(ok ? 1u : 0u)
        : "memory");
    return all != 0;
}

// A lane's 16 bytes of the scale blocks of one pair stage.
struct ScaleRegs {
    uint4 w[2], x[2][3];
    int rot, block;
    bool valid;
};
// Words rot .. rot + 3 of the eight words a, b (rot <= 4).
__device__ __forceinline__ uint4 rotate_words(const uint4& a, const uint4& b, int rot) {
    uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 4; k >= 1; k /= 2)
#pragma unroll
        for (int j = 0; j + k < 8; ++j) v[j] = rot & k ? v[j + k] : v[j];
    return make_uint4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void sts_masked(uint32_t dst, const uint4& v, uint32_t mask) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x & mask),
                 "r"(v.y & mask), "r"(v.z & mask), "r"(v.w & mask)
                 : "memory");
}
// 16 lanes x 16 columns as the fragments of 8 x 8 matrices: for columns 8 j ..
// r[4 j], r[4 j + 1] are lane t / 4, columns 2 (t % 4) and + 1, the next two
// lane t / 4 + 8.
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7])
        : "r"(taddr));
}
// Four 8 x 8 matrices of 16-bit values, transposed, to the row addresses that
// lanes 0-7, 8-15, 16-23 and 24-31 give.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c,
                                                  uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr),
                 "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(uint32_t lo, uint32_t hi, float alpha) {
    const __nv_bfloat162 h =
        __floats2bfloat162_rn(__uint_as_float(lo) * alpha, __uint_as_float(hi) * alpha);
    return *reinterpret_cast<const uint32_t*>(&h);
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
        int v = i <= p.experts ? min(max(static_cast<int>(ld_after_wait(reinterpret_cast<const uint32_t*>(p.offsets + i))), 0), p.rows) : 0;
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

template <bool FP4, GroupedMode MODE>
__global__ void __launch_bounds__(kGrpThreads, 1)
    tinym_grouped_kernel(const __grid_constant__ GroupedMaps maps, const GroupedParams p) {
    constexpr bool PAIR = MODE == kPair, FOLD = MODE == kFold;
    using Ops = Tc<PAIR ? 2 : 1>;
    constexpr int kCtas = PAIR ? 2 : 1;
    constexpr int kChunks = grouped_chunks(MODE);  // 128-byte chunks of K per stage
    constexpr int kMmaK = 32;              // bytes of K per MMA (32 E4M3 or 64 E2M1 elements)
    constexpr int kSfPerChunk = 2;         // MXFP4: scale blocks (128 elements) per chunk
    constexpr int kXsBlocks = grouped_x_scale_blocks(PAIR);
    constexpr int kWsBytes = kChunks * kSfPerChunk * kScaleBlock;  // W scales of a stage

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = align1024(smem_raw);
    const uint32_t s_base = smem_u32(smem);
    const int stages = p.stages;
    const uint32_t x_ring = s_base;
    const uint32_t sf_ring = s_base + p.sf_off;
    const uint32_t w_ring = s_base + p.w_off;
    const uint32_t bars = s_base + p.bar_off;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (stages + s); };
    auto acc_full = [&](int b) { return bars + 8u * (2 * stages + b); };
    auto acc_empty = [&](int b) { return bars + 8u * (2 * stages + 2 + b); };
    const uint32_t drain_bar = bars + 8u * (2 * stages + 4);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + p.bar_off + 8u * (2 * stages + kGrpBars));
    volatile uint32_t* abort_flag = tmem_slot + 1;
    // Pair, written by the other CTA: at CTA 0 the stages that CTA 1 has
    // issued, at CTA 1 whether CTA 0 has given up.
    volatile uint32_t* peer = tmem_slot + 2;
    int32_t* off = reinterpret_cast<int32_t*>(smem + p.tab_off);
    int32_t* prefix = off + p.experts + 1;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int rank = PAIR ? static_cast<int>(cluster_ctarank()) : 0;  // 0 issues the pair's MMAs
    const WaitGuard guard{abort_flag, &g_err_word, p.timeout_ns, p.err_host};
    // of K, or of a segment of it
    const int k_chunks = FOLD ? p.k_bytes / kBlockK / p.fold : (p.k_bytes + kBlockK - 1) / kBlockK;
    const int nkb = (k_chunks + kChunks - 1) / kChunks;
    auto at_rank = [&](uint32_t addr, int r) { return PAIR ? dsmem_map(addr, r) : addr; };

    if (warp == 3) {
        // What the producer will need first: the maps that the first stage is
        // likely to use, and the parameters (a miss of the constant cache
        // costs some hundred cycles, and the walk would take them one by one).
        if (lane == 0) {
            tma_prefetch_desc(&maps.w[p.piece_units - 1]);
            tma_prefetch_desc(&maps.x[0]);
        }
        asm volatile("" ::"r"(p.rows), "r"(p.units), "r"(p.stages), "r"(p.sf_off), "r"(p.by_grid.mul),
                     "r"(p.by_band.mul), "r"(p.by_width[2].mul), "r"(p.by_width[7].mul), "r"(p.flags)
                     : "memory");
    }
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            // full: the producer's expect_tx (and the bytes), the scales.  A
            // pair uses that of CTA 0, for both CTAs' bytes and scales.
            mbar_init(full_bar(s), 1 + (FP4 ? kCtas : 0));
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full(b), p.flags & kGrpNoCommit ? 2 : 1);
            mbar_init(acc_empty(b), 4 * kCtas);  // one arrival per epilogue warp
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0u;
        *peer = 0u;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    // Everything above overlaps the previous kernel's tail (programmatic
    // dependent launch); no global memory is read before it has completed.
    grid_dependency_wait();
    if (warp == 1) {
        // Tensor memory is taken behind that wait, and the next kernel may
        // start only when it has been: a CTA that held some while it waits
        // for the grid before, beside one of that grid that waits for some,
        // would wait for good.
        Ops::alloc(smem_u32(tmem_slot), p.tmem_cols);
        grid_launch_dependents();
    }
    if (warp == 0) grouped_tables(p, off, prefix, lane);
    uint32_t tmem = 0u;
    if constexpr (PAIR) {
        tc_fence_before_sync();
        __syncthreads();
        // the other CTA's barriers exist before anything arrives on them
        cluster_arrive_release();
        cluster_wait_acquire();
        tc_fence_after_sync();
        tmem = *tmem_slot;
    } else if (warp == 0) {
        // The producer made the barriers and the tables itself: it loads the
        // first stages while the others come to the barrier.
        __syncwarp();
        asm volatile("barrier.cta.arrive 2, 256;" ::: "memory");
    } else {
        tc_fence_before_sync();
        asm volatile("barrier.cta.sync 2, 256;" ::: "memory");
        tc_fence_after_sync();
        tmem = *tmem_slot;
    }

    GroupedAhead<PAIR> walk(p, off, prefix, blockIdx.x / kCtas, gridDim.x / kCtas);
    GroupedPiece w;
    // MMA row of a stream piece's first W row (0 unless scales are blocked).
    auto first_row = [&]() { return MODE == kStream && FP4 ? w.w0 % kTileRows : 0; };
    // X rows that this CTA loads, and the box that holds them.
    auto x_cols = [&]() { return PAIR ? ((w.rows + 31) & ~31) / 2 : FOLD ? p.fold_x : w.rows; };
    auto x_box = [&](int cols) {
        return 32 - __clz((cols - 1) / grouped_x_box(PAIR, 0));  // log2 of the boxes of 8 or 16, rounded up
    };
    const int segs = FOLD ? p.fold : 1;
    int issued = 0;  // producer: stages

    if (warp == 0) {
        // ---------------- TMA producer (the whole warp walks, one lane issues)
        const uint64_t pol_w = PAIR ? l2_policy_evict_normal() : l2_policy_w();
        const uint64_t pol_x = l2_policy_evict_last();
        int s = 0;
        uint32_t ph = 1u;  // the first pass over the ring does not wait
        bool ok = !(p.flags & kGrpNoLoads);
        while (ok && walk.next(&w)) {
            const int cols = x_cols();
            const int xi = x_box(cols);
            const int x_rows = grouped_x_box(PAIR, xi);
            const int x_row = w.row0 + rank * cols;
            const int w_rows = PAIR ? kTileRows : w.h;
            const int w_row = w.w0 + rank * kTileRows;
            const CUtensorMap* mw = &maps.w[w_rows / 8 - 1];
            const CUtensorMap* mx = &maps.x[xi];
            for (int i = 0; i < nkb; ++i) {
                if (issued >= stages &&
                    !(ok = warp_wait<PAIR>(empty_bar(s), ph, guard, kErrProducerWait)))
                    break;
                const uint32_t wd = w_ring + s * p.w_stage, xd = x_ring + s * p.x_stage;
                const uint32_t bar = full_bar(s);
                const int c0 = i * kChunks;
                if (elect_one()) {
                    if constexpr (PAIR) {
                        // Both CTAs' copies complete on CTA 0's barrier, which
                        // may get CTA 1's bytes ahead of its own expect_tx.
                        const uint32_t pair_bar = at_rank(bar, 0);
                        if (rank == 0) mbar_expect_tx(bar, kCtas * (kTileRows + x_rows) * kBlockK);
                        tma_load_3d_pair(wd, mw, pair_bar, c0 * kBlockK, w_row, w.e, pol_w);
                        tma_load_3d_pair(xd, mx, pair_bar, c0 * kBlockK, x_row, 0, pol_x);
                    } else if constexpr (FOLD) {
                        mbar_expect_tx(bar, segs * (w_rows + x_rows) * kChunks * kBlockK);
                        tma_load_5d(wd, mw, bar, 0, w_row, 0, c0, w.e, pol_w);
                        tma_load_4d(xd, mx, bar, 0, x_row, 0, c0, pol_x);
                    } else if (p.chunked || i < nkb - 1) {
                        mbar_expect_tx(bar, (w_rows + x_rows) * kChunks * kBlockK);
                        tma_load_4d(wd, mw, bar, 0, w_row, c0, w.e, pol_w);
                        tma_load_4d(xd, mx, bar, 0, x_row, c0, 0, pol_x);
                    } else {
                        // K ends inside a chunk: the last stage's boxes are chunks
                        const int nc = min(kChunks, k_chunks - c0);
                        const CUtensorMap* tw = &maps.w_tail[w_rows / 8 - 1];
                        mbar_expect_tx(bar, (w_rows + x_rows) * nc * kBlockK);
                        for (int c = 0; c < nc; ++c) {
                            tma_load_3d(wd + c * w_rows * kBlockK, tw, bar, (c0 + c) * kBlockK, w_row,
                                        w.e, pol_w);
                            tma_load_3d(xd + c * x_rows * kBlockK, &maps.x_tail[xi], bar, (c0 + c) * kBlockK,
                                        x_row, 0, pol_x);
                        }
                    }
                }
                __syncwarp();
                if (i == 0) walk.ahead();
                ++issued;
                if (++s == stages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        }
        // CTA 0's commits arrive at CTA 1's slots: it stays until the last has.
        if (rank)
            for (int j = 0; ok && j < stages; ++j) {
                ok = warp_wait<PAIR>(empty_bar(s), ph, guard, kErrProducerWait);
                if (++s == stages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
        if (rank && lane == 0) dsmem_st_u32(at_rank(smem_u32(tmem_slot + 2), 0), issued);
    } else if (warp == 1) {
        // ---------------- MMA issuer (the whole warp walks, one lane issues)
        if (rank == 0) {
            const uint32_t tmem_u = __shfl_sync(0xFFFFFFFFu, tmem, 0);
            const uint64_t da0 = sw128_kmajor_desc(w_ring);
            const uint64_t db0 = sw128_kmajor_desc(x_ring);
            int s = 0, piece = 0, slot = 0;
            uint32_t ph = 0u;
            bool ok = !(p.flags & kGrpNoMma);
            while (ok && walk.next(&w)) {
                const int b = piece & 1;
                const uint32_t mma_n = PAIR ? (w.rows + 31) & ~31
                                            : ((FOLD ? segs * p.fold_x : w.rows) + 15) & ~15;
                const uint32_t idesc = FP4 ? idesc_mxf4(kCtas * 128, mma_n)
                                           : idesc_e4m3_f32(kCtas * 128, mma_n);
                const uint32_t acc = tmem_u + b * p.acc_cols;
                const bool two = PAIR && mma_n > 128;  // X scale blocks of the tile
                if (!(ok = warp_wait<PAIR>(acc_empty(b), ((piece >> 1) & 1) ^ 1u, guard, kErrMmaWait)))
                    break;
                tc_fence_after_sync();
                // Bytes from chunk to chunk of a stage, and of the rows that
                // stand in front of a blocked piece's first one.
                const int w_chunk = segs * (PAIR ? kTileRows : w.h) * kBlockK;
                const int x_chunk = segs * grouped_x_box(PAIR, x_box(x_cols())) * kBlockK;
                const uint64_t da1 = da0 - static_cast<uint64_t>((first_row() * kBlockK) >> 4);
                for (int i = 0; i < nkb; ++i) {
                    if (!(ok = warp_wait<PAIR>(full_bar(s), ph, guard, kErrMmaWait))) break;
                    tc_fence_after_sync();
                    const uint64_t da = da1 + static_cast<uint64_t>((s * p.w_stage) >> 4);
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
#pragma unroll
                                for (int q = 0; q < kSfPerChunk; ++q) {
                                    const int blk = c * kSfPerChunk + q;
                                    const uint32_t xs = sf + kWsBytes + blk * kXsBlocks * kScaleBlock;
                                    Ops::cp_scales(sfa + 4 * q, scale_desc(sf + blk * kScaleBlock));
                                    Ops::cp_scales(sfb + 8 * q, scale_desc(xs));
                                    if (PAIR && two)
                                        Ops::cp_scales(sfb + 8 * q + 4, scale_desc(xs + kScaleBlock));
                                }
                            }
#pragma unroll
                            for (int kk = 0; kk < kBlockK / kMmaK; ++kk) {
                                const uint64_t ak = da + static_cast<uint64_t>((c * w_chunk + kk * kMmaK) >> 4);
                                const uint64_t bk = db + static_cast<uint64_t>((c * x_chunk + kk * kMmaK) >> 4);
                                const uint32_t accumulate = (i | c | kk) ? 1u : 0u;
                                if constexpr (FP4) {
                                    // 64 elements: scales 2 (kk % 2), +1 of block kk / 2
                                    const uint32_t id = (kk & 1) * 2;
                                    Ops::mma_mxf4(acc, ak, bk, idesc | (id << 4) | (id << 29),
                                                  sfa + 4 * (kk >> 1), sfb + 8 * (kk >> 1), accumulate);
                                } else {
                                    Ops::mma_e4m3(acc, ak, bk, idesc, accumulate);
                                }
                            }
                        }
                        // both CTAs of a pair wait for the MMAs
#pragma unroll
                        for (int r = 0; r < kCtas; ++r) {
                            Ops::commit(r ? at_rank(empty_bar(s), r) : empty_bar(s));
                            if (i == nkb - 1) Ops::commit(r ? at_rank(acc_full(b), r) : acc_full(b));
                        }
                    }
                    __syncwarp();
                    if (i == 0) walk.ahead();
                    slot += kChunks;
                    if (++s == stages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                ++piece;
            }
        }
    } else if (warp < 4) {
        // ---------------- MXFP4 scales
        const int blocks = (p.k_bytes * 2 + 127) / 128;  // scale blocks along K
        const int tail = (p.k_bytes * 2 % 128) / 32;     // scales in the last one, 0: all
        const uint32_t tail_mask = tail ? (1u << (8 * tail)) - 1u : 0xFFFFFFFFu;
        // Scales past K become 2^-127 (the data there are zeros).
        auto block_mask = [&](int b) {
            return b < blocks - 1 ? 0xFFFFFFFFu : b < blocks ? tail_mask : 0u;
        };
        if constexpr (FP4 && PAIR) {
            // Warps 2 and 3 take alternate stages, each with the scales of its
            // next two in registers: a stage's are stored when its slot is
            // free, and those of four stages later loaded.  A W block is
            // stored as it is.  An X tile that starts at row r0 of the blocks
            // needs from lane i the words of rows r0 + 32 j + i: those of
            // block row (i + r0) % 32, rotated, from two or three blocks.
            // (Words copied one by one, by cp.async, took ~900 cycles a stage.)
            ScaleRegs ra, rb;
            const uint8_t *ws = nullptr, *xs[3] = {nullptr, nullptr, nullptr};
            int i = warp - 2, rot = 0;
            auto enter = [&]() {  // a piece
                const int w0 = min(w.w0 + rank * kTileRows, p.n - 1);
                ws = p.w_scales + w.e * p.w_scale_stride +
                     static_cast<int64_t>(w0 >> 7) * blocks * kScaleBlock + lane * 16;
                const int first = w.row0 >> 7, last = (w.row0 + w.rows - 1) >> 7;
                const int src = lane + (w.row0 & 31);
                rot = ((w.row0 & 127) >> 5) + (src >> 5);
#pragma unroll
                for (int j = 0; j < 3; ++j)
                    xs[j] = p.x_scales + static_cast<int64_t>(min(first + j, last)) * blocks * kScaleBlock +
                            (src & 31) * 16;
            };
            auto load = [&](ScaleRegs* r) {
                r->rot = rot;
                r->block = i * kSfPerChunk;
#pragma unroll
                for (int q = 0; q < kSfPerChunk; ++q) {
                    const int64_t at = static_cast<int64_t>(min(r->block + q, blocks - 1)) * kScaleBlock;
                    r->w[q] = ld_after_wait(reinterpret_cast<const uint4*>(ws + at));
#pragma unroll
                    for (int j = 0; j < 3; ++j)
                        r->x[q][j] = ld_after_wait(reinterpret_cast<const uint4*>(xs[j] + at));
                }
            };
            bool more = walk.next(&w);
            if (more) enter();
            auto fetch = [&](ScaleRegs* r) {  // this warp's next stage, if there is one
                while (more && i >= nkb) {
                    i -= nkb;
                    if ((more = walk.next(&w))) enter();
                }
                r->valid = more;
                if (more) load(r);
                i += 2;
            };
            fetch(&ra);
            fetch(&rb);
            int s = warp - 2;
            uint32_t ph = 1u;
            auto step = [&](ScaleRegs& r) {
                if (!r.valid || !warp_wait<true>(empty_bar(s), ph, guard, kErrProducerWait)) return false;
                const uint32_t wd = sf_ring + s * p.sf_stage + lane * 16;
                const uint32_t xd = wd + kWsBytes;
#pragma unroll
                for (int q = 0; q < kSfPerChunk; ++q) {
                    const uint32_t mask = block_mask(r.block + q);
                    sts_masked(wd + q * kScaleBlock, r.w[q], mask);
                    sts_masked(xd + q * kXsBlocks * kScaleBlock,
                               rotate_words(r.x[q][0], r.x[q][1], r.rot), mask);
                    sts_masked(xd + (q * kXsBlocks + 1) * kScaleBlock,
                               rotate_words(r.x[q][1], r.x[q][2], r.rot), mask);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (elect_one()) {
                    if (rank) mbar_arrive_remote(at_rank(full_bar(s), 0));
                    else mbar_arrive(full_bar(s));
                }
                __syncwarp();
                if ((s += 2) >= stages) {
                    s -= stages;
                    ph ^= 1u;
                }
                fetch(&r);
                return true;
            };
            while (step(ra) && step(rb)) {
            }
        }
        if constexpr (FP4 && !PAIR) {
            // Warps 2 and 3 take alternate stages, each with the scales of its
            // next one in registers.  X words, and folded the W words of every
            // MMA row (W row r of segment a), are gathered one by one; else a
            // W block is stored as it is.  (4-byte cp.async took ~50 cycles
            // each: 0.7 us a stage of 32 X rows or more.)
            constexpr int kBlocks = kChunks * kSfPerChunk;
            const int seg_blocks = blocks / segs;
            uint32_t v[kBlocks][6];
            const uint8_t* ws[FOLD ? 4 : 1] = {};
            const uint8_t* xs[2] = {};
            int i = warp - 2, first = 0;
            // The scale word of 128-column group 0 of row r (of a segment).
            auto word_at = [&](const uint8_t* base, int r, int a) {
                return base + (static_cast<int64_t>(r >> 7) * blocks + a * seg_blocks) * kScaleBlock +
                       (r & 31) * 16 + ((r >> 5) & 3) * 4;
            };
            auto enter = [&]() {  // a piece
                const uint8_t* base = p.w_scales + w.e * p.w_scale_stride;
                if constexpr (FOLD) {
                    const uint32_t by_h = (65536u + w.h - 1) / w.h;  // exact quotients below 128
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int m = j * 32 + lane, a = static_cast<int>((m * by_h) >> 16);
                        ws[j] = word_at(base, min(w.w0 + m - a * w.h, p.n - 1), a < segs ? a : 0);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int c = j * 32 + lane, a = c / (p.fold_x == 8 ? 8 : 16);
                        xs[j] = word_at(p.x_scales, w.row0 + min(c - a * p.fold_x, w.rows - 1),
                                        a < segs ? a : 0);
                    }
                } else {
                    ws[0] = base + static_cast<int64_t>(w.w0 >> 7) * blocks * kScaleBlock + lane * 16;
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        xs[j] = word_at(p.x_scales, w.row0 + min(j * 32 + lane, w.rows - 1), 0);
                }
            };
            bool more = walk.next(&w);
            if (more) enter();
            auto fetch = [&]() {  // this warp's next stage, if there is one
                while (more && i >= nkb) {
                    i -= nkb;
                    if ((more = walk.next(&w))) enter();
                }
                if (!more) return;
                first = i * kBlocks;
                i += 2;
#pragma unroll
                for (int q = 0; q < kBlocks; ++q) {
                    const int64_t at = static_cast<int64_t>(min(first + q, seg_blocks - 1)) * kScaleBlock;
                    if constexpr (FOLD) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            v[q][j] = ld_after_wait(reinterpret_cast<const uint32_t*>(ws[j] + at));
                    } else {
                        const uint4 o = ld_after_wait(reinterpret_cast<const uint4*>(ws[0] + at));
                        v[q][0] = o.x, v[q][1] = o.y, v[q][2] = o.z, v[q][3] = o.w;
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        v[q][4 + j] = ld_after_wait(reinterpret_cast<const uint32_t*>(xs[j] + at));
                }
            };
            fetch();
            int s = warp - 2;
            uint32_t ph = 1u;
            while (more) {
                if (!warp_wait(empty_bar(s), ph, guard, kErrProducerWait)) break;
                const uint32_t wd = sf_ring + s * p.sf_stage + lane * 16;
#pragma unroll
                for (int q = 0; q < kBlocks; ++q) {
                    const uint32_t mask = FOLD ? 0xFFFFFFFFu : block_mask(first + q);
                    sts_masked(wd + q * kScaleBlock, make_uint4(v[q][0], v[q][1], v[q][2], v[q][3]), mask);
                    sts_masked(wd + kWsBytes + q * kScaleBlock, make_uint4(v[q][4], v[q][5], 0u, 0u), mask);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (elect_one()) mbar_arrive(full_bar(s));
                __syncwarp();
                if ((s += 2) >= stages) {
                    s -= stages;
                    ph ^= 1u;
                }
                fetch();
            }
        }
    } else {
        // ---------------- epilogue: warp w reads TMEM lanes 32 (w % 4) ..
        const int q = warp & 3;
        int piece = 0;
        while (walk.next(&w)) {
            const int b = piece & 1;
            // ahead of the wait, so that its latency is hidden
            float alpha = 1.0f;
            if (p.alpha)
                asm volatile("ld.global.f32 %0, [%1];" : "=f"(alpha) : "l"(p.alpha + w.e * p.alpha_stride) : "memory");
            walk.ahead();
            bool ready = warp_wait<PAIR>(acc_full(b), (piece >> 1) & 1, guard, kErrEpilogueWait);
            if constexpr (FOLD) ready = epilogue_all(ready);  // the warps meet below: all or none
            if (!ready) break;
            tc_fence_after_sync();
            const uint32_t taddr = tmem + b * p.acc_cols + (static_cast<uint32_t>(q * 32) << 16);
            __nv_bfloat16* row0 = p.y + static_cast<int64_t>(w.row0) * p.ldy;
            if constexpr (FOLD) {
                // Lane a h + r holds W row r in segment a: the columns of that
                // segment go to shared memory, and the segments are added in
                // order.
                float* sums = reinterpret_cast<float*>(smem + p.out_off);
                const int m = q * 32 + lane;
                const uint32_t by_h = (65536u + w.h - 1) / w.h;  // exact quotients below 1,024 (h <= 64)
                const int a = static_cast<int>((m * by_h) >> 16);
                for (int i = 0; i < segs; ++i) {
                    float v[8];
                    for (int c = 0; c < p.fold_x; c += 8) {
                        tmem_ld_x8(taddr + i * p.fold_x + c, v);
                        if (i == a)
#pragma unroll
                            for (int t = 0; t < 8; ++t) sums[m * 17 + c + t] = v[t];
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(acc_empty(b));
                epilogue_bar_sync();
                for (int i = m; i < w.h * w.rows; i += 128) {
                    const int t = static_cast<int>((i * by_h) >> 16);
                    const int r = i - t * w.h;
                    float sum = sums[r * 17 + t];
                    for (int k = 1; k < segs; ++k) sum += sums[(k * w.h + r) * 17 + t];
                    if (w.w0 + r < p.n) row0[t * p.ldy + w.w0 + r] = __float2bfloat16_rn(sum * alpha);
                }
                ++piece;
                continue;
            }
            // W rows of this warp's TMEM lanes, and those of them in the piece.
            const int n0 = w.w0 + rank * kTileRows - first_row() + q * 32;
            const int n_lo = PAIR ? n0 : w.w0;
            const int n_hi = min(p.n, PAIR ? n0 + 32 : w.w0 + w.h);
            // kCols X rows at a time through shared memory, [X row][32 W rows]
            // of BF16 with the 16-byte chunks of a row exchanged so that
            // neither side has bank conflicts, to 16-byte stores.
            constexpr int kCols = PAIR ? 32 : 16;
            uint8_t* buf = smem + p.out_off + q * kOutBytes;
            for (int c = 0; c < w.rows; c += kCols) {
                uint32_t v[2][kCols / 2];
#pragma unroll
                for (int g = 0; g < kCols; g += 16) {
                    tmem_ld_frag(taddr + c + g, v[0] + g / 2);
                    tmem_ld_frag(taddr + (16u << 16) + c + g, v[1] + g / 2);
                }
                tmem_ld_wait();
                if (c + kCols >= w.rows) {  // everything is read: the accumulator is free
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        if (rank) mbar_arrive_remote(at_rank(acc_empty(b), 0));
                        else mbar_arrive(acc_empty(b));
                    }
                }
                if (n0 >= n_hi || n0 + 32 <= n_lo) continue;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int g = 0; g < kCols / 8; g += 2) {
                        const int r = 8 * (g + (lane >> 4)) + (lane & 7);
                        const int ch = 2 * h + ((lane >> 3) & 1);
                        const uint32_t* f = v[h] + 4 * g;
                        stmatrix_x4_trans(smem_u32(buf) + r * 64 + ((ch ^ ((r >> 1) & 3)) * 16),
                                          pack_bf16(f[0], f[1], alpha), pack_bf16(f[2], f[3], alpha),
                                          pack_bf16(f[4], f[5], alpha), pack_bf16(f[6], f[7], alpha));
                    }
                __syncwarp();
                if (p.wide_y) {
#pragma unroll
                    for (int k = 0; k < kCols / 8; ++k) {
                        const int r = 8 * k + (lane >> 2), ch = lane & 3;
                        const int n = n0 + ch * 8;
                        const uint4 o = *reinterpret_cast<const uint4*>(
                            buf + r * 64 + ((ch ^ ((r >> 1) & 3)) * 16));
                        if (c + r < w.rows && n >= n_lo && n < n_hi) {
                            __nv_bfloat16* dst = row0 + (c + r) * p.ldy + n;
                            if (n + 8 <= n_hi) {
                                *reinterpret_cast<uint4*>(dst) = o;
                            } else {
                                const uint32_t ow[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                                for (int i = 0; i < 8; ++i)
                                    if (n + i < n_hi)
                                        reinterpret_cast<uint16_t*>(dst)[i] =
                                            static_cast<uint16_t>(ow[i / 2] >> (16 * (i & 1)));
                            }
                        }
                    }
                } else {
                    // Y's rows do not start on 16 bytes: one value per lane,
                    // 64 bytes of a row per warp.
                    const int n = n0 + lane;
#pragma unroll
                    for (int r = 0; r < kCols; ++r) {
                        if (c + r < w.rows && n >= n_lo && n < n_hi)
                            row0[(c + r) * p.ldy + n] = *reinterpret_cast<const __nv_bfloat16*>(
                                buf + r * 64 + (((lane >> 3) ^ ((r >> 1) & 3)) * 16) + (lane & 7) * 2);
                    }
                }
                __syncwarp();
            }
            ++piece;
        }
        if (p.flags & kGrpZeroRest) {
            // rows before the first group and behind the last
            const int lo = off[0], hi = off[p.experts];
            const int rest = lo + p.rows - hi;
            for (int i = blockIdx.x; i < rest; i += gridDim.x) {
                __nv_bfloat16* dst = p.y + static_cast<int64_t>(i < lo ? i : hi + i - lo) * p.ldy;
                const int whole = p.wide_y ? p.n / 8 : 0;  // 16-byte stores, then what is left
                for (int n = threadIdx.x - 128; n < whole; n += 128)
                    reinterpret_cast<uint4*>(dst)[n] = make_uint4(0u, 0u, 0u, 0u);
                for (int n = whole * 8 + threadIdx.x - 128; n < p.n; n += 128)
                    dst[n] = __float2bfloat16_rn(0.0f);
            }
        }
    }
    // The roles meet.  Neither CTA of a pair leaves while the other may still
    // use its shared memory or arrive on its barriers.
    auto meet = [&]() {
        __syncwarp();
        tc_fence_before_sync();
        if constexpr (PAIR) {
            cluster_arrive_release();
            cluster_wait_acquire();
        } else {
            __syncthreads();
        }
        tc_fence_after_sync();
    };
    if (PAIR && rank == 0 && lane == 0 && *abort_flag) dsmem_st_u32(at_rank(smem_u32(tmem_slot + 2), 1), 1u);
    meet();
    // Every accumulator has been stored, so every MMA and copy is over, unless
    // a wait ran out: then wait (bounded) for what is still in flight before
    // shared and tensor memory are released.
    if (PAIR && rank ? *peer != 0 : *abort_flag != 0) {
        if (warp == 0 && lane == 0 && rank == 0) {
            // A stage that lacks another arrival runs into the limit, long
            // after every copy has landed.
            bool ok = true;
            for (int j = max(0, issued - stages); ok && j < issued; ++j)
                ok = mbar_drain(full_bar(j % stages), (j / stages) & 1, guard, kErrDrain);
            if (PAIR && ok && static_cast<int>(*peer) > issued)  // CTA 1's alone
                mbar_drain(full_bar(issued % stages), (issued / stages) & 1, guard, kErrDrain);
        }
        if (warp == 1 && rank == 0) {
            if (elect_one()) Ops::commit(drain_bar);
            __syncwarp();
            if (lane == 0) mbar_drain(drain_bar, 0, guard, kErrDrain);
        }
        if constexpr (PAIR) meet();
        __syncwarp();
    }
    if (warp == 1) Ops::dealloc(tmem, p.tmem_cols);
}

}  // namespace tinym
