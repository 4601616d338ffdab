// Host-side checks of the grouped product's work list and carve-up
// (csrc/tinym_grouped.cuh: grouped_plan, GroupedWalk), over shapes and group
// sizes.  Built with nvcc and run on the CPU by tests/test_grouped_layout.py;
// no GPU is touched.
//
//  * Every (row of a group, W row) is computed by exactly one piece, pieces
//    stay inside their group's rows and hold at most tn rows and 128 W rows
//    that start inside N.
//  * The rings, scale slots, barriers and tables lie end to end inside the
//    allocation, stages on 1024-byte and scale blocks on 512-byte boundaries,
//    and the MMA's 128-row reads end inside it.
//  * Accumulators and scale columns fit the tensor memory that is allocated.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "tinym_grouped.cuh"
#include "tinym_mxfp4.cuh"

namespace {

long g_checks = 0;
int g_failures = 0;

void expect(bool ok, const char* what, long a = 0, long b = 0, long c = 0) {
    ++g_checks;
    if (!ok && ++g_failures <= 20) std::printf("FAIL %s (%ld, %ld, %ld)\n", what, a, b, c);
}

// The kernel's tables, one after the other instead of by a warp.
void tables(const tinym::GroupedParams& p, const std::vector<int>& raw, std::vector<int>* off,
            std::vector<int>* prefix) {
    int start = 0, tiles = 0;
    for (int i = 0; i <= p.experts; ++i) {
        const int before = start;
        start = std::max(start, std::min(std::max(raw[i], 0), p.rows));
        if (i) tiles += (start - before + p.tn - 1) / p.tn;
        off->push_back(start);
        prefix->push_back(tiles);
    }
}

template <bool PAIR>
void check_walk(const tinym::GroupedPlan& g, const std::vector<int>& raw) {
    const tinym::GroupedParams& p = g.prm;
    std::vector<int> off, prefix;
    tables(p, raw, &off, &prefix);
    const int unit = PAIR ? 256 : 8;
    const int n_units = (p.n + unit - 1) / unit;
    const int ctas = PAIR ? g.grid / 2 : g.grid;
    std::vector<std::vector<unsigned char>> seen(p.rows, std::vector<unsigned char>(n_units, 0));
    int least = 1 << 30, most = 0;
    for (int b = 0; b < ctas; ++b) {
        tinym::GroupedWalk<PAIR> walk(p, off.data(), prefix.data(), b, ctas);
        tinym::GroupedPiece w;
        int units = 0;
        while (walk.next(&w)) {
            expect(w.e >= 0 && w.e < p.experts, "expert", w.e);
            expect(w.rows >= 1 && w.rows <= p.tn, "rows of a piece", w.rows, p.tn);
            expect(w.row0 >= off[w.e] && w.row0 + w.rows <= off[w.e + 1], "piece inside its group",
                   w.row0, w.rows, w.e);
            expect(w.h >= unit && w.h <= std::max(128, unit) && w.h % unit == 0 && w.w0 % unit == 0, "W rows",
                   w.w0, w.h);
            expect(w.w0 >= 0 && w.w0 < p.n && w.w0 + w.h <= n_units * unit, "W range", w.w0, w.h);
            if (!PAIR) expect(w.h <= p.piece_units * 8, "piece fits its stage", w.h, p.piece_units);
            if (!PAIR && p.blocked) {
                expect(w.w0 / 128 == (w.w0 + w.h - 1) / 128, "piece inside a block", w.w0, w.h);
                // the MMA reads from the block's first row, ahead of the stage
                expect(w.w0 % 128 * 128 <= static_cast<int>(p.w_off), "read before the stage", w.w0, p.w_off);
            }
            for (int r = 0; r < w.rows; ++r)
                for (int u = 0; u < w.h / unit; ++u) ++seen[w.row0 + r][w.w0 / unit + u];
            units += w.h / unit;
        }
        least = std::min(least, units);
        most = std::max(most, units);
    }
    const int total = prefix[p.experts] * p.units, share = (total + ctas - 1) / ctas;
    if (PAIR) expect(most - least <= 1, "equal shares", least, most);
    else if (!p.part_units) expect(most <= share || (!p.blocked && most <= p.piece_units && 2 * most <= 3 * (share + 1)),
                                   "shares", most, share);
    else expect(most <= p.part_units * std::max(1, (prefix[p.experts] * p.units + ctas - 1) / ctas),
                "shares of parts", least, most);
    for (int r = 0; r < p.rows; ++r)
        for (int u = 0; u < n_units; ++u)
            expect(seen[r][u] == (r >= off[0] && r < off[p.experts] ? 1 : 0), "computed once", r, u,
                   seen[r][u]);
}

void check_plan(const tinym::GroupedPlan& g, bool fp4, uint32_t limit) {
    const tinym::GroupedParams& p = g.prm;
    expect(g.smem <= limit && p.stages >= 2, "shared memory", g.smem, p.stages);
    expect(p.w_stage % 1024 == 0 && p.x_stage % 1024 == 0, "stage alignment", p.w_stage, p.x_stage);
    expect(p.sf_off >= static_cast<uint32_t>(p.stages * p.x_stage) && p.sf_off % 512 == 0 && p.sf_stage % 512 == 0,
           "scale ring", p.sf_off, p.sf_stage);
    expect(p.w_off >= p.sf_off + p.stages * p.sf_stage && p.w_off % 1024 == 0, "W ring", p.w_off);
    expect(p.out_off >= p.w_off + p.stages * p.w_stage && p.out_off % 16 == 0, "output", p.out_off);
    expect(p.bar_off >= p.out_off + (p.fold ? tinym::kFoldOutBytes : 4 * tinym::kOutBytes) && p.bar_off % 8 == 0, "barriers", p.bar_off);
    expect(p.tab_off >= p.bar_off + 8u * (2 * p.stages + tinym::kGrpBars) + 8u && p.tab_off % 4 == 0, "tables",
           p.tab_off);
    expect(p.tab_off + 8u * (p.experts + 1) + 1024 <= g.smem, "tables inside", p.tab_off, g.smem);
    const uint32_t chunks = tinym::grouped_chunks(g.mode);
    // every W read is 128 rows of a chunk that starts inside its stage, every
    // X read at most 8 rows longer than the box
    expect(p.w_off + p.stages * p.w_stage + (g.pair ? 0 : 128 * 128) + 1024 <= g.smem, "W read inside", p.w_stage,
           g.smem);
    const int segs = std::max(1, p.fold);
    expect(p.w_stage == segs * p.piece_units * 8 * 128 * static_cast<int>(chunks), "W stage", p.w_stage);
    expect((p.fold != 0) == (g.mode == tinym::kFold), "mode", p.fold, g.mode);
    if (p.fold) {
        expect(p.fold >= 2 && p.fold * p.piece_units <= 16 && p.fold * p.fold_x <= 64 && p.tn == 16 &&
                   (p.fold_x == 8 || p.fold_x == 16) && p.fold_x >= std::min(p.rows, 16),
               "folded rows and columns", p.fold, p.fold_x, p.piece_units);
        expect(p.k_bytes % (128 * p.fold) == 0 && !p.blocked && !p.part_units, "segments", p.k_bytes, p.fold);
        expect(p.x_stage == p.fold * p.fold_x * 128 * static_cast<int>(chunks), "folded X stage", p.x_stage);
        expect(static_cast<int>(p.acc_cols) >= p.fold * p.fold_x && p.acc_cols % 16 == 0, "columns", p.acc_cols);
        expect(p.bar_off >= p.out_off + 128 * 17 * 4, "folded sums", p.out_off, p.bar_off);
        for (int h = 8; h <= p.piece_units * 8; h += 8)  // the kernels' quotients
            for (int i = 0; i < 16 * h || i < 128; ++i)
                expect(static_cast<int>((i * ((65536u + h - 1) / h)) >> 16) == i / h, "quotient", i, h);
    }
    int box = 0;
    while (box < 4 && tinym::grouped_x_box(g.pair, box) * (g.pair ? 2 : 1) < (p.fold ? p.fold_x : p.tn)) ++box;
    expect(box < 4 && segs * tinym::grouped_x_box(g.pair, box) * 128 * static_cast<int>(chunks) <= p.x_stage, "X box", box,
           p.x_stage);
    expect(p.tn % 16 == 0 && p.tn >= 16 && p.tn <= 256 && (!g.pair || p.tn % 32 == 0) &&
               p.tn <= 128 * tinym::grouped_x_scale_blocks(g.pair),
           "tile width", p.tn);
    expect((p.fold || p.acc_cols >= static_cast<uint32_t>(p.tn)) && p.tmem_cols <= 512 && (p.tmem_cols & (p.tmem_cols - 1)) == 0,
           "tensor memory", p.acc_cols, p.tmem_cols);
    expect((fp4 ? p.sf_col + 2 * tinym::kSfSlotCols : 2 * p.acc_cols) <= p.tmem_cols &&
               (!fp4 || (p.sf_col >= 2 * p.acc_cols && p.sf_col % 4 == 0)),
           "scale columns", p.sf_col, p.tmem_cols);
    expect(g.grid >= 1 && (!g.pair || g.grid % 2 == 0), "grid", g.grid);
}

void check_div() {
    const uint32_t ds[] = {1, 2, 3, 5, 7, 8, 40, 48, 127, 128, 129, 5120, 65537, 1000003, (1u << 30) - 1, 1u << 30};
    for (uint32_t d : ds) {
        const tinym::FastDiv f = tinym::FastDiv::make(d);
        auto div = [&](uint32_t n) {
            return static_cast<uint32_t>((static_cast<uint64_t>(n) * f.mul) >> f.shift);
        };
        for (uint64_t q = 0; q * d < (1ull << 31); q += 1 + (1ull << 31) / d / 997)
            for (int64_t s = -1; s <= 1; ++s) {
                const int64_t n = static_cast<int64_t>(q * d) + s;
                if (n < 0 || n >= (1ll << 31)) continue;
                expect(div(static_cast<uint32_t>(n)) == static_cast<uint32_t>(n) / d, "division", n, d);
            }
    }
}

}  // namespace

int main() {
    const uint32_t limit = 232448;
    std::srand(7);
    const int row_counts[] = {1, 2, 3, 15, 16, 17, 64, 65, 130, 257, 700};
    const int expert_counts[] = {1, 2, 5, 31, 32, 33, 64, 100};
    const int ns[] = {1, 7, 8, 100, 129, 1000, 2050, 6000};
    for (int rows : row_counts)
        for (int experts : expert_counts)
            for (int n : ns)
                for (int mode = 0; mode < 5; ++mode)
                    for (int fp4 = 0; fp4 < 2; ++fp4) {
                        tinym::GroupedPlan g;
                        const char* why = tinym::grouped_plan(fp4, rows, experts, n,
                                                              mode % 2 ? 128 * (1 + std::rand() % 48)
                                                                       : 16 * (1 + std::rand() % 300),
                                                              mode == 4 ? 3 : 148, limit, &g);
                        expect(!why, "plan", rows, experts, n);
                        if (why) continue;
                        check_plan(g, fp4, limit);
                        std::vector<int> off(experts + 1);
                        for (int i = 0; i <= experts; ++i) {
                            if (mode == 0) off[i] = static_cast<int>(static_cast<long>(rows) * i / experts);
                            if (mode == 1) off[i] = i > experts / 2 ? rows : 0;           // one group
                            if (mode == 2) off[i] = std::rand() % (rows + 20) - 10;       // not sorted, outside
                            if (mode == 3) off[i] = std::min(rows, 1 + i / 2);            // spare rows
                            if (mode == 4) off[i] = 0;                                    // no rows
                        }
                        if (g.pair) check_walk<true>(g, off);
                        else check_walk<false>(g, off);
                    }
    // large shapes: the plan alone
    for (int64_t rows : {int64_t(1), int64_t(4096), int64_t(1) << 20, (int64_t(1) << 31) - 1024})
        for (int64_t experts : {1, 64, 1024})
            for (int64_t n : {int64_t(1), int64_t(16384), int64_t(1) << 24})
                for (int fp4 = 0; fp4 < 2; ++fp4) {
                    tinym::GroupedPlan g;
                    if (!tinym::grouped_plan(fp4, rows, experts, n, 8192, 148, limit, &g)) {
                        check_plan(g, fp4, limit);
                        expect((std::min(experts, rows) + rows / g.prm.tn) * g.prm.units < (int64_t(1) << 31),
                               "tiles fit 32 bits", rows, experts, n);
                    }
                }
    check_div();
    if (g_failures) {
        std::printf("%d of %ld checks failed\n", g_failures, g_checks);
        return 1;
    }
    std::printf("grouped layout checks ok (%ld checks)\n", g_checks);
    return 0;
}
