// Choice of the kernel for a grouped product.
#ifndef KUDNN_GROUPED_H
#define KUDNN_GROUPED_H

#include <cmath>
#include <initializer_list>

#include "moe.h"

// A tiled kernel of the forward product.
struct GroupedTile {
    enum { STREAM, RING, PINGPONG } kind;
    int bm, bn;        // rows and columns of a tile
    int form;          // STREAM: waves; RING: stages
    bool native;       // e4m3 products by the e4m3 matrix instruction
    bool hint;         // the weights are read by one row tile: non-temporal copies
};

// e4m3 operands. The e4m3 matrix instruction aligns the products of 8 consecutive indices to the largest of them and drops
// what lies more than 13 bits below it (measured: beside 2^16 a product of 2^2 is lost, at a distance of 8 indices it is kept);
// bf16 holds e4m3 exactly, and its instruction sums in f32, at half the rate and with the widening to do. Products into f32 and f16
// are formed that way, and so are those of less than 2^33 operations, whose time is the weight's way from HBM and the launch
// (8 experts of 32 rows, 2048 x 4096: 21 us exact, 18 us native). Larger ones into bf16, whose rounding is 32 times coarser than what
// is dropped, take the native instruction (4096 x 4096 x 4096: 66 us native, 166 exact; 64 experts of 64 rows, 2048 x 4096: 144 and 207):
// the error against 64 bits in norm is 0.001658 either way at 4096 x 4096 x 11008 (203 us native, 425 exact). f16's rounding is only 4 times
// coarser, and there it grew from 2.072e-4 to 2.098e-4 (203 us native, 450 to 520 exact).
inline bool kudnn_grouped_native(int64_t R, int64_t N, int64_t K, int c_dt)
{
    return c_dt == KUDNN_DT_BF16 && static_cast<double>(R) * static_cast<double>(N) * static_cast<double>(K) >= 4294967296.0;
}

// The tile with the least estimate for R rows in `groups` groups of weights N x K (rows of `es` bytes an element). A tile's
// work is the blocks of 128 bytes of a row (dealt to its waves, where they split the sum) times what a block takes the busiest
// CU, plus the tile's own start and end. With u = tiles / (tiles the chip holds at once) a block takes from `alone` (u near 0:
// latency) to `full` us (u = 1), and a multiple of `full` beyond. The call takes 2.2 us, the longer of that work and the
// weight's way from HBM, and a third of the shorter. Rows are rarely dealt evenly: a group is taken to have up to 1.25 r + 4
// of an average of r, and half a tile more than r rows fill.
// The figures are a fit to 322 products timed on MI355X on every kernel (1 to 128 groups of 1 to 4096 rows, K and N = 256 to
// 8192, 16-bit and e4m3; weights rotated past the Infinity Cache): the choice takes 1.012 times the best kernel's time on average,
// and more than 1.1 times in 14 of them (1.21 at most); on 144 more with skewed sizes (a softmax over normal numbers) 1.037 times
// (timed after the ring's e4m3 tiles had become a tenth faster than the fit has them).
// Always 256 x 256 tiles, or one tile of 64 x 64, would take 2 to 5 times.
// any: operands that are not whole 16-byte chunks. They pass through registers, which the 256 x 256 tiles and the 64 x 64 tiles
// of 8 waves have none left for and the longer ring has no use for; the others stay in the order that the figures give them.
inline GroupedTile kudnn_grouped_rule(int64_t R, int64_t groups, int64_t N, int64_t K, int dt, int c_dt, bool any)
{
    struct Kind {
        int kind, bm, bn, form, waves;   // waves: that split the sum
        double slots;
        double alone[3], full[3];        // 16-bit; e4m3 exact; e4m3 native (0: none)
        double ends;
        bool any;
    };
    static const Kind kKinds[] = {
        {GroupedTile::STREAM, 16, 32, 8, 8, 768, {0.06, 0.13, 0}, {0.26, 0.30, 0}, 1.53, true},
        {GroupedTile::STREAM, 16, 64, 8, 8, 512, {0.19, 0.22, 0}, {0.32, 0.38, 0}, 0.91, true},
        {GroupedTile::STREAM, 64, 64, 4, 4, 512, {0.29, 0.41, 0}, {0.59, 0.76, 0}, 1.78, true},
        {GroupedTile::STREAM, 64, 64, 8, 8, 256, {0.19, 0.25, 0}, {0.31, 0.41, 0}, 2.11, false},
        {GroupedTile::RING, 64, 128, 2, 1, 768, {0.78, 1.05, 0.49}, {1.25, 1.85, 1.82}, 1.12, true},
        {GroupedTile::RING, 128, 128, 2, 1, 512, {0.84, 1.19, 0.85}, {1.18, 2.56, 1.51}, 0.79, true},
        {GroupedTile::RING, 128, 128, 4, 1, 256, {0.53, 1.03, 0.72}, {0.62, 1.30, 0.99}, 2.37, false},
        {GroupedTile::PINGPONG, 256, 256, 0, 1, 256, {1.11, 0, 1.44}, {1.11, 0, 2.15}, 1.88, false},
    };
    const bool f8 = dt == KUDNN_DT_F8E4M3, native = f8 && kudnn_grouped_native(R, N, K, c_dt);
    const int col = f8 ? (native ? 2 : 1) : 0;
    const double r = static_cast<double>(R) / static_cast<double>(groups), es = f8 ? 1.0 : 2.0;
    const double cover = groups == 1 ? r : 1.25 * r + 4.0;
    const double stream = static_cast<double>(groups) * static_cast<double>(N) * static_cast<double>(K) * es / 8.1e6;
    GroupedTile best{GroupedTile::STREAM, 16, 64, 8, false, false};
    double bestUs = 0.0;
    for (const Kind &k : kKinds) {
        if (k.full[col] == 0.0 || (any && !k.any)) {
            continue;
        }
        const double blocks = std::ceil(std::ceil(static_cast<double>(K) * es / 128.0) / k.waves) * k.waves;
        const double rowTiles = cover <= k.bm ? 1.0 : (groups == 1 ? std::ceil(r / k.bm) : r / k.bm + 0.54);
        const double u = static_cast<double>(groups) * rowTiles * std::ceil(static_cast<double>(N) / k.bn) / k.slots;
        const double rounds = 0.5 * (u + std::ceil(u));
        const double work = blocks * (u <= 1.0 ? k.alone[col] + (k.full[col] - k.alone[col]) * u : k.full[col] * rounds) +
                            k.ends * (rounds > 1.0 ? rounds : 1.0);
        const double us = 2.2 + (work > stream ? work + 0.36 * stream : stream + 0.36 * work);
        if (bestUs == 0.0 || us < bestUs) {
            bestUs = us;
            best = GroupedTile{static_cast<decltype(best.kind)>(k.kind), k.bm, k.bn, k.form, native, cover <= k.bm};
        }
    }
    return best;
}

// Threads of a workgroup of the tile's kernel.
inline int kudnn_grouped_threads(const GroupedTile &t)
{
    return t.kind == GroupedTile::STREAM ? t.form * 64 : (t.kind == GroupedTile::RING && t.bm == 64 ? 256 : 512);
}

// A grid's threads must stay below 2^32.
inline bool kudnn_grid_fits(int64_t workgroups, int64_t threads) { return workgroups < (int64_t(1) << 32) / threads; }

// Whether the grid of every kernel that a product of these sizes may take holds it: the rule's tiles for operands of either alignment and the
// generic kernel's 64 x 64; `backward`: also those of its gradients.
inline bool kudnn_grouped_fits(int64_t R, int64_t E, int64_t N, int64_t K, int dt, int c_dt, bool grouped, bool backward)
{
    const auto up = [](int64_t n, int64_t by) { return (n + by - 1) / by; };
    const auto rows = [&](int64_t bm) { return kudnn_max_row_tiles(R, E, bm, grouped); };
    const int64_t cut = 128;      // whole 256 x 256 tiles that may be cut in two
    if (R > 0) {
        for (const bool any : {false, true}) {
            const GroupedTile t = kudnn_grouped_rule(R, grouped ? (E < R ? E : R) : 1, N, K, dt, c_dt, any);
            if (!kudnn_grid_fits(rows(t.bm) * up(N, t.bn) + (t.kind == GroupedTile::PINGPONG ? cut : 0), kudnn_grouped_threads(t))) return false;
        }
        if (!kudnn_grid_fits(rows(64) * up(N, 64), 256)) return false;
    }
    return !backward || (kudnn_grid_fits(rows(64) * up(K, 64), 256) && kudnn_grid_fits(rows(256) * up(K, 256) + cut, 512) &&
                         kudnn_grid_fits(E * up(N, 64) * up(K, 64), 256) && kudnn_grid_fits(E * up(N, 256) * up(K, 256), 512));
}

// Whether an e4m3 product of R rows leaves the quantisation of x to the workgroups: each takes the whole of its rows (up to 48 KB
// of e4m3 in LDS) before its first block of weights has arrived, where a launch of its own and the wait for it cost 3.5 us of 15
// (1 x 4096 x 14336).
inline bool kudnn_grouped_fused(int64_t R, int64_t groups, int64_t N, int64_t K, int c_dt, bool any)
{
    if (R > 16 || K < 16 || R * kudnn_fp8_pitch(K) > 49152) {
        return false;
    }
    const GroupedTile t = kudnn_grouped_rule(R, groups, N, K, KUDNN_DT_F8E4M3, c_dt, any);
    return t.kind == GroupedTile::STREAM && t.bm == 16;
}

inline int kudnn_launch_grouped(const GroupedArgs &g, hipStream_t stream)
{
    const bool whole = kudnn_grouped_tiled(g, true);
    if (g.form != GROUPED_FWD && whole) {
        return kudnn_launch_grouped_pingpong(g, stream);
    }
    const int64_t rowBytes = g.C * (g.dt == KUDNN_DT_F8E4M3 ? 1 : 2);
    if (g.form != GROUPED_FWD || (!whole && (rowBytes < 16 || !kudnn_grouped_tiled(g, false)))) {
        return kudnn_launch_grouped_generic(g, stream);
    }
    const int64_t groups = g.offsets == nullptr ? 1 : (g.E < g.R ? g.E : g.R);
    const GroupedTile t = kudnn_grouped_rule(g.R, groups, g.J, g.C, g.dt, g.c_dt, !whole);
    switch (t.kind) {
        case GroupedTile::STREAM: return kudnn_launch_grouped_stream(g, t.bm, t.bn, t.form, t.hint, !whole, stream);
        case GroupedTile::RING: return kudnn_launch_grouped_ring(g, t.bm, t.form, t.native, t.hint, !whole, stream);
        default: return kudnn_launch_grouped_pingpong(g, stream);
    }
}

#endif  // KUDNN_GROUPED_H
