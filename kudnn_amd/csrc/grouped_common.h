// Device helpers shared by the grouped product kernels: which rows a workgroup has.
#ifndef KUDNN_GROUPED_COMMON_H
#define KUDNN_GROUPED_COMMON_H

#include "device_common.h"
#include "moe.h"

namespace kudnn_dev {

// A tile of rows of one expert. e == E: the rows that belong to no expert (past offsets[E]).
struct RowTile {
    int e, begin, end;   // the expert's rows
    int r0;              // first row of the tile
    int index;           // the tile's place among the experts' tiles (for the order of workgroups)
};

__device__ __forceinline__ int clamp_row(int v, int R) { return v < 0 ? 0 : (v > R ? R : v); }

// Row tiles of all experts and of the rest, by one wave: 64 experts at a time, a scan over the lanes. Returns whether tile
// number `want` exists and fills it in; `total` gets the number of tiles. Offsets are clamped to [0, R], so any contents
// stay inside the buffers.
__device__ __forceinline__ bool find_row_tile(const int32_t *offsets, int E, int R, int bm, int want, RowTile &t, int &total)
{
    const int lane = threadIdx.x & 63;
    bool found = false;
    int carry = 0;
    if (offsets == nullptr) {   // one group of all rows
        total = (R + bm - 1) / bm;
        t = RowTile{0, 0, R, want * bm, want};
        return want < total;
    }
    for (int base = 0; base <= E; base += 64) {
        const int e = base + lane;
        int lo = 0, hi = 0;
        if (e <= E) {
            lo = clamp_row(offsets[e], R);
            hi = e < E ? clamp_row(offsets[e + 1], R) : R;
        }
        const int tiles = hi > lo ? (hi - lo + bm - 1) / bm : 0;
        int incl = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            incl += lane >= d ? o : 0;
        }
        const bool mine = tiles > 0 && want >= carry + incl - tiles && want < carry + incl;
        const unsigned long long who = __ballot(mine);
        if (who != 0ull) {
            const int src = __ffsll(static_cast<unsigned long long>(who)) - 1;
            const int first = carry + __shfl(incl - tiles, src);
            t.e = base + src;
            t.begin = __shfl(lo, src);
            t.end = __shfl(hi, src);
            t.r0 = t.begin + (want - first) * bm;
            t.index = want;
            found = true;
        }
        carry += __shfl(incl, 63);
    }
    total = carry;
    return found;
}

// Most row tiles that offsets of any contents in order can make: each group of rows leaves at most one part tile.
inline int64_t max_row_tiles(int64_t R, int64_t E, int64_t bm, bool grouped)
{
    if (!grouped) return (R + bm - 1) / bm;
    const int64_t groups = E + 1 < R ? E + 1 : R;
    // n groups of which every one has a part tile: (R - n) / bm whole ones besides, at most
    return groups + (R - groups) / bm;
}

// Row of the gathered operand that row r takes, or -1.
__device__ __forceinline__ int64_t source_row(const GroupedArgs &g, int64_t r)
{
    if (g.rows == nullptr) return r;
    const int64_t s = g.rows[r];
    return s >= 0 && s < g.S ? s : -1;
}

}  // namespace kudnn_dev

#endif  // KUDNN_GROUPED_COMMON_H
