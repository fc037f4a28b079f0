// Choice of the kernel for a grouped product.
#ifndef KUDNN_GROUPED_H
#define KUDNN_GROUPED_H

#include "moe.h"

// Whether the grids of every kernel hold a product of these sizes (a grid's threads must stay below 2^32: 2^24
// workgroups of 256); `backward`: also those of its gradients.
inline bool kudnn_grouped_fits(int64_t R, int64_t E, int64_t N, int64_t K, bool backward)
{
    const int64_t most = int64_t(1) << 24;
    const auto tiles = [](int64_t n) { return (n + 63) / 64; };
    const int64_t rows = tiles(R) + (E + 1 < R ? E + 1 : R);
    const auto fits = [&](int64_t a, int64_t b) { return a == 0 || b < most / a; };
    return fits(rows, tiles(N)) && (!backward || (fits(rows, tiles(K)) && tiles(N) < most && fits(tiles(N) * tiles(K), E)));
}

inline int kudnn_launch_grouped(const GroupedArgs &g, hipStream_t stream)
{
    if (!kudnn_grouped_pingpong_eligible(g)) {
        return kudnn_launch_grouped_generic(g, stream);
    }
    if (g.form == GROUPED_FWD) {
        const int64_t groups = g.offsets == nullptr ? 1 : (g.E < g.R ? g.E : g.R);
        const int64_t rows = (g.R + groups - 1) / groups;   // of an expert, on average
        const int64_t tiles = groups * ((rows + 255) / 256) * ((g.J + 255) / 256);
        const bool f8 = g.dt == KUDNN_DT_F8E4M3;
        if (rows <= 64 || (f8 && (g.c_dt == KUDNN_DT_F32 || tiles < 128))) {
            const int bm = rows <= 16 ? 16 : (rows <= 32 ? 32 : 64);
            const int64_t narrow = groups * ((rows + bm - 1) / bm) * ((g.J + 63) / 64);
            return kudnn_launch_grouped_stream(g, bm, bm == 16 && narrow < 512 ? 32 : 64, stream);
        }
    }
    return kudnn_launch_grouped_pingpong(g, stream);
}

#endif  // KUDNN_GROUPED_H
