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
    return kudnn_launch_grouped_generic(g, stream);
}

#endif  // KUDNN_GROUPED_H
