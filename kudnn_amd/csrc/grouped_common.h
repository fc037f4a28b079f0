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
};

__device__ __forceinline__ int clamp_row(int v, int R) { return v < 0 ? 0 : (v > R ? R : v); }

// Row tiles of all experts and of the rest, as one wave sees them: 64 experts at a time, a scan over the lanes. Offsets are
// clamped to [0, R], so any contents stay inside the buffers. With up to 63 experts the offsets are read once.
class RowTiles {
public:
    __device__ __forceinline__ RowTiles(const int32_t *offsets, int E, int R, int bm) : offsets_(offsets), E_(E), R_(R), bm_(bm)
    {
        if (offsets == nullptr) {   // one group of all rows
            total_ = (R + bm - 1) / bm;
            return;
        }
        int carry = 0;
        for (int base = 0; base <= E; base += 64) {
            scan(base, carry);
            carry += __shfl(first_ + tiles_ - carry, 63);
        }
        total_ = __builtin_amdgcn_readfirstlane(carry);
    }
    __device__ __forceinline__ int total() const { return total_; }
    // Tile number `want` < total(). Its members are the same in every lane.
    __device__ __forceinline__ RowTile find(int want)
    {
        RowTile t{0, 0, 0, 0};
        if (offsets_ == nullptr) {
            t.end = R_;
            t.r0 = want * bm_;
            return t;
        }
        int carry = 0;
        for (int base = 0; base <= E_; base += 64) {
            if (E_ >= 64) scan(base, carry);
            const unsigned long long who = __ballot(tiles_ > 0 && want >= first_ && want < first_ + tiles_);
            if (who != 0ull) {
                const int src = __ffsll(who) - 1;
                t.e = base + src;
                t.begin = __builtin_amdgcn_readlane(lo_, src);
                t.end = __builtin_amdgcn_readlane(hi_, src);
                t.r0 = t.begin + (want - __builtin_amdgcn_readlane(first_, src)) * bm_;
                break;
            }
            carry += __shfl(first_ + tiles_ - carry, 63);
        }
        return t;
    }

private:
    // Expert base + lane: its rows, its tiles, and how many tiles there are before.
    __device__ __forceinline__ void scan(int base, int carry)
    {
        const int lane = threadIdx.x & 63, e = base + lane;
        lo_ = hi_ = 0;
        if (e <= E_) {
            lo_ = clamp_row(offsets_[e], R_);
            hi_ = e < E_ ? clamp_row(offsets_[e + 1], R_) : R_;
        }
        tiles_ = hi_ > lo_ ? (hi_ - lo_ + bm_ - 1) / bm_ : 0;
        int incl = tiles_;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            incl += lane >= d ? o : 0;
        }
        first_ = carry + incl - tiles_;
    }
    const int32_t *offsets_;
    int E_, R_, bm_, total_ = 0;
    int lo_ = 0, hi_ = 0, tiles_ = 0, first_ = 0;
};

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
