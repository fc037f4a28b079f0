// Grouped products of few rows: the experts' Linear layers of one token or a decode batch, in 16 bits or e4m3.
//
// A workgroup has a tile of BM rows of one expert and BN columns; its waves split the sum: wave w of W takes the blocks
// w, w + W, ... of 128 bytes of each row and accumulates the whole tile over them. A wave copies a block's rows into LDS of
// its own, reads them into registers once they are there, sends the copies of its next block and multiplies while they fly.
// Nothing is shared and no barrier orders the waves until their sums meet in LDS at the end, in wave order (the same bits
// every run).
//
// What bounds it is the weight's way from HBM. A copy covers 8 rows of whole 128-byte lines: reading 16 rows of 64 bytes, the
// layout the MFMAs want, straight into registers streamed 90 MB at 4.4 TB/s where this pattern gave 5.2, and 5.7 with
// the non-temporal hint (1 GB: 6.2, 6.1 and 7.0; a plain read of whole rows 7.1). The hint is for weights that one row tile
// reads. Measured: 8 experts of one row each, 2048 x 4096 bf16 (134 MB): 21.4 us a call back to back (6.3 TB/s).
//
// v_mfma_f32_16x16x32: lane l has row l % 16 of an operand and 8 of its 32 summed indices. A block's row is 8 chunks of 16
// bytes; lane group l / 16 takes chunks g and g + 4. Which index of the sum a lane has does not matter as long as both operands
// agree. Rows are held with chunk c in slot c ^ ((row / 2) % 8), so that 16 lanes read 16 different slots.
//
// e4m3: the matrix instruction for e4m3 aligns the products of 8 consecutive indices to the largest of them and drops what
// lies more than 13 bits below (measured; groups of 8 are then added in f32). Here, where the weight's way from HBM or the
// launch takes the time, the values are widened to bf16, which holds them exactly, and multiplied by the bf16 instruction, whose
// sums are f32's. A block of 128 is four chained MFMAs; its sum times sx[row] sw[block] is added to the running sum.
//
// Copies go through buffer resources: rows past the group's end or without a token, columns past the last and chunks past
// the end of the sum have an offset outside and read as zeros.
#include <type_traits>

#include "e4m3.h"
#include "grouped_common.h"

using namespace kudnn_dev;

namespace {

// BM x BN tile, W waves. HINT: the weights are read by one row tile (non-temporal). REG: rows of any alignment and length (16
// bytes at least) go to LDS through registers, a block ahead, since a copy moves whole aligned chunks only. XDT (e4m3, 16 rows):
// 0, or the type of rows of x that this workgroup quantises itself, into `rowsLds`, while its first weights are on their way.
template <int CT, int BM, int BN, int W, bool HINT, bool REG, int XDT>
__global__ __launch_bounds__(W * 64) void grouped_stream_kernel(GroupedArgs g, int tilesJ)
{
    constexpr bool F8 = CT == KUDNN_DT_F8E4M3;
    constexpr int ES = F8 ? 1 : 2, MT = BM / 16, NT = BN / 16, kPitch = BN + 4;
    constexpr int kStage = (BM + BN) * 8;                        // 16-byte chunks of a wave's block: A's rows, then B's
    constexpr int kSums = W * BM * kPitch / 4;                   // the sums reuse the stages
    __shared__ uint4 lds[W * kStage > kSums ? W * kStage : kSums];
    extern __shared__ uint4 rowsLds[];                           // XDT: the tile's rows as e4m3, then their scales
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row16 = lane & 15, grp = lane >> 4;

    const int E = static_cast<int>(g.E);
    RowTiles<> tiles(g.offsets, E, static_cast<int>(g.R), BM);
    const int actual = tiles.total() * tilesJ;
    if (static_cast<int>(blockIdx.x) >= actual) return;
    // the row tiles of one block of columns are neighbours: those of one expert read the same weights
    const int lid = xcd_remap(blockIdx.x, actual);
    const int tj = lid / tiles.total();
    const RowTile t = tiles.find(lid - tj * tiles.total());
    const int j0 = tj * BN;
    const bool none = g.offsets != nullptr && t.e == E;   // rows of no expert: zero
    const int e = none ? 0 : t.e;

    const uint32_t lda = static_cast<uint32_t>(g.lda) * ES, ldb = static_cast<uint32_t>(g.ldb) * ES;
    const uint32_t rowBytes = static_cast<uint32_t>(g.C) * ES;
    const int blocks = none ? 0 : static_cast<int>((rowBytes + 127) / 128);
    const bool gather = g.rows != nullptr;
    // (XDT: A is not copied)
    const uint8_t *baseA = static_cast<const uint8_t *>(g.a) + (gather ? 0u : static_cast<uint64_t>(t.r0) * lda);
    const uint8_t *baseB = static_cast<const uint8_t *>(g.b) + static_cast<uint64_t>(e) * static_cast<uint64_t>(g.be) * ES + static_cast<uint64_t>(j0) * ldb;
    const i32x4_t ra = resource(baseA, static_cast<uint64_t>(gather ? g.S : t.end - t.r0) * lda);
    const i32x4_t rb = resource(baseB, static_cast<uint64_t>(BN) * ldb);
    // copy i has rows 8 i .. 8 i + 7: lane -> row l / 8, slot l % 8, chunk slot ^ ((row / 2) % 8)
    uint32_t va[BM / 8], vb[BN / 8];
    const uint32_t chunk0 = static_cast<uint32_t>((lane & 7) ^ (lane >> 4));
#pragma unroll
    for (int i = 0; i < BM / 8; ++i) {
        const int row = i * 8 + (lane >> 3), r = t.r0 + row;
        const int64_t s = r < t.end ? source_row(g, r) : -1;
        va[i] = s < 0 ? kOut : (gather ? static_cast<uint32_t>(s) : static_cast<uint32_t>(row)) * lda + (chunk0 ^ (4u * (i & 1))) * 16u;
    }
#pragma unroll
    for (int i = 0; i < BN / 8; ++i) {
        const int row = i * 8 + (lane >> 3);
        vb[i] = j0 + row < g.J ? static_cast<uint32_t>(row) * ldb + (chunk0 ^ (4u * (i & 1))) * 16u : kOut;
    }
    const uint32_t stage = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)(lds + wave * kStage)));
    auto copy = [&](int kb) __attribute__((always_inline)) {
        const uint32_t at = static_cast<uint32_t>(kb) * 128u;
        const bool tail = at + 128u > rowBytes;     // chunks past the end of the sum
        const uint32_t left = rowBytes - at;
#pragma unroll
        for (int i = 0; i < BN / 8; ++i) {
            const bool in = !tail || (chunk0 ^ (4u * (i & 1))) * 16u < left;
            copy_lds<HINT>(rb, in ? vb[i] : kOut, at, stage + static_cast<uint32_t>(BM / 8 + i) * 1024u);
        }
#pragma unroll
        for (int i = 0; i < (XDT ? 0 : BM / 8); ++i) {
            const bool in = !tail || (chunk0 ^ (4u * (i & 1))) * 16u < left;
            copy_lds<false>(ra, in ? va[i] : kOut, at, stage + static_cast<uint32_t>(i) * 1024u);
        }
    };
    // the same through registers
    constexpr int kCopies = (BM + BN) / 8;
    u32x4_t held[REG ? kCopies : 1];
    auto load = [&](int kb) __attribute__((always_inline)) {
        const uint32_t at = static_cast<uint32_t>(kb) * 128u;
        const bool tail = at + 128u > rowBytes;
#pragma unroll
        for (int q = XDT ? BM / 8 : 0; q < kCopies; ++q) {
            const uint32_t v = q < BM / 8 ? va[q < BM / 8 ? q : 0] : vb[q < BM / 8 ? 0 : q - BM / 8];
            const uint8_t *p = (q < BM / 8 ? baseA : baseB) + at + v;
            u32x4_t x{0u, 0u, 0u, 0u};
            if (v != kOut) {
                x = tail ? load16_tail<ES>(p, static_cast<int>(rowBytes) - static_cast<int>(at + (chunk0 ^ (4u * (q & 1))) * 16u)) : load16_any<ES>(p);
            }
            held[REG ? q : 0] = x;
        }
    };
    auto put = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int q = XDT ? BM / 8 : 0; q < kCopies; ++q) lds[wave * kStage + q * 64 + lane] = __builtin_bit_cast(uint4, held[REG ? q : 0]);
    };
    // scales: lane l has the row of x that its results have, 16 i + l % 16
    const_float *sw = nullptr;
    uint32_t sxAt[MT];
    const uint32_t KB = static_cast<uint32_t>((g.C + 127) / 128);
    if constexpr (F8) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int r = t.r0 + i * 16 + row16;
            const int64_t s = r < t.end ? source_row(g, r) : -1;
            sxAt[i] = s < 0 ? kOut : static_cast<uint32_t>(s) * KB;
        }
        sw = (const_float *)(g.b_scale + (static_cast<int64_t>(e) * ((g.J + 127) / 128) + j0 / 128) * KB);
    }
    struct Block {
        u32x4_t a[MT][2], b[NT][2];
        float sx[MT], sw;
    };
    const uint4 *mine = lds + wave * kStage;
    const int sw16 = (row16 >> 1) & 7;
    const int pitch = static_cast<int>(KB) * 8;                  // XDT: 16-byte chunks of a row
    const int held16 = t.end - t.r0 < BM ? t.end - t.r0 : BM;     // rows of the tile
    auto fetch = [&](Block &x, int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int slot = (grp + 4 * h) ^ sw16;
#pragma unroll
            for (int j = 0; j < NT; ++j) x.b[j][h] = __builtin_bit_cast(u32x4_t, mine[(BM + j * 16 + row16) * 8 + slot]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if constexpr (XDT != 0) {
                    x.a[i][h] = u32x4_t{0u, 0u, 0u, 0u};
                    if (row16 < held16) x.a[i][h] = __builtin_bit_cast(u32x4_t, rowsLds[row16 * pitch + kb * 8 + grp + 4 * h]);
                } else {
                    x.a[i][h] = __builtin_bit_cast(u32x4_t, mine[(i * 16 + row16) * 8 + slot]);
                }
            }
        }
    };
    auto scales = [&](Block &x, int kb) __attribute__((always_inline)) {
        if constexpr (F8) {
            x.sw = sw[kb];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if constexpr (XDT != 0) {
                    const float *scale = reinterpret_cast<const float *>(rowsLds + g.R * pitch);
                    x.sx[i] = row16 < held16 ? scale[row16 * KB + static_cast<uint32_t>(kb)] : 0.0f;
                } else {
                    x.sx[i] = sxAt[i] != kOut ? g.a_scale[sxAt[i] + static_cast<uint32_t>(kb)] : 0.0f;
                }
            }
        }
    };
    // XDT: 16 lanes quantise a block of a row
    auto quantize = [&]() __attribute__((always_inline)) {
        if constexpr (XDT != 0) {
            const bool aligned = g.lda % 8 == 0 && reinterpret_cast<uintptr_t>(g.a) % 16 == 0;
            const int units = none ? 0 : held16 * static_cast<int>(KB), sub = threadIdx.x & 15;
            for (int u = threadIdx.x >> 4; u < units; u += W * 4) {
                const int r = u / static_cast<int>(KB), kb = u - r * static_cast<int>(KB);
                const int64_t s = source_row(g, t.r0 + r), col = kb * 128 + sub * 8;
                float v[8];
                load_eight<XDT>(g.a, s * g.lda + col, s < 0 ? 0 : g.C - col, aligned, v);
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
                for (int d = 1; d < 16; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
                const float sc = block_scale(amax);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = v[i] / sc;
                reinterpret_cast<uint2 *>(rowsLds)[(r * pitch + kb * 8) * 2 + sub] =
                    make_uint2(pack_e4m3(v[0], v[1], v[2], v[3]), pack_e4m3(v[4], v[5], v[6], v[7]));
                if (sub == 0) reinterpret_cast<float *>(rowsLds + g.R * pitch)[r * KB + kb] = sc;
            }
            __syncthreads();
        }
    };

    f32x4_t acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    auto multiply = [&](const Block &x) __attribute__((always_inline)) {
        // the first operand's index runs over a lane's registers: four consecutive columns of one row
        if constexpr (F8) {
            u32x4_t a[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int s = 0; s < 4; ++s) a[i][s] = operand<CT>(x.a[i][s / 2], s & 1);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                u32x4_t b[4];
#pragma unroll
                for (int s = 0; s < 4; ++s) b[s] = operand<CT>(x.b[j][s / 2], s & 1);
                f32x4_t part[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) part[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < 4; ++s) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) part[i] = mfma<CT>(b[s], a[i][s], part[i]);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const float s = x.sx[i] * x.sw;
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(s, part[i][r], acc[j][i][r]);
                }
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) acc[j][i] = mfma<CT>(x.b[j][h], x.a[i][h], acc[j][i]);
                }
            }
        }
    };
    if (wave < blocks) {
        if constexpr (REG) {
            load(wave);
        } else {
            copy(wave);
        }
    }
    quantize();
    if (REG && wave < blocks) {
        for (int kb = wave; kb < blocks; kb += W) {
            Block x;
            scales(x, kb);
            put();
            wave_sync();
            fetch(x, kb);
            wave_sync();
            if (kb + W < blocks) load(kb + W);
            multiply(x);
        }
    } else if (wave < blocks) {
        for (int kb = wave; kb < blocks; kb += W) {
            Block x;
            scales(x, kb);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // this wave's copies of block kb have landed
            fetch(x, kb);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and left LDS before the next ones arrive there
            if (kb + W < blocks) copy(kb + W);
            multiply(x);
        }
    }

    __syncthreads();   // the sums lie over all waves' stages
    float *sums = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            *reinterpret_cast<float4 *>(sums + (wave * BM + i * 16 + row16) * kPitch + j * 16 + grp * 4) =
                make_float4(acc[j][i][0], acc[j][i][1], acc[j][i][2], acc[j][i][3]);
        }
    }
    __syncthreads();
    const bool wide = g.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(g.c) % 16 == 0;
    for (int x = threadIdx.x; x < BM * BN / 4; x += W * 64) {
        const int r = x / (BN / 4), c = x % (BN / 4) * 4;
        const int64_t row = t.r0 + r, col = j0 + c;
        if (row >= t.end || col >= g.J) continue;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float4 p = *reinterpret_cast<const float4 *>(sums + (w * BM + r) * kPitch + c);
            v[0] += p.x, v[1] += p.y, v[2] += p.z, v[3] += p.w;
        }
        store4(g, row * g.ldc + col, col, v, wide);
    }
}

template <int CT, int BM, int BN, int W, bool ANY = true, int XDT = 0>
void launch(const GroupedArgs &g, bool hint, bool any, hipStream_t stream)
{
    const int64_t tilesJ = (g.J + BN - 1) / BN;
    const unsigned tiles = static_cast<unsigned>(kudnn_max_row_tiles(g.R, g.E, BM, g.offsets != nullptr) * tilesJ);
    // the rows of a tile and their scales
    const size_t lds = XDT != 0 ? static_cast<size_t>(g.R * (kudnn_fp8_pitch(g.C) + (g.C + 127) / 128 * 4)) : 0;
    if (ANY && any) {
        grouped_stream_kernel<CT, BM, BN, W, false, ANY, XDT><<<tiles, W * 64, lds, stream>>>(g, static_cast<int>(tilesJ));
    } else if (hint) {
        grouped_stream_kernel<CT, BM, BN, W, true, false, XDT><<<tiles, W * 64, lds, stream>>>(g, static_cast<int>(tilesJ));
    } else {
        grouped_stream_kernel<CT, BM, BN, W, false, false, XDT><<<tiles, W * 64, lds, stream>>>(g, static_cast<int>(tilesJ));
    }
}

template <int CT>
void launch_tile(const GroupedArgs &g, int bm, int bn, int waves, bool hint, bool any, hipStream_t stream)
{
    if (bm == 16 && bn == 32) {
        launch<CT, 16, 32, 8>(g, hint, any, stream);
    } else if (bm == 16) {
        launch<CT, 16, 64, 8>(g, hint, any, stream);
    } else if (waves == 4) {
        launch<CT, 64, 64, 4>(g, hint, any, stream);
    } else {
        launch<CT, 64, 64, 8, false>(g, hint, any, stream);
    }
}

template <int XDT>
void launch_fused(const GroupedArgs &g, int bn, bool any, hipStream_t stream)
{
    // at most 16 rows: the weights are read once
    if (bn == 32) {
        launch<KUDNN_DT_F8E4M3, 16, 32, 8, true, XDT>(g, true, any, stream);
    } else {
        launch<KUDNN_DT_F8E4M3, 16, 64, 8, true, XDT>(g, true, any, stream);
    }
}

}  // namespace

int kudnn_launch_grouped_stream(const GroupedArgs &g, int bm, int bn, int waves, bool hint, bool any, hipStream_t stream)
{
    if (g.x_dt == KUDNN_DT_BF16) {
        launch_fused<KUDNN_DT_BF16>(g, bn, any, stream);
        return hipGetLastError() == hipSuccess ? 0 : -1;
    }
    if (g.x_dt == KUDNN_DT_F16) {
        launch_fused<KUDNN_DT_F16>(g, bn, any, stream);
        return hipGetLastError() == hipSuccess ? 0 : -1;
    }
    switch (g.dt) {
        case KUDNN_DT_BF16: launch_tile<KUDNN_DT_BF16>(g, bm, bn, waves, hint, any, stream); break;
        case KUDNN_DT_F16: launch_tile<KUDNN_DT_F16>(g, bm, bn, waves, hint, any, stream); break;
        case KUDNN_DT_F8E4M3: launch_tile<KUDNN_DT_F8E4M3>(g, bm, bn, waves, hint, any, stream); break;
        default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
