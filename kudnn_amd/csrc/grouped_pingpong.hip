// Grouped products on 256 x 256 tiles: the experts' Linear layers, their gradients, and the e4m3 product with block scales.
//
// The tile's sum runs over k-tiles of 128 bytes of each operand row (64 16-bit or 128 8-bit values; in the forms that sum
// over an operand's rows, 64 rows of 512 bytes). Eight waves in two groups of four: while a wave of one group issues MFMAs
// on a SIMD, its partner of the other group reads its fragments from LDS and sends the copies of later k-tiles, and a
// barrier swaps the roles (group 1 runs one phase behind). Group 0 streams operand A (double-buffered), group 1 operand B
// (triple-buffered: its partner group reads a B tile one phase longer); 5 x 32 KB fill the CU's LDS. Wave (p, g) has A's
// 64 indices from 64 p and B's 128 from 128 g of the tile.
//
//   GROUPED_FWD     A = rows of x (gathered), B = rows of W[e]; both contiguous along the sum.
//   GROUPED_BWD_IN  A = rows of dy, B = W[e] with the summed index as rows: read from LDS by transposing reads.
//   GROUPED_BWD_W   A = dy, B = x (gathered), both with the summed index, the expert's rows, as rows. Any count of rows: those
//                   past the expert's last read as zero.
//
// Every copy is a buffer load into LDS of 64 x 16 bytes. A lane's row and chunk are its vector offset, the k-tile is the
// scalar one. What lies outside - rows past the group's end or without a token, chunks past the last column or past the end
// of the sum - has a vector offset beyond the resource's range and is written as zeros, so ragged groups cost no extra
// code in the loop, and a neighbour's NaN cannot come in.
//
// e4m3: one v_mfma_*_16x16x128 covers a block of 128 for 16 x 16 outputs; its result is added to the running f32 sum times
// sx[row] sw[block]. A lane's four results share the row of x, so a k-tile costs a wave 32 MFMAs (1024 cycles), 128 fused
// multiply-adds (512) and 4 products of scales. The row scales are loaded for three k-tiles at once, a lane a row, and pass to the
// lanes that need them through ds_bpermute.
//
// Tiles of at most 128 rows ("halves") have a form of their own: their waves lie 2 x 4 over 128 x 256, and A takes half the room,
// so it is triple-buffered too. They come last in the grid, behind the whole tiles, where they fill what the last round of
// those leaves free; where that round's whole tiles, cut in two, fit one round with them, they are cut.
//
// The MFMAs bound the tiles that fill the chip several times, at the clock that the card's power leaves them (1.8 to 1.97 of 2.4
// GHz); with 256 rows of one expert or fewer a tile it is the weight's stream (grouped.h says where smaller tiles take over).
// Measured: 16384 rows of 8 experts (700 to 4700 each), 4096 x 4096 bf16: forward 495 us (1.11 PFLOP/s of the rows there are), input
// gradient 505, weight gradient 506; 16384 rows of one expert 418, 426 and 396 us (1.31 to 1.39 PFLOP/s); e4m3 4096 x 4096 x
// 11008 217 us (1.70 PFLOP/s).
#include <type_traits>
#include <utility>

#include "grouped_common.h"

using namespace kudnn_dev;

namespace {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

constexpr int kBM = 256, kBN = 256, kKC = 8, kTile = 256 * kKC;  // kTile: 16-byte chunks of a buffer (32 KB)
constexpr int kCUs = 256;         // of which each holds one workgroup
constexpr int kPitch = 68;                                        // epilogue staging: 64 columns + 4 (floats)

template <int... I, typename F>
__device__ __forceinline__ void sfor_impl(std::integer_sequence<int, I...>, F &&f)
{
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void sfor(F &&f)
{
    sfor_impl(std::make_integer_sequence<int, N>{}, f);
}

template <int N>
__device__ __forceinline__ void wait_vmcnt()
{
    // s_waitcnt: vmcnt[3:0] bits 3:0, vmcnt[5:4] bits 15:14; expcnt (7) and lgkmcnt (15) left unconstrained
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
}
__device__ __forceinline__ void wait_lgkmcnt0() { __builtin_amdgcn_s_waitcnt(0xC07F); }

__device__ __forceinline__ uint32_t lds_addr(const uint4 *p)
{
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)p));
}

// Eight outputs of a row from column j: one or two 16-byte stores where the row allows it, else element by element.
__device__ __forceinline__ void store8(const GroupedArgs &g, int64_t at, int64_t j, const float (&v)[8], bool wide)
{
    if (wide && j + 8 <= g.J) {
        if (g.c_dt == KUDNN_DT_F32) {
            float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(g.c) + at);
            p[0] = make_float4(v[0], v[1], v[2], v[3]);
            p[1] = make_float4(v[4], v[5], v[6], v[7]);
            return;
        }
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            w[q] = g.c_dt == KUDNN_DT_BF16 ? pack_bf16x2_rne(v[2 * q], v[2 * q + 1])
                                           : static_cast<uint32_t>(f32_to_f16_rne(v[2 * q])) |
                                                 (static_cast<uint32_t>(f32_to_f16_rne(v[2 * q + 1])) << 16);
        }
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(g.c) + at) = make_uint4(w[0], w[1], w[2], w[3]);
        return;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        if (j + q < g.J) store_elem(g.c, g.c_dt, at + q, v[q]);
    }
}

template <int CT, int FORM>
__global__ __launch_bounds__(512, 1) void grouped_pingpong_kernel(GroupedArgs ga, int tilesJ, int order)
{
    constexpr bool F8 = CT == KUDNN_DT_F8E4M3;
    constexpr uint32_t ES = F8 ? 1u : 2u;
    constexpr bool AK = FORM == GROUPED_BWD_W;      // A is read with the summed index as rows
    constexpr bool BK = FORM != GROUPED_FWD;        // so is B
    // tiles of at most 128 rows, or columns, take less than a whole one's time (e4m3 has no registers left for it)
    constexpr bool PARTS = !F8 && FORM != GROUPED_BWD_W;
    __shared__ uint4 a0[kTile], a1[kTile], b0[kTile], b1[kTile], b2[kTile];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = wave >> 2, p = wave & 3;
    const int R = static_cast<int>(ga.R), E = static_cast<int>(ga.E);

    // ---- which tile: A's and B's first index, the group's rows, the k-tiles
    int e, aFirst, bFirst, begin, end, sumLen;
    bool half = false;   // at most 128 of A's indices are the tile's
    if constexpr (FORM == GROUPED_BWD_W) {
        const int tilesI = static_cast<int>((ga.I + kBM - 1) / kBM), perExpert = tilesI * tilesJ;
        // all XCDs on one expert at a time: its tiles take as long as it has rows, so an expert of its own would leave the XCD
        // of the fullest one behind (8 experts of 700 to 4000 rows, 4096 x 4096: 768 us that way)
        e = static_cast<int>(blockIdx.x) / perExpert;
        int ti, tj;
        grouped_tile(xcd_remap(static_cast<int>(blockIdx.x) - e * perExpert, perExpert), tilesI, tilesJ, order, ti, tj);
        begin = clamp_row(ga.offsets[e], R);
        end = clamp_row(ga.offsets[e + 1], R);
        aFirst = ti * kBM;                          // columns of dy, C's rows
        bFirst = tj * kBN;                          // columns of x, C's columns
        sumLen = end > begin ? end - begin : 0;
    } else {
        RowTiles<PARTS> tiles(ga.offsets, E, R, kBM);
        // The halves come last, where they fill what the whole tiles' last round leaves free. If that round's tiles, cut in two,
        // and the halves fit into one round together, they are cut: a round of halves takes 0.66 of the time.
        const int whole = tiles.total() * tilesJ, halves = tiles.halves() * tilesJ, last = whole % kCUs;
        const int cut = PARTS && 2 * last + halves <= kCUs ? last : 0, uncut = whole - cut;
        int lid = static_cast<int>(blockIdx.x), ti, tj;
        if (lid >= uncut + 2 * cut + halves) return;
        half = PARTS && lid >= uncut;
        RowTile t;
        if (lid >= uncut + 2 * cut) {
            grouped_tile(xcd_remap(lid - uncut - 2 * cut, halves), tiles.halves(), tilesJ, order, ti, tj);
            t = tiles.find_half(ti);
        } else {
            const int part = lid < uncut ? 0 : lid >= uncut + cut;
            lid -= part * cut;
            const int place = lid < uncut ? xcd_remap(lid, uncut) : uncut + xcd_remap(lid - uncut, cut);
            grouped_tile(place, tiles.total(), tilesJ, order, ti, tj);
            t = tiles.find(ti);
            if (half) {
                t.r0 += part * 128;
                t.end = t.end < t.r0 + 128 ? t.end : t.r0 + 128;
            }
        }
        e = t.e;
        begin = t.r0;
        end = t.end;
        aFirst = begin;                             // rows
        bFirst = tj * kBN;                          // columns of C
        sumLen = ga.offsets != nullptr && e == E ? 0 : static_cast<int>(ga.C);   // rows of no expert: zero
    }
    constexpr int kPerTile = BK && AK ? 64 : static_cast<int>(128u / ES);       // summed indices of a k-tile
    const int nk = (sumLen + kPerTile - 1) / kPerTile;
    const int tailLen = sumLen - (nk - 1) * kPerTile;                            // summed indices of the last k-tile
    // a wave's part of the tile: from A's index aWave on and B's bWave
    const int aWave = (half ? p & 1 : p) * 64, bWave = g * 128 + (half ? (p >> 1) * 64 : 0);
    // group 1 has nothing to multiply where the tile has at most 128 of B's indices
    const int bLeft = static_cast<int>(ga.J) - bFirst;
    const bool active = !PARTS || g == 0 || bLeft > 128;
    // and the operand rows past 128 need no copies
    const bool copies = !PARTS || (g == 0 ? !half || p < 2 : BK || bLeft > 128 || p < 2);

    // ---- this wave's stream: group 0 copies A, group 1 copies B; wave p copies pieces 8 p .. 8 p + 7 of a tile.
    // Contiguous along the sum: piece q holds rows 8 q .. 8 q + 7, 128 bytes each; lane -> row l / 8, LDS slot l % 8, source
    // chunk slot ^ ((row / 2) % 8), so that the 16 lanes of a quarter-wave read 16 different slots.
    // Summed index as rows: piece q holds rows 2 q and 2 q + 1 of 512 bytes; lane -> row l / 32, source chunk
    // (l % 32) ^ (4 (row % 4)).
    const uint32_t lda = static_cast<uint32_t>(ga.lda) * ES, ldb = static_cast<uint32_t>(ga.ldb) * ES;
    uint32_t vo[8];
    int tailAt[2];      // the first summed index (or row) that this lane's chunk holds, in even and odd pieces
    uint32_t kStep;     // scalar offset of a k-tile
    i32x4_t rs;
    const uint8_t *ax = static_cast<const uint8_t *>(ga.a), *bx = static_cast<const uint8_t *>(ga.b);
    if (g == 0) {
        const uint8_t *base;
        uint64_t bytes;
        if constexpr (AK) {
            // dy [rows][N], the expert's rows
            base = ax + static_cast<uint64_t>(begin) * lda;
            bytes = static_cast<uint64_t>(sumLen) * lda;
            kStep = 64u * lda;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t q = static_cast<uint32_t>(p * 8 + j), row = 2u * q + (static_cast<uint32_t>(lane) >> 5);
                const uint32_t col = static_cast<uint32_t>(aFirst) + (((static_cast<uint32_t>(lane) & 31u) ^ (4u * (row & 3u))) * 8u);
                vo[j] = col < static_cast<uint32_t>(ga.I) ? row * lda + col * ES : kOut;
            }
            tailAt[0] = tailAt[1] = 2 * p * 8 + (lane >> 5);
        } else {
            const bool gather = ga.rows != nullptr;
            base = ax + (gather ? 0u : static_cast<uint64_t>(aFirst) * lda);
            bytes = gather ? static_cast<uint64_t>(ga.S) * lda : static_cast<uint64_t>(end - aFirst) * lda;
            kStep = 128u;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int q = p * 8 + j, row = q * 8 + (lane >> 3), r = aFirst + row;
                const uint32_t chunk = static_cast<uint32_t>((lane & 7) ^ ((row >> 1) & 7));
                uint32_t at = kOut;
                if (r < end) {
                    if (FORM == GROUPED_FWD && gather) {
                        const int64_t s = source_row(ga, r);
                        at = s >= 0 ? static_cast<uint32_t>(s) * lda + chunk * 16u : kOut;
                    } else {
                        at = static_cast<uint32_t>(row) * lda + chunk * 16u;
                    }
                }
                vo[j] = at;
            }
            tailAt[0] = ((lane & 7) ^ (lane >> 4)) * static_cast<int>(16u / ES);
            tailAt[1] = ((lane & 7) ^ (4 + (lane >> 4))) * static_cast<int>(16u / ES);
        }
        rs = resource(base, bytes);
    } else {
        if constexpr (AK) {
            // x [rows][K]: the expert's rows, or rows of all tokens when gathered
            const bool gather = ga.rows != nullptr;
            rs = resource(bx + (gather ? 0u : static_cast<uint64_t>(begin) * ldb), static_cast<uint64_t>(gather ? ga.S : sumLen) * ldb);
            kStep = gather ? 0u : 64u * ldb;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t q = static_cast<uint32_t>(p * 8 + j), row = 2u * q + (static_cast<uint32_t>(lane) >> 5);
                const uint32_t col = static_cast<uint32_t>(bFirst) + (((static_cast<uint32_t>(lane) & 31u) ^ (4u * (row & 3u))) * 8u);
                vo[j] = col < static_cast<uint32_t>(ga.J) ? (gather ? 0u : row * ldb) + col * ES : kOut;
            }
            tailAt[0] = tailAt[1] = 2 * p * 8 + (lane >> 5);
        } else if constexpr (BK) {
            // W[e] [C][J]
            rs = resource(bx + static_cast<uint64_t>(e < E ? e : 0) * static_cast<uint64_t>(ga.be) * ES, static_cast<uint64_t>(ga.C) * ldb);
            kStep = 64u * ldb;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t q = static_cast<uint32_t>(p * 8 + j), row = 2u * q + (static_cast<uint32_t>(lane) >> 5);
                const uint32_t col = static_cast<uint32_t>(bFirst) + (((static_cast<uint32_t>(lane) & 31u) ^ (4u * (row & 3u))) * 8u);
                vo[j] = col < static_cast<uint32_t>(ga.J) ? row * ldb + col * ES : kOut;
            }
            tailAt[0] = tailAt[1] = 2 * p * 8 + (lane >> 5);
        } else {
            // W[e] [J][C]
            rs = resource(bx + static_cast<uint64_t>(e < E ? e : 0) * static_cast<uint64_t>(ga.be) * ES + static_cast<uint64_t>(bFirst) * ldb,
                           static_cast<uint64_t>(kBN) * ldb);
            kStep = 128u;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int q = p * 8 + j, row = q * 8 + (lane >> 3);
                const uint32_t chunk = static_cast<uint32_t>((lane & 7) ^ ((row >> 1) & 7));
                vo[j] = bFirst + row < ga.J ? static_cast<uint32_t>(row) * ldb + chunk * 16u : kOut;
            }
            tailAt[0] = ((lane & 7) ^ (lane >> 4)) * static_cast<int>(16u / ES);
            tailAt[1] = ((lane & 7) ^ (4 + (lane >> 4))) * static_cast<int>(16u / ES);
        }
    }
    // Gathered rows of x in the weight's gradient change with the k-tile. Lane l holds the offset of row l % 16 of the wave's 16 in
    // k-tile l / 16 of four; the numbers of the next four are loaded meanwhile.
    const bool gatherK = AK && g == 1 && ga.rows != nullptr;
    uint32_t rowOff = kOut;
    int rowNext = -1;
    auto load_rows = [&](int four) __attribute__((always_inline)) {
        const int r = begin + (four * 4 + (lane >> 4)) * 64 + p * 16 + (lane & 15);
        rowNext = -1;
        if (r < end) rowNext = ga.rows[r];
    };
    auto next_rows = [&]() __attribute__((always_inline)) {
        rowOff = static_cast<uint32_t>(rowNext) < static_cast<uint32_t>(ga.S) ? static_cast<uint32_t>(rowNext) * ldb : kOut;
    };
    auto stream = [&](int t, uint32_t lds) __attribute__((always_inline)) {
        if (!copies) return;
        const uint32_t soff = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(t) * kStep);
        lds = __builtin_amdgcn_readfirstlane(lds + static_cast<uint32_t>(p * 8) * 1024u);
        if (AK && gatherK) {
            const int from = ((t & 3) * 16 + (lane >> 5)) * 4;
            uint32_t at[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) at[j] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(from + 8 * j, static_cast<int>(rowOff)));
            sfor<8>([&](auto jc) __attribute__((always_inline)) {
                constexpr int j = decltype(jc)::value;
                // the sum of offsets saturates: kOut stays kOut
                copy_lds<false>(rs, __builtin_elementwise_add_sat(at[j], vo[j]), soff, lds + static_cast<uint32_t>(j) * 1024u);
            });
        } else if (t == nk - 1 && tailLen < kPerTile) {
            // past the end of the sum: rows (2 apart from piece to piece), or chunks (whole ones: the sum is a multiple of one)
            sfor<8>([&](auto jc) __attribute__((always_inline)) {
                constexpr int j = decltype(jc)::value;
                const bool rowsAreSummed = g == 0 ? AK : BK;
                const int at = rowsAreSummed ? tailAt[0] + 2 * j : tailAt[j & 1];
                copy_lds<false>(rs, at < tailLen ? vo[j] : kOut, soff, lds + static_cast<uint32_t>(j) * 1024u);
            });
        } else {
            sfor<8>([&](auto jc) __attribute__((always_inline)) {
                constexpr int j = decltype(jc)::value;
                copy_lds<false>(rs, vo[j], soff, lds + static_cast<uint32_t>(j) * 1024u);
            });
        }
    };

    // ---- scales (e4m3): lane l holds sx of row 64 p + l for these three k-tiles and the next
    const int KB = static_cast<int>((ga.C + 127) / 128);
    float sx[2][3];
    uint32_t sxAt = kOut;
    const_float *sw = nullptr;
    if constexpr (F8) {
        const int r = aFirst + aWave + lane;
        const int64_t s = r < end ? source_row(ga, r) : -1;
        sxAt = s >= 0 ? static_cast<uint32_t>(s) * static_cast<uint32_t>(KB) : kOut;
        const int64_t NB = (ga.J + 127) / 128;
        int64_t nb = bFirst / 128 + g;
        nb = nb < NB ? nb : NB - 1;                 // a half tile past the last column: its results are not stored
        sw = (const_float *)(ga.b_scale + ((e < E ? e : 0) * NB + nb) * KB);
    }
    auto load_sx = [&](int t, float (&v)[3]) __attribute__((always_inline)) {
        v[0] = v[1] = v[2] = 0.0f;
        if (sxAt == kOut) return;
        const float *at = ga.a_scale + sxAt + static_cast<uint32_t>(t);
        if (t + 2 < nk) {
            v[0] = at[0], v[1] = at[1], v[2] = at[2];
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if (t + q < nk) v[q] = at[q];
            }
        }
    };

    // ---- fragments
    const int lrow = lane & 31, lh = lane >> 5;
    const int fsw = (lrow >> 1) & 7;
    const uint32_t kmJJ = static_cast<uint32_t>((lane & 15) >> 2);
    // transposing reads: row 8 (l / 32) + jj of the 16-row step, column bytes within 64: 16 (2 ((l / 16) & 1) + (l & 3) / 2) +
    // 8 (l & 1), the 64-byte strip XOR jj
    const uint32_t trRow = (8u * static_cast<uint32_t>(lane >> 5) + kmJJ) * 512u;
    const uint32_t trCol = 16u * (2u * static_cast<uint32_t>((lane >> 4) & 1) + static_cast<uint32_t>((lane & 3) >> 1)) + 8u * static_cast<uint32_t>(lane & 1);
    auto read_tr = [&](const uint4 *buf, uint32_t strip, int s) __attribute__((always_inline)) -> uint4 {
        typedef short v4i16_t __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) v4i16_t lds_v4i16;
        typedef __attribute__((address_space(3))) char lds_char;
        lds_char *at = (lds_char *)(const_cast<uint4 *>(buf)) + (trRow + ((strip * 64u) ^ (64u * kmJJ)) + trCol);
        const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16 *)(at + (16 * s) * 512));
        const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16 *)(at + (16 * s + 4) * 512));
        const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
        return make_uint4(l2.x, l2.y, h2.x, h2.y);
    };
    const int offA = (aWave + lrow) * kKC, offB = (bWave + lrow) * kKC;
    // e4m3: 16 rows, lane group l / 16 has chunks 2 (l / 16) and + 1
    const int row16 = lane & 15, c16 = (lane >> 4) * 2, sw16 = (row16 >> 1) & 7;
    auto read16 = [&](const uint4 *buf, int row0) __attribute__((always_inline)) -> i32x8_t {
        const uint4 lo = buf[(row0 + row16) * kKC + (c16 ^ sw16)], hi = buf[(row0 + row16) * kKC + ((c16 + 1) ^ sw16)];
        return join(__builtin_bit_cast(u32x4_t, lo), __builtin_bit_cast(u32x4_t, hi));
    };

    f32x16_t acc[4][2];      // [strip of 32 of B][strip of 32 of A]
    f32x4_t acc8[8][4];      // e4m3: [16 of B][16 of A]
    if constexpr (F8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc8[j][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[j][i][r] = 0.0f;
            }
        }
    }

    // HALF: of A's 128 indices and B's 256, a wave has 64 and 64, and A is triple-buffered as well: its tiles take half the room,
    // and half the products do not cover a copy's latency
    auto step = [&](auto ic, int t, auto halfc) __attribute__((always_inline)) {
        constexpr int I = decltype(ic)::value;
        constexpr bool HALF = decltype(halfc)::value;
        constexpr int NB = HALF ? 2 : 4, NB8 = 2 * NB;      // strips of B
        const uint4 *at = HALF ? (I % 3 == 0 ? a0 : (I % 3 == 1 ? a0 + kTile / 2 : a1)) : (I % 2 == 0 ? a0 : a1);
        const uint4 *bt = I % 3 == 0 ? b0 : (I % 3 == 1 ? b1 : b2);
        const uint32_t la = lds_addr(HALF ? (I % 3 == 0 ? a1 : (I % 3 == 1 ? a0 : a0 + kTile / 2)) : (I % 2 == 0 ? a1 : a0));
        const uint32_t lb = lds_addr(I % 3 == 0 ? b2 : (I % 3 == 1 ? b0 : b1));
        // ---- memory phase
        uint4 fa[4][2], fb[2][4];
        i32x8_t fa8[4], fb8[2];
        float s8[4];
        if constexpr (F8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) fa8[i] = read16(at, aWave + i * 16);
            const float swt = sw[t];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s8[i] = u2f(static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute((i * 16 + row16) * 4, static_cast<int>(f2u(sx[I / 3][I % 3]))))) * swt;
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (AK) {
                        fa[s][i] = read_tr(at, static_cast<uint32_t>(p * 2 + i), s);
                    } else {
                        fa[s][i] = at[offA + i * 32 * kKC + ((2 * s + lh) ^ fsw)];
                    }
                }
            }
        }
        const int tt = HALF ? t + 2 : t + 1 + g;  // group 0 copies A(t + 1), or A(t + 2) of a half, group 1 copies B(t + 2)
        if (AK && gatherK && (tt & 3) == 0) {
            next_rows();
        }
        if (tt < nk) {
            stream(tt, g == 0 ? la : lb);
        }
        // group 1 lets this phase's copies (B(t + 2)) fly and waits for the previous phase's (B(t + 1)), which group 0 reads
        // in the next phase
        if (g == 1) {
            if (t + 2 < nk) {
                wait_vmcnt<8>();
            } else {
                wait_vmcnt<0>();
            }
        }
        if constexpr (F8 && I % 3 == 0) {
            load_sx(t + 3, sx[1 - I / 3]);
        }
        if (AK && gatherK && (tt & 3) == 0) {
            load_rows((tt >> 2) + 1);
        }
        auto read_b = [&](auto slotc, auto stepc) __attribute__((always_inline)) {
            constexpr int slot = decltype(slotc)::value, s = decltype(stepc)::value;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if constexpr (BK) {
                    fb[slot][j] = read_tr(bt, static_cast<uint32_t>(bWave / 32 + j), s);
                } else {
                    fb[slot][j] = bt[offB + j * 32 * kKC + ((2 * s + lh) ^ fsw)];
                }
            }
        };
        if constexpr (F8) {
            fb8[0] = read16(bt, bWave);
        } else {
            read_b(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{});
        }
        wait_lgkmcnt0();
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        // ---- compute phase, at raised wave priority
        __builtin_amdgcn_s_setprio(1);
        if (!active) {
        } else if constexpr (F8) {
            // product m = 4 j + i of strips j of B and i of A; the sums of product m - 2 run under it
            f32x4_t part[4];
            sfor<NB8>([&](auto jc) __attribute__((always_inline)) {
                constexpr int j = decltype(jc)::value;
                if constexpr (j + 1 < NB8) {
                    fb8[(j + 1) & 1] = read16(bt, bWave + (j + 1) * 16);
                }
                asm volatile("" ::: "memory");   // keeps the later strips' reads, and their registers, behind this one's
                __builtin_amdgcn_sched_barrier(0);
                sfor<4>([&](auto ic2) __attribute__((always_inline)) {
                    constexpr int i = decltype(ic2)::value, m = 4 * j + i - 2;
                    part[i] = mfma_e4m3(fb8[j & 1], fa8[i]);
                    if constexpr (m >= 0) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc8[m / 4][m % 4][r] = fmaf(s8[m % 4], part[m % 4][r], acc8[m / 4][m % 4][r]);
                        // the sums belong here: nothing else keeps the compiler from moving all of them to the next k-tile
                        asm volatile("" : "+v"(acc8[m / 4][m % 4]));
                    }
                    __builtin_amdgcn_sched_barrier(0);
                });
                __builtin_amdgcn_sched_barrier(0);
            });
#pragma unroll
            for (int i = 2; i < 4; ++i) {
#pragma unroll
                for (int r = 0; r < 4; ++r) acc8[NB8 - 1][i][r] = fmaf(s8[i], part[i][r], acc8[NB8 - 1][i][r]);
                asm volatile("" : "+v"(acc8[NB8 - 1][i]));
            }
        } else {
            sfor<4>([&](auto sc) __attribute__((always_inline)) {
                constexpr int s = decltype(sc)::value;
                if constexpr (s + 1 < 4) {
                    read_b(std::integral_constant<int, (s + 1) & 1>{}, std::integral_constant<int, s + 1>{});
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < NB; ++j) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // the first operand's index runs over a lane's registers: the one that is contiguous in C
                        const uint4 first = fb[s & 1][j], second = fa[s][i];
                        if constexpr (CT == KUDNN_DT_BF16) {
                            acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, first),
                                                                                __builtin_bit_cast(bf16x8_t, second), acc[j][i], 0, 0, 0);
                        } else {
                            acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, first),
                                                                               __builtin_bit_cast(f16x8_t, second), acc[j][i], 0, 0, 0);
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        }
        __builtin_amdgcn_s_setprio(0);
        if (g == 0) {          // A(t + 1), which this group reads in the next phase
            if (HALF && t + 2 < nk) {
                wait_vmcnt<8>();
            } else {
                wait_vmcnt<0>();
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };

    if (nk > 0) {
        if constexpr (F8) {
            load_sx(0, sx[0]);
        }
        if (AK && gatherK) {
            load_rows(0);
            next_rows();
            load_rows(1);
        }
        stream(0, g == 0 ? lds_addr(a0) : lds_addr(b0));
        if ((g == 1 || (PARTS && half)) && nk > 1) {
            stream(1, g == 0 ? lds_addr(a0 + kTile / 2) : lds_addr(b1));
            wait_vmcnt<8>();
        } else {
            wait_vmcnt<0>();
        }
        __builtin_amdgcn_s_barrier();
        if (g == 1) {
            __builtin_amdgcn_s_barrier();  // group 1 runs one phase behind
        }
        auto run = [&](auto halfc) __attribute__((always_inline)) {
            for (int t = 0; t < nk; t += 6) {
                sfor<6>([&](auto ic) __attribute__((always_inline)) {
                    if (t + decltype(ic)::value < nk) step(ic, t + decltype(ic)::value, halfc);
                });
            }
        };
        if constexpr (PARTS) {
            if (half) {
                run(std::true_type{});
            } else {
                run(std::false_type{});
            }
        } else {
            run(std::false_type{});
        }
        if (g == 0) {
            __builtin_amdgcn_s_barrier();  // matches group 1's extra barrier at the start
        }
    }

    // ---- epilogue: units of 32 rows x 64 columns of C pass through LDS (32 x 68 floats a wave, in the tile buffers) and come
    // back 8 columns a lane: stores of whole 128-byte lines
    __syncthreads();   // every wave is done with the tile buffers
    float *stage = reinterpret_cast<float *>(wave < 3 ? a0 : (wave < 6 ? a1 : b0)) + (wave % 3) * (32 * kPitch);
    const int64_t rowW = aFirst + aWave, colW = bFirst + bWave;
    const int64_t rowEnd = FORM == GROUPED_BWD_W ? ga.I : end;
    const int64_t cBase = FORM == GROUPED_BWD_W ? e * ga.ce : 0;
    const bool wide = ga.ldc % 8 == 0 && ga.ce % 8 == 0 && reinterpret_cast<uintptr_t>(ga.c) % 16 == 0;
    const int col8 = (lane & 7) * 8, rl = lane >> 3;
    sfor<4>([&](auto uc) __attribute__((always_inline)) {
        constexpr int u = decltype(uc)::value;
        if (PARTS && u >= 2 && half) return;
        constexpr int rowU = (u % 2) * 32, colU = (u / 2) * 64;
        if constexpr (F8) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const f32x4_t v = acc8[(u / 2) * 4 + j][(u % 2) * 2 + i];
                    *reinterpret_cast<float4 *>(stage + (i * 16 + row16) * kPitch + j * 16 + (lane >> 4) * 4) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
        } else {
#pragma unroll
            for (int sh = 0; sh < 2; ++sh) {
                const f32x16_t &v = acc[2 * (u / 2) + sh][u % 2];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    *reinterpret_cast<float4 *>(stage + lrow * kPitch + sh * 32 + q * 8 + lh * 4) =
                        make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                }
            }
        }
        // the bias of this lane's columns, the same for its rows
        float bias[8];
        if constexpr (F8) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                bias[q] = ga.bias != nullptr && colW + colU + col8 + q < ga.J ? load_elem(ga.bias, ga.c_dt, colW + colU + col8 + q) : 0.0f;
            }
        }
        wave_sync();
#pragma unroll
        for (int ps = 0; ps < 4; ++ps) {
            const int64_t row = rowW + rowU + rl + ps * 8, col = colW + colU + col8;
            const float *sp = stage + (rl + ps * 8) * kPitch + col8;
            const float4 lo = *reinterpret_cast<const float4 *>(sp), hi = *reinterpret_cast<const float4 *>(sp + 4);
            float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
            if (row < rowEnd && col < ga.J) {
                if constexpr (F8) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) v[q] += bias[q];
                }
                store8(ga, cBase + row * ga.ldc + col, col, v, wide);
            }
        }
        wave_sync();
    });
}

template <int CT, int FORM>
void launch(const GroupedArgs &g, hipStream_t stream)
{
    const int64_t tilesJ = (g.J + 255) / 256;
    const int64_t tiles = FORM == GROUPED_BWD_W ? g.E * ((g.I + 255) / 256) : kudnn_max_row_tiles(g.R, g.E, 256, g.offsets != nullptr);
    // up to a round of tiles may be cut in two
    const int64_t grid = tiles * tilesJ + (CT != KUDNN_DT_F8E4M3 && FORM != GROUPED_BWD_W ? (tiles * tilesJ < kCUs / 2 ? tiles * tilesJ : kCUs / 2) : 0);
    grouped_pingpong_kernel<CT, FORM><<<static_cast<unsigned>(grid), 512, 0, stream>>>(g, static_cast<int>(tilesJ), 4);
}

template <int CT>
void launch_form(const GroupedArgs &g, hipStream_t stream)
{
    switch (g.form) {
        case GROUPED_FWD: launch<CT, GROUPED_FWD>(g, stream); break;
        case GROUPED_BWD_IN: launch<CT, GROUPED_BWD_IN>(g, stream); break;
        default: launch<CT, GROUPED_BWD_W>(g, stream); break;
    }
}

}  // namespace

bool kudnn_grouped_tiled(const GroupedArgs &g, bool whole)
{
    const int64_t es = g.dt == KUDNN_DT_F8E4M3 ? 1 : 2, chunk = whole ? 16 / es : 1;
    const int64_t span = (int64_t(1) << 32) - (int64_t(1) << 20);
    if (whole && (reinterpret_cast<uintptr_t>(g.a) % 16 != 0 || reinterpret_cast<uintptr_t>(g.b) % 16 != 0)) {
        return false;
    }
    bool ok = g.lda % chunk == 0 && g.ldb % chunk == 0;
    if (g.form == GROUPED_BWD_W) {
        // the chunks lie along both of C's indices (of a last part chunk the columns past the end are not stored); offsets of any row
        // of x and of the expert's rows
        return ok && g.offsets != nullptr && (g.a_padded || g.I % chunk == 0) && (g.b_padded || g.J % chunk == 0) &&
               g.R < span / (g.lda * es) && (g.S > g.R ? g.S : g.R) < span / (g.ldb * es);
    }
    // chunks of A lie along the sum; those of B too in the forward form, else along C's columns
    ok = ok && g.be % chunk == 0 && (g.a_padded || g.C % chunk == 0) && (g.form == GROUPED_FWD || g.b_padded || g.J % chunk == 0);
    const int64_t rowsA = g.rows != nullptr ? g.S : 256, rowsB = g.form == GROUPED_FWD ? 256 : g.C;
    return ok && rowsA < span / (g.lda * es) && rowsB < span / (g.ldb * es);
}

int kudnn_launch_grouped_pingpong(const GroupedArgs &g, hipStream_t stream)
{
    switch (g.dt) {
        case KUDNN_DT_BF16: launch_form<KUDNN_DT_BF16>(g, stream); break;
        case KUDNN_DT_F16: launch_form<KUDNN_DT_F16>(g, stream); break;
        case KUDNN_DT_F8E4M3: launch<KUDNN_DT_F8E4M3, GROUPED_FWD>(g, stream); break;
        default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
