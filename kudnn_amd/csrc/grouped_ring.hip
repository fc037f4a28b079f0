// Grouped products of some 30 to 200 rows of an expert: tiles of BM = 64 or 128 rows and 128 columns.
//
// Between the few rows whose sum is dealt to the waves (grouped_stream.hip), where a wave that holds the whole tile would need
// too many registers, and the 256 x 256 tiles (grouped_pingpong.hip), of which so few rows fill a part only, the weight's way
// from HBM still bounds the product. The waves share the tile's blocks of 128 bytes a row in a ring of S stages in LDS; wave
// (wm, wn) has 1 / WM of the rows and 1 / WN of the columns. Per block: wait for this wave's own copies of it, one barrier (now
// everyone's have landed, and everyone is done with the block before), send the copies of the block S - 1 ahead into the
// stage that the barrier freed, read the fragments, multiply.
// Fragments, swizzle, exact e4m3 (by bf16 MFMAs) and what lies outside the operands: as in grouped_stream.hip. The row scales
// are copied to LDS as well, so that no load of the compiler's own waits for the ring.
//
// Two blocks leave room for three workgroups of 64-row tiles a CU or two of 128, whose starts and ends hide under one another's
// blocks; four blocks (one workgroup a CU) pay where there are fewer tiles than that. Measured: 64 experts of 64 rows on
// average, 2048 x 4096 e4m3 (537 MB): 137 us on 128 x 128 tiles of two blocks (4.2 TB/s); a fifth of it is the tiles' starts and ends.
#include "grouped_common.h"

using namespace kudnn_dev;

namespace {

// Waits until at most N of this wave's copies are on their way and its LDS reads are done (a block's products may sink below
// the barrier, and their reads' wait with them; the stage is overwritten after it). No LDS access moves across.
template <int N>
__device__ __forceinline__ void wait_copies()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(N) : "memory");
}

// HINT: the weights are read by one row tile (non-temporal). NATIVE: e4m3 products by the e4m3 matrix instruction.
// REG (two stages): rows of any alignment and length (16 bytes at least) go to LDS through registers, a block ahead, since a
// copy moves whole aligned chunks only.
template <int CT, int BM, int WM, int WN, int S, bool HINT, bool NATIVE, bool REG>
__global__ __launch_bounds__(WM * WN * 64) void grouped_ring_kernel(GroupedArgs g, int tilesJ)
{
    constexpr bool F8 = CT == KUDNN_DT_F8E4M3;
    constexpr int BN = 128, W = WM * WN, ES = F8 ? 1 : 2;
    constexpr int MT = BM / WM / 16, NT = BN / WN / 16;            // 16 x 16 results of a wave
    constexpr int kRows = (BM + BN) / 8, kCopies = kRows / W;       // 8-row copies of a block, and of a wave
    static_assert(kRows % W == 0, "copies are dealt evenly");
    constexpr int kScaleWaves = F8 ? BM / 64 : 0;                   // each copies the scales of 64 rows
    constexpr int kStage = (BM + BN) * 8;                           // 16-byte chunks of a stage
    __shared__ uint4 lds[S * kStage];
    __shared__ uint4 scales[F8 ? 2 * BM : 1];                       // [two runs of four blocks][row]: a word a block
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN, row16 = lane & 15, grp = lane >> 4;

    const int E = static_cast<int>(g.E);
    RowTiles<> tiles(g.offsets, E, static_cast<int>(g.R), BM);
    const int actual = tiles.total() * tilesJ;
    if (static_cast<int>(blockIdx.x) >= actual) return;
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
    const uint8_t *baseA = static_cast<const uint8_t *>(g.a) + (gather ? 0u : static_cast<uint64_t>(t.r0) * lda);
    const uint8_t *baseB = static_cast<const uint8_t *>(g.b) + static_cast<uint64_t>(e) * static_cast<uint64_t>(g.be) * ES + static_cast<uint64_t>(j0) * ldb;
    const i32x4_t ra = resource(baseA, static_cast<uint64_t>(gather ? g.S : t.end - t.r0) * lda);
    const i32x4_t rb = resource(baseB, static_cast<uint64_t>(BN) * ldb);
    // copy q = wave kCopies + i has rows 8 q .. 8 q + 7 of the stage, A's before B's: lane -> row l / 8, slot l % 8, chunk
    // slot ^ ((row / 2) % 8)
    uint32_t vo[kCopies];
    const uint32_t chunk0 = static_cast<uint32_t>((lane & 7) ^ (lane >> 4));
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
        const int q = wave * kCopies + i, row = q * 8 + (lane >> 3);
        const uint32_t c = (chunk0 ^ (4u * (q & 1))) * 16u;
        if (q < BM / 8) {
            const int r = t.r0 + row;
            const int64_t s = r < t.end ? source_row(g, r) : -1;
            vo[i] = s < 0 ? kOut : (gather ? static_cast<uint32_t>(s) : static_cast<uint32_t>(row)) * lda + c;
        } else {
            vo[i] = j0 + row - BM < g.J ? static_cast<uint32_t>(row - BM) * ldb + c : kOut;
        }
    }
    // Row scales: those of four blocks at once (of the row's last four at its end), by one lane a row. A word a block and row, copied
    // by every wave, were more requests than the operands' copies: 64 experts of 64 rows on average, 2048 x 4096, took 152 us
    // instead of 137.
    const uint32_t KB = static_cast<uint32_t>((g.C + 127) / 128);
    const int lastRun = KB > 4u ? static_cast<int>(KB) - 4 : 0;
    auto run_of = [&](int kb) __attribute__((always_inline)) { return (kb & ~3) < lastRun ? kb & ~3 : lastRun; };   // its first block
    uint32_t vs = kOut;
    i32x4_t rsc = ra;
    const_float *sw = nullptr;
    if constexpr (F8) {
        const int r = t.r0 + wave * 64 + lane;
        const int64_t s = wave < kScaleWaves && r < t.end ? source_row(g, r) : -1;
        vs = s < 0 ? kOut : static_cast<uint32_t>(s) * KB * 4u;
        rsc = resource(g.a_scale, static_cast<uint64_t>(g.S) * KB * 4u);
        sw = (const_float *)(g.b_scale + (static_cast<int64_t>(e) * ((g.J + 127) / 128) + tj) * KB);
    }
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)lds));
    auto copy = [&](int kb, int stage) __attribute__((always_inline)) {
        const uint32_t at = static_cast<uint32_t>(kb) * 128u, to = base + static_cast<uint32_t>(stage * kStage) * 16u;
        const bool tail = at + 128u > rowBytes;     // chunks past the end of the sum
        const uint32_t left = rowBytes - at;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int q = wave * kCopies + i;
            const bool in = !tail || (chunk0 ^ (4u * (q & 1))) * 16u < left;
            const uint32_t v = in ? vo[i] : kOut, at16 = to + static_cast<uint32_t>(q) * 1024u;
            if (q < BM / 8) {
                copy_lds<false>(ra, v, at, at16);
            } else {
                copy_lds<HINT>(rb, v, at, at16);
            }
        }
    };
    const uint32_t baseScales = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void *)scales));
    auto copy_scales = [&](int kb) __attribute__((always_inline)) {
        if (wave >= kScaleWaves) return;
        const int buffer = ((kb >> 2) & 1) * BM + wave * 64;
        if (KB >= 4u) {
            copy_lds<false>(rsc, vs, static_cast<uint32_t>(run_of(kb)) * 4u, baseScales + static_cast<uint32_t>(buffer) * 16u);
        } else {                                                    // rows of less than 16 bytes
            float *to = reinterpret_cast<float *>(scales + buffer + lane);
            for (uint32_t q = 0; q < KB; ++q) to[q] = vs != kOut ? g.a_scale[vs / 4u + q] : 0.0f;
        }
    };

    // the same through registers
    u32x4_t held[REG ? kCopies : 1];
    u32x4_t heldScales{0u, 0u, 0u, 0u};
    auto load = [&](int kb) __attribute__((always_inline)) {
        const uint32_t at = static_cast<uint32_t>(kb) * 128u;
        const bool tail = at + 128u > rowBytes;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
            const int q = wave * kCopies + i;
            const uint8_t *p = (q < BM / 8 ? baseA : baseB) + at + vo[i];
            u32x4_t x{0u, 0u, 0u, 0u};
            if (vo[i] != kOut) {
                x = tail ? load16_tail<ES>(p, static_cast<int>(rowBytes) - static_cast<int>(at + (chunk0 ^ (4u * (q & 1))) * 16u)) : load16_any<ES>(p);
            }
            held[REG ? i : 0] = x;
        }
        if constexpr (F8) {
            if (vs != kOut && (kb & 3) == 0) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if (static_cast<uint32_t>(run_of(kb) + q) < KB) heldScales[q] = f2u(g.a_scale[vs / 4u + static_cast<uint32_t>(run_of(kb) + q)]);
                }
            }
        }
    };
    auto put = [&](int kb, int stage) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) lds[stage * kStage + (wave * kCopies + i) * 64 + lane] = __builtin_bit_cast(uint4, held[REG ? i : 0]);
        if constexpr (F8) {
            if (wave < kScaleWaves && (kb & 3) == 0) scales[((kb >> 2) & 1) * BM + wave * 64 + lane] = __builtin_bit_cast(uint4, heldScales);
        }
    };

    f32x4_t acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int sw16 = (row16 >> 1) & 7;
    auto multiply = [&](int kb, int stage) __attribute__((always_inline)) {
        const uint4 *at = lds + stage * kStage;
        u32x4_t a[MT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < MT; ++i) a[i][h] = __builtin_bit_cast(u32x4_t, at[((wm * MT + i) * 16 + row16) * 8 + ((grp + 4 * h) ^ sw16)]);
        }
        if constexpr (F8) {
            const float *sx = reinterpret_cast<const float *>(scales + ((kb >> 2) & 1) * BM) + (kb - run_of(kb));
            const float swb = sw[kb];
            float s[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) s[i] = sx[((wm * MT + i) * 16 + row16) * 4] * swb;
            if constexpr (NATIVE) {
                // one instruction a block and 16 x 16 results; lane group g has the 16 indices of chunk g and those of g + 4
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int r = (BM + (wn * NT + j) * 16 + row16) * 8;
                    const i32x8_t b = join(__builtin_bit_cast(u32x4_t, at[r + (grp ^ sw16)]), __builtin_bit_cast(u32x4_t, at[r + ((grp + 4) ^ sw16)]));
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        const f32x4_t part = mfma_e4m3(b, join(a[i][0], a[i][1]));
#pragma unroll
                        for (int q = 0; q < 4; ++q) acc[j][i][q] = fmaf(s[i], part[q], acc[j][i][q]);
                    }
                }
                return;
            }
            u32x4_t wide[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i) {
#pragma unroll
                for (int q = 0; q < 4; ++q) wide[i][q] = operand<CT>(a[i][q / 2], q & 1);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                u32x4_t b[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4_t raw = __builtin_bit_cast(u32x4_t, at[(BM + (wn * NT + j) * 16 + row16) * 8 + ((grp + 4 * h) ^ sw16)]);
                    b[2 * h] = operand<CT>(raw, 0);
                    b[2 * h + 1] = operand<CT>(raw, 1);
                }
                f32x4_t part[MT];
#pragma unroll
                for (int i = 0; i < MT; ++i) part[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
#pragma unroll
                    for (int i = 0; i < MT; ++i) part[i] = mfma<CT>(b[q], wide[i][q], part[i]);
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[j][i][r] = fmaf(s[i], part[i][r], acc[j][i][r]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x4_t b = __builtin_bit_cast(u32x4_t, at[(BM + (wn * NT + j) * 16 + row16) * 8 + ((grp + 4 * h) ^ sw16)]);
#pragma unroll
                    for (int i = 0; i < MT; ++i) acc[j][i] = mfma<CT>(b, a[i][h], acc[j][i]);
                }
            }
        }
    };

    if constexpr (REG) {
        static_assert(S == 2, "one block in use, one written");
        if (blocks > 0) {
            load(0);
            put(0, 0);
            if (blocks > 1) load(1);
        }
        for (int kb = 0; kb < blocks; ++kb) {
            __syncthreads();     // block kb is written, block kb - 1 has been read
            if (kb + 1 < blocks) put(kb + 1, (kb + 1) & 1);
            if (kb + 2 < blocks) load(kb + 2);
            multiply(kb, kb & 1);
        }
    }
    if (F8 && !REG && blocks > 0) copy_scales(0);
#pragma unroll
    for (int s = 0; s < S - 1 && !REG; ++s) {
        if (s < blocks) copy(s, s);
    }
    int stage = 0;
    for (int kb = 0; kb < blocks && !REG; ++kb) {
        // blocks kb + 1 .. kb + S - 2 may still be on their way (scales were sent at least S - 1 blocks ago)
        if (kb + S - 2 < blocks) {
            wait_copies<(S - 2) * kCopies>();
        } else {
            wait_copies<0>();
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int freed = stage == 0 ? S - 1 : stage - 1;
        if (F8 && (kb & 3) == 0 && kb + 4 < blocks) copy_scales(kb + 4);
        if (kb + S - 1 < blocks) copy(kb + S - 1, freed);
        multiply(kb, stage);
        stage = stage == S - 1 ? 0 : stage + 1;
    }

    const bool wide = g.ldc % 4 == 0 && reinterpret_cast<uintptr_t>(g.c) % 16 == 0;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t row = t.r0 + (wm * MT + i) * 16 + row16;
        if (row >= t.end) continue;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int64_t col = j0 + (wn * NT + j) * 16 + grp * 4;
            if (col >= g.J) continue;
            float v[4] = {acc[j][i][0], acc[j][i][1], acc[j][i][2], acc[j][i][3]};
            store4(g, row * g.ldc + col, col, v, wide);
        }
    }
}

template <int CT, int BM, int WM, int WN, int S, bool NATIVE>
void launch(const GroupedArgs &g, bool hint, hipStream_t stream)
{
    const int64_t tilesJ = (g.J + 127) / 128;
    const unsigned tiles = static_cast<unsigned>(kudnn_max_row_tiles(g.R, g.E, BM, g.offsets != nullptr) * tilesJ);
    if (hint) {
        grouped_ring_kernel<CT, BM, WM, WN, S, true, NATIVE, false><<<tiles, WM * WN * 64, 0, stream>>>(g, static_cast<int>(tilesJ));
    } else {
        grouped_ring_kernel<CT, BM, WM, WN, S, false, NATIVE, false><<<tiles, WM * WN * 64, 0, stream>>>(g, static_cast<int>(tilesJ));
    }
}

template <int CT, int BM, int WM, int WN, bool NATIVE>
void launch_any(const GroupedArgs &g, hipStream_t stream)
{
    const int64_t tilesJ = (g.J + 127) / 128;
    const unsigned tiles = static_cast<unsigned>(kudnn_max_row_tiles(g.R, g.E, BM, g.offsets != nullptr) * tilesJ);
    grouped_ring_kernel<CT, BM, WM, WN, 2, false, NATIVE, true><<<tiles, WM * WN * 64, 0, stream>>>(g, static_cast<int>(tilesJ));
}

template <int CT, bool NATIVE = false>
void launch_tile(const GroupedArgs &g, int bm, int stages, bool hint, bool any, hipStream_t stream)
{
    if (any && bm == 64) {
        launch_any<CT, 64, 2, 2, NATIVE>(g, stream);
    } else if (any) {
        launch_any<CT, 128, 2, 4, NATIVE>(g, stream);
    } else if (bm == 64) {
        launch<CT, 64, 2, 2, 2, NATIVE>(g, hint, stream);
    } else if (stages == 2) {
        launch<CT, 128, 2, 4, 2, NATIVE>(g, hint, stream);
    } else {
        launch<CT, 128, 2, 4, 4, NATIVE>(g, hint, stream);
    }
}

}  // namespace

int kudnn_launch_grouped_ring(const GroupedArgs &g, int bm, int stages, bool native, bool hint, bool any, hipStream_t stream)
{
    switch (g.dt) {
        case KUDNN_DT_BF16: launch_tile<KUDNN_DT_BF16>(g, bm, stages, hint, any, stream); break;
        case KUDNN_DT_F16: launch_tile<KUDNN_DT_F16>(g, bm, stages, hint, any, stream); break;
        case KUDNN_DT_F8E4M3:
            if (native) {
                launch_tile<KUDNN_DT_F8E4M3, true>(g, bm, stages, hint, any, stream);
            } else {
                launch_tile<KUDNN_DT_F8E4M3>(g, bm, stages, hint, any, stream);
            }
            break;
        default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
