// Grouped products of any sizes, pitches and alignments: 64 x 64 tiles, the operands read one element at a time.
//
// This is the kernel behind every form for what the others leave: rows of less than 16 bytes, operands past 32-bit offsets, and gradients of
// misaligned bases or more than 65535 experts (other rows off 16-byte chunks pass through registers in the forward products and are packed for
// the gradients). A workgroup of four waves holds a 64 x 64 tile of C, each wave a 32 x 32 quarter in four 16 x 16 MFMA accumulators; 32 of the summed index at a time pass
// through LDS, masked to the operand's bounds. e4m3 values are widened to bf16, which holds them exactly; their products are
// summed within a block of 128 and then scaled into the running sum.
// Bound by the element-wise copies: the index arithmetic of 16 elements a thread and step outweighs its MFMAs (16384 rows of 32
// experts, 2048 x 2824 f16: 2.2 ms, ten times the tiled kernels' time).
#include "grouped_common.h"

using namespace kudnn_dev;

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kT = 64, kC = 32, kPitch = 40;   // tile side, summed indices a step, LDS pitch (16-bit elements)

template <int DT>
__device__ __forceinline__ uint16_t load16(const void *p, int64_t i)
{
    if constexpr (DT == KUDNN_DT_F8E4M3) {
        const uint32_t b = static_cast<const uint8_t *>(p)[i];
        return static_cast<uint16_t>(f2u(__builtin_amdgcn_cvt_f32_fp8(static_cast<int>(b), 0)) >> 16);
    } else {
        return static_cast<const uint16_t *>(p)[i];
    }
}

template <int DT, int FORM>
__global__ __launch_bounds__(256) void grouped_generic_kernel(GroupedArgs g, int tilesJ)
{
    __shared__ __align__(16) uint16_t sa[kT * kPitch], sb[kT * kPitch];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t j0 = static_cast<int64_t>(blockIdx.x % tilesJ) * kT;
    int64_t i0, iEnd, c0 = 0, cEnd = g.C, e;
    if constexpr (FORM == GROUPED_BWD_W) {
        const int64_t tilesI = (g.I + kT - 1) / kT, t = blockIdx.x / tilesJ;
        e = t / tilesI;
        i0 = (t - e * tilesI) * kT;
        iEnd = g.I;
        const int R = static_cast<int>(g.R);
        c0 = g.offsets == nullptr ? 0 : clamp_row(g.offsets[e], R);
        cEnd = g.offsets == nullptr ? R : clamp_row(g.offsets[e + 1], R);
    } else {
        RowTiles<> tiles(g.offsets, static_cast<int>(g.E), static_cast<int>(g.R), kT);
        const int want = static_cast<int>(blockIdx.x) / tilesJ;
        if (want >= tiles.total()) return;
        const RowTile t = tiles.find(want);
        e = t.e;
        i0 = t.r0;
        iEnd = t.end;
        if (g.offsets != nullptr && e == g.E) cEnd = 0;   // rows of no expert: zero
    }
    // element (row, c) of each operand: A by its row i (FWD, BWD_IN) or column i (BWD_W), B by its row or column j
    f32x4_t acc[2][2] = {}, sum[2][2] = {};
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    const int64_t KB = (g.C + 127) / 128, NB = (g.J + 127) / 128;
    for (int64_t c = c0; c < cEnd; c += kC) {
        __syncthreads();
#pragma unroll 1
        for (int x = threadIdx.x; x < kT * kC; x += 256) {
            // consecutive threads along the index that is contiguous in memory
            {
                const int ti = FORM == GROUPED_BWD_W ? x % kT : x / kC, tc = FORM == GROUPED_BWD_W ? x / kT : x % kC;
                const int64_t i = i0 + ti, cc = c + tc;
                uint16_t v = 0;
                if (i < iEnd && cc < cEnd) {
                    if constexpr (FORM == GROUPED_BWD_W) {
                        v = load16<DT>(g.a, cc * g.lda + i);
                    } else {
                        const int64_t r = FORM == GROUPED_FWD ? source_row(g, i) : i;
                        if (r >= 0) v = load16<DT>(g.a, r * g.lda + cc);
                    }
                }
                sa[ti * kPitch + tc] = v;
            }
            {
                const int tj = FORM == GROUPED_FWD ? x / kC : x % kT, tc = FORM == GROUPED_FWD ? x % kC : x / kT;
                const int64_t j = j0 + tj, cc = c + tc;
                uint16_t v = 0;
                if (j < g.J && cc < cEnd) {
                    if constexpr (FORM == GROUPED_FWD) {
                        v = load16<DT>(g.b, e * g.be + j * g.ldb + cc);
                    } else if constexpr (FORM == GROUPED_BWD_IN) {
                        v = load16<DT>(g.b, e * g.be + cc * g.ldb + j);
                    } else {
                        const int64_t r = source_row(g, cc);
                        if (r >= 0) v = load16<DT>(g.b, r * g.ldb + j);
                    }
                }
                sb[tj * kPitch + tc] = v;
            }
        }
        __syncthreads();
        uint4 fa[2], fb[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            fa[q] = *reinterpret_cast<const uint4 *>(&sa[(wi + q * 16 + (lane & 15)) * kPitch + (lane >> 4) * 8]);
            fb[q] = *reinterpret_cast<const uint4 *>(&sb[(wj + q * 16 + (lane & 15)) * kPitch + (lane >> 4) * 8]);
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                // the first operand gives the rows of the result: B's index runs over a lane's four registers
                if constexpr (DT == KUDNN_DT_F16) {
                    acc[p][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, fb[q]),
                                                                      __builtin_bit_cast(f16x8_t, fa[p]), acc[p][q], 0, 0, 0);
                } else {
                    acc[p][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, fb[q]),
                                                                       __builtin_bit_cast(bf16x8_t, fa[p]), acc[p][q], 0, 0, 0);
                }
            }
        }
        if constexpr (DT == KUDNN_DT_F8E4M3) {
            if (c % 128 == 96 || c + kC >= cEnd) {   // the end of a block of 128
                const int64_t kb = c / 128;
                const float sw = g.b_scale[(e * NB + j0 / 128) * KB + kb];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int64_t i = i0 + wi + p * 16 + (lane & 15);
                    const int64_t r = i < iEnd ? source_row(g, i) : -1;
                    const float s = r >= 0 ? g.a_scale[r * KB + kb] * sw : 0.0f;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
#pragma unroll
                        for (int v = 0; v < 4; ++v) {
                            sum[p][q][v] = fmaf(s, acc[p][q][v], sum[p][q][v]);
                            acc[p][q][v] = 0.0f;
                        }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int64_t i = i0 + wi + p * 16 + (lane & 15);
        if (i >= iEnd) continue;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int64_t j = j0 + wj + q * 16 + (lane >> 4) * 4 + v;
                if (j >= g.J) continue;
                float y = DT == KUDNN_DT_F8E4M3 ? sum[p][q][v] : acc[p][q][v];
                if (g.bias != nullptr) y += load_elem(g.bias, g.c_dt, j);
                store_elem(g.c, g.c_dt, (FORM == GROUPED_BWD_W ? e * g.ce : 0) + i * g.ldc + j, y);
            }
        }
    }
}

template <int DT, int FORM>
void launch(const GroupedArgs &g, hipStream_t stream)
{
    const int64_t tilesJ = (g.J + kT - 1) / kT;
    const int64_t tilesI = FORM == GROUPED_BWD_W ? g.E * ((g.I + kT - 1) / kT)
                                                 : kudnn_max_row_tiles(g.R, g.E, kT, g.offsets != nullptr);
    grouped_generic_kernel<DT, FORM><<<static_cast<unsigned>(tilesI * tilesJ), 256, 0, stream>>>(g, static_cast<int>(tilesJ));
}

template <int DT>
void launch_form(const GroupedArgs &g, hipStream_t stream)
{
    switch (g.form) {
        case GROUPED_FWD: launch<DT, GROUPED_FWD>(g, stream); break;
        case GROUPED_BWD_IN: launch<DT, GROUPED_BWD_IN>(g, stream); break;
        default: launch<DT, GROUPED_BWD_W>(g, stream); break;
    }
}

}  // namespace

int kudnn_launch_grouped_generic(const GroupedArgs &g, hipStream_t stream)
{
    switch (g.dt) {
        case KUDNN_DT_BF16: launch_form<KUDNN_DT_BF16>(g, stream); break;
        case KUDNN_DT_F16: launch_form<KUDNN_DT_F16>(g, stream); break;
        case KUDNN_DT_F8E4M3: launch<KUDNN_DT_F8E4M3, GROUPED_FWD>(g, stream); break;
        default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
