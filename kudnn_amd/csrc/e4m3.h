// Block scales and e4m3 values: shared by the quantisers and the products that quantise their rows themselves.
#ifndef KUDNN_E4M3_H
#define KUDNN_E4M3_H

#include "device_common.h"

namespace kudnn_dev {

constexpr float kInvMax = 1.0f / 448.0f, kTiny = 1.17549435e-38f;

__device__ __forceinline__ float block_scale(float amax) { return fmaxf(amax * kInvMax, kTiny); }

// Four values as e4m3 bytes, lowest first.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d)
{
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

// Eight elements from index `at` on, of which `valid` belong to the row (the rest are zeros); wide: 16-byte loads are aligned.
template <int DT>
__device__ __forceinline__ void load_eight(const void *x, int64_t at, int64_t valid, bool wide, float (&v)[8])
{
    if (wide && valid >= 8) {
        if constexpr (DT == KUDNN_DT_F32) {
            const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(x) + at);
            const float4 lo = p[0], hi = p[1];
            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
        } else {
            const uint4 r = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(x) + at);
            const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = DT == KUDNN_DT_BF16 ? u2f(w[i] << 16) : f16_to_f32(static_cast<uint16_t>(w[i]));
                v[2 * i + 1] = DT == KUDNN_DT_BF16 ? u2f(w[i] & 0xffff0000u) : f16_to_f32(static_cast<uint16_t>(w[i] >> 16));
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? load_elem(x, DT, at + i) : 0.0f;
}

}  // namespace kudnn_dev

#endif  // KUDNN_E4M3_H
