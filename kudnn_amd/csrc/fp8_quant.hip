// e4m3 values with a f32 scale for each block: 1 x 128 of a row, 128 x 128 of a weight.
//   s = max(amax * r, 2^-126) with r = 1 / 448 rounded to f32,  q = round to nearest even of x / s
// The product is rounded to f32 and the division is an IEEE f32 division, so the values are the same on every machine that
// follows the definition. (A bf16 x lies on a tie between two e4m3 values in one of 16 cases where s is a power of two, so the last
// bit of s decides many roundings: the product, and not a quotient, is what torch's division by a number gives on a GPU.)
// s is at most 2^-23 of itself off amax / 448, so |x / s| stays below 464, where e4m3 would leave its range: no clamp is needed. A NaN in a block
// stays NaN and an infinity becomes one (inf / inf), which the product hands on.
// Rows are bound by HBM: x is read once, a byte an element is written (4096 x 4096 bf16: 13.6 us, 3.7 TB/s; the 50 MB leave the launch's start
// and end a third of that).
#include "e4m3.h"
#include "moe.h"

using namespace kudnn_dev;

namespace {

constexpr int kThreads = 256;

// 16 lanes a block of a row, 8 elements a lane; 16 blocks a workgroup.
template <int DT, bool WIDE>
__global__ __launch_bounds__(kThreads) void quantize_rows_kernel(const void *x, int64_t M, int64_t K, int64_t ldx, uint8_t *q,
                                                                int64_t ldq, float *scale, int zeroTail)
{
    const int64_t KB = (K + 127) / 128;
    const int64_t block = static_cast<int64_t>(blockIdx.x) * (kThreads / 16) + threadIdx.x / 16;
    if (block >= M * KB) return;   // a block's 16 lanes leave together
    const int64_t row = block / KB, kb = block - row * KB;
    const int64_t col = kb * 128 + (threadIdx.x % 16) * 8;
    float v[8];
    load_eight<DT>(x, row * ldx + col, K - col, WIDE, v);
    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
    const float s = block_scale(amax);
    if (threadIdx.x % 16 == 0) scale[row * KB + kb] = s;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] / s;
    const uint32_t lo = pack_e4m3(v[0], v[1], v[2], v[3]), hi = pack_e4m3(v[4], v[5], v[6], v[7]);
    uint8_t *out = q + row * ldq + col;
    if ((WIDE && col + 8 <= K) || (zeroTail && col + 8 <= ldq)) {
        // rows of the library's own have whole blocks; others are wide only where 8 bytes are aligned
        *reinterpret_cast<uint2 *>(out) = make_uint2(lo, hi);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (col + i < K) out[i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
        }
    }
}

// A workgroup a block of 128 x 128: 16 neighbouring elements of 16 rows at a time, one a thread, read once for the largest and again for the values.
// It runs once for a weight, not in a call: 14336 x 4096 bf16 take 98 us (1.8 TB/s of reading it once and writing the bytes).
template <int DT>
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(const void *w, int64_t N, int64_t K, int64_t we, int64_t ldw,
                                                                  uint8_t *q, float *scale)
{
    __shared__ float part[kThreads / 64];
    const int64_t kb = blockIdx.x, nb = blockIdx.y, e = blockIdx.z;
    const int64_t c0 = kb * 128 + (threadIdx.x & 15), r0 = nb * 128 + (threadIdx.x >> 4);
    float amax = 0.0f;
    for (int64_t r = r0; r < nb * 128 + 128 && r < N; r += 16) {
        for (int64_t c = c0; c < kb * 128 + 128 && c < K; c += 16) amax = fmaxf(amax, fabsf(load_elem(w, DT, e * we + r * ldw + c)));
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = amax;
    __syncthreads();
    const float s = block_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
    if (threadIdx.x == 0) scale[(e * gridDim.y + nb) * gridDim.x + kb] = s;
    for (int64_t r = r0; r < nb * 128 + 128 && r < N; r += 16) {
        for (int64_t c = c0; c < kb * 128 + 128 && c < K; c += 16) {
            const float v = load_elem(w, DT, e * we + r * ldw + c) / s;
            q[(e * N + r) * K + c] = static_cast<uint8_t>(pack_e4m3(v, v, v, v) & 255u);
        }
    }
}

template <int DT>
void launch_rows(bool wide, unsigned grid, const void *x, int64_t M, int64_t K, int64_t ldx, void *q, int64_t ldq,
                 float *scale, int zeroTail, hipStream_t stream)
{
    if (wide) {
        quantize_rows_kernel<DT, true><<<grid, kThreads, 0, stream>>>(x, M, K, ldx, static_cast<uint8_t *>(q), ldq, scale, zeroTail);
    } else {
        quantize_rows_kernel<DT, false><<<grid, kThreads, 0, stream>>>(x, M, K, ldx, static_cast<uint8_t *>(q), ldq, scale, zeroTail);
    }
}

}  // namespace

int kudnn_launch_quantize_rows(const void *x, int dt, int64_t M, int64_t K, int64_t ldx, void *q, int64_t ldq,
                               float *scale, bool zero_tail, hipStream_t stream)
{
    const int64_t blocks = M * ((K + 127) / 128);
    const unsigned grid = static_cast<unsigned>((blocks + kThreads / 16 - 1) / (kThreads / 16));
    const bool wide = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ldx % (dt == KUDNN_DT_F32 ? 4 : 8) == 0 &&
                      reinterpret_cast<uintptr_t>(q) % 8 == 0 && ldq % 8 == 0;
    switch (dt) {
        case KUDNN_DT_F32: launch_rows<KUDNN_DT_F32>(wide, grid, x, M, K, ldx, q, ldq, scale, zero_tail, stream); break;
        case KUDNN_DT_BF16: launch_rows<KUDNN_DT_BF16>(wide, grid, x, M, K, ldx, q, ldq, scale, zero_tail, stream); break;
        case KUDNN_DT_F16: launch_rows<KUDNN_DT_F16>(wide, grid, x, M, K, ldx, q, ldq, scale, zero_tail, stream); break;
        default: return -1;
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int kudnn_launch_quantize_blocks(const void *w, int dt, int64_t E, int64_t N, int64_t K, int64_t we, int64_t ldw, void *q,
                                 float *scale, hipStream_t stream)
{
    const int64_t nb = (N + 127) / 128, kb = (K + 127) / 128;
    // the grid's third dimension holds 65535: more experts go in several launches
    for (int64_t e0 = 0; e0 < E; e0 += 65535) {
        const int64_t n = E - e0 < 65535 ? E - e0 : 65535;
        const dim3 grid(static_cast<unsigned>(kb), static_cast<unsigned>(nb), static_cast<unsigned>(n));
        const int64_t size = dt == KUDNN_DT_F32 ? 4 : 2;
        const void *src = static_cast<const char *>(w) + e0 * we * size;
        uint8_t *dst = static_cast<uint8_t *>(q) + e0 * N * K;
        float *sc = scale + e0 * nb * kb;
        switch (dt) {
            case KUDNN_DT_F32: quantize_blocks_kernel<KUDNN_DT_F32><<<grid, kThreads, 0, stream>>>(src, N, K, we, ldw, dst, sc); break;
            case KUDNN_DT_BF16: quantize_blocks_kernel<KUDNN_DT_BF16><<<grid, kThreads, 0, stream>>>(src, N, K, we, ldw, dst, sc); break;
            case KUDNN_DT_F16: quantize_blocks_kernel<KUDNN_DT_F16><<<grid, kThreads, 0, stream>>>(src, N, K, we, ldw, dst, sc); break;
            default: return -1;
        }
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
