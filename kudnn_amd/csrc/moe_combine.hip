// Weighted sum of a token's experts, out[t] = sum over j of w[t][j] y[slots[t][j]], and its gradients. Both are bound by
// HBM: the forward pass reads each row of y once and writes a row per token; the backward pass reads y and dout and writes
// dy, taking the dot products of dweights on the way.
//
// A thread holds 16 bytes of a row (8 16-bit or 4 f32 values) and walks the token's k rows, so every access is a whole
// line of consecutive lanes; rows that are not whole 16-byte pieces take the same kernel with one element a thread.
// Sums over j run in j's order and dot products in a fixed tree, so results do not depend on timing.
// What passes through once is read and written non-temporally: 8192 tokens x 4 rows of 4096 bf16 take 60 us forward
// (335 MB, 5.6 TB/s; 73 us with cached accesses) and 112 us backward (604 MB, 5.4 TB/s), where a plain copy of 2 GiB reaches 4.9
// TB/s.
#include "device_common.h"
#include "moe.h"

using namespace kudnn_dev;

namespace {

constexpr int kThreads = 256;

typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef uint32_t v4u_t __attribute__((ext_vector_type(4)));

// STREAM: read or written once, so it need not stay in the caches (non-temporal).
template <int DT, int VEC, bool STREAM>
__device__ __forceinline__ void load_vec(const void *p, int64_t i, float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        v[0] = load_elem(p, DT, i);
    } else if constexpr (DT == KUDNN_DT_F32) {
        const v4f_t *at = reinterpret_cast<const v4f_t *>(static_cast<const float *>(p) + i);
#pragma unroll
        for (int h = 0; h < VEC / 4; ++h) {
            const v4f_t r = STREAM ? __builtin_nontemporal_load(at + h) : at[h];
            v[4 * h] = r.x, v[4 * h + 1] = r.y, v[4 * h + 2] = r.z, v[4 * h + 3] = r.w;
        }
    } else {
        const v4u_t *at = reinterpret_cast<const v4u_t *>(static_cast<const uint16_t *>(p) + i);
        const v4u_t r = STREAM ? __builtin_nontemporal_load(at) : *at;
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            v[2 * q] = DT == KUDNN_DT_BF16 ? u2f(w[q] << 16) : f16_to_f32(static_cast<uint16_t>(w[q]));
            v[2 * q + 1] = DT == KUDNN_DT_BF16 ? u2f(w[q] & 0xffff0000u) : f16_to_f32(static_cast<uint16_t>(w[q] >> 16));
        }
    }
}

template <int DT, int VEC>
__device__ __forceinline__ void store_vec(void *p, int64_t i, const float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        store_elem(p, DT, i, v[0]);
    } else if constexpr (DT == KUDNN_DT_F32) {
        __builtin_nontemporal_store(v4f_t{v[0], v[1], v[2], v[3]}, reinterpret_cast<v4f_t *>(static_cast<float *>(p) + i));
    } else {
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            w[q] = DT == KUDNN_DT_BF16 ? pack_bf16x2_rne(v[2 * q], v[2 * q + 1])
                                       : static_cast<uint32_t>(f32_to_f16_rne(v[2 * q])) |
                                             (static_cast<uint32_t>(f32_to_f16_rne(v[2 * q + 1])) << 16);
        }
        __builtin_nontemporal_store(v4u_t{w[0], w[1], w[2], w[3]}, reinterpret_cast<v4u_t *>(static_cast<uint16_t *>(p) + i));
    }
}

template <int DT, bool WIDE>
constexpr int vec_of() { return !WIDE ? 1 : (DT == KUDNN_DT_F32 ? 4 : 8); }

__device__ __forceinline__ int64_t slot_of(const CombineArgs &a, int64_t t, int j)
{
    const int64_t s = a.slots[t * a.k + j];
    return s >= 0 && s < a.R ? s : -1;
}

// grid: (column pieces, tokens). ODT: out's type, DT or a 16-bit type of f32 rows (a gradient whose sum over a token's slots is to be
// rounded once: 8192 x 2 rows of 4096 take 59 us so (335 MB, 5.7 TB/s), and 39 of bf16 rows).
template <int DT, int ODT, bool WIDE>
__global__ __launch_bounds__(kThreads) void combine_kernel(CombineArgs a)
{
    constexpr int VEC = vec_of<ODT, WIDE>();
    const int64_t col = (static_cast<int64_t>(blockIdx.y) * blockDim.x + threadIdx.x) * VEC;
    if (col >= a.N) return;
    for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
        float sum[VEC];
#pragma unroll
        for (int q = 0; q < VEC; ++q) sum[q] = 0.0f;
        // four rows at a time on their way; a row without a slot is not read
        for (int j0 = 0; j0 < a.k; j0 += 4) {
            float v[4][VEC], w[4];
            bool there[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t s = j0 + j < a.k ? slot_of(a, t, j0 + j) : -1;
                there[j] = s >= 0;
                w[j] = 1.0f;
                if (there[j]) {
                    if (a.weights != nullptr) w[j] = a.weights[t * a.k + j0 + j];
                    load_vec<DT, VEC, true>(a.y, s * a.ldy + col, v[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (there[j]) {
#pragma unroll
                    for (int q = 0; q < VEC; ++q) sum[q] = fmaf(w[j], v[j][q], sum[q]);
                }
            }
        }
        store_vec<ODT, VEC>(a.out, t * a.ldo + col, sum);
    }
}

// Rows of dy that no slot names are zero: workgroup `id` of `1 << shift` has the rows r with r % (1 << shift) == id, marks in LDS those that
// are named, and clears the others. Rows are dealt in turn, since a router leaves its unused rows together at the end. These workgroups
// start first and read under the others' traffic: 8192 x 4 rows of 4096 bf16 with 0, a 16th and half of the tokens without experts take 112, 110
// and 85 us (130, 231 and 956 where one workgroup counted the slots and cleared the rows past the count).
constexpr int kMarks = 131072;       // rows of a workgroup that one reading of the slots can mark: 2^25 rows of y in one

template <int DT, int VEC>
__device__ __forceinline__ void clear_unnamed(const CombineArgs &a, uint32_t id, int shift, uint32_t *named)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t slots = a.T * a.k, mine = ((a.R - 1 - id) >> shift) + 1;   // id < R
    const bool quads = reinterpret_cast<uintptr_t>(a.slots) % 16 == 0;
    float zero[VEC];
#pragma unroll
    for (int q = 0; q < VEC; ++q) zero[q] = 0.0f;
    for (int64_t base = 0; base < mine; base += kMarks) {
        const int rows = static_cast<int>(mine - base < kMarks ? mine - base : kMarks), words = (rows + 31) / 32;
        for (int w = threadIdx.x; w < words; w += kThreads) named[w] = 0u;
        __syncthreads();
        auto mark = [&](int s) __attribute__((always_inline)) {
            const int64_t at = (static_cast<int64_t>(s) >> shift) - base;
            if (s >= 0 && s < a.R && (static_cast<uint32_t>(s) & ((1u << shift) - 1u)) == id && at >= 0 && at < rows) {
                atomicOr(&named[at >> 5], 1u << (at & 31));
            }
        };
        const int64_t whole = quads ? slots / 4 : 0;
        const int4 *four = reinterpret_cast<const int4 *>(a.slots);
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < whole; i += kThreads) {
            const int4 s = four[i];
            mark(s.x), mark(s.y), mark(s.z), mark(s.w);
        }
        for (int64_t i = whole * 4 + threadIdx.x; i < slots; i += kThreads) mark(a.slots[i]);
        __syncthreads();
        for (int w = wave; w < words; w += kThreads / 64) {
            uint32_t free = ~named[w] & (rows - w * 32 >= 32 ? ~0u : (1u << (rows - w * 32)) - 1u);
            while (free != 0u) {
                const int64_t row = ((base + w * 32 + __ffs(free) - 1) << shift) + id;
                free &= free - 1u;
                for (int64_t col = lane * VEC; col < a.N; col += 64 * VEC) store_vec<DT, VEC>(a.dy, row * a.N + col, zero);
            }
        }
        __syncthreads();   // before the next marks
    }
}

// The first `1 << shift` workgroups (none with shift < 0) clear the rows that no slot names, as long as the others take; then a workgroup
// a token (at a time). Thread partials of the k dot products meet in LDS.
template <int DT, bool WIDE>
__global__ __launch_bounds__(kThreads) void combine_backward_kernel(CombineArgs a, int shift)
{
    constexpr int VEC = vec_of<DT, WIDE>();
    constexpr int kWaves = kThreads / 64;
    __shared__ float part[64][kWaves];
    __shared__ uint32_t named[kMarks / 32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t clearing = shift < 0 ? 0u : 1u << shift;
    if (blockIdx.x < clearing) {
        clear_unnamed<DT, VEC>(a, blockIdx.x, shift, named);
        return;
    }
    for (int64_t t = blockIdx.x - clearing; t < a.T; t += gridDim.x - clearing) {
        for (int j = 0; j < a.k; ++j) {
            const int64_t s = slot_of(a, t, j);
            const float w = a.weights == nullptr ? 1.0f : a.weights[t * a.k + j];
            float dot = 0.0f;
            if (s >= 0) {
                for (int64_t col = threadIdx.x * VEC; col < a.N; col += kThreads * VEC) {
                    float g[VEC], v[VEC];
                    load_vec<DT, VEC, false>(a.dout, t * a.N + col, g);
                    if (a.dweights != nullptr) {
                        load_vec<DT, VEC, true>(a.y, s * a.ldy + col, v);
#pragma unroll
                        for (int q = 0; q < VEC; ++q) dot = fmaf(g[q], v[q], dot);
                    }
                    if (a.dy != nullptr) {
#pragma unroll
                        for (int q = 0; q < VEC; ++q) v[q] = w * g[q];
                        store_vec<DT, VEC>(a.dy, s * a.N + col, v);
                    }
                }
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) dot += __shfl_xor(dot, d);
            if (lane == 0) part[j][wave] = dot;
        }
        if (a.dweights == nullptr) continue;
        __syncthreads();
        if (static_cast<int>(threadIdx.x) < a.k) {
            float dot = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) dot += part[threadIdx.x][w];
            a.dweights[t * a.k + threadIdx.x] = dot;
        }
        __syncthreads();   // before the next token's parts
    }
}

constexpr int64_t kMostTokens = int64_t(1) << 23;   // of a grid, half of what its 2^32 threads allow; more in turns

template <int DT, int ODT>
int launch(const CombineArgs &a, bool wide, hipStream_t stream)
{
    const int64_t each = wide ? vec_of<ODT, true>() : 1, waves = (a.N + 64 * each - 1) / (64 * each);
    const unsigned threads = waves < kThreads / 64 ? static_cast<unsigned>(waves) * 64 : kThreads;   // none that has no columns
    const int64_t piece = threads * each, pieces = (a.N + piece - 1) / piece;
    const dim3 grid(static_cast<unsigned>(a.T < kMostTokens ? a.T : kMostTokens), static_cast<unsigned>(pieces));
    if (wide) {
        combine_kernel<DT, ODT, true><<<grid, threads, 0, stream>>>(a);
    } else {
        combine_kernel<DT, ODT, false><<<grid, threads, 0, stream>>>(a);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

template <int DT>
int launch_backward(const CombineArgs &a, bool wide, hipStream_t stream)
{
    // clearing workgroups: a power of two, up to 256, of 64 rows each or more where there are that few
    int shift = a.dy != nullptr && a.R > 0 && a.N > 0 ? 0 : -1;
    while (shift >= 0 && shift < 8 && (int64_t(64) << shift) < a.R) ++shift;
    const unsigned grid = static_cast<unsigned>((a.T < kMostTokens ? a.T : kMostTokens) + (shift < 0 ? 0 : 1 << shift));
    if (grid == 0) {
        return 0;
    }
    if (wide) {
        combine_backward_kernel<DT, true><<<grid, kThreads, 0, stream>>>(a, shift);
    } else {
        combine_backward_kernel<DT, false><<<grid, kThreads, 0, stream>>>(a, shift);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

bool whole(const CombineArgs &a)
{
    const int64_t v = a.dt == KUDNN_DT_F32 && a.out_dt == KUDNN_DT_F32 ? 4 : 8;
    return a.N % v == 0 && a.ldy % v == 0 && a.ldo % v == 0 && aligned16(a.y) && aligned16(a.out) && aligned16(a.dout) && aligned16(a.dy);
}

}  // namespace

int kudnn_launch_moe_combine(const CombineArgs &a, hipStream_t stream)
{
    const bool wide = whole(a);
    switch (a.dt) {
        case KUDNN_DT_F32:
            switch (a.out_dt) {
                case KUDNN_DT_F32: return launch<KUDNN_DT_F32, KUDNN_DT_F32>(a, wide, stream);
                case KUDNN_DT_BF16: return launch<KUDNN_DT_F32, KUDNN_DT_BF16>(a, wide, stream);
                default: return launch<KUDNN_DT_F32, KUDNN_DT_F16>(a, wide, stream);
            }
        case KUDNN_DT_BF16: return launch<KUDNN_DT_BF16, KUDNN_DT_BF16>(a, wide, stream);
        case KUDNN_DT_F16: return launch<KUDNN_DT_F16, KUDNN_DT_F16>(a, wide, stream);
        default: return -1;
    }
}

int kudnn_launch_moe_combine_backward(const CombineArgs &a, hipStream_t stream)
{
    const bool wide = whole(a);
    switch (a.dt) {
        case KUDNN_DT_F32: return launch_backward<KUDNN_DT_F32>(a, wide, stream);
        case KUDNN_DT_BF16: return launch_backward<KUDNN_DT_BF16>(a, wide, stream);
        case KUDNN_DT_F16: return launch_backward<KUDNN_DT_F16>(a, wide, stream);
        default: return -1;
    }
}
