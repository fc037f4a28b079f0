// Router of a mixture of experts: softmax over the experts of each token, its k largest, and the tokens in the order of
// their experts; and the gradient of the weights.
//
// A workgroup takes 64 tokens. A group of L lanes holds a token's logits in registers (V = up to 16 neighbours a lane, in
// 16-byte loads where the rows allow it) and picks the largest k times, each time by a butterfly over the L lanes: the larger key
// (the logit's bits, made to order as signed integers) wins, of equal ones the lower index, so the result is unique. Butterflies
// within 16 lanes are DPP moves.
//
// The order by expert is a counting sort without atomics whose order could change the result. A token takes an expert at
// most once, so a row's place among its workgroup's rows of one expert is the number of earlier tokens that took it: each
// expert has a 64-bit mask of the workgroup's tokens (set by atomic OR, which commutes), and the place is a population
// count. A second launch adds the counts of the earlier workgroups (bytes, at most 64 each) and of all experts before;
// a call of at most 64 tokens is one launch. The counts are read by every workgroup again (T / 64 x E bytes from L2), which
// at 16384 tokens and 128 experts costs less than launches that would sum and scan them (16.0 against 21.0 us a call). That grows as the square of T,
// so above 768 workgroups a launch sums each run of 128 of them, another scans those sums, and the last one reads its own run's counts
// only: 65536 tokens 40.5 us against 45.5, 262144 tokens 117 against 270, 2^20 tokens 433 against 3009 (32768 tokens: 26.2 against 23.1).
#include <type_traits>

#include "device_common.h"
#include "moe.h"

using namespace kudnn_dev;

namespace {

constexpr int kTokens = KUDNN_ROUTE_TOKENS;
// 8 lanes a token for all 64 tokens at once: with 256 threads, two after the other, 16384 x 128 took 15.6 us instead of 10.6
constexpr int kThreads = KUDNN_ROUTE_THREADS;
constexpr int kEach = KUDNN_ROUTE_MAX_EXPERTS / kThreads;   // experts of a thread in the scan over them
constexpr int kClosed = INT32_MIN;

// The logit's order as a signed integer: -0 is 0, NaN the largest.
__device__ __forceinline__ int order_key(float x)
{
    const int u = static_cast<int>(f2u(x == 0.0f ? 0.0f : x));
    return x != x ? INT32_MAX : (u < 0 ? u ^ 0x7fffffff : u);
}
__device__ __forceinline__ float key_value(int key)
{
    return key == INT32_MAX ? u2f(0x7fc00000u) : u2f(static_cast<uint32_t>(key < 0 ? key ^ 0x7fffffff : key));
}

// The value of the lane across: distance 1 and 2 within a quad; at 4 and 8 the mirrored lane, which stands for the group across
// once all lanes of each smaller group hold the same; 16 and 32 by the permute network.
template <int D>
__device__ __forceinline__ int across(int v)
{
    if constexpr (D == 1) {
        return __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, false);     // quad_perm [1, 0, 3, 2]
    } else if constexpr (D == 2) {
        return __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, false);     // quad_perm [2, 3, 0, 1]
    } else if constexpr (D == 4) {
        return __builtin_amdgcn_mov_dpp(v, 0x141, 0xf, 0xf, false);    // row_half_mirror
    } else if constexpr (D == 8) {
        return __builtin_amdgcn_mov_dpp(v, 0x140, 0xf, 0xf, false);    // row_mirror
    } else {
        return __shfl_xor(v, D);
    }
}
template <int D>
__device__ __forceinline__ float across(float v) { return u2f(static_cast<uint32_t>(across<D>(static_cast<int>(f2u(v))))); }

// f(distance) for the steps of a butterfly over L lanes.
template <int L, int D = 1, typename F>
__device__ __forceinline__ void butterfly(F &&f)
{
    if constexpr (D < L) {
        f(std::integral_constant<int, D>{});
        butterfly<L, 2 * D>(f);
    }
}

// V logits of a row from index i0 on as f32 and whether each is there and open by the mask. wide: 16-byte loads of logits, and
// loads of V mask bytes, are aligned and inside the row.
template <int V>
__device__ __forceinline__ void load_logits(const void *logits, int dt, int64_t row, int64_t ld, const uint8_t *mask, int64_t maskRow,
                                            int64_t mask_se, int i0, int E, bool wide, float (&x)[V], bool (&open)[V])
{
    if (wide && i0 + V <= E) {
        if constexpr (V >= 4) {
            if (dt == KUDNN_DT_F32) {
                const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(logits) + row * ld + i0);
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    const float4 r = p[q];
                    x[4 * q] = r.x, x[4 * q + 1] = r.y, x[4 * q + 2] = r.z, x[4 * q + 3] = r.w;
                }
            } else {
                const uint2 *p = reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(logits) + row * ld + i0);
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    const uint2 r = p[q];
                    const uint32_t w[4] = {r.x & 0xffffu, r.x >> 16, r.y & 0xffffu, r.y >> 16};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        x[4 * q + i] = dt == KUDNN_DT_BF16 ? u2f(w[i] << 16) : f16_to_f32(static_cast<uint16_t>(w[i]));
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) open[i] = true;
        if (mask != nullptr) {
            if constexpr (V >= 4) {
                const uint32_t *m = reinterpret_cast<const uint32_t *>(mask + maskRow + i0);
#pragma unroll
                for (int q = 0; q < V / 4; ++q) {
                    const uint32_t r = m[q];
#pragma unroll
                    for (int i = 0; i < 4; ++i) open[4 * q + i] = ((r >> (8 * i)) & 255u) != 0u;
                }
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = i0 + i;
        open[i] = e < E && (mask == nullptr || mask[maskRow + e * mask_se] != 0);
        x[i] = open[i] ? load_elem(logits, dt, row * ld + e) : 0.0f;
    }
}

struct Shared {
    unsigned long long mask[KUDNN_ROUTE_MAX_EXPERTS];  // tokens of this workgroup that took the expert
    int base[KUDNN_ROUTE_MAX_EXPERTS];                 // first row of this workgroup's rows of the expert
    int key[kTokens * KUDNN_ROUTE_MAX_K];
    short expert[kTokens * KUDNN_ROUTE_MAX_K];
    float sum[kTokens];
    int scan[kThreads / 64 + 1];
    int total;
};

// Exclusive scan over the experts of total[e], in place, by the whole workgroup; total -> offsets.
__device__ __forceinline__ void scan_experts(int (&v)[kEach], Shared &sh)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) mine += v[i];
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(incl, d);
        incl += lane >= d ? o : 0;
    }
    if (lane == 63) sh.scan[wave] = incl;
    __syncthreads();
    int run = incl - mine;
    for (int w = 0; w < wave; ++w) run += sh.scan[w];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int c = v[i];
        v[i] = run;
        run += c;
    }
    if (threadIdx.x == kThreads - 1) sh.total = run;
    __syncthreads();
}

// Slots and rows of this workgroup's tokens, once sh.mask and sh.base are set. `experts` as written before.
__device__ __forceinline__ void place(const RouteArgs &a, Shared &sh, int64_t t0, int n, const short *fromLds)
{
    for (int i = threadIdx.x; i < n * a.k; i += kThreads) {
        const int t = i / a.k;
        const int e = fromLds != nullptr ? fromLds[i] : a.experts[t0 * a.k + i];
        int slot = -1;
        if (e >= 0) {
            slot = sh.base[e] + __popcll(sh.mask[e] & ((1ull << t) - 1ull));
            a.rows[slot] = static_cast<int32_t>(t0 + t);
        }
        a.slots[t0 * a.k + i] = slot;
    }
    // rows that no token takes
    const int64_t all = a.T * a.k;
    for (int64_t r = sh.total + static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; r < all;
         r += static_cast<int64_t>(gridDim.x) * kThreads) {
        a.rows[r] = -1;
    }
}

// L lanes a token, V logits a lane.
template <int L, int V>
__global__ __launch_bounds__(kThreads) void route_kernel(RouteArgs a, int single)
{
    __shared__ Shared sh;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTokens;
    const int n = static_cast<int>(a.T - t0 < kTokens ? a.T - t0 : kTokens);
    for (int e = threadIdx.x; e < a.E; e += kThreads) sh.mask[e] = 0ull;
    __syncthreads();

    const int sub = threadIdx.x % L;
    for (int t = threadIdx.x / L; t < n; t += kThreads / L) {
        const int64_t tok = t0 + t;
        int key[V];
        {
            float x[V];
            bool open[V];
            load_logits<V>(a.logits, a.dt, tok, a.ld, a.mask, tok * a.mask_st, a.mask_se, sub * V, a.E, a.wide, x, open);
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = open[i] && x[i] != -__builtin_inff() ? order_key(x[i]) : kClosed;
        }
        if (!a.normalize) {
            int m = kClosed;
#pragma unroll
            for (int i = 0; i < V; ++i) m = max(m, key[i]);
            butterfly<L>([&](auto d) __attribute__((always_inline)) { m = max(m, across<decltype(d)::value>(m)); });
            const float top = key_value(m);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) s += key[i] == kClosed ? 0.0f : fast_exp(key_value(key[i]) - top);
            butterfly<L>([&](auto d) __attribute__((always_inline)) { s += across<decltype(d)::value>(s); });
            if (sub == 0) sh.sum[t] = s;
        }
        for (int j = 0; j < a.k; ++j) {
            int bk = key[0], bi = 0;
#pragma unroll
            for (int i = 1; i < V; ++i) {
                if (key[i] > bk) {
                    bk = key[i];
                    bi = i;
                }
            }
            int be = sub * V + bi;
            butterfly<L>([&](auto d) __attribute__((always_inline)) {
                const int ok = across<decltype(d)::value>(bk), oe = across<decltype(d)::value>(be);
                const bool take = ok > bk || (ok == bk && oe < be);
                bk = take ? ok : bk;
                be = take ? oe : be;
            });
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = sub * V + i == be ? kClosed : key[i];
            if (sub == 0) {
                sh.key[t * a.k + j] = bk;
                sh.expert[t * a.k + j] = static_cast<short>(bk == kClosed ? -1 : be);
                if (bk != kClosed) atomicOr(&sh.mask[be], 1ull << t);
            }
        }
    }
    __syncthreads();

    for (int i = threadIdx.x; i < n * a.k; i += kThreads) {
        const int t = i / a.k;
        float w = 0.0f;
        if (sh.key[i] != kClosed) {
            const float top = key_value(sh.key[t * a.k]);
            float s = 0.0f;
            if (a.normalize) {
                for (int j = 0; j < a.k; ++j) {
                    const int kj = sh.key[t * a.k + j];
                    s += kj == kClosed ? 0.0f : fast_exp(key_value(kj) - top);
                }
            } else {
                s = sh.sum[t];
            }
            w = fast_exp(key_value(sh.key[i]) - top) / s;
        }
        a.weights[t0 * a.k + i] = w;
        a.experts[t0 * a.k + i] = sh.expert[i];
    }
    if (!single) {
        uint8_t *out = a.counts + static_cast<int64_t>(blockIdx.x) * a.counts_ld;
        for (int e = threadIdx.x; e < a.counts_ld; e += kThreads) {
            out[e] = static_cast<uint8_t>(e < a.E ? __popcll(sh.mask[e]) : 0);
        }
        return;
    }
    int v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int e = threadIdx.x * kEach + i;
        v[i] = e < a.E ? __popcll(sh.mask[e]) : 0;
    }
    scan_experts(v, sh);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int e = threadIdx.x * kEach + i;
        if (e < a.E) {
            sh.base[e] = v[i];
            a.offsets[e] = v[i];
        }
    }
    if (threadIdx.x == 0) a.offsets[a.E] = sh.total;
    __syncthreads();
    place(a, sh, t0, n, sh.expert);
}

// Adds the counts of workgroups b0 up to b1 of the whole launch into total[], and those of them before workgroup `own` into before[] (both in
// LDS, cleared): thread (column c, slice s) sums 4 experts' bytes over every S-th workgroup.
template <bool BEFORE>
__device__ __forceinline__ void add_counts(const RouteArgs &a, int b0, int b1, int own, int *total, int *before)
{
    const int words = a.counts_ld / 4;             // at most 256
    const int S = kThreads / words, c = threadIdx.x % words, s = threadIdx.x / words;
    if (s >= S) return;
    // pairs of 16-bit sums: experts 0 and 2, 1 and 3 of the four
    static_assert(KUDNN_ROUTE_DIRECT * kTokens < 65536 && KUDNN_ROUTE_RUN <= KUDNN_ROUTE_DIRECT, "a sum of 16 bits holds the workgroups' rows");
    const uint32_t *p = reinterpret_cast<const uint32_t *>(a.counts) + c;
    uint32_t all[2] = {0u, 0u}, bef[2] = {0u, 0u};
#pragma unroll 8
    for (int b = b0 + s; b < b1; b += S) {
        const uint32_t w = p[static_cast<int64_t>(b) * words];
        const uint32_t lo = w & 0x00ff00ffu, hi = (w >> 8) & 0x00ff00ffu;
        all[0] += lo;
        all[1] += hi;
        if constexpr (BEFORE) {
            const bool early = b < own;
            bef[0] += early ? lo : 0u;
            bef[1] += early ? hi : 0u;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        atomicAdd(&total[c * 4 + i], static_cast<int>((all[i & 1] >> (16 * (i >> 1))) & 0xffffu));   // integers: in any order
        if constexpr (BEFORE) atomicAdd(&before[c * 4 + i], static_cast<int>((bef[i & 1] >> (16 * (i >> 1))) & 0xffffu));
    }
}

// Many workgroups: the rows of each run of them into sums[1 + run].
__global__ __launch_bounds__(kThreads) void route_sum_kernel(RouteArgs a, int blocks)
{
    __shared__ int total[KUDNN_ROUTE_MAX_EXPERTS];
    for (int e = threadIdx.x; e < a.counts_ld; e += kThreads) total[e] = 0;
    __syncthreads();
    const int b0 = static_cast<int>(blockIdx.x * KUDNN_ROUTE_RUN), b1 = b0 + static_cast<int>(KUDNN_ROUTE_RUN);
    add_counts<false>(a, b0, b1 < blocks ? b1 : blocks, 0, total, nullptr);
    __syncthreads();
    for (int e = threadIdx.x; e < a.counts_ld; e += kThreads) a.sums[(blockIdx.x + int64_t(1)) * a.counts_ld + e] = total[e];
}

// A lane an expert: sums[1 + run] becomes the rows of the runs before, sums[0] those of all.
__global__ __launch_bounds__(64) void route_scan_kernel(RouteArgs a, int64_t runs)
{
    const int e = static_cast<int>(blockIdx.x * 64 + threadIdx.x);
    if (e >= a.counts_ld) return;
    int32_t *at = a.sums + a.counts_ld + e;
    int before = 0;
    int64_t run = 0;
    for (; run + 16 <= runs; run += 16, at += 16 * a.counts_ld) {
        int v[16];                                   // on their way together
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = at[i * a.counts_ld];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            at[i * a.counts_ld] = before;
            before += v[i];
        }
    }
    for (; run < runs; ++run, at += a.counts_ld) {
        const int v = *at;
        *at = before;
        before += v;
    }
    a.sums[e] = before;
}

// Places the rows. SUMS: from the scanned sums of the runs and the counts of this run's workgroups, else from the counts of all workgroups.
template <bool SUMS>
__global__ __launch_bounds__(kThreads) void route_place_kernel(RouteArgs a, int blocks)
{
    __shared__ Shared sh;
    __shared__ int before[KUDNN_ROUTE_MAX_EXPERTS], total[KUDNN_ROUTE_MAX_EXPERTS];
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kTokens;
    const int n = static_cast<int>(a.T - t0 < kTokens ? a.T - t0 : kTokens);
    for (int e = threadIdx.x; e < KUDNN_ROUTE_MAX_EXPERTS; e += kThreads) {
        sh.mask[e] = 0ull;
        before[e] = 0;
        total[e] = 0;
        if (SUMS && e < a.counts_ld) {
            before[e] = a.sums[(blockIdx.x / KUDNN_ROUTE_RUN + 1) * a.counts_ld + e];
            total[e] = a.sums[e];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.k; i += kThreads) {
        const int e = a.experts[t0 * a.k + i];
        if (e >= 0) atomicOr(&sh.mask[e], 1ull << (i / a.k));
    }
    const int own = static_cast<int>(blockIdx.x);
    if constexpr (SUMS) {
        add_counts<false>(a, own / static_cast<int>(KUDNN_ROUTE_RUN) * static_cast<int>(KUDNN_ROUTE_RUN), own, 0, before, nullptr);
    } else {
        add_counts<true>(a, 0, blocks, own, total, before);
    }
    __syncthreads();
    int v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) v[i] = total[threadIdx.x * kEach + i];
    scan_experts(v, sh);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int e = threadIdx.x * kEach + i;
        sh.base[e] = v[i] + before[e];
        if (blockIdx.x == 0 && e < a.E) a.offsets[e] = v[i];
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.E] = sh.total;
    __syncthreads();
    place(a, sh, t0, n, nullptr);
}

// Gradient of the logits. L lanes a token as in the forward pass; the whole softmax p is formed again where it counts.
//   normalize: dx_e = w_e (d_e - sum d w) for the chosen, else 0.  Otherwise: dx_e = p_e (d_e - sum d p), d_e = 0 unless chosen.
template <int L, int V>
__device__ __forceinline__ void route_backward_token(const RouteBackwardArgs &a, int64_t tok)
{
    const int sub = threadIdx.x % L;
    float d[V], p[V];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = p[i] = 0.0f;
    for (int j = 0; j < a.k; ++j) {
        const int e = a.experts[tok * a.k + j];
        if (e < 0) continue;
        const float g = a.dweights[tok * a.k + j], w = a.weights[tok * a.k + j];
        dot += g * w;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (sub * V + i == e) {
                d[i] = g;
                p[i] = w;
            }
        }
    }
    if (!a.normalize) {
        float x[V], top = -__builtin_inff(), s = 0.0f;
        bool open[V];
        load_logits<V>(a.logits, a.dt, tok, a.ld, a.mask, tok * a.mask_st, a.mask_se, sub * V, a.E, a.wide, x, open);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            x[i] = open[i] ? x[i] : -__builtin_inff();
            top = fmaxf(top, x[i]);
        }
        butterfly<L>([&](auto m) __attribute__((always_inline)) { top = fmaxf(top, across<decltype(m)::value>(top)); });
#pragma unroll
        for (int i = 0; i < V; ++i) {
            p[i] = x[i] == -__builtin_inff() ? 0.0f : fast_exp(x[i] - top);
            s += p[i];
        }
        butterfly<L>([&](auto m) __attribute__((always_inline)) { s += across<decltype(m)::value>(s); });
        const float inv = s == 0.0f ? 0.0f : 1.0f / s;
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = p[i] == 0.0f ? 0.0f : p[i] * inv;  // 0 stays 0 beside a NaN in the sum
    }
    float dx[V];
#pragma unroll
    for (int i = 0; i < V; ++i) dx[i] = p[i] == 0.0f ? 0.0f : p[i] * (d[i] - dot);
    const int e0 = sub * V;
    if (V % 4 == 0 && a.wide_out && e0 + V <= a.E) {
#pragma unroll
        for (int q = 0; q < V / 4; ++q) {
            if (a.dt == KUDNN_DT_F32) {
                reinterpret_cast<float4 *>(static_cast<float *>(a.dlogits) + tok * a.E + e0)[q] =
                    make_float4(dx[4 * q], dx[4 * q + 1], dx[4 * q + 2], dx[4 * q + 3]);
            } else {
                uint32_t w[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float lo = dx[4 * q + 2 * i], hi = dx[4 * q + 2 * i + 1];
                    w[i] = a.dt == KUDNN_DT_BF16 ? pack_bf16x2_rne(lo, hi) : static_cast<uint32_t>(f32_to_f16_rne(lo)) | (static_cast<uint32_t>(f32_to_f16_rne(hi)) << 16);
                }
                reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.dlogits) + tok * a.E + e0)[q] = make_uint2(w[0], w[1]);
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (e0 + i < a.E) store_elem(a.dlogits, a.dt, tok * a.E + e0 + i, dx[i]);
    }
}

template <int L, int V>
__global__ __launch_bounds__(kThreads) void route_backward_kernel(RouteBackwardArgs a)
{
    // a token's lanes leave together: the shuffles stay within L lanes
    for (int64_t tok = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / L; tok < a.T;
         tok += static_cast<int64_t>(gridDim.x) * (kThreads / L)) {
        route_backward_token<L, V>(a, tok);
    }
}

// Whether a row's logits and mask bytes can be read 4 values at a time.
bool wide_rows(const void *logits, int dt, int64_t ld, const uint8_t *mask, int64_t mask_st, int64_t mask_se)
{
    const uintptr_t size = dt == KUDNN_DT_F32 ? 16 : 8;
    return reinterpret_cast<uintptr_t>(logits) % size == 0 && ld % 4 == 0 &&
           (mask == nullptr || (reinterpret_cast<uintptr_t>(mask) % 4 == 0 && mask_st % 4 == 0 && mask_se == 1));
}

// The lanes and registers a token takes: 8 lanes up to 128 experts, so that a wave holds 8 tokens.
template <typename F>
int with_shape(int E, F &&f)
{
    if (E <= 32) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 4>{});
    if (E <= 64) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
    if (E <= 128) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 16>{});
    if (E <= 256) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 16>{});
    if (E <= 512) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 16>{});
    return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
}

}  // namespace

int kudnn_launch_moe_route(const RouteArgs &args, hipStream_t stream)
{
    RouteArgs a = args;
    a.wide = wide_rows(a.logits, a.dt, a.ld, a.mask, a.mask_st, a.mask_se);
    const int blocks = a.T <= kTokens ? 1 : static_cast<int>((a.T + kTokens - 1) / kTokens);  // no tokens: zero offsets
    const int single = blocks <= 1 ? 1 : 0;
    with_shape(a.E, [&](auto l, auto v) {
        route_kernel<decltype(l)::value, decltype(v)::value><<<blocks, kThreads, 0, stream>>>(a, single);
        return 0;
    });
    if (blocks > KUDNN_ROUTE_DIRECT) {
        const int64_t runs = (blocks + KUDNN_ROUTE_RUN - 1) / KUDNN_ROUTE_RUN;
        route_sum_kernel<<<static_cast<unsigned>(runs), kThreads, 0, stream>>>(a, blocks);
        route_scan_kernel<<<(a.counts_ld + 63) / 64, 64, 0, stream>>>(a, runs);
        route_place_kernel<true><<<blocks, kThreads, 0, stream>>>(a, blocks);
    } else if (!single) {
        route_place_kernel<false><<<blocks, kThreads, 0, stream>>>(a, blocks);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int kudnn_launch_moe_route_backward(const RouteBackwardArgs &args, hipStream_t stream)
{
    RouteBackwardArgs a = args;
    a.wide = wide_rows(a.logits, a.dt, a.ld, a.mask, a.mask_st, a.mask_se);
    a.wide_out = a.E % 4 == 0 && reinterpret_cast<uintptr_t>(a.dlogits) % 16 == 0;
    with_shape(a.E, [&](auto l, auto v) {
        constexpr int perBlock = kThreads / decltype(l)::value;
        constexpr int64_t most = int64_t(1) << 22;    // half of what a grid's 2^32 threads allow; more tokens in turns
        const int64_t blocks = (a.T + perBlock - 1) / perBlock;
        route_backward_kernel<decltype(l)::value, decltype(v)::value>
            <<<static_cast<unsigned>(blocks < most ? blocks : most), kThreads, 0, stream>>>(a);
        return 0;
    });
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
