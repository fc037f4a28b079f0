// Router of a mixture of experts: softmax over the experts of each token, its k largest, and the tokens in the order of
// their experts; and the gradient of the weights.
//
// A workgroup takes 64 tokens. A group of L lanes holds a token's logits in registers (V = up to 16 a lane) and picks the
// largest k times, each time by a butterfly over the L lanes of a 64-bit key: the logit's bits, made to order as signed
// integers, above the complement of the expert's index, so that ties go to the lowest index and the result is unique.
//
// The order by expert is a counting sort without atomics whose order could change the result. A token takes an expert at
// most once, so a row's place among its workgroup's rows of one expert is the number of earlier tokens that took it: each
// expert has a 64-bit mask of the workgroup's tokens (set by atomic OR, which commutes), and the place is a population
// count. A second launch adds the counts of the earlier workgroups (bytes, at most 64 each) and of all experts before;
// a call of at most 64 tokens is one launch. The counts are read by every workgroup again (T / 64 x E bytes from L2), which
// at 16384 tokens and 128 experts costs less than a third launch that would scan them.
#include <type_traits>

#include "device_common.h"
#include "moe.h"

using namespace kudnn_dev;

namespace {

constexpr int kTokens = KUDNN_ROUTE_TOKENS, kThreads = 256;
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

struct Shared {
    unsigned long long mask[KUDNN_ROUTE_MAX_EXPERTS];  // tokens of this workgroup that took the expert
    int base[KUDNN_ROUTE_MAX_EXPERTS];                 // first row of this workgroup's rows of the expert
    int key[kTokens * KUDNN_ROUTE_MAX_K];
    short expert[kTokens * KUDNN_ROUTE_MAX_K];
    float sum[kTokens];
    int scan[kThreads / 64 + 1];
    int total;
};

// Exclusive scan over the experts of total[e], in place, by the whole workgroup (4 experts a thread); total -> offsets.
__device__ __forceinline__ void scan_experts(int (&v)[4], Shared &sh)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int mine = v[0] + v[1] + v[2] + v[3];
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
    for (int i = 0; i < 4; ++i) {
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
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = i * L + sub;
            key[i] = kClosed;
            if (e < a.E && (a.mask == nullptr || a.mask[tok * a.mask_st + e * a.mask_se] != 0)) {
                const float x = load_elem(a.logits, a.dt, tok * a.ld + e);
                key[i] = x == -__builtin_inff() ? kClosed : order_key(x);
            }
        }
        float top = 0.0f;
        if (!a.normalize) {
            int m = kClosed;
#pragma unroll
            for (int i = 0; i < V; ++i) m = max(m, key[i]);
#pragma unroll
            for (int d = 1; d < L; d <<= 1) m = max(m, __shfl_xor(m, d));
            top = key_value(m);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) s += key[i] == kClosed ? 0.0f : fast_exp(key_value(key[i]) - top);
#pragma unroll
            for (int d = 1; d < L; d <<= 1) s += __shfl_xor(s, d);
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
            int be = bi * L + sub;
#pragma unroll
            for (int d = 1; d < L; d <<= 1) {
                const int ok = __shfl_xor(bk, d), oe = __shfl_xor(be, d);
                const bool take = ok > bk || (ok == bk && oe < be);
                bk = take ? ok : bk;
                be = take ? oe : be;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = i * L + sub == be ? kClosed : key[i];
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
    int v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = threadIdx.x * 4 + i;
        v[i] = e < a.E ? __popcll(sh.mask[e]) : 0;
    }
    scan_experts(v, sh);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = threadIdx.x * 4 + i;
        if (e < a.E) {
            sh.base[e] = v[i];
            a.offsets[e] = v[i];
        }
    }
    if (threadIdx.x == 0) a.offsets[a.E] = sh.total;
    __syncthreads();
    place(a, sh, t0, n, sh.expert);
}

// Adds the counts of the workgroups: thread (column c, slice s) sums 4 experts' bytes over every S-th workgroup.
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
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * a.k; i += kThreads) {
        const int e = a.experts[t0 * a.k + i];
        if (e >= 0) atomicOr(&sh.mask[e], 1ull << (i / a.k));
    }
    const int words = a.counts_ld / 4;             // at most 256
    const int S = kThreads / words, c = threadIdx.x % words, s = threadIdx.x / words;
    if (s < S) {
        int all[4] = {0, 0, 0, 0}, bef[4] = {0, 0, 0, 0};
        const uint32_t *p = reinterpret_cast<const uint32_t *>(a.counts) + c;
#pragma unroll 8
        for (int b = s; b < blocks; b += S) {
            const uint32_t w = p[static_cast<int64_t>(b) * words];
            const bool early = b < static_cast<int>(blockIdx.x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int x = static_cast<int>((w >> (8 * i)) & 255u);
                all[i] += x;
                bef[i] += early ? x : 0;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            atomicAdd(&total[c * 4 + i], all[i]);   // integers: the order does not matter
            atomicAdd(&before[c * 4 + i], bef[i]);
        }
    }
    __syncthreads();
    int v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = total[threadIdx.x * 4 + i];
    scan_experts(v, sh);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = threadIdx.x * 4 + i;
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
__global__ __launch_bounds__(kThreads) void route_backward_kernel(RouteBackwardArgs a)
{
    const int64_t tok = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / L;
    const int sub = threadIdx.x % L;
    if (tok >= a.T) return;   // a token's lanes leave together: the shuffles below stay within L lanes
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
            if (i * L + sub == e) {
                d[i] = g;
                p[i] = w;
            }
        }
    }
    if (!a.normalize) {
        float x[V], top = -__builtin_inff(), s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = i * L + sub;
            const bool open = e < a.E && (a.mask == nullptr || a.mask[tok * a.mask_st + e * a.mask_se] != 0);
            x[i] = open ? load_elem(a.logits, a.dt, tok * a.ld + e) : -__builtin_inff();
            top = fmaxf(top, x[i]);
        }
#pragma unroll
        for (int m = 1; m < L; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            p[i] = x[i] == -__builtin_inff() ? 0.0f : fast_exp(x[i] - top);
            s += p[i];
        }
#pragma unroll
        for (int m = 1; m < L; m <<= 1) s += __shfl_xor(s, m);
        const float inv = s == 0.0f ? 0.0f : 1.0f / s;
#pragma unroll
        for (int i = 0; i < V; ++i) p[i] = p[i] == 0.0f ? 0.0f : p[i] * inv;  // 0 stays 0 beside a NaN in the sum
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = i * L + sub;
        if (e < a.E) store_elem(a.dlogits, a.dt, tok * a.E + e, p[i] == 0.0f ? 0.0f : p[i] * (d[i] - dot));
    }
}

// The lanes and registers a token takes: 8 lanes up to 128 experts, so that a wave holds 8 tokens.
template <typename F>
int with_shape(int E, F &&f)
{
    if (E <= 16) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 2>{});
    if (E <= 64) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 8>{});
    if (E <= 128) return f(std::integral_constant<int, 8>{}, std::integral_constant<int, 16>{});
    if (E <= 256) return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 16>{});
    if (E <= 512) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 16>{});
    return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{});
}

}  // namespace

int kudnn_launch_moe_route(const RouteArgs &a, hipStream_t stream)
{
    const int blocks = a.T <= kTokens ? 1 : static_cast<int>((a.T + kTokens - 1) / kTokens);  // no tokens: zero offsets
    const int single = blocks <= 1 ? 1 : 0;
    with_shape(a.E, [&](auto l, auto v) {
        route_kernel<decltype(l)::value, decltype(v)::value><<<blocks, kThreads, 0, stream>>>(a, single);
        return 0;
    });
    if (!single) {
        route_place_kernel<<<blocks, kThreads, 0, stream>>>(a, blocks);
    }
    return hipGetLastError() == hipSuccess ? 0 : -1;
}

int kudnn_launch_moe_route_backward(const RouteBackwardArgs &a, hipStream_t stream)
{
    with_shape(a.E, [&](auto l, auto v) {
        constexpr int perBlock = kThreads / decltype(l)::value;
        route_backward_kernel<decltype(l)::value, decltype(v)::value>
            <<<static_cast<unsigned>((a.T + perBlock - 1) / perBlock), kThreads, 0, stream>>>(a);
        return 0;
    });
    return hipGetLastError() == hipSuccess ? 0 : -1;
}
