// Device helpers shared by the grouped product kernels: copies to LDS, operands, and which rows a workgroup has.
#ifndef KUDNN_GROUPED_COMMON_H
#define KUDNN_GROUPED_COMMON_H

#include "device_common.h"
#include "moe.h"

namespace kudnn_dev {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2v_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(4))) float const_float;

constexpr uint32_t kOut = 0xffffffffu;   // a vector offset outside every resource

// Raw buffer resource: base address, no stride, `bytes` in range, 32-bit data format.
__device__ __forceinline__ i32x4_t resource(const void *base, uint64_t bytes)
{
    const uint64_t p = reinterpret_cast<uint64_t>(base);
    i32x4_t rs;
    rs.x = __builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(p)));
    rs.y = __builtin_amdgcn_readfirstlane(static_cast<int>((p >> 32) & 0xffffu));
    rs.z = __builtin_amdgcn_readfirstlane(static_cast<int>(bytes < 0xfffffff0ull ? static_cast<uint32_t>(bytes) : 0xfffffff0u));
    rs.w = 0x00020000;
    return rs;
}

// One copy to LDS: lane l's 16 bytes at voff + soff of the resource land at lds + 16 l, zeros where voff is out of range.
// Inline asm, so that the compiler does not wait for it before other LDS reads; the waits below order it. The s_nops are the
// wait states a copy needs after VALU writes of the SGPRs it reads (v_readfirstlane) and after the write of M0.
template <bool NT>
__device__ __forceinline__ void copy_lds(i32x4_t rs, uint32_t voff, uint32_t soff, uint32_t lds)
{
    if constexpr (NT) {
        asm volatile("s_nop 4\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen nt lds"
                     ::"v"(voff), "s"(rs), "s"(lds), "s"(soff) : "memory");
    } else {
        asm volatile("s_nop 4\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen lds"
                     ::"v"(voff), "s"(rs), "s"(lds), "s"(soff) : "memory");
    }
}

// Orders LDS accesses of one wave to memory of its own.
__device__ __forceinline__ void wave_sync()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// 16 bytes at an address that is a multiple of the element size ES only.
template <int ES>
__device__ __forceinline__ u32x4_t load16_any(const uint8_t *p)
{
    struct __attribute__((packed, aligned(ES))) Any16 {
        uint32_t w[4];
    };
    const Any16 v = *reinterpret_cast<const Any16 *>(p);
    return u32x4_t{v.w[0], v.w[1], v.w[2], v.w[3]};
}

// The 16 bytes at p of which only the first `valid` (any number, also none) belong to the row, which is at least 16 long: the
// rest are zeros. It reads the row's last 16 bytes and shifts them down, so no byte past the row's end is touched.
template <int ES>
__device__ __forceinline__ u32x4_t load16_tail(const uint8_t *p, int valid)
{
    if (valid >= 16) return load16_any<ES>(p);
    if (valid <= 0) return u32x4_t{0u, 0u, 0u, 0u};
    const u32x4_t v = load16_any<ES>(p + valid - 16);
    uint64_t lo = v.x | static_cast<uint64_t>(v.y) << 32, hi = v.z | static_cast<uint64_t>(v.w) << 32;
    const int drop = (16 - valid) * 8;      // bits of the row's earlier elements
    if (drop >= 64) {
        lo = hi >> (drop - 64);
        hi = 0;
    } else {
        lo = lo >> drop | hi << (64 - drop);
        hi >>= drop;
    }
    return u32x4_t{static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi), static_cast<uint32_t>(hi >> 32)};
}

// Four e4m3 bytes as four bf16, exactly.
__device__ __forceinline__ uint2 widen4(uint32_t w)
{
    const bf16x2v_t lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
    return make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// Operand registers of one MFMA from a chunk: 16-bit types the chunk itself, e4m3 its half h.
template <int CT>
__device__ __forceinline__ u32x4_t operand(const u32x4_t &chunk, int h)
{
    if constexpr (CT == KUDNN_DT_F8E4M3) {
        const uint2 a = widen4(chunk[2 * h]), b = widen4(chunk[2 * h + 1]);
        return u32x4_t{a.x, a.y, b.x, b.y};
    } else {
        return chunk;
    }
}

__device__ __forceinline__ i32x8_t join(const u32x4_t &lo, const u32x4_t &hi)
{
    return i32x8_t{static_cast<int>(lo.x), static_cast<int>(lo.y), static_cast<int>(lo.z), static_cast<int>(lo.w),
                   static_cast<int>(hi.x), static_cast<int>(hi.y), static_cast<int>(hi.z), static_cast<int>(hi.w)};
}

// 16 x 16 sums over 128 e4m3 products (block exponents of 1).
__device__ __forceinline__ f32x4_t mfma_e4m3(const i32x8_t &a, const i32x8_t &b)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}

template <int CT>
__device__ __forceinline__ f32x4_t mfma(const u32x4_t &a, const u32x4_t &b, const f32x4_t &c)
{
    if constexpr (CT == KUDNN_DT_F16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
}


// A tile of rows of one expert. e == E: the rows that belong to no expert (before offsets[0], and past offsets[E]).
struct RowTile {
    int e, begin, end;   // the expert's rows
    int r0;              // first row of the tile
};

__device__ __forceinline__ int clamp_row(int v, int R) { return v < 0 ? 0 : (v > R ? R : v); }

// Row tiles of all experts and of the rest, as one wave sees them: 64 experts at a time, a scan over the lanes. Offsets are
// clamped to [0, R], so any contents stay inside the buffers. With up to 64 experts the offsets are read once.
// HALVES: an expert's last tile, if it has at most bm / 2 rows, is not counted among the tiles but among the halves.
template <bool HALVES = false>
class RowTiles {
public:
    __device__ __forceinline__ RowTiles(const int32_t *offsets, int E, int R, int bm) : offsets_(offsets), E_(E), R_(R), bm_(bm)
    {
        if (offsets == nullptr) {   // one group of all rows
            total_ = experts_ = whole(R);
            halves_ = half(R) ? 1 : 0;
            return;
        }
        for (int base = 0; base < E; base += 64) {
            experts_ = scan(base, experts_);
            if (base == 0) lead_ = __builtin_amdgcn_readfirstlane(lo_);    // the first expert's begin
        }
        experts_ = __builtin_amdgcn_readfirstlane(experts_);
        rest_ = __builtin_amdgcn_readlane(hi_, (E - 1) & 63);    // the last expert's end
        total_ = experts_ + (lead_ + bm - 1) / bm + (R - rest_ + bm - 1) / bm;
    }
    __device__ __forceinline__ int total() const { return total_; }
    __device__ __forceinline__ int halves() const { return halves_; }
    // Half number `want` < halves().
    __device__ __forceinline__ RowTile find_half(int want)
    {
        RowTile t{0, 0, R_, whole(R_) * bm_};
        for (int base = 0; offsets_ != nullptr && base < E_; base += 64) {
            if (E_ > 64) scan(base, 0);
            const bool mine = half(hi_ - lo_);
            const unsigned long long who = __ballot(mine);
            const int before = __builtin_popcountll(who & ((1ull << (threadIdx.x & 63)) - 1ull));
            const unsigned long long is = __ballot(mine && before == want);
            if (is != 0ull) {
                const int src = __ffsll(is) - 1;
                t.e = base + src;
                t.begin = __builtin_amdgcn_readlane(lo_, src);
                t.end = __builtin_amdgcn_readlane(hi_, src);
                t.r0 = t.begin + whole(t.end - t.begin) * bm_;
                break;
            }
            want -= __builtin_popcountll(who);
        }
        return t;
    }
    // Tile number `want` < total(). Its members are the same in every lane.
    __device__ __forceinline__ RowTile find(int want)
    {
        if (offsets_ == nullptr) {
            return RowTile{0, 0, R_, want * bm_};
        }
        // behind the experts' tiles those of the rows before them, then those past them
        const int none = want - experts_, lead = (lead_ + bm_ - 1) / bm_;
        RowTile t{E_, rest_, R_, rest_ + (none - lead) * bm_};
        if (none < lead) {
            t.begin = 0;
            t.end = lead_;
            t.r0 = none * bm_;
        }
        int before = 0;
        for (int base = 0; base < E_ && want < experts_; base += 64) {
            if (E_ > 64) before = scan(base, before);
            const unsigned long long who = __ballot(tiles_ > 0 && want >= first_ && want < first_ + tiles_);
            if (who != 0ull) {
                const int src = __ffsll(who) - 1;
                t.e = base + src;
                t.begin = __builtin_amdgcn_readlane(lo_, src);
                t.end = __builtin_amdgcn_readlane(hi_, src);
                t.r0 = t.begin + (want - __builtin_amdgcn_readlane(first_, src)) * bm_;
                break;
            }
        }
        return t;
    }

private:
    __device__ __forceinline__ bool half(int n) const { return HALVES && n > 0 && (n - 1) % bm_ < bm_ / 2; }
    __device__ __forceinline__ int whole(int n) const { return n <= 0 ? 0 : (n + bm_ - 1) / bm_ - (half(n) ? 1 : 0); }
    // Expert base + lane: its rows, its tiles, and the number of tiles before; returns the number up to the 64th.
    __device__ __forceinline__ int scan(int base, int before)
    {
        const int lane = threadIdx.x & 63, e = base + lane;
        lo_ = hi_ = 0;
        if (e < E_) {
            lo_ = clamp_row(offsets_[e], R_);
            hi_ = clamp_row(offsets_[e + 1], R_);
        }
        tiles_ = whole(hi_ - lo_);
        if constexpr (HALVES) halves_ += __builtin_popcountll(__ballot(half(hi_ - lo_)));
        int incl = tiles_;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d);
            incl += lane >= d ? o : 0;
        }
        first_ = before + incl - tiles_;
        return before + __shfl(incl, 63);
    }
    const int32_t *offsets_;
    int E_, R_, bm_, total_ = 0, experts_ = 0, lead_ = 0, rest_ = 0, halves_ = 0;
    int lo_ = 0, hi_ = 0, tiles_ = 0, first_ = 0;
};

// Four outputs of a row from column j at element `at` of C, with the bias; `wide`: a 16- or 8-byte store is aligned.
__device__ __forceinline__ void store4(const GroupedArgs &g, int64_t at, int64_t j, float (&v)[4], bool wide)
{
    if (g.bias != nullptr) {
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] += j + q < g.J ? load_elem(g.bias, g.c_dt, j + q) : 0.0f;
    }
    if (wide && j + 4 <= g.J) {
        if (g.c_dt == KUDNN_DT_F32) {
            *reinterpret_cast<float4 *>(static_cast<float *>(g.c) + at) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint32_t w[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                w[q] = g.c_dt == KUDNN_DT_BF16 ? pack_bf16x2_rne(v[2 * q], v[2 * q + 1])
                                               : static_cast<uint32_t>(f32_to_f16_rne(v[2 * q])) |
                                                     (static_cast<uint32_t>(f32_to_f16_rne(v[2 * q + 1])) << 16);
            }
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(g.c) + at) = make_uint2(w[0], w[1]);
        }
        return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (j + q < g.J) store_elem(g.c, g.c_dt, at + q, v[q]);
    }
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
