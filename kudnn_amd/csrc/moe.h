// Kernel arguments and launchers of the mixture-of-experts operators. A launcher returns 0, or -1 if the launch failed.
#ifndef KUDNN_MOE_H
#define KUDNN_MOE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/kudnn_hip.h"

// ---- router (moe_route.hip)

constexpr int KUDNN_ROUTE_MAX_EXPERTS = 1024, KUDNN_ROUTE_MAX_K = 32;
constexpr int KUDNN_ROUTE_TOKENS = 64;  // tokens of a workgroup: one bit each in an expert's 64-bit mask
constexpr int KUDNN_ROUTE_THREADS = 512;  // of a workgroup
// Calls of more workgroups sum the counts of each run of KUDNN_ROUTE_RUN and scan the sums in launches of their own (moe_route.hip).
constexpr int64_t KUDNN_ROUTE_DIRECT = 768, KUDNN_ROUTE_RUN = 128;

struct RouteArgs {
    const void *logits;
    const uint8_t *mask;          // nullptr: every expert is open
    int64_t T, ld, mask_st, mask_se;
    int E, k, dt, normalize;
    float *weights;
    int32_t *experts, *offsets, *rows, *slots;
    uint8_t *counts;              // [workgroups][counts_ld]: a workgroup's rows of each expert; unused with one workgroup
    int counts_ld;
    int32_t *sums;                // more than KUDNN_ROUTE_DIRECT workgroups: [1 + runs][counts_ld], all rows of each expert, then those before a run
    bool wide;                    // set by the launcher: rows can be read 4 values at a time
};
int kudnn_launch_moe_route(const RouteArgs &a, hipStream_t stream);

struct RouteBackwardArgs {
    const void *logits;
    const uint8_t *mask;
    int64_t T, ld, mask_st, mask_se;
    int E, k, dt, normalize;
    const float *weights, *dweights;
    const int32_t *experts;
    void *dlogits;                // dense [T][E]
    bool wide, wide_out;          // set by the launcher: rows can be read and written 4 values at a time
};
int kudnn_launch_moe_route_backward(const RouteBackwardArgs &a, hipStream_t stream);

// ---- weighted sum (moe_combine.hip)

struct CombineArgs {
    const void *y, *dout;
    const float *weights;         // nullptr: ones
    const int32_t *slots;
    void *out, *dy;
    float *dweights;
    int64_t T, R, N, ldy, ldo;    // ldo: row pitch of out (dout and dy are dense)
    int k, dt, out_dt;            // out_dt: dt, or 16 bits of f32 rows (forward)
};
int kudnn_launch_moe_combine(const CombineArgs &a, hipStream_t stream);
int kudnn_launch_moe_combine_backward(const CombineArgs &a, hipStream_t stream);

// ---- block quantisation (fp8_quant.hip)

// 8-bit rows made by the library for its own products: whole blocks of 128, zero past K.
inline int64_t kudnn_fp8_pitch(int64_t K) { return (K + 127) / 128 * 128; }
// zero_tail: columns K .. ldq - 1 (up to the end of the last block) are written as zeros.
int kudnn_launch_quantize_rows(const void *x, int dt, int64_t M, int64_t K, int64_t ldx, void *q, int64_t ldq,
                               float *scale, bool zero_tail, hipStream_t stream);
int kudnn_launch_quantize_blocks(const void *w, int dt, int64_t E, int64_t N, int64_t K, int64_t we, int64_t ldw, void *q,
                                 float *scale, hipStream_t stream);

// ---- grouped products (grouped_*.hip)

// C = A x B^T in one of three forms. Rows r of expert e are offsets[e] .. offsets[e + 1] - 1 of [0, R).
//   GROUPED_FWD     C[r][j] = sum over c of A[row(r)][c] B[e][j][c]       I = rows, J = N, C = K
//   GROUPED_BWD_IN  C[r][j] = sum over c of A[r][c] B[e][c][j]            I = rows, J = K, C = N
//   GROUPED_BWD_W   C[e][i][j] = sum over r of A[r][i] B[row(r)][j]       I = N, J = K, C = rows
// row(r) = rows[r] if rows is given, else r.
enum { GROUPED_FWD = 0, GROUPED_BWD_IN = 1, GROUPED_BWD_W = 2 };

struct GroupedArgs {
    const void *a, *b;
    void *c;
    const float *a_scale, *b_scale;  // e4m3 operands: [S][KB] and [E][NB][KB]
    const void *bias;                // of C's type, or nullptr
    const int32_t *offsets;          // nullptr: one group of all rows
    const int32_t *rows;             // nullptr: row(r) = r
    int64_t R, S;                    // rows of the order by expert; rows of the gathered operand
    int64_t E, I, J, C;              // I: R for the first two forms; C: unused for the last
    int64_t lda, ldb, ldc;           // row pitches in elements
    int64_t be, ce;                  // pitch of an expert in B (first two forms), in C (last)
    int form, dt, c_dt;              // dt: BF16, F16 or F8E4M3 (GROUPED_FWD only)
    int x_dt;                        // not 0: A is not quantised yet but of this 16-bit type (a_scale unused); see below
    bool a_padded, b_padded;         // the operand's rows (packed by the library) hold zeros up to a whole 16-byte chunk
};

// Most row tiles that offsets of any contents in order can make: each group of rows leaves at most one part tile.
inline int64_t kudnn_max_row_tiles(int64_t R, int64_t E, int64_t bm, bool grouped)
{
    if (!grouped) return (R + bm - 1) / bm;
    const int64_t groups = E + 2 < R ? E + 2 : R;   // with the rows before the experts' and those past them
    // n groups of which every one has a part tile: (R - n) / bm whole ones besides, at most
    return groups + (R - groups) / bm;
}

// Any sizes, pitches and alignments (grouped_generic.hip).
int kudnn_launch_grouped_generic(const GroupedArgs &g, hipStream_t stream);
// Whether offsets within an operand fit 32 bits, as every kernel but the generic one needs, and (`whole`) the operands are whole
// 16-byte chunks, as the copies to LDS need (grouped_pingpong.hip).
bool kudnn_grouped_tiled(const GroupedArgs &g, bool whole);
// 256 x 256 tiles (grouped_pingpong.hip); e4m3 products by the e4m3 matrix instruction.
int kudnn_launch_grouped_pingpong(const GroupedArgs &g, hipStream_t stream);
// GROUPED_FWD of few rows, the sum dealt to the waves (grouped_stream.hip); products exact in f32. Tiles (bm, bn) and waves:
// (16, 32) and (16, 64) with 8, (64, 64) with 4 or (not `any`) 8. hint: the weights are read by one row tile. any: operands that are not
// whole chunks, of rows of 16 bytes or more.
// With g.x_dt: e4m3 products whose workgroups quantise their rows of x themselves, 16 rows a tile (kudnn_grouped_fused).
int kudnn_launch_grouped_stream(const GroupedArgs &g, int bm, int bn, int waves, bool hint, bool any, hipStream_t stream);
// GROUPED_FWD on tiles of bm (64 or 128) rows and 128 columns, a ring of 2 or (128 rows, not `any`) 4 stages (grouped_ring.hip).
// native: e4m3 products by the e4m3 matrix instruction, else exact in f32.
int kudnn_launch_grouped_ring(const GroupedArgs &g, int bm, int stages, bool native, bool hint, bool any, hipStream_t stream);

#endif  // KUDNN_MOE_H
