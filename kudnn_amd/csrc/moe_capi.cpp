// C ABI of the mixture-of-experts operators: descriptor checks in *_create, pointer checks and the launch in *_run.
// Plans hold sizes only, so a plan may run on several streams at once; workspaces are the caller's.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <new>
#include <string>

#include "../../include/kudnn_hip.h"
#include "grouped.h"
#include "kernels.h"
#include "moe.h"
#include "plan_base.h"

using kudnn_host::DeviceMemory;

struct kudnn_moe_route_plan : PlanBase {
    kudnn_moe_route_plan() : PlanBase(PLAN_MOE_ROUTE) {}
    int64_t T = 0, ld = 0, maskSt = 0, maskSe = 0, sumsAt = 0, workspace = 0;
    int E = 0, k = 0, dt = 0, normalize = 0, countsLd = 0;
    bool masked = false;
};

struct kudnn_grouped_linear_plan : PlanBase {
    kudnn_grouped_linear_plan() : PlanBase(PLAN_GROUPED_LINEAR) {}
    int64_t S = 0, R = 0, E = 0, K = 0, N = 0, ldx = 0, ldw = 0, we = 0, ldy = 0;
    int dt = 0;
    bool gather = false;
    // gradients: rows that are not whole 16-byte chunks are packed to a pitch that is (0: read in place). Byte offsets in
    // the workspace: dy at 0, then w (gradient of x) or x (gradient of w)
    int64_t packDy = 0, packW = 0, packX = 0, second = 0, workspace = 0;
};

struct kudnn_linear_fp8_plan : PlanBase {
    kudnn_linear_fp8_plan() : PlanBase(PLAN_LINEAR_FP8) {}
    int64_t S = 0, R = 0, E = 0, K = 0, N = 0, ldx = 0, ldw = 0, we = 0, ldy = 0, scaleOffset = 0, workspace = 0;
    int xdt = 0, ydt = 0;
    bool grouped = false, gather = false, hasBias = false, fused = false;   // fused: the product quantises x itself
};

struct kudnn_moe_combine_plan : PlanBase {
    kudnn_moe_combine_plan() : PlanBase(PLAN_MOE_COMBINE) {}
    int64_t T = 0, R = 0, N = 0, ldy = 0, ldo = 0;
    int k = 0, dt = 0, outDt = 0;
};

namespace {

using kudnn_host::SetError;

int Bad(const char *msg) { return SetError(KUDNN_STATUS_BAD_ARGUMENTS, msg); }
int Unsupported(const char *msg) { return SetError(KUDNN_STATUS_UNSUPPORTED, msg); }
int Null(const char *msg) { return SetError(KUDNN_STATUS_NULL_POINTER, msg); }

bool IsFloat(int dt) { return dt == KUDNN_DT_F32 || dt == KUDNN_DT_F16 || dt == KUDNN_DT_BF16; }
bool IsHalf(int dt) { return dt == KUDNN_DT_F16 || dt == KUDNN_DT_BF16; }

constexpr int64_t kMaxRows = INT32_MAX;      // row numbers are 32-bit
constexpr int64_t kMaxSide = int64_t(1) << 24;  // widths
constexpr int64_t kMaxExperts = int64_t(1) << 20;

// A {rows, cols} matrix with contiguous rows: its row pitch, or -1.
int64_t RowPitch(const kudnn_tensor_desc &d)
{
    if (d.ndims != 2 || d.dims[0] < 0 || d.dims[1] < 0 || (d.dims[1] > 1 && d.strides[1] != 1)) {
        return -1;
    }
    if (d.dims[0] <= 1) {
        return d.dims[1];
    }
    return d.strides[0] >= d.dims[1] ? d.strides[0] : -1;
}

// A {E, K, N} weight held as [N][K] for each expert, rows contiguous: its row and expert pitch.
bool WeightPitch(const kudnn_tensor_desc &d, int64_t &ldw, int64_t &we)
{
    if (d.ndims != 3 || (d.dims[1] > 1 && d.strides[1] != 1)) {
        return false;
    }
    ldw = d.dims[2] <= 1 ? d.dims[1] : d.strides[2];
    we = d.dims[0] <= 1 ? d.dims[2] * ldw : d.strides[0];
    return ldw >= d.dims[1] && (d.dims[0] <= 1 || we >= (d.dims[2] - 1) * ldw + d.dims[1]);
}

// Aligned for the element type: kernels read elements whole.
bool ElemAligned(const void *p, int dt)
{
    const uintptr_t a = dt == KUDNN_DT_F32 || dt == KUDNN_DT_S32 ? 4 : (dt == KUDNN_DT_F8E4M3 || dt == KUDNN_DT_U8 ? 1 : 2);
    return reinterpret_cast<uintptr_t>(p) % a == 0;
}

struct Buffer {
    const void *p;
    int dt;
};
// Every buffer is device memory and aligned to its elements (null ones have been refused where they are needed).
template <int N>
int CheckBuffers(const Buffer (&b)[N])
{
    for (const Buffer &x : b) {
        if (x.p == nullptr) {
            continue;
        }
        if (!DeviceMemory(x.p)) {
            return Bad("mixture of experts: every buffer must be device memory");
        }
        if (!ElemAligned(x.p, x.dt)) {
            return Bad("mixture of experts: a buffer is not aligned to its element type");
        }
    }
    return KUDNN_STATUS_SUCCESS;
}

// The forward kernel of a product from aligned bases, for describe().
std::string TileName(int64_t R, int64_t groups, int64_t N, int64_t K, int64_t lda, int64_t ldb, int dt, int c_dt)
{
    const int64_t whole = dt == KUDNN_DT_F8E4M3 ? 16 : 8;
    if (R == 0) {
        return "";
    }
    if (K < whole) {
        return " tile=generic";
    }
    const bool any = K % whole != 0 || lda % whole != 0 || ldb % whole != 0;
    const GroupedTile t = kudnn_grouped_rule(R, groups < R ? groups : R, N, K, dt, c_dt, any);
    return std::string(" tile=") + (t.kind == GroupedTile::STREAM ? "stream" : (t.kind == GroupedTile::RING ? "ring" : "pingpong")) +
           std::to_string(t.bm) + "x" + std::to_string(t.bn) + (t.form > 0 ? "/" + std::to_string(t.form) : "") + (any ? " any" : "") +
           (t.native || (dt == KUDNN_DT_F8E4M3 && t.kind == GroupedTile::PINGPONG) ? " e4m3" : "");
}

// Rows of a 16-bit operand packed to a pitch of `pitch` elements, zeros past the row.
int Pack(const void *src, int dt, int64_t rows, int64_t cols, int64_t ld, int64_t batches, int64_t bs, void *dst, int64_t pitch,
         hipStream_t stream)
{
    PackArgs p{};
    p.src = src;
    p.src_dt = p.dst_dt = dt;
    p.rows = rows;
    p.cols = cols;
    p.s_r = ld;
    p.s_k = 1;
    p.bdim[0] = p.bdim[1] = 1;
    p.bdim[2] = batches;
    p.bs[2] = bs;
    p.dst = dst;
    p.kp = pitch;
    p.dst_bstride = rows * pitch;
    return rows == 0 ? 0 : kudnn_launch_pack(p, batches, stream);
}

int Launched(int rc, const char *what)
{
    return rc == 0 ? KUDNN_STATUS_SUCCESS : SetError(KUDNN_STATUS_HIP_ERROR, what);
}

// No exception leaves a C entry.
template <typename F>
int Guard(F &&f) noexcept
{
    try {
        return f();
    } catch (const std::bad_alloc &) {
        return SetError(KUDNN_STATUS_ALLOC_FAILED, "out of host memory");
    } catch (...) {
        return SetError(KUDNN_STATUS_INTERNAL, "unexpected exception");
    }
}

}  // namespace

extern "C" {

// ---- router

int kudnn_moe_route_create(const kudnn_tensor_desc *logits, const kudnn_tensor_desc *mask, int top_k, int normalize,
                           kudnn_moe_route_t *plan)
{
    return Guard([&]() -> int {
        if (logits == nullptr || plan == nullptr) {
            return Null("router: null argument");
        }
        *plan = nullptr;
        const int64_t ld = RowPitch(*logits);
        if (ld < 0) {
            return Bad("router: logits must be a {tokens, experts} matrix with contiguous rows");
        }
        const int64_t T = logits->dims[0], E = logits->dims[1];
        if (!IsFloat(logits->dtype)) {
            return Unsupported("router: logits must be f32, bf16 or f16");
        }
        if (E < 1 || E > KUDNN_ROUTE_MAX_EXPERTS) {
            return Unsupported("router: 1 to 1024 experts");
        }
        if (top_k < 1 || top_k > E) {
            return Bad("router: top_k must be between 1 and the number of experts");
        }
        if (top_k > KUDNN_ROUTE_MAX_K) {
            return Unsupported("router: top_k of at most 32");
        }
        // the grid's threads must stay below 2^32 (the gradient's goes over the tokens in turns)
        if (T > kMaxRows || T * top_k > kMaxRows ||
            !kudnn_grid_fits((T + KUDNN_ROUTE_TOKENS - 1) / KUDNN_ROUTE_TOKENS, KUDNN_ROUTE_THREADS)) {
            return Unsupported("router: too many tokens");
        }
        auto p = new kudnn_moe_route_plan();
        if (mask != nullptr && mask->ndims != 0) {
            if (mask->ndims != 2 || mask->dtype != KUDNN_DT_U8 || (mask->dims[0] != T && mask->dims[0] != 1) ||
                (mask->dims[1] != E && mask->dims[1] != 1)) {
                delete p;
                return Bad("router: mask must be u8 of {tokens or 1, experts or 1}");
            }
            p->masked = true;
            p->maskSt = mask->dims[0] == 1 ? 0 : mask->strides[0];
            p->maskSe = mask->dims[1] == 1 ? 0 : mask->strides[1];
        }
        p->T = T;
        p->E = static_cast<int>(E);
        p->ld = ld;
        p->k = top_k;
        p->dt = logits->dtype;
        p->normalize = normalize != 0 ? 1 : 0;
        p->countsLd = static_cast<int>((E + 3) / 4 * 4);
        const int64_t blocks = (T + KUDNN_ROUTE_TOKENS - 1) / KUDNN_ROUTE_TOKENS;
        const int64_t runs = blocks > KUDNN_ROUTE_DIRECT ? (blocks + KUDNN_ROUTE_RUN - 1) / KUDNN_ROUTE_RUN : 0;
        p->sumsAt = blocks * p->countsLd;
        p->workspace = blocks > 1 ? p->sumsAt + (runs > 0 ? (runs + 1) * p->countsLd * static_cast<int64_t>(sizeof(int32_t)) : 0) : 0;
        p->desc = "moe_route T=" + std::to_string(T) + " E=" + std::to_string(E) + " k=" + std::to_string(top_k) +
                  (runs > 0 ? " launches=4" : (p->workspace > 0 ? " launches=2" : " launches=1"));
        *plan = p;
        return KUDNN_STATUS_SUCCESS;
    });
}

int64_t kudnn_moe_route_workspace_bytes(kudnn_moe_route_t plan) { return plan == nullptr ? 0 : plan->workspace; }

int kudnn_moe_route_run(kudnn_moe_route_t plan, const void *logits, const void *mask, float *weights, int32_t *experts,
                        int32_t *offsets, int32_t *rows, int32_t *slots, void *workspace, void *stream)
{
    if (plan == nullptr) {
        return Null("router: null plan");
    }
    const bool some = plan->T > 0;
    if (offsets == nullptr || (some && (logits == nullptr || weights == nullptr || experts == nullptr || rows == nullptr ||
                                        slots == nullptr)) ||
        (some && plan->masked && mask == nullptr) || (plan->workspace > 0 && workspace == nullptr)) {
        return Null("router: one of the buffers is nullptr");
    }
    if (!plan->masked && mask != nullptr) {
        return Bad("router: a mask was given to a plan made without one");
    }
    const int s = CheckBuffers({Buffer{logits, plan->dt}, Buffer{mask, KUDNN_DT_U8}, Buffer{weights, KUDNN_DT_F32},
                                Buffer{experts, KUDNN_DT_S32}, Buffer{offsets, KUDNN_DT_S32}, Buffer{rows, KUDNN_DT_S32},
                                Buffer{slots, KUDNN_DT_S32}, Buffer{workspace, KUDNN_DT_S32}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    RouteArgs a{};
    a.logits = logits;
    a.mask = plan->masked ? static_cast<const uint8_t *>(mask) : nullptr;
    a.T = plan->T;
    a.ld = plan->ld;
    a.mask_st = plan->maskSt;
    a.mask_se = plan->maskSe;
    a.E = plan->E;
    a.k = plan->k;
    a.dt = plan->dt;
    a.normalize = plan->normalize;
    a.weights = weights;
    a.experts = experts;
    a.offsets = offsets;
    a.rows = rows;
    a.slots = slots;
    a.counts = static_cast<uint8_t *>(workspace);
    a.counts_ld = plan->countsLd;
    a.sums = reinterpret_cast<int32_t *>(a.counts + plan->sumsAt);
    return Launched(kudnn_launch_moe_route(a, static_cast<hipStream_t>(stream)), "router: launch failed");
}

int kudnn_moe_route_backward(kudnn_moe_route_t plan, const void *logits, const void *mask, const float *weights,
                             const int32_t *experts, const float *dweights, void *dlogits, void *stream)
{
    if (plan == nullptr) {
        return Null("router: null plan");
    }
    if (plan->T == 0) {
        return KUDNN_STATUS_SUCCESS;
    }
    const bool whole = plan->normalize == 0;   // forms the softmax again
    if (weights == nullptr || experts == nullptr || dweights == nullptr || dlogits == nullptr || (whole && logits == nullptr) ||
        (whole && plan->masked && mask == nullptr)) {
        return Null("router: one of the buffers is nullptr");
    }
    const int s = CheckBuffers({Buffer{logits, plan->dt}, Buffer{mask, KUDNN_DT_U8}, Buffer{weights, KUDNN_DT_F32},
                                Buffer{experts, KUDNN_DT_S32}, Buffer{dweights, KUDNN_DT_F32}, Buffer{dlogits, plan->dt}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    RouteBackwardArgs a{};
    a.logits = logits;
    a.mask = plan->masked ? static_cast<const uint8_t *>(mask) : nullptr;
    a.T = plan->T;
    a.ld = plan->ld;
    a.mask_st = plan->maskSt;
    a.mask_se = plan->maskSe;
    a.E = plan->E;
    a.k = plan->k;
    a.dt = plan->dt;
    a.normalize = plan->normalize;
    a.weights = weights;
    a.dweights = dweights;
    a.experts = experts;
    a.dlogits = dlogits;
    return Launched(kudnn_launch_moe_route_backward(a, static_cast<hipStream_t>(stream)), "router: launch failed");
}

int kudnn_moe_route_destroy(kudnn_moe_route_t plan)
{
    delete plan;
    return KUDNN_STATUS_SUCCESS;
}

// ---- grouped Linear

int kudnn_grouped_linear_create(const kudnn_tensor_desc *x, const kudnn_tensor_desc *w, const kudnn_tensor_desc *y, int gather,
                                kudnn_grouped_linear_t *plan)
{
    return Guard([&]() -> int {
        if (x == nullptr || w == nullptr || y == nullptr || plan == nullptr) {
            return Null("grouped Linear: null argument");
        }
        *plan = nullptr;
        int64_t ldw = 0, we = 0;
        const int64_t ldx = RowPitch(*x), ldy = RowPitch(*y);
        if (ldx < 0 || ldy < 0) {
            return Bad("grouped Linear: x and y must be matrices with contiguous rows");
        }
        if (!WeightPitch(*w, ldw, we)) {
            return Bad("grouped Linear: w must be {experts, K, N} with K contiguous (layout ACB)");
        }
        if (!IsHalf(x->dtype) || w->dtype != x->dtype || y->dtype != x->dtype) {
            return Unsupported("grouped Linear: x, w and y must be of one type, bf16 or f16");
        }
        if (w->dims[1] != x->dims[1] || w->dims[2] != y->dims[1] || (gather == 0 && x->dims[0] != y->dims[0])) {
            return Bad("grouped Linear: shapes of x, w and y do not fit");
        }
        const int64_t E = w->dims[0], K = w->dims[1], N = w->dims[2], R = y->dims[0], S = x->dims[0];
        if (E < 1 || K < 1 || N < 1) {
            return Bad("grouped Linear: no experts, or a width of zero");
        }
        if (R > kMaxRows || S > kMaxRows || E > kMaxExperts || K > kMaxSide || N > kMaxSide ||
            !kudnn_grouped_fits(R, E, N, K, x->dtype, y->dtype, true, true)) {
            return Unsupported("grouped Linear: sizes beyond the grid's");
        }
        auto p = new kudnn_grouped_linear_plan();
        p->S = S;
        p->R = R;
        p->E = E;
        p->K = K;
        p->N = N;
        p->ldx = ldx;
        p->ldw = ldw;
        p->we = we;
        p->ldy = ldy;
        p->dt = x->dtype;
        p->gather = gather != 0;
        // few rows, or more experts than a launch of the pack takes, are left to the generic kernel
        if (E <= 65535 && K >= 8 && N >= 8 && ldw < kMaxSide) {
            const auto up = [](int64_t v, int64_t to) { return (v + to - 1) / to * to; };
            p->packDy = N % 8 != 0 ? up(N, 8) : 0;
            p->packW = K % 8 != 0 || ldw % 8 != 0 || (E > 1 && we % 8 != 0) ? up(K, 8) : 0;
            p->packX = K % 8 != 0 || (S > 1 && ldx % 8 != 0) ? up(K, 8) : 0;
            p->second = up(R * p->packDy * 2, 256);
            const int64_t w2 = E * N * p->packW * 2, x2 = S * p->packX * 2;
            p->workspace = p->second + (w2 > x2 ? w2 : x2);
        }
        p->desc = "grouped_linear E=" + std::to_string(E) + " R=" + std::to_string(R) + " N=" + std::to_string(N) + " K=" +
                  std::to_string(K) + (p->gather ? " gather" : "") + TileName(R, E, N, K, ldx, ldw, p->dt, p->dt);
        *plan = p;
        return KUDNN_STATUS_SUCCESS;
    });
}

int64_t kudnn_grouped_linear_workspace_bytes(kudnn_grouped_linear_t plan) { return plan == nullptr ? 0 : plan->workspace; }

int kudnn_grouped_linear_run(kudnn_grouped_linear_t plan, const void *x, const void *w, const int32_t *offsets,
                             const int32_t *rows, void *y, void *stream)
{
    if (plan == nullptr) {
        return Null("grouped Linear: null plan");
    }
    if (plan->R == 0) {
        return KUDNN_STATUS_SUCCESS;
    }
    if ((x == nullptr && plan->S > 0) || w == nullptr || offsets == nullptr || y == nullptr || (plan->gather && rows == nullptr)) {
        return Null("grouped Linear: one of the buffers is nullptr");
    }
    if (!plan->gather && rows != nullptr) {
        return Bad("grouped Linear: rows were given to a plan made without gather");
    }
    const int s = CheckBuffers({Buffer{x, plan->dt}, Buffer{w, plan->dt}, Buffer{offsets, KUDNN_DT_S32},
                                Buffer{rows, KUDNN_DT_S32}, Buffer{y, plan->dt}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    GroupedArgs g{};
    g.a = x;
    g.b = w;
    g.c = y;
    g.offsets = offsets;
    g.rows = rows;
    g.R = plan->R;
    g.S = plan->S;
    g.E = plan->E;
    g.I = plan->R;
    g.J = plan->N;
    g.C = plan->K;
    g.lda = plan->ldx;
    g.ldb = plan->ldw;
    g.ldc = plan->ldy;
    g.be = plan->we;
    g.form = GROUPED_FWD;
    g.dt = g.c_dt = plan->dt;
    return Launched(kudnn_launch_grouped(g, static_cast<hipStream_t>(stream)), "grouped Linear: launch failed");
}

int kudnn_grouped_linear_backward_input(kudnn_grouped_linear_t plan, const void *dy, const void *w, const int32_t *offsets,
                                        void *dx, int dx_dt, void *workspace, void *stream)
{
    if (plan == nullptr) {
        return Null("grouped Linear: null plan");
    }
    if (dx_dt == KUDNN_DT_UNDEFINED) {
        dx_dt = plan->dt;
    }
    if (dx_dt != plan->dt && dx_dt != KUDNN_DT_F32) {
        return Unsupported("grouped Linear: dx must be of the operands' type or f32");
    }
    if (plan->R == 0) {
        return KUDNN_STATUS_SUCCESS;
    }
    if (dy == nullptr || w == nullptr || offsets == nullptr || dx == nullptr || (plan->workspace > 0 && workspace == nullptr)) {
        return Null("grouped Linear: one of the buffers is nullptr");
    }
    const int s = CheckBuffers({Buffer{dy, plan->dt}, Buffer{w, plan->dt}, Buffer{offsets, KUDNN_DT_S32}, Buffer{dx, dx_dt},
                                Buffer{workspace, KUDNN_DT_S32}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
        return Bad("grouped Linear: the workspace must be 16-byte aligned");
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    GroupedArgs g{};
    g.a = dy;
    g.b = w;
    g.c = dx;
    g.offsets = offsets;
    g.R = g.S = g.I = plan->R;
    g.E = plan->E;
    g.J = plan->K;
    g.C = plan->N;
    g.lda = plan->N;
    g.ldb = plan->ldw;
    g.ldc = plan->K;
    g.be = plan->we;
    g.form = GROUPED_BWD_IN;
    g.dt = plan->dt;
    g.c_dt = dx_dt;
    char *ws = static_cast<char *>(workspace);
    int rc = 0;
    if (plan->packDy > 0) {
        rc = Pack(dy, plan->dt, plan->R, plan->N, plan->N, 1, 0, ws, plan->packDy, st);
        g.a = ws;
        g.lda = plan->packDy;
        g.a_padded = true;
    }
    if (rc == 0 && plan->packW > 0) {
        rc = Pack(w, plan->dt, plan->N, plan->K, plan->ldw, plan->E, plan->we, ws + plan->second, plan->packW, st);
        g.b = ws + plan->second;
        g.ldb = plan->packW;
        g.be = plan->N * plan->packW;
        g.b_padded = true;
    }
    return Launched(rc == 0 ? kudnn_launch_grouped(g, st) : rc, "grouped Linear: launch failed");
}

int kudnn_grouped_linear_backward_weight(kudnn_grouped_linear_t plan, const void *dy, const void *x, const int32_t *offsets,
                                         const int32_t *rows, void *dw, void *workspace, void *stream)
{
    if (plan == nullptr) {
        return Null("grouped Linear: null plan");
    }
    const bool some = plan->R > 0;
    if ((some && dy == nullptr) || (x == nullptr && some && plan->S > 0) || offsets == nullptr || dw == nullptr ||
        (some && plan->gather && rows == nullptr) || (some && plan->workspace > 0 && workspace == nullptr)) {
        return Null("grouped Linear: one of the buffers is nullptr");
    }
    if (!plan->gather && rows != nullptr) {
        return Bad("grouped Linear: rows were given to a plan made without gather");
    }
    const int s = CheckBuffers({Buffer{dy, plan->dt}, Buffer{x, plan->dt}, Buffer{offsets, KUDNN_DT_S32},
                                Buffer{rows, KUDNN_DT_S32}, Buffer{dw, plan->dt}, Buffer{workspace, KUDNN_DT_S32}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
        return Bad("grouped Linear: the workspace must be 16-byte aligned");
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    GroupedArgs g{};
    g.a = dy;
    g.b = x;
    g.c = dw;
    g.offsets = offsets;
    g.rows = rows;
    g.R = plan->R;
    g.S = plan->S;
    g.E = plan->E;
    g.I = plan->N;
    g.J = plan->K;
    g.lda = plan->N;
    g.ldb = plan->ldx;
    g.ldc = plan->K;
    g.ce = plan->N * plan->K;
    g.form = GROUPED_BWD_W;
    g.dt = g.c_dt = plan->dt;
    char *ws = static_cast<char *>(workspace);
    int rc = 0;
    if (some && plan->packDy > 0) {
        rc = Pack(dy, plan->dt, plan->R, plan->N, plan->N, 1, 0, ws, plan->packDy, st);
        g.a = ws;
        g.lda = plan->packDy;
        g.a_padded = true;
    }
    if (some && rc == 0 && plan->packX > 0) {
        rc = Pack(x, plan->dt, plan->S, plan->K, plan->ldx, 1, 0, ws + plan->second, plan->packX, st);
        g.b = ws + plan->second;
        g.ldb = plan->packX;
        g.b_padded = true;
    }
    return Launched(rc == 0 ? kudnn_launch_grouped(g, st) : rc, "grouped Linear: launch failed");
}

int kudnn_grouped_linear_destroy(kudnn_grouped_linear_t plan)
{
    delete plan;
    return KUDNN_STATUS_SUCCESS;
}

// ---- block scales and the 8-bit Linear

int kudnn_quantize_rows(const kudnn_tensor_desc *x_desc, const void *x, void *q, int64_t ldq, float *scale, void *stream)
{
    if (x_desc == nullptr) {
        return Null("quantize: null descriptor");
    }
    const int64_t ldx = RowPitch(*x_desc);
    if (ldx < 0) {
        return Bad("quantize: x must be a matrix with contiguous rows");
    }
    if (!IsFloat(x_desc->dtype)) {
        return Unsupported("quantize: x must be f32, bf16 or f16");
    }
    const int64_t M = x_desc->dims[0], K = x_desc->dims[1];
    if (ldq < K) {
        return Bad("quantize: the row pitch of the values is less than a row");
    }
    if (M == 0 || K == 0) {
        return KUDNN_STATUS_SUCCESS;
    }
    // 16 threads a block of 128: the grid's threads must stay below 2^32
    if (K > kMaxSide || M > (int64_t(1) << 27) / ((K + 127) / 128)) {
        return Unsupported("quantize: too large");
    }
    if (x == nullptr || q == nullptr || scale == nullptr) {
        return Null("quantize: one of the buffers is nullptr");
    }
    const int s = CheckBuffers({Buffer{x, x_desc->dtype}, Buffer{q, KUDNN_DT_F8E4M3}, Buffer{scale, KUDNN_DT_F32}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    return Launched(kudnn_launch_quantize_rows(x, x_desc->dtype, M, K, ldx, q, ldq, scale, false, static_cast<hipStream_t>(stream)),
                    "quantize: launch failed");
}

int kudnn_quantize_blocks(const kudnn_tensor_desc *w_desc, const void *w, void *q, float *scale, void *stream)
{
    if (w_desc == nullptr) {
        return Null("quantize: null descriptor");
    }
    int64_t ldw = 0, we = 0;
    if (!WeightPitch(*w_desc, ldw, we)) {
        return Bad("quantize: w must be {experts, K, N} with K contiguous (layout ACB)");
    }
    if (!IsFloat(w_desc->dtype)) {
        return Unsupported("quantize: w must be f32, bf16 or f16");
    }
    const int64_t E = w_desc->dims[0], K = w_desc->dims[1], N = w_desc->dims[2];
    if (E == 0 || K == 0 || N == 0) {
        return KUDNN_STATUS_SUCCESS;
    }
    if (E > kMaxExperts || N > int64_t(65535) * 128 || K > kMaxSide) {   // the grid's second dimension holds 65535
        return Unsupported("quantize: too large");
    }
    if (w == nullptr || q == nullptr || scale == nullptr) {
        return Null("quantize: one of the buffers is nullptr");
    }
    const int s = CheckBuffers({Buffer{w, w_desc->dtype}, Buffer{q, KUDNN_DT_F8E4M3}, Buffer{scale, KUDNN_DT_F32}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    return Launched(kudnn_launch_quantize_blocks(w, w_desc->dtype, E, N, K, we, ldw, q, scale, static_cast<hipStream_t>(stream)),
                    "quantize: launch failed");
}

int kudnn_linear_fp8_create(const kudnn_tensor_desc *x, const kudnn_tensor_desc *w, const kudnn_tensor_desc *y,
                            const kudnn_tensor_desc *bias, int grouped, int gather, kudnn_linear_fp8_t *plan)
{
    return Guard([&]() -> int {
        if (x == nullptr || w == nullptr || y == nullptr || plan == nullptr) {
            return Null("8-bit Linear: null argument");
        }
        *plan = nullptr;
        const int64_t ldx = RowPitch(*x), ldy = RowPitch(*y);
        if (ldx < 0 || ldy < 0) {
            return Bad("8-bit Linear: x and y must be matrices with contiguous rows");
        }
        kudnn_tensor_desc w3 = *w;
        if (w->ndims == 2) {   // {K, N} BA: one expert
            w3.ndims = 3;
            w3.dims[0] = 1;
            w3.strides[0] = 0;
            for (int i = 0; i < 2; ++i) {
                w3.dims[i + 1] = w->dims[i];
                w3.strides[i + 1] = w->strides[i];
            }
        }
        int64_t ldw = 0, we = 0;
        if (!WeightPitch(w3, ldw, we)) {
            return Bad("8-bit Linear: w must be {K, N} BA or {experts, K, N} ACB, K contiguous");
        }
        const int64_t E = w3.dims[0], K = w3.dims[1], N = w3.dims[2], S = x->dims[0], R = y->dims[0];
        if (w->dtype != KUDNN_DT_F8E4M3 || !(x->dtype == KUDNN_DT_F8E4M3 || IsHalf(x->dtype)) || !IsFloat(y->dtype)) {
            return Unsupported("8-bit Linear: w must be e4m3, x e4m3, bf16 or f16, y bf16, f16 or f32");
        }
        if (K != x->dims[1] || N != y->dims[1] || ((grouped == 0 || gather == 0) && S != R) || (grouped == 0 && (E != 1 || gather != 0))) {
            return Bad("8-bit Linear: shapes of x, w and y do not fit");
        }
        if (E < 1 || K < 1 || N < 1) {
            return Bad("8-bit Linear: no weight, or a width of zero");
        }
        const bool hasBias = bias != nullptr && bias->ndims != 0;
        if (hasBias) {
            if (grouped != 0 || bias->dtype != y->dtype) {
                return Unsupported("8-bit Linear: a bias is taken without groups and of y's type");
            }
            if (bias->ndims != 2 || bias->dims[0] != 1 || bias->dims[1] != N || (N > 1 && bias->strides[1] != 1)) {
                return Bad("8-bit Linear: bias must be {1, N}");
            }
        }
        if (R > kMaxRows || S > kMaxRows || E > kMaxExperts || K > kMaxSide || N > kMaxSide ||
            S > (int64_t(1) << 27) / ((K + 127) / 128) || !kudnn_grouped_fits(R, E, N, K, w->dtype, y->dtype, grouped != 0, false)) {
            return Unsupported("8-bit Linear: sizes beyond the grid's");
        }
        auto p = new kudnn_linear_fp8_plan();
        p->S = S;
        p->R = R;
        p->E = E;
        p->K = K;
        p->N = N;
        p->ldx = ldx;
        p->ldw = ldw;
        p->we = we;
        p->ldy = ldy;
        p->xdt = x->dtype;
        p->ydt = y->dtype;
        p->grouped = grouped != 0;
        p->gather = gather != 0;
        p->hasBias = hasBias;
        // weights that 32-bit offsets do not reach go through the generic kernel, which takes e4m3 rows
        p->fused = R > 0 && p->xdt != KUDNN_DT_F8E4M3 && ldw < kMaxSide &&
                   kudnn_grouped_fused(R, p->grouped ? (E < R ? E : R) : 1, N, K, p->ydt, K % 16 != 0 || ldw % 16 != 0);
        if (p->xdt != KUDNN_DT_F8E4M3 && !p->fused) {
            p->scaleOffset = S * kudnn_fp8_pitch(K);
            p->workspace = p->scaleOffset + S * ((K + 127) / 128) * static_cast<int64_t>(sizeof(float));
        }
        p->desc = "linear_fp8 E=" + std::to_string(E) + " R=" + std::to_string(R) + " N=" + std::to_string(N) + " K=" +
                  std::to_string(K) + (p->grouped ? (p->gather ? " grouped gather" : " grouped") : "") + (p->fused ? " fused" : "") + TileName(R, E, N, K, p->xdt == KUDNN_DT_F8E4M3 ? ldx : kudnn_fp8_pitch(K), ldw, KUDNN_DT_F8E4M3, p->ydt);
        *plan = p;
        return KUDNN_STATUS_SUCCESS;
    });
}

int64_t kudnn_linear_fp8_workspace_bytes(kudnn_linear_fp8_t plan) { return plan == nullptr ? 0 : plan->workspace; }

int kudnn_linear_fp8_run(kudnn_linear_fp8_t plan, const void *x, const float *x_scale, const void *w, const float *w_scale,
                         const void *bias, const int32_t *offsets, const int32_t *rows, void *y, void *workspace, void *stream)
{
    if (plan == nullptr) {
        return Null("8-bit Linear: null plan");
    }
    if (plan->R == 0) {
        return KUDNN_STATUS_SUCCESS;
    }
    const bool quantized = plan->xdt == KUDNN_DT_F8E4M3;
    if ((x == nullptr && plan->S > 0) || (quantized && x_scale == nullptr && plan->S > 0) || w == nullptr || w_scale == nullptr ||
        y == nullptr || (plan->hasBias && bias == nullptr) || (plan->grouped && offsets == nullptr) ||
        (plan->gather && rows == nullptr) || (plan->workspace > 0 && workspace == nullptr)) {
        return Null("8-bit Linear: one of the buffers is nullptr");
    }
    if ((!quantized && x_scale != nullptr) || (!plan->hasBias && bias != nullptr) || (!plan->gather && rows != nullptr) ||
        (!plan->grouped && offsets != nullptr)) {
        return Bad("8-bit Linear: a buffer was given that the plan was made without");
    }
    const int s = CheckBuffers({Buffer{x, plan->xdt}, Buffer{x_scale, KUDNN_DT_F32}, Buffer{w, KUDNN_DT_F8E4M3},
                                Buffer{w_scale, KUDNN_DT_F32}, Buffer{bias, plan->ydt}, Buffer{offsets, KUDNN_DT_S32},
                                Buffer{rows, KUDNN_DT_S32}, Buffer{y, plan->ydt}, Buffer{workspace, KUDNN_DT_S32}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    if (plan->workspace > 0 && reinterpret_cast<uintptr_t>(workspace) % 16 != 0) {
        return Bad("8-bit Linear: the workspace must be 16-byte aligned");
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    GroupedArgs g{};
    g.a = x;
    g.a_scale = x_scale;
    g.lda = plan->ldx;
    if (plan->fused) {
        g.x_dt = plan->xdt;
    } else if (!quantized) {
        char *ws = static_cast<char *>(workspace);
        float *scale = reinterpret_cast<float *>(ws + plan->scaleOffset);
        if (plan->S > 0 &&
            kudnn_launch_quantize_rows(x, plan->xdt, plan->S, plan->K, plan->ldx, ws, kudnn_fp8_pitch(plan->K), scale, true, st) != 0) {
            return Launched(-1, "8-bit Linear: launch failed");
        }
        g.a = ws;
        g.a_scale = scale;
        g.lda = kudnn_fp8_pitch(plan->K);
    }
    g.b = w;
    g.c = y;
    g.b_scale = w_scale;
    g.bias = bias;
    g.offsets = offsets;
    g.rows = rows;
    g.R = g.I = plan->R;
    g.S = plan->S;
    g.E = plan->E;
    g.J = plan->N;
    g.C = plan->K;
    g.ldb = plan->ldw;
    g.ldc = plan->ldy;
    g.be = plan->we;
    g.form = GROUPED_FWD;
    g.dt = KUDNN_DT_F8E4M3;
    g.c_dt = plan->ydt;
    if (plan->fused) {
        const bool any = plan->K % 16 != 0 || plan->ldw % 16 != 0 || (plan->E > 1 && plan->we % 16 != 0) || reinterpret_cast<uintptr_t>(w) % 16 != 0;
        const GroupedTile t = kudnn_grouped_rule(g.R, plan->grouped ? (g.E < g.R ? g.E : g.R) : 1, g.J, g.C, g.dt, g.c_dt, any);
        return Launched(kudnn_launch_grouped_stream(g, 16, t.bm == 16 ? t.bn : 64, 8, true, any, st), "8-bit Linear: launch failed");
    }
    return Launched(kudnn_launch_grouped(g, st), "8-bit Linear: launch failed");
}

int kudnn_linear_fp8_destroy(kudnn_linear_fp8_t plan)
{
    delete plan;
    return KUDNN_STATUS_SUCCESS;
}

// ---- weighted sum

int kudnn_moe_combine_create(const kudnn_tensor_desc *y, const kudnn_tensor_desc *out, int top_k, kudnn_moe_combine_t *plan)
{
    return Guard([&]() -> int {
        if (y == nullptr || out == nullptr || plan == nullptr) {
            return Null("weighted sum: null argument");
        }
        *plan = nullptr;
        const int64_t ldy = RowPitch(*y), ldo = RowPitch(*out);
        if (ldy < 0 || ldo < 0) {
            return Bad("weighted sum: y and out must be matrices with contiguous rows");
        }
        if (!IsFloat(y->dtype) || !(out->dtype == y->dtype || (y->dtype == KUDNN_DT_F32 && IsFloat(out->dtype)))) {
            return Unsupported("weighted sum: y and out must be of one type, f32, bf16 or f16, or y of f32 and out of 16 bits");
        }
        if (y->dims[1] != out->dims[1]) {
            return Bad("weighted sum: y and out have different widths");
        }
        if (top_k < 1) {
            return Bad("weighted sum: top_k must be at least 1");
        }
        // a grid has at most 65535 pieces of a row of 256 columns
        if (top_k > 64 || out->dims[0] > kMaxRows || y->dims[0] > kMaxRows || y->dims[1] > kMaxSide / 2) {
            return Unsupported("weighted sum: at most 64 experts a token, 2^31 - 1 tokens and 2^23 columns");
        }
        auto p = new kudnn_moe_combine_plan();
        p->T = out->dims[0];
        p->R = y->dims[0];
        p->N = y->dims[1];
        p->ldy = ldy;
        p->ldo = ldo;
        p->k = top_k;
        p->dt = y->dtype;
        p->outDt = out->dtype;
        p->desc = "moe_combine T=" + std::to_string(p->T) + " R=" + std::to_string(p->R) + " N=" + std::to_string(p->N) +
                  " k=" + std::to_string(top_k);
        *plan = p;
        return KUDNN_STATUS_SUCCESS;
    });
}

int kudnn_moe_combine_run(kudnn_moe_combine_t plan, const void *y, const float *weights, const int32_t *slots, void *out,
                          void *stream)
{
    if (plan == nullptr) {
        return Null("weighted sum: null plan");
    }
    if (plan->T == 0 || plan->N == 0) {
        return KUDNN_STATUS_SUCCESS;
    }
    if ((y == nullptr && plan->R > 0) || slots == nullptr || out == nullptr) {
        return Null("weighted sum: one of the buffers is nullptr");
    }
    const int s = CheckBuffers({Buffer{y, plan->dt}, Buffer{weights, KUDNN_DT_F32}, Buffer{slots, KUDNN_DT_S32}, Buffer{out, plan->outDt}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    CombineArgs a{};
    a.y = y;
    a.weights = weights;
    a.slots = slots;
    a.out = out;
    a.T = plan->T;
    a.R = plan->R;
    a.N = plan->N;
    a.ldy = plan->ldy;
    a.ldo = plan->ldo;
    a.k = plan->k;
    a.dt = plan->dt;
    a.out_dt = plan->outDt;
    return Launched(kudnn_launch_moe_combine(a, static_cast<hipStream_t>(stream)), "weighted sum: launch failed");
}

int kudnn_moe_combine_backward(kudnn_moe_combine_t plan, const void *y, const float *weights, const int32_t *slots,
                               const void *dout, void *dy, float *dweights, void *stream)
{
    if (plan == nullptr) {
        return Null("weighted sum: null plan");
    }
    if (plan->outDt != plan->dt) {
        return Unsupported("weighted sum: the gradients need y and out of one type");
    }
    if (dy == nullptr && dweights == nullptr) {
        return KUDNN_STATUS_SUCCESS;
    }
    if ((plan->T > 0 && (slots == nullptr || dout == nullptr)) || (dweights != nullptr && y == nullptr && plan->R > 0)) {
        return Null("weighted sum: one of the buffers is nullptr");
    }
    const int s = CheckBuffers({Buffer{y, plan->dt}, Buffer{weights, KUDNN_DT_F32}, Buffer{slots, KUDNN_DT_S32},
                                Buffer{dout, plan->dt}, Buffer{dy, plan->dt}, Buffer{dweights, KUDNN_DT_F32}});
    if (s != KUDNN_STATUS_SUCCESS) {
        return s;
    }
    CombineArgs a{};
    a.y = y;
    a.dout = dout;
    a.weights = weights;
    a.slots = slots;
    a.dy = dy;
    a.dweights = dweights;
    a.T = plan->T;
    a.R = plan->R;
    a.N = plan->N;
    a.ldy = plan->ldy;
    a.ldo = plan->N;
    a.k = plan->k;
    a.dt = a.out_dt = plan->dt;
    return Launched(kudnn_launch_moe_combine_backward(a, static_cast<hipStream_t>(stream)), "weighted sum: launch failed");
}

int kudnn_moe_combine_destroy(kudnn_moe_combine_t plan)
{
    delete plan;
    return KUDNN_STATUS_SUCCESS;
}

}  // extern "C"
