// Mixture of experts (MI355X addition, no KuDNN counterpart): the router, the experts' Linear products over ragged groups of
// rows, the 8-bit products with a scale for each block of 128, and the weighted sum of a token's experts.
//
// The operators run on the device alone: every pointer is device memory, Run is asynchronous on `stream` (a hipStream_t,
// nullptr = the default stream), allocates nothing and changes nothing in the object, so one object may run on several
// streams at once and under graph capture. Where WorkspaceBytes() is not 0 the caller gives that much device memory, 16-byte
// aligned, which is in use until the run's work on the stream is done. Unsupported descriptors throw Service::Unsupported,
// mismatched ones and null pointers Service::LogicError.
//
// With T tokens and k experts each there are R = T * k rows, sorted by expert:
//   offsets int32[E + 1]  expert e has the rows offsets[e] .. offsets[e + 1] - 1
//   rows    int32[R]      the token of each row, -1 past the last
//   slots   int32[T * k]  the row of each of a token's experts, -1 where it has none
// Weights are {E, K, N} with Layout::ACB: each expert's held as [N][K].
#ifndef KUDNN_MOE_HPP
#define KUDNN_MOE_HPP

#include <cstdint>
#include <memory>

#include "types/kudnn_tensor_info.hpp"

namespace KuDNN {

namespace Detail {
class MoeRouteImpl;
class GroupedLinearImpl;
class LinearFp8Impl;
class MoeCombineImpl;
}  // namespace Detail

// Softmax over each token's open experts, its topK largest, and the rows in the experts' order.
class KUDNN_API_PUBLIC MoeRoute final {
public:
    // logits {T, E} AB of F32, BF16 or F16; mask {T or 1, E or 1} of U8, or a descriptor of size 0 for none.
    MoeRoute(const TensorInfo &logits, const TensorInfo &mask, int topK, bool normalize) noexcept(false);
    MoeRoute(const MoeRoute &other) = delete;
    MoeRoute(MoeRoute &&other) noexcept;
    MoeRoute &operator=(MoeRoute &&other) noexcept;
    ~MoeRoute() noexcept;
    std::int64_t WorkspaceBytes() const noexcept(false);
    void Run(const void *logits, const void *mask, float *weights, std::int32_t *experts, std::int32_t *offsets, std::int32_t *rows,
             std::int32_t *slots, void *workspace, void *stream = nullptr) const noexcept(false);
    // dlogits {T, E} dense, of the logits' type.
    void Backward(const void *logits, const void *mask, const float *weights, const std::int32_t *experts, const float *dweights,
                  void *dlogits, void *stream = nullptr) const noexcept(false);

private:
    std::unique_ptr<Detail::MoeRouteImpl> pImpl;
};

// y[r] = x[rows[r]] x w[e] for the rows r of expert e (x[r] without gather); zero for rows of no expert.
class KUDNN_API_PUBLIC GroupedLinear final {
public:
    // x {S, K} AB, w {E, K, N} ACB, y {R, N} AB, all BF16 or all F16.
    GroupedLinear(const TensorInfo &x, const TensorInfo &w, const TensorInfo &y, bool gather) noexcept(false);
    GroupedLinear(const GroupedLinear &other) = delete;
    GroupedLinear(GroupedLinear &&other) noexcept;
    GroupedLinear &operator=(GroupedLinear &&other) noexcept;
    ~GroupedLinear() noexcept;
    // Of the two gradients; Run needs none.
    std::int64_t WorkspaceBytes() const noexcept(false);
    void Run(const void *x, const void *w, const std::int32_t *offsets, const std::int32_t *rows, void *y,
             void *stream = nullptr) const noexcept(false);
    // dx {R, K} dense, in the experts' order, of the operands' type (UNDEFINED) or F32; with gather, MoeCombine without weights adds a
    // token's rows.
    void BackwardInput(const void *dy, const void *w, const std::int32_t *offsets, void *dx, void *workspace, void *stream = nullptr,
                       Element::TypeT dxType = Element::TypeT::UNDEFINED) const noexcept(false);
    // dw dense [E][N][K].
    void BackwardWeight(const void *dy, const void *x, const std::int32_t *offsets, const std::int32_t *rows, void *dw, void *workspace,
                        void *stream = nullptr) const noexcept(false);

private:
    std::unique_ptr<Detail::GroupedLinearImpl> pImpl;
};

// Linear with e4m3 operands and a scale for each block of 128, for one weight or, grouped, one an expert.
class KUDNN_API_PUBLIC LinearFp8 final {
public:
    // x {S, K} AB of F8E4M3 (with scales), BF16 or F16 (quantised by Run); w {K, N} BA or {E, K, N} ACB of F8E4M3; y {R, N} AB of
    // BF16, F16 or F32; bias {1, N} of y's type, or a descriptor of size 0 for none (none when grouped).
    LinearFp8(const TensorInfo &x, const TensorInfo &w, const TensorInfo &y, const TensorInfo &bias, bool grouped,
              bool gather) noexcept(false);
    LinearFp8(const LinearFp8 &other) = delete;
    LinearFp8(LinearFp8 &&other) noexcept;
    LinearFp8 &operator=(LinearFp8 &&other) noexcept;
    ~LinearFp8() noexcept;
    std::int64_t WorkspaceBytes() const noexcept(false);
    void Run(const void *x, const float *xScale, const void *w, const float *wScale, const void *bias, const std::int32_t *offsets,
             const std::int32_t *rows, void *y, void *workspace, void *stream = nullptr) const noexcept(false);
    // x {M, K} AB -> q e4m3 [M][K] with a row pitch of ldq bytes, scale float[M][ceil(K / 128)].
    static void QuantizeRows(const TensorInfo &xInfo, const void *x, void *q, std::int64_t ldq, float *scale,
                             void *stream = nullptr) noexcept(false);
    // w {E, K, N} ACB -> q e4m3 [E][N][K], scale float[E][ceil(N / 128)][ceil(K / 128)].
    static void QuantizeBlocks(const TensorInfo &wInfo, const void *w, void *q, float *scale, void *stream = nullptr) noexcept(false);

private:
    std::unique_ptr<Detail::LinearFp8Impl> pImpl;
};

// out[t] = sum over j of weights[t][j] y[slots[t][j]] (weights nullptr: ones).
class KUDNN_API_PUBLIC MoeCombine final {
public:
    // y {R, N} AB and out {T, N} AB of one type: F32, BF16 or F16; or y of F32 and out of 16 bits (Run only).
    MoeCombine(const TensorInfo &y, const TensorInfo &out, int topK) noexcept(false);
    MoeCombine(const MoeCombine &other) = delete;
    MoeCombine(MoeCombine &&other) noexcept;
    MoeCombine &operator=(MoeCombine &&other) noexcept;
    ~MoeCombine() noexcept;
    void Run(const void *y, const float *weights, const std::int32_t *slots, void *out, void *stream = nullptr) const noexcept(false);
    // dy dense {R, N} and dweights float[T][k]; either may be nullptr.
    void Backward(const void *y, const float *weights, const std::int32_t *slots, const void *dout, void *dy, float *dweights,
                  void *stream = nullptr) const noexcept(false);

private:
    std::unique_ptr<Detail::MoeCombineImpl> pImpl;
};

}  // namespace KuDNN

#endif  // KUDNN_MOE_HPP
