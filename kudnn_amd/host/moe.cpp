// KuDNN's mixture-of-experts classes (operations/kudnn_moe.hpp) on top of the C ABI of libkudnn_hip.so.
#include "../../include/kudnn.hpp"
#include "../../include/kudnn_hip.h"
#include "abi.h"

namespace KuDNN {

namespace Detail {

// Owner of one C ABI plan handle.
template <typename H, int (*Destroy)(H)>
class Handle {
public:
    Handle() = default;
    Handle(const Handle &) = delete;
    Handle &operator=(const Handle &) = delete;
    ~Handle() { Destroy(h); }
    H h = nullptr;
};

class MoeRouteImpl final : public Handle<kudnn_moe_route_t, kudnn_moe_route_destroy> {};
class GroupedLinearImpl final : public Handle<kudnn_grouped_linear_t, kudnn_grouped_linear_destroy> {};
class LinearFp8Impl final : public Handle<kudnn_linear_fp8_t, kudnn_linear_fp8_destroy> {};
class MoeCombineImpl final : public Handle<kudnn_moe_combine_t, kudnn_moe_combine_destroy> {};

}  // namespace Detail

namespace {

// The plan of an object that has not been moved from.
template <typename Impl>
auto Get(const std::unique_ptr<Impl> &p)
{
    if (p == nullptr) {
        throw Service::LogicError{"mixture of experts: the object was moved from"};
    }
    return p->h;
}

// A descriptor of size 0 means "none".
const kudnn_tensor_desc *OrNone(const TensorInfo &info, const kudnn_tensor_desc &d) { return info.GetTotalTensorSize() == 0 ? nullptr : &d; }

}  // namespace

MoeRoute::MoeRoute(const TensorInfo &logits, const TensorInfo &mask, int topK, bool normalize) noexcept(false)
    : pImpl(new Detail::MoeRouteImpl)
{
    const kudnn_tensor_desc dl = Abi::ToDesc(logits), dm = Abi::ToDesc(mask);
    Abi::Check(kudnn_moe_route_create(&dl, OrNone(mask, dm), topK, normalize ? 1 : 0, &pImpl->h));
}
MoeRoute::MoeRoute(MoeRoute &&other) noexcept = default;
MoeRoute &MoeRoute::operator=(MoeRoute &&other) noexcept = default;
MoeRoute::~MoeRoute() noexcept = default;
std::int64_t MoeRoute::WorkspaceBytes() const noexcept(false) { return kudnn_moe_route_workspace_bytes(Get(pImpl)); }
void MoeRoute::Run(const void *logits, const void *mask, float *weights, std::int32_t *experts, std::int32_t *offsets,
                   std::int32_t *rows, std::int32_t *slots, void *workspace, void *stream) const noexcept(false)
{
    Abi::Check(kudnn_moe_route_run(Get(pImpl), logits, mask, weights, experts, offsets, rows, slots, workspace, stream));
}
void MoeRoute::Backward(const void *logits, const void *mask, const float *weights, const std::int32_t *experts, const float *dweights,
                        void *dlogits, void *stream) const noexcept(false)
{
    Abi::Check(kudnn_moe_route_backward(Get(pImpl), logits, mask, weights, experts, dweights, dlogits, stream));
}

GroupedLinear::GroupedLinear(const TensorInfo &x, const TensorInfo &w, const TensorInfo &y, bool gather) noexcept(false)
    : pImpl(new Detail::GroupedLinearImpl)
{
    const kudnn_tensor_desc dx = Abi::ToDesc(x), dw = Abi::ToDesc(w), dy = Abi::ToDesc(y);
    Abi::Check(kudnn_grouped_linear_create(&dx, &dw, &dy, gather ? 1 : 0, &pImpl->h));
}
GroupedLinear::GroupedLinear(GroupedLinear &&other) noexcept = default;
GroupedLinear &GroupedLinear::operator=(GroupedLinear &&other) noexcept = default;
GroupedLinear::~GroupedLinear() noexcept = default;
std::int64_t GroupedLinear::WorkspaceBytes() const noexcept(false) { return kudnn_grouped_linear_workspace_bytes(Get(pImpl)); }
void GroupedLinear::Run(const void *x, const void *w, const std::int32_t *offsets, const std::int32_t *rows, void *y,
                        void *stream) const noexcept(false)
{
    Abi::Check(kudnn_grouped_linear_run(Get(pImpl), x, w, offsets, rows, y, stream));
}
void GroupedLinear::BackwardInput(const void *dy, const void *w, const std::int32_t *offsets, void *dx, void *workspace,
                                  void *stream, Element::TypeT dxType) const noexcept(false)
{
    Abi::Check(kudnn_grouped_linear_backward_input(Get(pImpl), dy, w, offsets, dx, static_cast<int>(dxType), workspace, stream));
}
void GroupedLinear::BackwardWeight(const void *dy, const void *x, const std::int32_t *offsets, const std::int32_t *rows, void *dw,
                                   void *workspace, void *stream) const noexcept(false)
{
    Abi::Check(kudnn_grouped_linear_backward_weight(Get(pImpl), dy, x, offsets, rows, dw, workspace, stream));
}

LinearFp8::LinearFp8(const TensorInfo &x, const TensorInfo &w, const TensorInfo &y, const TensorInfo &bias, bool grouped,
                     bool gather) noexcept(false)
    : pImpl(new Detail::LinearFp8Impl)
{
    const kudnn_tensor_desc dx = Abi::ToDesc(x), dw = Abi::ToDesc(w), dy = Abi::ToDesc(y), db = Abi::ToDesc(bias);
    Abi::Check(kudnn_linear_fp8_create(&dx, &dw, &dy, OrNone(bias, db), grouped ? 1 : 0, gather ? 1 : 0, &pImpl->h));
}
LinearFp8::LinearFp8(LinearFp8 &&other) noexcept = default;
LinearFp8 &LinearFp8::operator=(LinearFp8 &&other) noexcept = default;
LinearFp8::~LinearFp8() noexcept = default;
std::int64_t LinearFp8::WorkspaceBytes() const noexcept(false) { return kudnn_linear_fp8_workspace_bytes(Get(pImpl)); }
void LinearFp8::Run(const void *x, const float *xScale, const void *w, const float *wScale, const void *bias,
                    const std::int32_t *offsets, const std::int32_t *rows, void *y, void *workspace, void *stream) const noexcept(false)
{
    Abi::Check(kudnn_linear_fp8_run(Get(pImpl), x, xScale, w, wScale, bias, offsets, rows, y, workspace, stream));
}
void LinearFp8::QuantizeRows(const TensorInfo &xInfo, const void *x, void *q, std::int64_t ldq, float *scale,
                             void *stream) noexcept(false)
{
    const kudnn_tensor_desc d = Abi::ToDesc(xInfo);
    Abi::Check(kudnn_quantize_rows(&d, x, q, ldq, scale, stream));
}
void LinearFp8::QuantizeBlocks(const TensorInfo &wInfo, const void *w, void *q, float *scale, void *stream) noexcept(false)
{
    const kudnn_tensor_desc d = Abi::ToDesc(wInfo);
    Abi::Check(kudnn_quantize_blocks(&d, w, q, scale, stream));
}

MoeCombine::MoeCombine(const TensorInfo &y, const TensorInfo &out, int topK) noexcept(false) : pImpl(new Detail::MoeCombineImpl)
{
    const kudnn_tensor_desc dy = Abi::ToDesc(y), dout = Abi::ToDesc(out);
    Abi::Check(kudnn_moe_combine_create(&dy, &dout, topK, &pImpl->h));
}
MoeCombine::MoeCombine(MoeCombine &&other) noexcept = default;
MoeCombine &MoeCombine::operator=(MoeCombine &&other) noexcept = default;
MoeCombine::~MoeCombine() noexcept = default;
void MoeCombine::Run(const void *y, const float *weights, const std::int32_t *slots, void *out, void *stream) const noexcept(false)
{
    Abi::Check(kudnn_moe_combine_run(Get(pImpl), y, weights, slots, out, stream));
}
void MoeCombine::Backward(const void *y, const float *weights, const std::int32_t *slots, const void *dout, void *dy, float *dweights,
                          void *stream) const noexcept(false)
{
    Abi::Check(kudnn_moe_combine_backward(Get(pImpl), y, weights, slots, dout, dy, dweights, stream));
}

}  // namespace KuDNN
