// What the operator classes share of the C ABI: descriptors, and statuses as the exceptions KuDNN throws.
#ifndef KUDNN_HOST_ABI_H
#define KUDNN_HOST_ABI_H

#include <cstring>
#include <stdexcept>

#include "../../include/kudnn.hpp"
#include "../../include/kudnn_hip.h"

namespace KuDNN {
namespace Abi {

inline kudnn_tensor_desc ToDesc(const TensorInfo &t)
{
    kudnn_tensor_desc d;
    std::memset(&d, 0, sizeof(d));
    const Shape dims = t.GetDims();
    const Shape strides = t.GetStrides();
    d.ndims = static_cast<int32_t>(dims.GetNumDims());
    d.dtype = static_cast<int32_t>(static_cast<Element::TypeT>(t.GetType()));
    d.layout = static_cast<int32_t>(t.GetLayout());
    for (SizeType i = 0; i < dims.GetNumDims(); ++i) {
        d.dims[i] = static_cast<int64_t>(dims[i]);
        d.strides[i] = i < strides.GetNumDims() ? static_cast<int64_t>(strides[i]) : 0;
    }
    return d;
}

inline void Check(int s)
{
    switch (s) {
        case KUDNN_STATUS_SUCCESS: return;
        case KUDNN_STATUS_UNSUPPORTED: throw Service::Unsupported{kudnn_last_error()};
        case KUDNN_STATUS_BAD_ARGUMENTS:
        case KUDNN_STATUS_NULL_POINTER: throw Service::LogicError{kudnn_last_error()};
        case KUDNN_STATUS_ALLOC_FAILED: throw Service::BadAlloc{};
        default: throw std::runtime_error{kudnn_last_error()};
    }
}

}  // namespace Abi
}  // namespace KuDNN

#endif  // KUDNN_HOST_ABI_H
