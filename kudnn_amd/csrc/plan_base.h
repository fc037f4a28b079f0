// What the C ABI's translation units share on the host: the base of every plan handle and the thread's last error.
#ifndef KUDNN_PLAN_BASE_H
#define KUDNN_PLAN_BASE_H

#include <string>

enum PlanKind {
    PLAN_GEMM = 1,
    PLAN_LINEAR_ACT,
    PLAN_LINEAR_RES,
    PLAN_LINEAR_POSTOPS,
    PLAN_MOE_ROUTE,
    PLAN_GROUPED_LINEAR,
    PLAN_LINEAR_FP8,
    PLAN_MOE_COMBINE
};

struct PlanBase {
    int kind;
    std::string desc;
    explicit PlanBase(int k) : kind(k) {}
    virtual ~PlanBase() = default;
};

namespace kudnn_host {

// Sets kudnn_last_error()'s message of this thread and returns `status`.
int SetError(int status, const char *msg) noexcept;
// Whether p is null or memory that a kernel can read (hipMalloc, managed).
bool DeviceMemory(const void *p) noexcept;

}  // namespace kudnn_host

#endif  // KUDNN_PLAN_BASE_H
