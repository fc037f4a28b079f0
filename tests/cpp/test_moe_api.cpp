// Tests of the C++ classes of the mixture of experts (operations/kudnn_moe.hpp).
//   test_moe_api          refusals and moves; no GPU needed
//   test_moe_api --gpu    also a batch of integers through router, experts and weighted sum, forward and backward, exactly
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <utility>
#include <vector>

#include "kudnn.hpp"

using namespace KuDNN;

static int g_failed = 0;

#define CHECK(cond)                                                       \
    do {                                                                  \
        if (!(cond)) {                                                    \
            std::printf("  FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond); \
            ++g_failed;                                                   \
        }                                                                 \
    } while (0)
#define CHECK_THROWS(E, call)         \
    do {                              \
        bool thrown = false;          \
        try {                         \
            call;                     \
        } catch (const E &) {         \
            thrown = true;            \
        }                             \
        CHECK(thrown && #call != nullptr); \
    } while (0)

static const Element::TypeT F32 = Element::TypeT::F32, BF16 = Element::TypeT::BF16, F8 = Element::TypeT::F8E4M3, U8 = Element::TypeT::U8;
static const TensorInfo kNone({0}, F32, Layout::A);

static void Refusals()
{
    const TensorInfo logits({6, 4}, F32, Layout::AB), x({6, 64}, BF16, Layout::AB), w({4, 64, 32}, BF16, Layout::ACB),
        y({12, 32}, BF16, Layout::AB), out({6, 32}, BF16, Layout::AB), wide({4, 48, 32}, BF16, Layout::ACB);
    MoeRoute route(logits, kNone, 2, true);
    CHECK(route.WorkspaceBytes() >= 0);
    CHECK_THROWS(Service::LogicError, MoeRoute(logits, kNone, 5, true));                              // more than there are experts
    CHECK_THROWS(Service::LogicError, MoeRoute(logits, TensorInfo({5, 4}, U8, Layout::AB), 2, true));  // mask of other tokens
    CHECK_THROWS(Service::LogicError, route.Run(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr));
    MoeRoute moved(std::move(route));
    CHECK_THROWS(Service::LogicError, route.WorkspaceBytes());
    route = std::move(moved);
    CHECK(route.WorkspaceBytes() >= 0);

    GroupedLinear grouped(x, w, y, true);
    CHECK(grouped.WorkspaceBytes() == 0);
    CHECK_THROWS(Service::LogicError, GroupedLinear(x, wide, y, true));                                // K differs
    CHECK_THROWS(Service::LogicError, GroupedLinear(x, w, y, false));                                  // 6 rows into 12
    CHECK_THROWS(Service::LogicError, grouped.Run(nullptr, nullptr, nullptr, nullptr, nullptr));

    const TensorInfo w8({64, 32}, F8, Layout::BA), y8({6, 32}, BF16, Layout::AB);
    LinearFp8 dense(x, w8, y8, kNone, false, false);
    CHECK_THROWS(Service::LogicError, LinearFp8(x, w8, y8, TensorInfo({1, 31}, BF16, Layout::AB), false, false));
    CHECK_THROWS(Service::LogicError, dense.Run(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr));

    MoeCombine combine(y, out, 2);
    CHECK_THROWS(Service::LogicError, MoeCombine(y, TensorInfo({6, 31}, BF16, Layout::AB), 2));
    CHECK_THROWS(Service::LogicError, combine.Run(nullptr, nullptr, nullptr, nullptr));
    std::vector<float> host(6 * 32);
    std::vector<std::int32_t> slots(12);
    CHECK_THROWS(Service::LogicError, combine.Run(host.data(), nullptr, slots.data(), host.data()));   // host memory
    // the other operators do not know the 8-bit type
    CHECK(Gemm::ValidateInput(TensorInfo({6, 64}, F8, Layout::AB), w8, y8, kNone) != Status::SUCCESS);
}

template <typename T>
struct Device {
    explicit Device(const std::vector<T> &v) : Device(v.size()) { Copied(hipMemcpy(p, v.data(), n * sizeof(T), hipMemcpyHostToDevice)); }
    explicit Device(std::size_t count) : n(count) { Copied(hipMalloc(reinterpret_cast<void **>(&p), n * sizeof(T))); }
    Device(const Device &) = delete;
    ~Device() { (void)hipFree(p); }
    std::vector<T> Host() const
    {
        std::vector<T> v(n);
        Copied(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return v;
    }
    static void Copied(hipError_t e)
    {
        if (e != hipSuccess) {
            std::printf("  FAIL %s\n", hipGetErrorString(e));
            std::exit(1);
        }
    }
    T *p = nullptr;
    std::size_t n;
};

static std::uint16_t Bf16(float v)
{
    std::uint32_t u;
    std::memcpy(&u, &v, 4);
    return static_cast<std::uint16_t>(u >> 16);   // integers of up to 8 bits: exact
}
static float F32Of(std::uint16_t v)
{
    const std::uint32_t u = static_cast<std::uint32_t>(v) << 16;
    float f;
    std::memcpy(&f, &u, 4);
    return f;
}

// One expert a token: every weight is 1, and sums of small integers are exact in any order.
static void Integers()
{
    const int T = 37, E = 5, K = 40, N = 24;
    std::vector<float> logits(T * E);
    std::vector<std::uint16_t> x(T * K), w(E * N * K), dy(T * N);
    std::vector<int> expert(T);
    for (int t = 0; t < T; ++t) {
        expert[t] = (t * 7 + t / 3) % E;
        for (int e = 0; e < E; ++e) logits[t * E + e] = e == expert[t] ? 3.0f : 0.25f * static_cast<float>((t + e) % 4);
        for (int k = 0; k < K; ++k) x[t * K + k] = Bf16(static_cast<float>((t + 3 * k) % 3 - 1));
        for (int n = 0; n < N; ++n) dy[t * N + n] = Bf16(static_cast<float>((2 * t + n) % 3 - 1));
    }
    for (int i = 0; i < E * N * K; ++i) w[i] = Bf16(static_cast<float>(i % 5 - 2));
    const Device<float> dLogits(logits);
    const Device<std::uint16_t> dX(x), dW(w), dOut(dy);
    Device<float> weights(T);
    Device<std::int32_t> experts(T), offsets(E + 1), rows(T), slots(T);
    Device<std::uint16_t> y(T * N), out(T * N), dyRows(T * N), dxRows(T * K), dx(T * K), dw(E * N * K);

    const TensorInfo xi({T, K}, BF16, Layout::AB), yi({T, N}, BF16, Layout::AB);
    const MoeRoute route(TensorInfo({T, E}, F32, Layout::AB), kNone, 1, true);
    const GroupedLinear linear(xi, TensorInfo({E, K, N}, BF16, Layout::ACB), yi, true);
    const MoeCombine combine(yi, yi, 1), back(xi, xi, 1);
    Device<char> workspace(static_cast<std::size_t>(route.WorkspaceBytes()) + 16);
    CHECK(linear.WorkspaceBytes() == 0);
    route.Run(dLogits.p, nullptr, weights.p, experts.p, offsets.p, rows.p, slots.p, workspace.p);
    linear.Run(dX.p, dW.p, offsets.p, rows.p, y.p);
    combine.Run(y.p, weights.p, slots.p, out.p);
    combine.Backward(y.p, weights.p, slots.p, dOut.p, dyRows.p, nullptr);
    linear.BackwardInput(dyRows.p, dW.p, offsets.p, dxRows.p, nullptr);
    back.Run(dxRows.p, nullptr, slots.p, dx.p);
    linear.BackwardWeight(dyRows.p, dX.p, offsets.p, rows.p, dw.p, nullptr);
    Device<char>::Copied(hipDeviceSynchronize());

    const auto gotExperts = experts.Host();
    const auto gotOut = out.Host(), gotDx = dx.Host(), gotDw = dw.Host();
    std::vector<float> wantDw(E * N * K, 0.0f);
    bool same = true;
    for (int t = 0; t < T; ++t) {
        same = same && gotExperts[t] == expert[t];
        const std::uint16_t *we = w.data() + expert[t] * N * K;
        for (int n = 0; n < N; ++n) {
            float sum = 0.0f;
            for (int k = 0; k < K; ++k) {
                sum += F32Of(x[t * K + k]) * F32Of(we[n * K + k]);
                wantDw[(expert[t] * N + n) * K + k] += F32Of(dy[t * N + n]) * F32Of(x[t * K + k]);
            }
            same = same && F32Of(gotOut[t * N + n]) == sum;
        }
        for (int k = 0; k < K; ++k) {
            float sum = 0.0f;
            for (int n = 0; n < N; ++n) sum += F32Of(dy[t * N + n]) * F32Of(we[n * K + k]);
            same = same && F32Of(gotDx[t * K + k]) == sum;
        }
    }
    for (int i = 0; i < E * N * K; ++i) same = same && F32Of(gotDw[i]) == wantDw[i];
    CHECK(same);
}

int main(int argc, char **argv)
{
    std::setvbuf(stdout, nullptr, _IONBF, 0);
    Refusals();
    std::printf("refusals done\n");
    if (argc > 1 && std::strcmp(argv[1], "--gpu") == 0) {
        Integers();
    }
    std::printf("%d failed\n", g_failed);
    return g_failed == 0 ? 0 : 1;
}
