// Runs the sequence-model operators through the C++ host veneer (DevTensor front-ends over gpgpu::dnn
// over the C ABI) on values worked out by hand.  Needs a GPU.  Exit code 0 when every check passes;
// failures are listed on stderr.
#include <cmath>
#include <cstdio>
#include <limits>

#include "dev_tensor.h"

using namespace dlf;
using gpgpu::blas::bfloat16;
using gpgpu::blas::half;

static int g_failed = 0, g_checked = 0;

#define CHECK(cond)                                                              \
    do {                                                                         \
        ++g_checked;                                                             \
        if (!(cond)) {                                                           \
            ++g_failed;                                                          \
            std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
        }                                                                        \
    } while (0)

template <typename E, typename F>
static bool throws(F f) {
    try {
        f();
    } catch (const E&) {
        return true;
    } catch (...) {
    }
    return false;
}

// Within a few fp32 roundings of numbers of this size.
static bool near(const Tensor<float>& a, const std::vector<double>& b) {
    if (a.size() != b.size()) return false;
    for (size_t i = 0; i < b.size(); ++i)
        if (!(std::fabs(a.values()[i] - b[i]) <= 8 * std::ldexp(1.0, -24) * std::max(1.0, std::fabs(b[i])))) return false;
    return true;
}

// Gates of one half: every number below is a sum of few powers of two, exact in all three types.
template <typename T>
static void test_gated_scan() {
    auto G = dev(Tensor<T>({2, 3}, {T(0.5f), T(0.5f), T(0.5f), T(0.5f), T(0.f), T(0.5f)}));
    auto X = dev(Tensor<T>({2, 3}, {T(1.f), T(1.f), T(1.f), T(2.f), T(4.f), T(8.f)}));
    DevTensor<T> Y;
    DevTensor<float> last;
    gated_scan(G, X, Y, last, 1);
    CHECK(Y.read() == Tensor<T>({2, 3}, {T(1.f), T(1.5f), T(1.75f), T(2.f), T(4.f), T(10.f)}));
    CHECK(last.read() == Tensor<float>({2}, {1.75f, 10.f}));
    gated_scan(G, X, Y, last, 1, "gated", nullptr, true);
    CHECK(Y.read() == Tensor<T>({2, 3}, {T(1.75f), T(1.5f), T(1.f), T(4.f), T(4.f), T(8.f)}));

    // along the first axis, from a state, which is updated in place
    auto S = dev(Tensor<float>({3}, {4.f, 8.f, 16.f}));
    gated_scan(G, X, Y, S, 0, "gated", &S);
    CHECK(Y.read() == Tensor<T>({2, 3}, {T(3.f), T(5.f), T(9.f), T(3.5f), T(4.f), T(12.5f)}));
    CHECK(S.read() == Tensor<float>({3}, {3.5f, 4.f, 12.5f}));

    // gradients of the sum of all outputs: lam = 1.75, 1.5, 1 and 1, 1.5, 1 from the last step on
    gated_scan(G, X, Y, last, 1);
    auto dY = dev(Tensor<T>({2, 3}, {T(1.f), T(1.f), T(1.f), T(1.f), T(1.f), T(1.f)}));
    DevTensor<T> dG, dX;
    DevTensor<float> dS;
    gated_scan_grad(G, X, Y, dY, dG, dX, dS, 1);
    CHECK(dX.read() == Tensor<T>({2, 3}, {T(1.75f), T(1.5f), T(1.f), T(1.f), T(1.5f), T(1.f)}));
    CHECK(dG.read() == Tensor<T>({2, 3}, {T(0.f), T(1.5f), T(1.5f), T(0.f), T(3.f), T(4.f)}));
    CHECK(dS.read() == Tensor<float>({2}, {0.875f, 0.5f}));

    // logistic gates of 0: a = 1 - a = 1/2
    auto Z = dev(Tensor<T>({2, 3}, {T(0.f), T(0.f), T(0.f), T(0.f), T(0.f), T(0.f)}));
    gated_scan(Z, X, Y, last, 1, "gated_blend");
    CHECK(Y.read() == Tensor<T>({2, 3}, {T(0.5f), T(0.75f), T(0.875f), T(1.f), T(2.5f), T(5.25f)}));
    gated_scan_grad(Z, X, Y, dY, dG, dX, dS, 1, "gated_blend");
    CHECK(dX.read() == Tensor<T>({2, 3}, {T(0.875f), T(0.75f), T(0.5f), T(0.875f), T(0.75f), T(0.5f)}));
    gated_scan(Z, X, Y, last, 1, "gated_exp");
    CHECK(Y.read() == Tensor<T>({2, 3}, {T(1.f), T(2.f), T(3.f), T(2.f), T(6.f), T(14.f)}));

    CHECK(throws<gpgpu::RuntimeErrorCode>([&] { gated_scan(G, X, Y, last, 1, "gru"); }));
    CHECK(throws<shape_error>([&] { gated_scan(G.slice(1, 0, 2), X, Y, last, 1); }));
    CHECK(throws<shape_error>([&] { gated_scan(G, X, Y, last, 2); }));
    CHECK(throws<shape_error>([&] { gated_scan(G, X, Y, last, 1, "gated", &S); }));
}

static void test_long_scan() {
    // cut into segments, with scratch from the context: h counts 1, 2, ... with gates of one
    const size_t n = 20000, m = 3;
    std::vector<float> ones(n * m, 1.f);
    auto G = dev(Tensor<float>(Shape({n, m}), ones)), X = dev(Tensor<float>(Shape({n, m}), ones));
    DevTensor<float> Y, last;
    gated_scan(G, X, Y, last, 0);
    const auto y = Y.read();
    bool all = true;
    for (size_t i = 0; i < y.size(); ++i) all = all && y.values()[i] == static_cast<float>(i / m + 1);
    CHECK(all);
    CHECK(last.read() == Tensor<float>({3}, {20000.f, 20000.f, 20000.f}));
    CHECK(gpgpu::current::context().temporary_bytes_in_use() == 0);
}

static void test_route() {
    const float low = -std::numeric_limits<float>::infinity();
    auto X = dev(Tensor<float>({2, 4}, {0.f, 3.f, 2.f, 1.f, low, 1.f, 1.f, low}));
    DevTensor<float> W;
    DevTensor<int32_t> I;
    dnn::Routing how;
    how.k = 2;
    how.renormalise = true;
    how.scale = 2.f;
    DevTensor<int32_t> loads = dev(Tensor<int32_t>({4}, {10, 10, 10, 10}));
    dnn::route(X, W, I, how, "softmax", nullptr, &loads);
    const double e = std::exp(1.0);
    CHECK(I.read() == Tensor<int32_t>({2, 2}, {1, 2, 1, 2}));
    CHECK(near(W.read(), {2 * e / (1 + e), 2 / (1 + e), 1, 1}));
    CHECK(loads.read() == Tensor<int32_t>({4}, {10, 12, 12, 10}));

    // a bias decides who is chosen, not what they weigh
    auto bias = dev(Tensor<float>({4}, {0.f, -5.f, 0.f, 0.9f}));
    how.renormalise = false;
    how.scale = 1.f;
    dnn::route(X, W, I, how, "sigmoid", &bias);
    CHECK(I.read() == Tensor<int32_t>({2, 2}, {3, 2, 2, 1}));
    auto sig = [](double v) { return 1 / (1 + std::exp(-v)); };
    CHECK(near(W.read(), {sig(1), sig(2), sig(1), sig(1)}));

    // two groups of two, one kept
    how.groups = 2;
    how.kept_groups = 1;
    how.group_best = 2;
    dnn::route(X, W, I, how, "softmax");
    CHECK(I.read() == Tensor<int32_t>({2, 2}, {1, 0, 1, 0}));

    how = dnn::Routing();
    how.k = 2;
    dnn::route(X, W, I, how, "sigmoid");
    auto dW = dev(Tensor<float>({2, 2}, {1.f, 2.f, 3.f, 4.f}));
    DevTensor<float> dX;
    dnn::route_grad(X, I, dW, dX, how, "sigmoid");
    auto slope = [&](double v) { return sig(v) * sig(-v); };
    CHECK(near(dX.read(), {0, slope(3), 2 * slope(2), 0, 0, 3 * slope(1), 4 * slope(1), 0}));
    how.k = 5;
    CHECK(throws<gpgpu::RuntimeErrorCode>([&] { dnn::route(X, W, I, how); }));
    CHECK(throws<shape_error>([&] { dnn::route_grad(X, I, dW, dX, how); }));
}

template <typename I>
static void test_cross_entropy() {
    const double ln4 = std::log(4.0);
    auto X = dev(Tensor<float>({3, 4}, {0.f, 0.f, 0.f, 0.f, 5.f, 5.f, 5.f, 5.f, 1.f, 2.f, 3.f, 4.f}));
    auto t = dev(Tensor<I>({3}, {I(1), I(0), I(-1)}));
    DevTensor<float> loss, dX;
    dnn::cross_entropy(X, t, loss);
    CHECK(near(loss.read(), {ln4, ln4, 0}));
    auto w = dev(Tensor<float>({3}, {1.f, 2.f, 3.f}));
    dnn::cross_entropy_grad(X, t, loss, dX, &w);
    CHECK(near(loss.read(), {ln4, ln4, 0}));
    CHECK(near(dX.read(), {0.25, -0.75, 0.25, 0.25, -1.5, 0.5, 0.5, 0.5, 0, 0, 0, 0}));

    DevTensor<float> state, joined, A, B;
    reorder(X.slice(1, 0, 1), A);
    reorder(X.slice(1, 1, 4), B);
    dnn::cross_entropy_piece(A, t, 0, state);
    dnn::cross_entropy_piece(B, t, 1, state);
    dnn::cross_entropy_join(t, state, joined);
    CHECK(near(joined.read(), {ln4, ln4, 0}));
    dnn::cross_entropy_piece_grad(B, t, 1, state, B, &w);                 // in place
    CHECK(near(B.read(), {-0.75, 0.25, 0.25, 0.5, 0.5, 0.5, 0, 0, 0}));
    dnn::cross_entropy_grad(X, t, loss, X, &w, 0.5f);                     // in place, with z loss
    CHECK(near(loss.read(), {ln4 + 0.5 * ln4 * ln4, ln4 + 0.5 * (5 + ln4) * (5 + ln4), 0}));
    CHECK(near(X.read(), {(1 + ln4) / 4, (1 + ln4) / 4 - 1, (1 + ln4) / 4, (1 + ln4) / 4, 2 * ((6 + ln4) / 4 - 1), (6 + ln4) / 2, (6 + ln4) / 2,
                          (6 + ln4) / 2, 0, 0, 0, 0}));
    auto one = dev(Tensor<I>({1}, {I(0)}));
    CHECK(throws<shape_error>([&] { dnn::cross_entropy(X, one, loss); }));
}

static void test_bfloat16() {
    CHECK(static_cast<float>(bfloat16(1.5f)) == 1.5f && static_cast<float>(bfloat16(-3.0e38f)) < -2.9e38f);
    CHECK(static_cast<float>(bfloat16(1.0f + std::ldexp(1.f, -8))) == 1.0f);                          // ties to even
    CHECK(static_cast<float>(bfloat16(1.0f + 3 * std::ldexp(1.f, -8))) == 1.0f + std::ldexp(1.f, -6));
    CHECK(std::isnan(static_cast<float>(bfloat16(std::numeric_limits<float>::quiet_NaN()))));
    CHECK(std::isinf(static_cast<float>(bfloat16(std::numeric_limits<float>::max()))));
    DevTensor<bfloat16> T;
    reorder(dev(Tensor<bfloat16>({2, 2}, {bfloat16(1.f), bfloat16(2.f), bfloat16(3.f), bfloat16(4.f)})).transpose(), T);
    CHECK(T.read() == Tensor<bfloat16>({2, 2}, {bfloat16(1.f), bfloat16(3.f), bfloat16(2.f), bfloat16(4.f)}));
}

int main() {
    try {
        test_gated_scan<float>();
        test_gated_scan<half>();
        test_gated_scan<bfloat16>();
        test_long_scan();
        test_route();
        test_cross_entropy<int32_t>();
        test_cross_entropy<int64_t>();
        test_bfloat16();
    } catch (const std::exception& e) {
        std::fprintf(stderr, "exception: %s\n", e.what());
        return 1;
    }
    std::printf("%d checked, %d failed\n", g_checked, g_failed);
    return g_failed ? 1 : 0;
}
