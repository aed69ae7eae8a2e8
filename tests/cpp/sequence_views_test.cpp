// Runs the sequence-model operators through the C++ host veneer on views: rows at a stride, results over their own
// inputs.  Needs a GPU.  Exit code 0 when every check passes; failures are listed on stderr.
#include <cmath>
#include <cstdio>

#include "dev_tensor.h"

using namespace dlf;

static int g_failed = 0, g_checked = 0;

#define CHECK(cond)                                                              \
    do {                                                                         \
        ++g_checked;                                                             \
        if (!(cond)) {                                                           \
            ++g_failed;                                                          \
            std::fprintf(stderr, "FAILED %s:%d: %s\n", __FILE__, __LINE__, #cond); \
        }                                                                        \
    } while (0)

template <typename F>
static bool refuses(F f) {
    try {
        f();
    } catch (const shape_error&) {
        return true;
    }
    return false;
}

// [rows, 8] of which columns 2 to 7 are the logits
static DevTensor<float> wide() {
    std::vector<float> v(6 * 8);
    for (size_t i = 0; i < v.size(); ++i) v[i] = 0.25f * static_cast<float>((i * 7) % 11) - 1.0f;
    return dev(Tensor<float>({6, 8}, v));
}

// Everything on a slice gives what it gives on the slice's dense copy; what lies beside the slice stays.
static void test_rows_at_a_stride() {
    const auto before = wide().read();
    auto W = wide();
    auto X = W.slice(1, 2, 7);
    DevTensor<float> D;
    reorder(X, D);
    dnn::Routing how;
    how.k = 2;
    how.renormalise = true;
    DevTensor<float> w0, w1, g0, g1;
    DevTensor<int32_t> i0, i1;
    dnn::route(D, w0, i0, how);
    dnn::route(X, w1, i1, how);
    CHECK(w0.read() == w1.read());
    CHECK(i0.read() == i1.read());
    dnn::route_grad(D, i0, w0, g0, how);
    dnn::route_grad(X, i0, w0, g1, how);
    CHECK(g0.read() == g1.read());

    const auto t = dev(Tensor<int32_t>({6}, {0, 4, -1, 2, 3, 1}));
    DevTensor<float> l0, l1, s0, s1;
    dnn::cross_entropy(D, t, l0);
    dnn::cross_entropy(X, t, l1);
    CHECK(l0.read() == l1.read());
    dnn::cross_entropy_grad(D, t, l0, g0);
    dnn::cross_entropy_grad(X, t, l1, g1);
    CHECK(l0.read() == l1.read() && g0.read() == g1.read());
    dnn::cross_entropy_piece(D, t, 0, s0);
    dnn::cross_entropy_piece(X, t, 0, s1);
    dnn::cross_entropy_join(t, s0, l0);
    dnn::cross_entropy_join(t, s1, l1);
    CHECK(l0.read() == l1.read());
    dnn::cross_entropy_piece_grad(D, t, 0, s0, g0);
    dnn::cross_entropy_piece_grad(X, t, 0, s1, g1);
    CHECK(g0.read() == g1.read());
    CHECK(W.read() == before);

    // over the slice itself
    dnn::cross_entropy_grad(X, t, l1, X);
    CHECK(X.read() == g0.read());
    const auto after = W.read();
    for (size_t r = 0; r < 6; ++r)
        for (size_t c : {0, 1, 7}) CHECK(after.values()[8 * r + c] == before.values()[8 * r + c]);

    // three axes whose rows lie at one stride, and views whose do not
    auto C = wide().view(Shape::as_strided({2, 3, 5}, {24, 8, 1}, 2));
    dnn::cross_entropy(C, dev(Tensor<int32_t>({2, 3}, {0, 4, -1, 2, 3, 1})), l1);
    dnn::cross_entropy(D, t, l0);
    CHECK(l1.shape() == Shape({2, 3}) && l1.read().values() == l0.read().values());
    CHECK(refuses([&] { dnn::cross_entropy(W.transpose(), dev(Tensor<int32_t>({8}, std::vector<int32_t>(8, 0))), l1); }));
    CHECK(refuses([&] { dnn::cross_entropy(flip(W, 0), t, l1); }));
    CHECK(refuses([&] { dnn::cross_entropy(W.slice(0, 0, 4).view(Shape::as_strided({2, 2, 5}, {8, 16, 1}, 0)),
                                           dev(Tensor<int32_t>({2, 2}, {0, 0, 0, 0})), l1); }));
    CHECK(refuses([&] { dnn::cross_entropy(W.view(Shape::as_strided({6, 8}, {0, 1}, 0)), t, l1); }));
}

// A gradient over an input that is a view: the input is read where it lies.
static void test_gradients_over_views() {
    const std::vector<float> gate = {0.5f, 0.25f, 1.f, 2.f, 0.5f, 1.f, 0.f, 0.5f}, dy = {1.f, 2.f, -1.f, 0.5f, 4.f, 1.f, 2.f, 8.f};
    auto dense_g = dev(Tensor<float>({2, 3}, {gate[1], gate[3], gate[5], gate[2], gate[4], gate[6]}));
    auto dense_dy = dev(Tensor<float>({2, 3}, {dy[1], dy[3], dy[5], dy[2], dy[4], dy[6]}));
    auto Y = dev(Tensor<float>({2, 3}, {1.f, 2.f, 3.f, 4.f, 5.f, 6.f}));
    auto dlast = dev(Tensor<float>({2}, {0.5f, -1.f}));
    DevTensor<float> dG, dX, dS;
    gated_scan_grad(dense_g, Y, Y, dense_dy, dG, dX, dS, 1, "gated", nullptr, &dlast);
    auto g = dev(Tensor<float>({8}, gate)).view(Shape::as_strided({2, 3}, {1, 2}, 1));
    auto d = dev(Tensor<float>({8}, dy)).view(Shape::as_strided({2, 3}, {1, 2}, 1));
    auto s = dev(Tensor<float>({4}, {9.f, 0.5f, 9.f, -1.f})).view(Shape::as_strided({2}, {2}, 1));
    gated_scan_grad(g, Y, Y, d, g, d, s, 1, "gated", nullptr, &s);
    CHECK(g.read() == dG.read());
    CHECK(d.read() == dX.read());
    CHECK(s.read() == dS.read());
}

int main() {
    try {
        test_rows_at_a_stride();
        test_gradients_over_views();
    } catch (const std::exception& e) {
        std::fprintf(stderr, "exception: %s\n", e.what());
        return 1;
    }
    std::printf("%d checked, %d failed\n", g_checked, g_failed);
    return g_failed ? 1 : 0;
}
