// Routing to experts: scores of a row of router logits, the k largest choices among the kept
// groups, their weights; and the gradient of the logits.
#include <cstring>

#include "sequence.hip.h"

namespace dlfx {
namespace {

enum ScoreKind { kSoftmaxScore = 0, kSigmoidScore = 1 };

template <typename S> __device__ __forceinline__ float lowest_of();
template <> __device__ __forceinline__ float lowest_of<float>() { return -3.40282346638528859812e38f; }
template <> __device__ __forceinline__ float lowest_of<half_t>() { return -65504.0f; }
template <> __device__ __forceinline__ float lowest_of<bf16_t>() { return -3.38953138925153547590e38f; }

// Choices are compared as unsigned images that keep the order of doubles: an expert outside the
// kept groups 0, an absent one (or a NaN) 1, every number above that.
__device__ __forceinline__ uint64_t image_of(double v) {
    if (v != v) return 1;
    v += 0.0;                              // -0.0 and +0.0 are one value
    const uint64_t u = bit_cast<uint64_t>(v);
    return (u >> 63) ? ~u : (u | 0x8000000000000000ull);
}

// One wavefront per row: item i of a lane is expert i * 64 + lane.
template <typename S, int KIND, int ITEMS>
__global__ __launch_bounds__(256) void route_rows(const S* x, int64_t m, int n, int64_t stride, const float* bias, int groups, int kept_groups,
                                                  int group_best, int k, int renormalise, float scale, float* weights, int32_t* indices,
                                                  int32_t* loads) {
    const int lane = threadIdx.x % kWave;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (r >= m) return;
    const S* xr = x + r * stride;
    double score[ITEMS], choice[ITEMS];
    bool present[ITEMS];
    double mx = -std::numeric_limits<double>::infinity();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int e = i * kWave + lane;
        const float v = e < n ? static_cast<float>(xr[e]) : -std::numeric_limits<float>::infinity();
        present[i] = !(v <= lowest_of<S>());
        score[i] = v;
        if (present[i]) mx = v > mx ? v : mx;
    }
    mx = wave_reduce(mx, [](double a, double b) { return b > a ? b : a; });
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        choice[i] = score[i];
        if constexpr (KIND == kSoftmaxScore) score[i] = present[i] ? exp(score[i] - mx) : 0.0;
        else score[i] = present[i] ? 1.0 / (1.0 + exp(-score[i])) : 0.0;
        sum += score[i];
    }
    if constexpr (KIND == kSoftmaxScore) {
        sum = wave_reduce(sum, [](double a, double b) { return a + b; });
        const double scale_by = sum == 0.0 ? 0.0 : 1.0 / sum;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) score[i] *= scale_by;
    }
    const bool by_score = bias || kept_groups < groups;
    uint64_t image[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int e = i * kWave + lane;
        if (by_score) choice[i] = score[i] + (bias && e < n ? static_cast<double>(bias[e]) : 0.0);
        image[i] = e >= n ? 0 : present[i] ? image_of(choice[i]) : 1;
    }
    if (kept_groups < groups) {
        const int size = n / groups;
        // one group at a time: its value; then the groups are kept best first
        uint64_t group_image[ITEMS];       // group i * 64 + lane
        for (int i = 0; i < ITEMS; ++i) group_image[i] = 0;
        for (int g = 0; g < groups; ++g) {
            uint64_t best = 0;
            int at = -1;
            double value = 0.0;
            bool any = false;
            for (int round = 0; round < group_best; ++round) {
                uint64_t mine = 0;
                int where = 0x7fffffff;
                for (int i = 0; i < ITEMS; ++i) {
                    const int e = i * kWave + lane;
                    if (e / size != g || e >= n || e == at || image[i] <= 1) continue;
                    if (image[i] > mine) mine = image[i], where = e;
                }
                best = wave_reduce(mine, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
                if (best <= 1) break;
                int first = mine == best ? where : 0x7fffffff;
                first = wave_reduce(first, [](int a, int b) { return a < b ? a : b; });
                at = first;
                value += (best >> 63) ? bit_cast<double>(best & 0x7fffffffffffffffull) : bit_cast<double>(~best);
                any = true;
            }
            const uint64_t gi = any ? image_of(value) : 1;
            for (int i = 0; i < ITEMS; ++i)
                if (i * kWave + lane == g) group_image[i] = gi;
        }
        uint64_t open[ITEMS];
        for (int i = 0; i < ITEMS; ++i) open[i] = 0;
        for (int t = 0; t < kept_groups; ++t) {
            uint64_t mine = 0;
            int where = 0x7fffffff;
            for (int i = 0; i < ITEMS; ++i)
                if (group_image[i] > mine) mine = group_image[i], where = i * kWave + lane;
            const uint64_t best = wave_reduce(mine, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
            int first = mine == best ? where : 0x7fffffff;
            first = wave_reduce(first, [](int a, int b) { return a < b ? a : b; });
            for (int i = 0; i < ITEMS; ++i) {
                if (i * kWave + lane == first) group_image[i] = 0;
                if ((i * kWave + lane) / size == first) open[i] = 1;
            }
        }
        for (int i = 0; i < ITEMS; ++i)
            if (!open[i]) image[i] = 0;
    }
    double total = 0.0, my_score = 0.0;
    int my_index = 0;
    for (int t = 0; t < k; ++t) {
        uint64_t mine = 0;
        int where = 0x7fffffff;
        double s = 0.0;
        for (int i = 0; i < ITEMS; ++i)
            if (image[i] > mine) mine = image[i], where = i * kWave + lane, s = score[i];
        const uint64_t best = wave_reduce(mine, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
        int first = mine == best ? where : 0x7fffffff;
        first = wave_reduce(first, [](int a, int b) { return a < b ? a : b; });
        const double chosen = lane_get(s, first % kWave);
        for (int i = 0; i < ITEMS; ++i)
            if (i * kWave + lane == first) image[i] = 0;
        total += chosen;
        if (lane == t) my_index = first, my_score = chosen;
    }
    if (lane < k) {
        double w = my_score;
        if (renormalise) w = total == 0.0 ? 0.0 : w / total;
        weights[r * k + lane] = static_cast<float>(w * static_cast<double>(scale));
        indices[r * k + lane] = my_index;
        if (loads) atomicAdd(&loads[my_index], 1);
    }
}

template <typename S, int KIND, int ITEMS>
__global__ __launch_bounds__(256) void route_grad_rows(const S* x, int64_t m, int n, int64_t stride, int k, const int32_t* indices,
                                                       const float* dweights, int renormalise, float scale, S* dx, int64_t dx_stride) {
    const int lane = threadIdx.x % kWave;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 4 + threadIdx.x / kWave;
    if (r >= m) return;
    const S* xr = x + r * stride;
    float s[ITEMS], ds[ITEMS], rest[ITEMS];
    float mx = -std::numeric_limits<float>::infinity();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int e = i * kWave + lane;
        s[i] = e < n ? static_cast<float>(xr[e]) : -std::numeric_limits<float>::infinity();
        if (s[i] <= lowest_of<S>()) s[i] = -std::numeric_limits<float>::infinity();
        mx = fmaxf(mx, s[i]);
        ds[i] = 0.0f;
    }
    mx = wave_reduce(mx, [](float a, float b) { return fmaxf(a, b); });
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const float v = s[i];
        const bool present = v != -std::numeric_limits<float>::infinity();
        if constexpr (KIND == kSoftmaxScore) {
            s[i] = present ? expf(v - mx) : 0.0f;
        } else {
            const float e = expf(-fabsf(v)), big = 1.0f / (1.0f + e), small = e * big;
            s[i] = !present ? 0.0f : v < 0.0f ? small : big;
            rest[i] = v < 0.0f ? big : small;
        }
        sum += s[i];
    }
    if constexpr (KIND == kSoftmaxScore) {
        sum = wave_reduce(sum, [](float a, float b) { return a + b; });
        const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) s[i] *= by;
    }
    // chosen[i]: how often the row's k places name the expert; ds its share of the weights' gradients
    float chosen[ITEMS];
    for (int i = 0; i < ITEMS; ++i) chosen[i] = 0.0f;
    for (int t = 0; t < k; ++t) {
        const int e = indices[r * k + t];
        const float d = dweights[r * k + t] * scale;
        for (int i = 0; i < ITEMS; ++i)
            if (i * kWave + lane == e && e < n) ds[i] += d, chosen[i] += 1.0f;
    }
    if (renormalise) {
        float total = 0.0f, dot = 0.0f;
        for (int i = 0; i < ITEMS; ++i) total += chosen[i] * s[i], dot += ds[i] * s[i];
        total = wave_reduce(total, [](float a, float b) { return a + b; });
        dot = wave_reduce(dot, [](float a, float b) { return a + b; });
        const float by = total == 0.0f ? 0.0f : 1.0f / total;
        for (int i = 0; i < ITEMS; ++i) ds[i] = (ds[i] - chosen[i] * dot * by) * by;
    }
    if constexpr (KIND == kSoftmaxScore) {
        float dot = 0.0f;
        // renormalised weights do not change with the scores' common factor: the sum is 0
        if (!renormalise) {
            for (int i = 0; i < ITEMS; ++i) dot += ds[i] * s[i];
            dot = wave_reduce(dot, [](float a, float b) { return a + b; });
        }
        for (int i = 0; i < ITEMS; ++i) s[i] *= ds[i] - dot;
    } else {
        for (int i = 0; i < ITEMS; ++i) s[i] *= ds[i] * rest[i];
    }
    for (int i = 0; i < ITEMS; ++i) {
        const int e = i * kWave + lane;
        if (e < n) dx[r * dx_stride + e] = static_cast<S>(s[i]);
    }
}

template <typename F>
int dispatch_items(int64_t n, F&& f) {
    if (n <= 64) return f(std::integral_constant<int, 1>());
    if (n <= 128) return f(std::integral_constant<int, 2>());
    if (n <= 256) return f(std::integral_constant<int, 4>());
    if (n <= 512) return f(std::integral_constant<int, 8>());
    return f(std::integral_constant<int, 16>());
}

int check(const char* name, int64_t m, int64_t n, int64_t k, const void* x, int64_t stride, int* kind) {
    if (!name || !x || m <= 0 || n <= 0 || k <= 0 || k > n || stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    if (!std::strcmp(name, "softmax")) *kind = kSoftmaxScore;
    else if (!std::strcmp(name, "sigmoid")) *kind = kSigmoidScore;
    else return DLFX_ERR_UNKNOWN_OP;
    if (n > DLFX_ROUTE_MAX_N || k > DLFX_ROUTE_MAX_K || ceil_div(m, 4) > 0x7fffffffLL) return DLFX_ERR_TOO_LARGE;
    return DLFX_OK;
}

}  // namespace
}  // namespace dlfx

using namespace dlfx;

extern "C" int dlfx_route(dlfx_stream_t stream, const char* name, int dtype, int64_t m, int64_t n,
                          const void* x, int64_t x_offset, int64_t row_stride, const float* bias,
                          int64_t groups, int64_t kept_groups, int group_best, int64_t k, int renormalise, float scale,
                          float* weights, int32_t* indices, int32_t* loads) {
    int kind;
    if (int e = check(name, m, n, k, x, row_stride, &kind)) return e;
    if (!weights || !indices) return DLFX_ERR_INVALID_ARGUMENT;
    if (groups <= 0 || n % groups || kept_groups <= 0 || kept_groups > groups || (group_best != 1 && group_best != 2)) return DLFX_ERR_INVALID_ARGUMENT;
    if (kept_groups * (n / groups) < k) return DLFX_ERR_INVALID_ARGUMENT;
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        return dispatch_items(n, [&](auto items) {
            constexpr int ITEMS = decltype(items)::value;
            auto run = [&](auto kernel) {
                kernel<<<dim3(static_cast<unsigned>(ceil_div(m, 4))), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                    static_cast<const S*>(x) + x_offset, m, static_cast<int>(n), row_stride, bias, static_cast<int>(groups),
                    static_cast<int>(kept_groups), group_best, static_cast<int>(k), renormalise, scale, weights, indices, loads);
                DLFX_CHECK_LAUNCH();
                return static_cast<int>(DLFX_OK);
            };
            return kind == kSoftmaxScore ? run(route_rows<S, kSoftmaxScore, ITEMS>) : run(route_rows<S, kSigmoidScore, ITEMS>);
        });
    });
}

extern "C" int dlfx_route_grad(dlfx_stream_t stream, const char* name, int dtype, int64_t m, int64_t n,
                               const void* x, int64_t x_offset, int64_t row_stride,
                               int64_t k, const int32_t* indices, const float* dweights, int renormalise, float scale,
                               void* dx, int64_t dx_offset, int64_t dx_row_stride) {
    int kind;
    if (int e = check(name, m, n, k, x, row_stride, &kind)) return e;
    if (!indices || !dweights || !dx || dx_row_stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        return dispatch_items(n, [&](auto items) {
            constexpr int ITEMS = decltype(items)::value;
            auto run = [&](auto kernel) {
                kernel<<<dim3(static_cast<unsigned>(ceil_div(m, 4))), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                    static_cast<const S*>(x) + x_offset, m, static_cast<int>(n), row_stride, static_cast<int>(k), indices, dweights, renormalise,
                    scale, static_cast<S*>(dx) + dx_offset, dx_row_stride);
                DLFX_CHECK_LAUNCH();
                return static_cast<int>(DLFX_OK);
            };
            return kind == kSoftmaxScore ? run(route_grad_rows<S, kSoftmaxScore, ITEMS>) : run(route_grad_rows<S, kSigmoidScore, ITEMS>);
        });
    });
}
