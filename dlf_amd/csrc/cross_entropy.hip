// Softmax cross entropy of the rows of a matrix of logits, whole or in pieces of the vocabulary,
// and its gradient.
#include "sequence.hip.h"

namespace dlfx {
namespace {

// Running maximum of a row and the sum of exp(x - maximum).
struct MaxSum {
    float mx, sum;
};
constexpr float kNone = -std::numeric_limits<float>::infinity();

__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
    const float mx = fmaxf(a.mx, b.mx);
    // an empty side (maximum -inf) adds its sum of 0, or the NaN that the side has met
    const float fa = a.mx == mx ? 1.0f : expf(a.mx - mx);
    const float fb = b.mx == mx ? 1.0f : expf(b.mx - mx);
    return {mx, a.sum * fa + b.sum * fb};
}
__device__ __forceinline__ void fold(MaxSum& s, float x) {
    if (x > s.mx) {
        s.sum = s.sum * expf(s.mx - x) + 1.0f;
        s.mx = x;
    } else if (x != kNone) {
        s.sum += x == s.mx ? 1.0f : expf(x - s.mx);        // NaN: the sum is NaN from here on
    }
}

template <int WAVES>
__device__ __forceinline__ MaxSum block_join(MaxSum v, MaxSum* lds) {
    v = wave_reduce(v, join);
    __syncthreads();
    if (lane_id() == 0) lds[threadIdx.x / kWave] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) v = join(v, lds[i]);
    return v;
}

// Loss of a finished row.  log(sum) + (maximum - logit) in this order: the difference is exact for
// nearby values, maximum + log(sum) would round at the maximum's size.
__device__ __forceinline__ float loss_of(MaxSum s, float logit, float z) {
    const float log_sum = logf(s.sum);
    if (s.sum == 0.0f) return std::numeric_limits<float>::infinity();
    float loss = log_sum + (s.mx - logit);
    if (z != 0.0f) {
        const float lse = s.mx + log_sum;
        loss += z * lse * lse;
    }
    return loss;
}

// What the elements of a row's gradient have in common: dx = up (factor exp(x - mx) - [target]).
struct RowGrad {
    float mx, factor, up;
    int64_t target;
};
__device__ __forceinline__ RowGrad row_grad(MaxSum s, int64_t target, float weight, float z) {
    RowGrad g = {s.mx, 0.0f, weight, target};
    if (target < 0) g.up = 0.0f;
    else if (s.sum == 0.0f) g.up = 0.0f;          // nothing but -inf
    else {
        g.factor = 1.0f / s.sum;
        if (z != 0.0f) g.factor *= 1.0f + 2.0f * z * (s.mx + logf(s.sum));
    }
    return g;
}
__device__ __forceinline__ float grad_of(const RowGrad& g, float x, int64_t j) {
    if (g.up == 0.0f && (g.target < 0 || g.factor == 0.0f)) return 0.0f;
    float p = g.factor * expf(x - g.mx);
    if (j == g.target) p -= 1.0f;
    return g.up * p;
}

// One workgroup per row.
template <typename S, typename I>
__global__ __launch_bounds__(256) void loss_rows(const S* x, int64_t n, int64_t stride, const I* targets, int64_t first, int resume,
                                                 float* state, int64_t m, float z, float* loss) {
    __shared__ MaxSum lds[4];
    const int64_t r = blockIdx.x;
    const S* xr = x + r * stride;
    const int64_t target = static_cast<int64_t>(targets[r]);
    if (target < 0) {
        if (threadIdx.x == 0) {
            if (loss) loss[r] = 0.0f;
            else if (!resume) state[r] = kNone, state[m + r] = 0.0f, state[2 * m + r] = std::numeric_limits<float>::quiet_NaN();
        }
        return;
    }
    MaxSum v = {kNone, 0.0f};
    for (int64_t j = threadIdx.x; j < n; j += 256) fold(v, static_cast<float>(xr[j]));
    v = block_join<4>(v, lds);
    if (threadIdx.x) return;
    float logit = std::numeric_limits<float>::quiet_NaN();
    if (!loss && resume) {
        v = join({state[r], state[m + r]}, v);
        logit = state[2 * m + r];
    }
    if (target >= first && target - first < n) logit = static_cast<float>(xr[target - first]);
    if (loss) {
        loss[r] = loss_of(v, logit, z);
    } else {
        state[r] = v.mx;
        state[m + r] = v.sum;
        state[2 * m + r] = logit;
    }
}

template <typename I>
__global__ __launch_bounds__(256) void loss_join(int64_t m, const I* targets, const float* state, float z, float* loss) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r >= m) return;
    loss[r] = targets[r] < 0 ? 0.0f : loss_of({state[r], state[m + r]}, state[2 * m + r], z);
}

template <typename S, typename I>
__global__ __launch_bounds__(256) void grad_rows(const S* x, int64_t n, int64_t stride, const I* targets, int64_t first, const float* state,
                                                 const float* weights, float z, int64_t m, float* loss, S* dx, int64_t dx_stride) {
    __shared__ MaxSum lds[4];
    const int64_t r = blockIdx.x;
    const S* xr = x + r * stride;
    S* dr = dx + r * dx_stride;
    const int64_t target = static_cast<int64_t>(targets[r]);
    MaxSum v = {kNone, 0.0f};
    if (state) {
        v = {state[r], state[m + r]};
    } else if (target >= 0) {
        for (int64_t j = threadIdx.x; j < n; j += 256) fold(v, static_cast<float>(xr[j]));
        v = block_join<4>(v, lds);
        if (loss && threadIdx.x == 0) loss[r] = loss_of(v, target < n ? static_cast<float>(xr[target]) : std::numeric_limits<float>::quiet_NaN(), z);
        __syncthreads();
    } else if (loss && threadIdx.x == 0) {
        loss[r] = 0.0f;
    }
    const RowGrad g = row_grad(v, target, weights ? weights[r] : 1.0f, z);
    for (int64_t j = threadIdx.x; j < n; j += 256) dr[j] = static_cast<S>(grad_of(g, static_cast<float>(xr[j]), first + j));
}

template <typename F>
int dispatch_index(int index_dtype, F&& f) {
    if (index_dtype == DLFX_I32) return f(int32_t());
    if (index_dtype == DLFX_I64) return f(int64_t());
    return DLFX_ERR_UNSUPPORTED_DTYPE;
}

int check(int64_t m, int64_t n, const void* x, int64_t row_stride, const void* targets) {
    if (m <= 0 || n <= 0 || !x || !targets || row_stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    if (m > 0x7fffffffLL || n > 0x7fffffffLL) return DLFX_ERR_TOO_LARGE;
    return DLFX_OK;
}

}  // namespace
}  // namespace dlfx

using namespace dlfx;

extern "C" size_t dlfx_cross_entropy_scratch_bytes(int, int64_t, int64_t) { return 0; }

extern "C" int dlfx_cross_entropy(dlfx_stream_t stream, int dtype, int index_dtype, int64_t m, int64_t n,
                                  const void* x, int64_t x_offset, int64_t row_stride, const void* targets,
                                  float z_loss, float* loss, void* scratch, size_t scratch_bytes) {
    if (int e = check(m, n, x, row_stride, targets)) return e;
    if (!loss) return DLFX_ERR_INVALID_ARGUMENT;
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        return dispatch_index(index_dtype, [&](auto index) {
            using I = decltype(index);
            loss_rows<S, I><<<dim3(static_cast<unsigned>(m)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const S*>(x) + x_offset, n, row_stride, static_cast<const I*>(targets), 0, 0, nullptr, m, z_loss, loss);
            DLFX_CHECK_LAUNCH();
            return static_cast<int>(DLFX_OK);
        });
    });
}

extern "C" int dlfx_cross_entropy_grad(dlfx_stream_t stream, int dtype, int index_dtype, int64_t m, int64_t n,
                                       const void* x, int64_t x_offset, int64_t row_stride, const void* targets,
                                       const float* weights, float z_loss, float* loss,
                                       void* dx, int64_t dx_offset, int64_t dx_row_stride,
                                       void* scratch, size_t scratch_bytes) {
    if (int e = check(m, n, x, row_stride, targets)) return e;
    if (!dx || dx_row_stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        return dispatch_index(index_dtype, [&](auto index) {
            using I = decltype(index);
            grad_rows<S, I><<<dim3(static_cast<unsigned>(m)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const S*>(x) + x_offset, n, row_stride, static_cast<const I*>(targets), 0, nullptr, weights, z_loss, m, loss,
                static_cast<S*>(dx) + dx_offset, dx_row_stride);
            DLFX_CHECK_LAUNCH();
            return static_cast<int>(DLFX_OK);
        });
    });
}

extern "C" int dlfx_cross_entropy_piece(dlfx_stream_t stream, int dtype, int index_dtype, int64_t m, int64_t n,
                                        const void* x, int64_t x_offset, int64_t row_stride, const void* targets,
                                        int64_t first, int resume, float* state, void* scratch, size_t scratch_bytes) {
    if (int e = check(m, n, x, row_stride, targets)) return e;
    if (!state || first < 0) return DLFX_ERR_INVALID_ARGUMENT;
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        return dispatch_index(index_dtype, [&](auto index) {
            using I = decltype(index);
            loss_rows<S, I><<<dim3(static_cast<unsigned>(m)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const S*>(x) + x_offset, n, row_stride, static_cast<const I*>(targets), first, resume, state, m, 0.0f, nullptr);
            DLFX_CHECK_LAUNCH();
            return static_cast<int>(DLFX_OK);
        });
    });
}

extern "C" int dlfx_cross_entropy_join(dlfx_stream_t stream, int index_dtype, int64_t m, const void* targets,
                                       const float* state, float z_loss, float* loss) {
    if (m <= 0 || !targets || !state || !loss) return DLFX_ERR_INVALID_ARGUMENT;
    if (m > 0x7fffffffLL) return DLFX_ERR_TOO_LARGE;
    return dispatch_index(index_dtype, [&](auto index) {
        using I = decltype(index);
        loss_join<I><<<dim3(static_cast<unsigned>(ceil_div(m, 256))), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
            m, static_cast<const I*>(targets), state, z_loss, loss);
        DLFX_CHECK_LAUNCH();
        return static_cast<int>(DLFX_OK);
    });
}

extern "C" int dlfx_cross_entropy_piece_grad(dlfx_stream_t stream, int dtype, int index_dtype, int64_t m, int64_t n,
                                             const void* x, int64_t x_offset, int64_t row_stride, const void* targets,
                                             int64_t first, const float* state, const float* weights, float z_loss,
                                             void* dx, int64_t dx_offset, int64_t dx_row_stride) {
    if (int e = check(m, n, x, row_stride, targets)) return e;
    if (!state || first < 0 || !dx || dx_row_stride < n) return DLFX_ERR_INVALID_ARGUMENT;
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        return dispatch_index(index_dtype, [&](auto index) {
            using I = decltype(index);
            grad_rows<S, I><<<dim3(static_cast<unsigned>(m)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                static_cast<const S*>(x) + x_offset, n, row_stride, static_cast<const I*>(targets), first, state, weights, z_loss, m, nullptr,
                static_cast<S*>(dx) + dx_offset, dx_row_stride);
            DLFX_CHECK_LAUNCH();
            return static_cast<int>(DLFX_OK);
        });
    });
}
