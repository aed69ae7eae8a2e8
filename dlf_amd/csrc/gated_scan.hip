// Gated linear recurrence h[t] = a[t] h[t-1] + b[t] along one axis of strided views, and its
// backward pass.
#include <cstring>

#include "sequence.hip.h"

namespace dlfx {
namespace {

enum GateKind { kGated = 0, kGatedExp = 1, kGatedSigmoid = 2, kGatedBlend = 3 };

// Everything of a call that a kernel walks: row r of a tensor starts at base + row.at(r), step t is
// t * step elements further on.
template <typename S>
struct Track {
    S* base;
    int64_t step;
    DimMap row;
};

// Factor a of the state and 1 - a (blend: the factor of x; sigmoid and blend: a' = a (1 - a)).
// The logistic function from e = exp(-|g|) <= 1: the larger of a and 1 - a is 1 / (1 + e), the
// smaller e / (1 + e), so neither is a difference of nearby numbers and g = +-inf gives 1 and 0.
template <typename S, int KIND>
__device__ __forceinline__ void gate_of(float g, float& a, float& keep) {
    if constexpr (KIND == kGated) {
        a = g;
    } else if constexpr (KIND == kGatedExp) {
        a = fast_exp<S>(g);
    } else {
        const float e = fast_exp<S>(-fabsf(g));
        const float r = fast_reciprocal<S>(1.0f + e);
        const float small = e * r;
        a = g < 0.0f ? small : r;
        keep = g < 0.0f ? r : small;
    }
}

// One lane per row, step after step.
template <typename S, int KIND>
__global__ __launch_bounds__(256) void gated_walk(int64_t m, int64_t n, Track<const S> g, Track<const S> x, Track<const float> initial,
                                                  Track<S> y, Track<float> last) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r >= m) return;
    const S* gp = g.base + g.row.at(r);
    const S* xp = x.base + x.row.at(r);
    S* yp = y.base + y.row.at(r);
    float h = initial.base ? initial.base[initial.row.at(r)] : 0.0f;
    for (int64_t t = 0; t < n; ++t) {
        float a, keep = 1.0f, b = static_cast<float>(xp[t * x.step]);
        gate_of<S, KIND>(static_cast<float>(gp[t * g.step]), a, keep);
        if constexpr (KIND == kGatedBlend) b *= keep;
        h = fmaf(a, h, b);
        yp[t * y.step] = static_cast<S>(h);
    }
    if (last.base) last.base[last.row.at(r)] = h;
}

template <typename S, int KIND>
__global__ __launch_bounds__(256) void gated_grad_walk(int64_t m, int64_t n, Track<const S> g, Track<const S> x, Track<const float> initial,
                                                       Track<const S> y, Track<const S> dy, Track<const float> dlast,
                                                       Track<S> dg, Track<S> dx, Track<float> dinitial) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (r >= m) return;
    const S* gp = g.base + g.row.at(r);
    const S* xp = KIND == kGatedBlend ? x.base + x.row.at(r) : nullptr;
    const S* yp = y.base + y.row.at(r);
    const S* dyp = dy.base + dy.row.at(r);
    S* dgp = dg.base + dg.row.at(r);
    S* dxp = dx.base + dx.row.at(r);
    float mu = dlast.base ? dlast.base[dlast.row.at(r)] : 0.0f;
    const float h0 = initial.base ? initial.base[initial.row.at(r)] : 0.0f;
    for (int64_t t = n - 1; t >= 0; --t) {
        float a, keep = 1.0f;
        gate_of<S, KIND>(static_cast<float>(gp[t * g.step]), a, keep);
        const float lam = static_cast<float>(dyp[t * dy.step]) + mu;
        float before = t > 0 ? static_cast<float>(yp[(t - 1) * y.step]) : h0;
        if constexpr (KIND == kGatedBlend) before -= static_cast<float>(xp[t * x.step]);
        float d = lam * before;
        if constexpr (KIND == kGatedExp) d *= a;
        if constexpr (KIND == kGatedSigmoid || KIND == kGatedBlend) d *= a * keep;
        mu = a * lam;
        dgp[t * dg.step] = static_cast<S>(d);
        dxp[t * dx.step] = static_cast<S>(KIND == kGatedBlend ? lam * keep : lam);
    }
    if (dinitial.base) dinitial.base[dinitial.row.at(r)] = mu;
}

template <typename S>
bool make_track(int rank, const int64_t* dims, const void* base, int64_t offset, const int64_t* strides, bool per_row, Track<S>* out) {
    using E = typename std::remove_const<S>::type;
    out->base = base ? const_cast<S*>(static_cast<const E*>(base) + offset) : nullptr;
    out->step = 0;
    if (!base) {
        out->row.rank = 0;
        return true;
    }
    if (!per_row) out->step = strides[rank - 1];
    return make_dim_map(dims, strides, 0, rank - 1, &out->row);
}

int kind_of(const char* name) {
    if (!std::strcmp(name, "gated")) return kGated;
    if (!std::strcmp(name, "gated_exp")) return kGatedExp;
    if (!std::strcmp(name, "gated_sigmoid")) return kGatedSigmoid;
    if (!std::strcmp(name, "gated_blend")) return kGatedBlend;
    return -1;
}

template <typename F>
int dispatch_kind(int kind, F&& f) {
    switch (kind) {
    case kGated: return f(std::integral_constant<int, kGated>());
    case kGatedExp: return f(std::integral_constant<int, kGatedExp>());
    case kGatedSigmoid: return f(std::integral_constant<int, kGatedSigmoid>());
    default: return f(std::integral_constant<int, kGatedBlend>());
    }
}

bool shape_ok(int64_t m, int64_t n, int rank, const int64_t* dims, const int64_t* some_strides) {
    if (m <= 0 || n <= 0 || rank < 1) return false;
    if (!view_ok(rank, dims, some_strides)) return false;
    return dims[rank - 1] == n && view_size(rank - 1, dims) == m;
}

}  // namespace
}  // namespace dlfx

using namespace dlfx;

extern "C" size_t dlfx_gated_scan_scratch_bytes(int, int64_t, int64_t) { return 0; }

extern "C" int dlfx_gated_scan(dlfx_stream_t stream, const char* name, int dtype, int64_t m, int64_t n,
                               int rank, const int64_t* dims,
                               const void* gate, int64_t gate_offset, const int64_t* gate_strides,
                               const void* x, int64_t x_offset, const int64_t* x_strides,
                               const float* initial, int64_t initial_offset, const int64_t* initial_strides,
                               void* y, int64_t y_offset, const int64_t* y_strides,
                               float* last, int64_t last_offset, const int64_t* last_strides,
                               void* scratch, size_t scratch_bytes) {
    if (!name || !gate || !x || !y || !gate_strides || !x_strides || !y_strides) return DLFX_ERR_INVALID_ARGUMENT;
    const int kind = kind_of(name);
    if (kind < 0) return DLFX_ERR_UNKNOWN_OP;
    if (!shape_ok(m, n, rank, dims, y_strides) || !strides_distinct(rank, dims, y_strides)) return DLFX_ERR_INVALID_ARGUMENT;
    if (rank > 1 && ((initial && !initial_strides) || (last && !last_strides))) return DLFX_ERR_INVALID_ARGUMENT;
    if (last && !strides_distinct(rank - 1, dims, last_strides)) return DLFX_ERR_INVALID_ARGUMENT;
    (void)scratch; (void)scratch_bytes;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        Track<const S> tg, tx;
        Track<S> ty;
        Track<const float> ti;
        Track<float> tl;
        if (!make_track(rank, dims, gate, gate_offset, gate_strides, false, &tg) || !make_track(rank, dims, x, x_offset, x_strides, false, &tx) ||
            !make_track(rank, dims, y, y_offset, y_strides, false, &ty) || !make_track(rank, dims, initial, initial_offset, initial_strides, true, &ti) ||
            !make_track(rank, dims, last, last_offset, last_strides, true, &tl))
            return static_cast<int>(DLFX_ERR_RANK);
        if (ceil_div(m, 256) > 0x7fffffffLL) return static_cast<int>(DLFX_ERR_TOO_LARGE);
        return dispatch_kind(kind, [&](auto k) {
            gated_walk<S, decltype(k)::value><<<dim3(static_cast<unsigned>(ceil_div(m, 256))), dim3(256), 0, s>>>(m, n, tg, tx, ti, ty, tl);
            DLFX_CHECK_LAUNCH();
            return static_cast<int>(DLFX_OK);
        });
    });
}

extern "C" int dlfx_gated_scan_grad(dlfx_stream_t stream, const char* name, int dtype, int64_t m, int64_t n,
                                    int rank, const int64_t* dims,
                                    const void* gate, int64_t gate_offset, const int64_t* gate_strides,
                                    const void* x, int64_t x_offset, const int64_t* x_strides,
                                    const float* initial, int64_t initial_offset, const int64_t* initial_strides,
                                    const void* y, int64_t y_offset, const int64_t* y_strides,
                                    const void* dy, int64_t dy_offset, const int64_t* dy_strides,
                                    const float* dlast, int64_t dlast_offset, const int64_t* dlast_strides,
                                    void* dgate, int64_t dgate_offset, const int64_t* dgate_strides,
                                    void* dx, int64_t dx_offset, const int64_t* dx_strides,
                                    float* dinitial, int64_t dinitial_offset, const int64_t* dinitial_strides,
                                    void* scratch, size_t scratch_bytes) {
    if (!name || !gate || !y || !dy || !dgate || !dx || !gate_strides || !y_strides || !dy_strides || !dgate_strides || !dx_strides)
        return DLFX_ERR_INVALID_ARGUMENT;
    const int kind = kind_of(name);
    if (kind < 0) return DLFX_ERR_UNKNOWN_OP;
    if (kind == kGatedBlend && (!x || !x_strides)) return DLFX_ERR_INVALID_ARGUMENT;
    if (!shape_ok(m, n, rank, dims, dx_strides) || !strides_distinct(rank, dims, dx_strides) || !strides_distinct(rank, dims, dgate_strides))
        return DLFX_ERR_INVALID_ARGUMENT;
    if (rank > 1 && ((initial && !initial_strides) || (dlast && !dlast_strides) || (dinitial && !dinitial_strides))) return DLFX_ERR_INVALID_ARGUMENT;
    if (dinitial && !strides_distinct(rank - 1, dims, dinitial_strides)) return DLFX_ERR_INVALID_ARGUMENT;
    if (kind != kGatedBlend) x = nullptr;
    (void)scratch; (void)scratch_bytes;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dispatch_sequence_dtype(dtype, [&](auto tag) {
        using S = decltype(tag);
        Track<const S> tg, tx, ty, tdy;
        Track<S> tdg, tdx;
        Track<const float> ti, tdl;
        Track<float> tdi;
        if (!make_track(rank, dims, gate, gate_offset, gate_strides, false, &tg) || !make_track(rank, dims, x, x_offset, x_strides, false, &tx) ||
            !make_track(rank, dims, y, y_offset, y_strides, false, &ty) || !make_track(rank, dims, dy, dy_offset, dy_strides, false, &tdy) ||
            !make_track(rank, dims, dgate, dgate_offset, dgate_strides, false, &tdg) || !make_track(rank, dims, dx, dx_offset, dx_strides, false, &tdx) ||
            !make_track(rank, dims, initial, initial_offset, initial_strides, true, &ti) ||
            !make_track(rank, dims, dlast, dlast_offset, dlast_strides, true, &tdl) ||
            !make_track(rank, dims, dinitial, dinitial_offset, dinitial_strides, true, &tdi))
            return static_cast<int>(DLFX_ERR_RANK);
        if (ceil_div(m, 256) > 0x7fffffffLL) return static_cast<int>(DLFX_ERR_TOO_LARGE);
        return dispatch_kind(kind, [&](auto k) {
            gated_grad_walk<S, decltype(k)::value><<<dim3(static_cast<unsigned>(ceil_div(m, 256))), dim3(256), 0, s>>>(
                m, n, tg, tx, ti, ty, tdy, tdl, tdg, tdx, tdi);
            DLFX_CHECK_LAUNCH();
            return static_cast<int>(DLFX_OK);
        });
    });
}
