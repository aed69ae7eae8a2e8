// What gated_scan.hip, route.hip and cross_entropy.hip share: bfloat16, the three element types
// of the sequence-model operators, exponentials, vectors on any element boundary.
#pragma once

#include <limits>

#include "common.hip.h"

namespace dlfx {

using bf16_t = __bf16;      // gfx950 converts from fp32 in hardware, to nearest, ties to even

// float, half and bfloat16: the types of the sequence-model operators.  All arithmetic is in fp32.
template <typename F>
inline int dispatch_sequence_dtype(int dtype, F&& f) {
    switch (dtype) {
    case DLFX_F32: return f(float());
    case DLFX_F16: return f(half_t());
    case DLFX_BF16: return f(bf16_t());
    default: return DLFX_ERR_UNSUPPORTED_DTYPE;
    }
}

constexpr float kLog2E = 1.44269504088896340736f;

// exp(v).  fp32 elements take the library function (under 1 ulp); for two-byte elements the
// hardware's 2^x of the rounded product is off by |v| 2^-24, far inside their own rounding.
template <typename S> __device__ __forceinline__ float fast_exp(float v) {
    if constexpr (sizeof(S) == 4) return expf(v);
    else return __builtin_amdgcn_exp2f(v * kLog2E);
}
template <typename S> __device__ __forceinline__ float fast_reciprocal(float v) {
    if constexpr (sizeof(S) == 4) return 1.0f / v;
    else return __builtin_amdgcn_rcpf(v);
}

// N elements that start on any element boundary, moved in one access (global memory takes a
// 128-bit access at any address).
template <typename S, int N>
struct AnyVec {
    typedef S type __attribute__((ext_vector_type(N), aligned(sizeof(S))));
};

// A launch counts its threads along an axis of the grid in 32 bits.
constexpr int64_t kMostThreads = 0xffffffffLL;

// The same matrix written over itself at another stride would be read where it has been written.  (By the address
// that an offset leads to: one start can be given as different pointers and offsets.)
template <typename S>
bool overwrites(const S* x, int64_t stride, const S* dx, int64_t dx_stride, int64_t m) { return x == dx && stride != dx_stride && m > 1; }

inline bool strides_distinct(int rank, const int64_t* dims, const int64_t* strides) {
    for (int i = 0; i < rank; ++i)
        if (dims[i] > 1 && strides[i] == 0) return false;
    return true;
}

}  // namespace dlfx
