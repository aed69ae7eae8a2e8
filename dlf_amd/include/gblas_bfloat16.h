// bfloat16 host type of the veneer (not in the reference): the upper half of a float, built from one
// with round-to-nearest-even, the rounding the device applies.
#ifndef DLFX_VENEER_GBLAS_BFLOAT16_H_
#define DLFX_VENEER_GBLAS_BFLOAT16_H_

#include <cstdint>
#include <cstring>
#include <ostream>

namespace gpgpu { namespace blas {

struct alignas(2) bfloat16 {
    unsigned short x;

    bfloat16() : x(0) {}
    bfloat16(const float f) : x(from_float(f)) {}
    bfloat16& operator=(const float f) { x = from_float(f); return *this; }
    operator float() const {
        const uint32_t u = static_cast<uint32_t>(x) << 16;
        float f;
        std::memcpy(&f, &u, 4);
        return f;
    }

    static unsigned short from_float(float value) {
        uint32_t u;
        std::memcpy(&u, &value, 4);
        if ((u & 0x7fffffffu) > 0x7f800000u) return static_cast<unsigned short>(u >> 16 | 0x40u);      // a NaN stays one
        return static_cast<unsigned short>((u + 0x7fffu + (u >> 16 & 1u)) >> 16);
    }
};

inline std::ostream& operator<<(std::ostream& os, const bfloat16& v) { return os << static_cast<float>(v); }

}}  // namespace gpgpu::blas

#endif
