// Row codes: the device side of the quantiser, shared by the kernels that write codes and those that form them for
// themselves.  See mz_quant8.hip for the definition.
#pragma once
#include "mz_elem.h"

namespace mze {

constexpr float kTiny = 0x1p-119f;

__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

struct RowScale {
    float scale, inverse;  // inverse 0: the row is held as zeros
};

__device__ __forceinline__ RowScale row_scale(unsigned amax_bits, int scale_bits) {
    if (amax_bits >= 0x7F800000u) return {__uint_as_float(0x7FC00000u), 0.0f};
    const float a = __uint_as_float(amax_bits);
    if (a < kTiny) return {0.0f, 0.0f};
    float s = a / 127.0f;
    if (scale_bits >= 24) return {s, 127.0f / a};
    s = __uint_as_float((__float_as_uint(s) + 0x1FFFFFu) & ~0x1FFFFFu);
    return {s, 1.0f / s};
}

// One pack's codes.  Adding 1.5 * 2^23 rounds to a whole number, half to even, and leaves it in the low bits; the product
// is rounded before (no fused multiply-add), as the definition says.
template <class T>
__device__ __forceinline__ void store_codes(int8_t *out, const Pack<T> &p, float inverse) {
#pragma clang fp contract(off)
    constexpr int n = Pack<T>::n;
    unsigned w[n / 4];
#pragma unroll
    for (int q = 0; q < n / 4; ++q) {
        unsigned b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float v = (float)p.v[4 * q + e] * inverse;
            b[e] = __float_as_uint(v + 12582912.0f) & 0xFFu;
        }
        w[q] = inverse == 0.0f ? 0u : b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
    }
    if constexpr (n == 4) *(unsigned *)out = w[0];
    else *(uint2 *)out = make_uint2(w[0], w[1]);
}

inline int check_rows(const char *what, const void *x, int type, int64_t ld, int64_t rows, int64_t K) {
    if (!type_ok(type)) return mz::fail(MZ_ERR_ARG, "%s: unknown element type %d", what, type);
    if (rows < 0 || rows > 0x7FFFFFFF || K <= 0 || K > (1 << 30))
        return mz::fail(MZ_ERR_ARG, "%s: bad dimensions rows=%lld K=%lld", what, (long long)rows, (long long)K);
    if (rows > 0 && !x) return mz::fail(MZ_ERR_ARG, "%s: NULL argument", what);
    if (ld < K) return mz::fail(MZ_ERR_ARG, "%s: row stride %lld below the %lld values of a row", what, (long long)ld, (long long)K);
    if (((uintptr_t)x & (type_bytes(type) - 1)) != 0) return mz::fail(MZ_ERR_ARG, "%s: misaligned elements", what);
    return MZ_OK;
}

}  // namespace mze
