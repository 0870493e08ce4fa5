// Element types of the row operators (policy scores, 8-bit codes): float32, bfloat16 and float16 in memory, float32 in
// registers.  Conversions to 16 bits round to nearest even, once, on the way out.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "mz_common.h"

namespace mze {

using bf16 = __bf16;
using f16 = _Float16;

inline int type_bytes(int type) { return type == MZ_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == MZ_TYPE_F32 || type == MZ_TYPE_BF16 || type == MZ_TYPE_F16; }

// Runs f(T{}) with the C++ type of a MZ_TYPE_* code (checked by the caller).
template <class F>
inline void with_type(int type, F &&f) {
    switch (type) {
        case MZ_TYPE_BF16: f(bf16{}); break;
        case MZ_TYPE_F16: f(f16{}); break;
        default: f(float{}); break;
    }
}

// 16 bytes of elements, the widest load of a lane.
template <class T>
struct alignas(16) Pack {
    static constexpr int n = 16 / sizeof(T);
    T v[n];
};

// Rows can be read 16 bytes at a time when every one of them starts on a 16-byte address.
template <class T>
inline bool rows_aligned(const void *p, int64_t ld) {
    return ((uintptr_t)p & 15) == 0 && (ld * (int64_t)sizeof(T)) % 16 == 0;
}

}  // namespace mze
