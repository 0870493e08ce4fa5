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

// Elements j .. j + n - 1 of a row of K, zeros behind its end; WHOLE: rows start on 16-byte addresses.
template <class T, bool WHOLE>
__device__ __forceinline__ Pack<T> load_pack(const T *__restrict__ row, int j, int K) {
    constexpr int n = Pack<T>::n;
    if (WHOLE && j + n <= K) return *(const Pack<T> *)(row + j);
    Pack<T> p;
#pragma unroll
    for (int e = 0; e < n; ++e) p.v[e] = j + e < K ? row[j + e] : (T)0.0f;
    return p;
}

template <class T, bool WHOLE>
__device__ __forceinline__ void store_pack(T *__restrict__ row, int j, int K, const Pack<T> &p) {
    constexpr int n = Pack<T>::n;
    if (WHOLE && j + n <= K) {
        *(Pack<T> *)(row + j) = p;
    } else {
#pragma unroll
        for (int e = 0; e < n; ++e)
            if (j + e < K) row[j + e] = p.v[e];
    }
}

// f(true / false as a type) with whether rows can be read in 16-byte packs.
template <class F>
inline void with_flag(bool flag, F &&f) {
    if (flag) f(std::true_type{});
    else f(std::false_type{});
}

}  // namespace mze
