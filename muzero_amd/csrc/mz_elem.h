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

// Elements j .. j + n - 1 of a row of K, zeros behind its end; WHOLE: rows start on 16-byte addresses; PAST: this is the
// last time the call reads them, their lines need not stay in cache.
template <class T, bool WHOLE, bool PAST = false>
__device__ __forceinline__ Pack<T> load_pack(const T *__restrict__ row, int j, int K) {
    constexpr int n = Pack<T>::n;
    if (WHOLE && j + n <= K) {
        using words = __attribute__((ext_vector_type(4))) unsigned;
        if (PAST) return __builtin_bit_cast(Pack<T>, __builtin_nontemporal_load((const words *)(row + j)));
        return *(const Pack<T> *)(row + j);
    }
    Pack<T> p;
#pragma unroll
    for (int e = 0; e < n; ++e) p.v[e] = j + e < K ? row[j + e] : (T)0.0f;
    return p;
}

// A store whose line need not stay in cache.
template <class T>
__device__ __forceinline__ void store_past(T *to, const T &v) {
    using words = __attribute__((ext_vector_type(sizeof(T) / 4))) unsigned;
    __builtin_nontemporal_store(__builtin_bit_cast(words, v), (words *)to);
}

// Results of this size go past the caches: written through them they push out the operands, of which other workgroups
// (or the next call) still need parts, and whoever reads them finds little of them in the 256 MB of the last level anyway.
// us with / without: int8 product of 8192 x 4096 x 8192 to bf16 (134 MB) 236 / 262, 113 MB of codes read back 53.5 / 55.5
// with their coding; but four layers in a row, each reading what the last one wrote, 256 x 4096 x 4096 22.4 / 22.0,
// 4096 x 4096 x 4096 to float32 (67 MB) 78 / 74, 8192 x 8192 x 8192 to bf16 465 / 471.
inline bool past_caches(int64_t bytes) { return bytes >= 100LL << 20; }

template <class T, bool WHOLE, bool PAST = false>
__device__ __forceinline__ void store_pack(T *__restrict__ row, int j, int K, const Pack<T> &p) {
    constexpr int n = Pack<T>::n;
    if (WHOLE && j + n <= K) {
        if constexpr (PAST) store_past((Pack<T> *)(row + j), p);
        else *(Pack<T> *)(row + j) = p;
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
