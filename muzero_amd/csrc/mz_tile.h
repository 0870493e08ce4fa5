// Matrix products of two row-major operands that both run along the reduction (out[o][i] = sum_k outer[o][k] inner[i][k]),
// on the matrix cores (gfx950), for int8 and fp16 elements alike: a fragment of either instruction is 16 consecutive
// bytes of an operand row per lane (16 int8 of 64, 8 fp16 of 32), so tiles are laid out in bytes and the element type
// only picks the instruction.
//
// The inner operand is the instruction's first one: its 16 rows are the accumulator's rows, four consecutive ones per
// lane, so that a lane holds four consecutive values of an output row and stores them together.
#pragma once
#include "mz_elem.h"

namespace mzt8 {

using u32x4 = __attribute__((ext_vector_type(4))) unsigned int;
using i32x4 = __attribute__((ext_vector_type(4))) int;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using h16x8 = __attribute__((ext_vector_type(8))) _Float16;

struct OpI8 {  // exact: |sum| <= 127 * 127 * K < 2^31 for K <= 131072
    using acc = i32x4;
    static __device__ __forceinline__ acc mfma(const u32x4 &a, const u32x4 &b, const acc &c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), c, 0, 0, 0);
    }
};

struct OpF16 {
    using acc = f32x4;
    static __device__ __forceinline__ acc mfma(const u32x4 &a, const u32x4 &b, const acc &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
    }
};

// One operand in memory: `rows` rows of `pitch` bytes (a multiple of 16), the reduction in bytes 0 .. wrap-1 of a row,
// repeated when the other operand's rows are longer.
struct Operand {
    const uint8_t *p;
    int64_t pitch;
    int rows;
    int wrap;
};

constexpr int kThreads = 256, kTile = 128, kStep = 128;  // 4 waves of 64 x 64; 128 bytes of the reduction per step

// Byte offset of the 16-byte chunk c (0..7) of tile row r: the chunks of a row are rotated so that the 16 lanes of a
// fragment read fall into different banks.
__device__ __forceinline__ int chunk_at(int r, int c) { return r * kStep + ((c ^ ((r >> 1) & 7)) << 4); }

// acc[a][b]: inner rows i0 + wave_i * 64 + 16 a + 4 (lane / 16) + 0..3, outer row o0 + wave_o * 64 + 16 b + lane % 16.
template <class Op>
__device__ __forceinline__ void tile_product(const Operand &inner, int i0, const Operand &outer, int o0, int kbytes,
                                             uint8_t *lds, typename Op::acc (&acc)[4][4]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = (wave & 1) * 64, wo = (wave >> 1) * 64;
    uint8_t *li = lds, *lo = lds + kTile * kStep;
    for (int a = 0; a < 4; ++a)
        for (int b = 0; b < 4; ++b) acc[a][b] = {};
    for (int k = 0; k < kbytes; k += kStep) {
        __syncthreads();
        for (int c = threadIdx.x; c < kTile * 8; c += kThreads) {
            const int r = c >> 3, ch = c & 7;
            const int ri = min(i0 + r, inner.rows - 1), ro = min(o0 + r, outer.rows - 1);
            *(u32x4 *)(li + chunk_at(r, ch)) = *(const u32x4 *)(inner.p + ri * inner.pitch + k % inner.wrap + ch * 16);
            *(u32x4 *)(lo + chunk_at(r, ch)) = *(const u32x4 *)(outer.p + ro * outer.pitch + k % outer.wrap + ch * 16);
        }
        __syncthreads();
        for (int s = 0; s < 2; ++s) {
            u32x4 fi[4], fo[4];
            for (int a = 0; a < 4; ++a) {
                fi[a] = *(const u32x4 *)(li + chunk_at(wi + 16 * a + (lane & 15), s * 4 + (lane >> 4)));
                fo[a] = *(const u32x4 *)(lo + chunk_at(wo + 16 * a + (lane & 15), s * 4 + (lane >> 4)));
            }
            for (int a = 0; a < 4; ++a)
                for (int b = 0; b < 4; ++b) acc[a][b] = Op::mfma(fi[a], fo[b], acc[a][b]);
        }
    }
}

}  // namespace mzt8
