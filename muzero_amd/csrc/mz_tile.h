// Matrix products of two row-major operands that both run along the reduction (out[o][i] = sum_k outer[o][k] inner[i][k]),
// on the matrix cores (gfx950), for int8 and fp16 elements alike: a fragment of either instruction is 16 consecutive
// bytes of an operand row per lane (16 int8 of 64, 8 fp16 of 32), so tiles are laid out in bytes and the element type
// only picks the instruction.
//
// The inner operand is the instruction's first one: its 16 rows are the accumulator's rows, four consecutive ones per
// lane, so that a lane holds four consecutive values of an output row and stores them together.
#pragma once
#include <algorithm>

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

// One operand in memory: `rows` rows of `pitch` bytes (a multiple of 16, below 2^23 so that 256 of them are named by 32
// bits), the reduction in bytes 0 .. wrap-1 of a row (a multiple of 128), run through again when the other operand's rows
// are longer.
struct Operand {
    const uint8_t *p;
    int64_t pitch;
    int rows;
    int wrap;
};

constexpr int kStep = 128;  // bytes of the reduction per step: one cache line of every row

// Byte offset of the 16-byte chunk c (0..7) of tile row r.  A ds_read_b128 is served in groups of 16 lanes that hold
// rows 0-3 and 12-15 of one chunk and rows 4-11 of its neighbour (and the reverse); rotating the chunks by half the row
// number gives every group 16 different 16-byte columns of the 256-byte bank row.
__device__ __forceinline__ int chunk_at(int r, int c) { return r * kStep + ((c ^ ((r >> 1) & 7)) << 4); }

// One workgroup's tile of TI inner x TO outer rows, WI x WO waves.  Two stages of LDS, filled from memory directly; a step
// is two halves of 64 bytes, and each half a read of its fragments and their products.
//   8 waves  two waves on every SIMD, half of them (`late`) one phase behind: while one reads LDS and starts the loads, the
//            other one multiplies, and a barrier ends every phase, so that the matrix pipe always has a wave to serve.
//            8192^2 x 16384 bytes, 256 x 256 tiles: 2880 TOP/s int8, 1440 TFLOP/s fp16; with all waves in the same phase
//            (the 4-wave form) 2700 and 1330.
//   4 waves  several workgroups share a compute unit and fill each other's gaps.  Fragments are double-buffered in
//            registers: the second half is read while the first is multiplied, and one barrier per step -- the next stage
//            has arrived, everybody is done reading this one -- comes before the loads that refill this stage.
template <class Op_, int TI_, int TO_, int WI_, int WO_>
struct Tile {
    using Op = Op_;
    static constexpr int TI = TI_, TO = TO_, WI = WI_, WO = WO_;
    static constexpr int threads = 64 * WI * WO;
    static constexpr int NI = TI / WI / 16, NO = TO / WO / 16;  // fragments of a wave
    static constexpr int stage = (TI + TO) * kStep;
    static constexpr int lds_bytes = 2 * stage;
    static constexpr int loads = (TI + TO) / 8 / (WI * WO);     // 1024-byte pieces (8 rows) per wave and step
    static_assert((TI + TO) % (8 * WI * WO) == 0 && TI % 8 == 0, "pieces divide among the waves");
    using Acc = typename Op::acc[NI][NO];

    // acc[a][b], element e: inner row i0 + wi() + 16 a + 4 (lane / 16) + e, outer row o0 + wo() + 16 b + lane % 16.
    static __device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
    static __device__ __forceinline__ int wi() { return (wave() % WI) * (TI / WI); }
    static __device__ __forceinline__ int wo() { return (wave() / WI) * (TO / WO); }

    // Steps step0 .. step1-1 (of 128 bytes) of the product of the rows from i0 and o0; rows behind the last one are
    // read as the last one (their results are never stored).
    static __device__ __forceinline__ void product(const Operand &inner, int i0, const Operand &outer, int o0, int step0, int step1,
                                                   uint8_t *lds, Acc &acc) {
        const int lane = threadIdx.x & 63, w = wave();
#pragma unroll
        for (int a = 0; a < NI; ++a)
#pragma unroll
            for (int b = 0; b < NO; ++b) acc[a][b] = typename Op::acc{};
        if (step0 >= step1) return;

        // where this lane's pieces come from: piece j = w + q * waves holds tile rows 8 j .. 8 j + 7 (inner rows first)
        const uint8_t *ip = inner.p + (int64_t)i0 * inner.pitch, *op = outer.p + (int64_t)o0 * outer.pitch;
        unsigned off[loads];
#pragma unroll
        for (int q = 0; q < loads; ++q) {
            const int r = 8 * (w + q * WI * WO) + (lane >> 3), c = ((lane & 7) ^ ((r >> 1) & 7)) << 4;
            if (8 * (w + q * WI * WO) < TI)
                off[q] = (unsigned)min(r, inner.rows - 1 - i0) * (unsigned)inner.pitch + c;
            else
                off[q] = (unsigned)min(r - TI, outer.rows - 1 - o0) * (unsigned)outer.pitch + c;
        }
        int ki = step0 * kStep % inner.wrap, ko = step0 * kStep % outer.wrap;
        const auto fetch = [&](int s) {
            uint8_t *st = lds + s * stage;
#pragma unroll
            for (int q = 0; q < loads; ++q) {
                const int j = w + q * WI * WO;
                const uint8_t *src = (8 * j < TI ? ip + ki : op + ko) + off[q];
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                                 (__attribute__((address_space(3))) void *)(st + j * 1024), 16, 0, 0);
            }
            ki += kStep, ko += kStep;
            if (ki == inner.wrap) ki = 0;
            if (ko == outer.wrap) ko = 0;
        };
        const int row_i = wi() + (lane & 15), row_o = TI + wo() + (lane & 15);
        const int at_i = chunk_at(row_i, lane >> 4), at_o = chunk_at(row_o, lane >> 4);
        const int n = step1 - step0;
        fetch(0);
        if (n > 1) {
            fetch(1);
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(loads) : "memory");  // the first stage has arrived
        } else {
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        }
        // the second half's chunks are the first one's with bit 2 flipped
        const auto read = [&](int s, int half, u32x4(&fi)[NI], u32x4(&fo)[NO]) {
            const uint8_t *bi = lds + s * stage + (at_i ^ (half * 64)), *bo = lds + s * stage + (at_o ^ (half * 64));
#pragma unroll
            for (int b = 0; b < NO; ++b) fo[b] = *(const u32x4 *)(bo + b * 16 * kStep);
#pragma unroll
            for (int a = 0; a < NI; ++a) fi[a] = *(const u32x4 *)(bi + a * 16 * kStep);
        };
        const auto multiply = [&](const u32x4(&fi)[NI], const u32x4(&fo)[NO]) {
#pragma unroll
            for (int a = 0; a < NI; ++a)
#pragma unroll
                for (int b = 0; b < NO; ++b) acc[a][b] = Op::mfma(fi[a], fo[b], acc[a][b]);
        };
        if constexpr (WI * WO == 8) {
            // Barriers of step t: early waves pass 4t+1 .. 4t+4, late ones 4t+2 .. 4t+5.  Step t's stage is complete at
            // barrier 4t, where every wave has waited for its own loads; the last reads of step t-1 are done before
            // barrier 4t, and the loads that overwrite its stage start behind it.
            const bool late = w >= 4;
            u32x4 fi[NI], fo[NO];
            const auto products = [&] {
                __builtin_amdgcn_sched_barrier(0);
                __builtin_amdgcn_s_setprio(1);
                multiply(fi, fo);
                __builtin_amdgcn_s_setprio(0);
                __builtin_amdgcn_sched_barrier(0);
            };
            if (late) asm volatile("s_barrier" ::: "memory");
            for (int t = 0; t < n; ++t) {
                read(t & 1, 0, fi, fo);
                if (t >= 1 && t + 1 < n) fetch((t & 1) ^ 1);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                products();
                asm volatile("s_barrier" ::: "memory");
                read(t & 1, 1, fi, fo);
                if (late) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                products();
                if (!late) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                asm volatile("s_barrier" ::: "memory");
            }
            if (!late) asm volatile("s_barrier" ::: "memory");
        } else {
            u32x4 fi[2][NI], fo[2][NO];
            const auto spread = [] {  // the reads between the products
#pragma unroll
                for (int z = 0; z < NI + NO; ++z) {
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, NI * NO / (NI + NO), 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, NI * NO, 0);
                __builtin_amdgcn_sched_barrier(0);
            };
            read(0, 0, fi[0], fo[0]);
            for (int t = 0; t < n; ++t) {
                const int s = t & 1;
                read(s, 1, fi[1], fo[1]);
                multiply(fi[0], fo[0]);
                spread();
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                if (t + 2 < n) fetch(s);
                if (t + 1 < n) read(s ^ 1, 0, fi[0], fo[0]);
                multiply(fi[1], fo[1]);
                spread();
            }
        }
    }

    // The tile on its way out: f(outer row, v) for every four consecutive inner values, in an order that lets a wave store
    // whole cache lines of an output row; the accumulator's layout (one outer row per lane) would store 16 to 64 bytes of
    // 16 rows at a time.  Sixteen outer rows of a wave at a time go through its own part of LDS, which is free after
    // product().  The rows are counted within the tile; a lane's inner row is the same in every call (inner_of()).
    // pre(b, v) maps an accumulator on the way in, where the lane's outer row is outer_of(b).
    static constexpr int WC = TI / WI, lanes_per_row = WC / 4, out_ld = WC + 4;
    static_assert(WI * WO * 16 * out_ld * 4 <= lds_bytes, "the outgoing rows fit the stages");
    static __device__ __forceinline__ int inner_of() { return wi() + 4 * (threadIdx.x % lanes_per_row); }
    static __device__ __forceinline__ int outer_of(int b) { return wo() + 16 * b + (threadIdx.x & 15); }

    template <bool UNROLL, class P, class F>
    static __device__ __forceinline__ void drain(uint8_t *lds, const Acc &acc, P &&pre, F &&f) {
        using V = decltype(pre(0, acc[0][0]));
        const int lane = threadIdx.x & 63;
        uint8_t *mine = lds + wave() * 16 * out_ld * 4;
        const auto pass = [&](int b, int r) {
            f(wo() + 16 * b + r, *(const V *)(mine + (r * out_ld + 4 * (lane % lanes_per_row)) * 4));
        };
#pragma unroll
        for (int b = 0; b < NO; ++b) {
            // lanes read what other lanes of their wave wrote: LDS keeps a wave's order, the compiler has to as well
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int a = 0; a < NI; ++a) *(V *)(mine + ((lane & 15) * out_ld + 16 * a + 4 * (lane >> 4)) * 4) = pre(b, acc[a][b]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if constexpr (UNROLL) {
#pragma unroll
                for (int q = 0; q < lanes_per_row / 4; ++q) pass(b, q * (64 / lanes_per_row) + lane / lanes_per_row);
            } else {
#pragma nounroll
                for (int q = 0; q < lanes_per_row / 4; ++q) pass(b, q * (64 / lanes_per_row) + lane / lanes_per_row);
            }
        }
    }
};

// Stores four consecutive values of an output row: at once where the row's address allows it.
template <class T>
struct alignas(4 * sizeof(T)) Quad {
    T v[4];
};

template <bool PAST, class T>
__device__ __forceinline__ void store_quad(T *row, int at, int n, bool aligned, const float (&v)[4]) {
    if (aligned && at + 4 <= n) {
        const Quad<T> q = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
        if constexpr (PAST) mze::store_past((Quad<T> *)(row + at), q);
        else *(Quad<T> *)(row + at) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (at + e < n) row[at + e] = (T)v[e];
    }
}

// Every row starts on a multiple of four elements.
template <class T>
inline bool quads_aligned(const T *p, int64_t ld) {
    return (uintptr_t)p % (4 * sizeof(T)) == 0 && ld % 4 == 0;
}

// Block b of `tiles` -> tile: consecutive blocks go to the 8 dies in turn, each with an L2 of its own, so die d takes the
// d-th eighth of the tiles; within that, tiles run through bands of `band` outer tiles so that the blocks at work together
// share rows of both operands.
struct TileAt {
    int inner, outer;
};

__device__ __forceinline__ TileAt tile_at(int b, int tiles_i, int tiles_o, int band) {
    const int tiles = tiles_i * tiles_o, per = tiles >> 3, rest = tiles & 7, die = b & 7;
    const int t = die * per + min(die, rest) + (b >> 3);
    const int size = band * tiles_i, g = t / size, o0 = g * band, h = min(band, tiles_o - o0), u = t - g * size;
    return {u / h, o0 + u % h};
}

// Four consecutive values summed over the parts of a split reduction, in the order of the parts, eight loads in flight:
// part p's quad q lies at partial + (p quads + q) * 4.
template <class V, class E>
__device__ __forceinline__ V sum_parts(const E *__restrict__ partial, int splits, int64_t quads, int64_t q) {
    V sum = *(const V *)(partial + q * 4);
    for (int p0 = 1; p0 < splits; p0 += 8) {
        V v[8];
#pragma unroll
        for (int p = 0; p < 8; ++p)
            if (p0 + p < splits) v[p] = *(const V *)(partial + ((p0 + p) * quads + q) * 4);
#pragma unroll
        for (int p = 0; p < 8; ++p)
            if (p0 + p < splits) sum += v[p];
    }
    return sum;
}

// Tile size and parts of the reduction for an output of `outer` x `inner` values and `steps` steps.
struct Shape {
    int tile;    // 64 x 64, 128 (inner) x 256 (outer) or 256 x 256, named by the inner size
    int splits;  // parts of the reduction, joined by a second kernel
};

inline int64_t tiles_of(int64_t n, int64_t t) { return n > 0 ? (n + t - 1) / t : 1; }

// Large tiles read each operand less often, small ones fill the 256 compute units with less work.  Measured (int8, us;
// 64 / 128 x 256 / 256 tiles, best number of parts in brackets):
//     8192 x 8192, 32 steps       - / 267 / 240              2048 x 4096, 32 steps      55 / 39 / 49
//     4096 x 4096,  4 steps      26 / 26 / 19                1024 x 4096, 32 steps      29 / 35 / 43 (3)
//      256 x 9216, 144 steps     81 / 66 (3) / 58 (7)         256 x 9216, 72 steps      41 / 43 (3) / 47 (4)
//       64 x 9216, 144 steps     34 (3) / 52 (3) / 45 (6)     128 x 4096, 32 steps      13 / 19 (4) / 23 (6)
//      100 x  500, 128 steps     13 (8), undivided 39         1024 x 1024, 8 steps     6.4 / 13 / 19
//       64 x 131072, 32 steps    142 / - / 175                 64 x 131072, 4 steps      21 / - / 34
inline Shape shape_of(int64_t outer, int64_t inner, int64_t steps) {
    const int64_t large = tiles_of(outer, 256) * tiles_of(inner, 256), medium = tiles_of(outer, 256) * tiles_of(inner, 128);
    if (outer > 64) {  // else most of a larger tile would be rows that are not there
        if (large >= 200) return {256, 1};
        if (medium >= 200) return {128, 1};
        if (outer * inner * steps >= 240LL * 1000 * 1000 && steps >= 64)  // a long reduction: the operands are what is read
            return {256, (int)std::max<int64_t>(1, std::min(256 / large, steps / 16))};
    }
    const int64_t small = tiles_of(outer, 64) * tiles_of(inner, 64);
    return {64, (int)std::max<int64_t>(1, std::min({(int64_t)32, 600 / small, steps / 16}))};
}

}  // namespace mzt8
