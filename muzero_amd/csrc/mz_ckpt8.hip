// Weight gradients from 8-bit activation checkpoints (gfx950): a dense layer z = x W^T + b keeps its input as row codes
// (mz_quant8_rows: x_rk about s_r q_rk), and its backward pass forms
//     dW_nk = sum_r dz_rn s_r q_rk,     db_n = sum_r dz_rn
// without writing x out again.
//
// Few rows, or a small dW, take a kernel of their own (k_weight_grad_few).  For the rest the product runs on the fp16
// matrix instruction.  Codes are whole numbers up to 127: exact in fp16.  The row scale lies
// along the reduction, so it goes to the other side: v_rn = dz_rn s_r, which fp16 cannot hold as it is.  Each output row n
// is first brought into range by a power of two c_n (the largest |v_rn c_n| lies in 2^14 .. 2^15) and then held as
//     one plane   hi = fp16(v c)                       bfloat16 dz with scales of 3 significant bits: 8 + 3 = 11 bits,
//                                                      which is what fp16 has -- exact
//     two planes  hi = fp16(v c), lo = fp16(v c - hi)  everything else: 22 bits
// (values below 2^-16 of their row's largest lose bits of the second plane, values below 2^-28 of the first one: an
// absolute error of at most 2^-25 c_n^-1 then, 2^-39 of the largest).  The two planes' products go to one float32
// accumulator, and 1 / c_n is applied at the end, exact.
// Both operands of the product run along the rows, so both are transposed on the way:
//   k_col_stats, k_col_factors   per column of dz: the largest |v|, hence c_n, and the sum of dz (db), from chunks of rows;
//                                up to 1024 rows k_prepare joins the chunks itself, up to 256 it reads the columns itself:
//                                a launch costs more than that
//   k_prepare                    dz -> planes [n][plane][r] and codes -> fp16 [k][r], 64 rows per workgroup
//   k_weight_grad                the product; k_weight_join the sum of its parts where the reduction is split
#include "mz_codes.h"
#include "mz_tile.h"

namespace {

using namespace mze;
using namespace mzt8;

constexpr int kCT = 256;
constexpr int kMaxChunks = 128, kFewRows = 256, kFewChunks = 16;

enum Stats { kOwn, kChunks, kReady };  // where k_prepare's column factors come from

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// The power of two that brings a column with largest magnitude `bits` to 2^14 .. 2^15, and its inverse; NaN for a column
// with an infinity or a NaN.
__device__ __forceinline__ float column_factor(unsigned bits, float *inverse) {
    if (bits >= 0x7F800000u) {
        *inverse = __uint_as_float(0x7FC00000u);
        return *inverse;
    }
    int e = 14 - (max((int)(bits >> 23), 1) - 127);  // ilogb of the largest (subnormal ones count as 2^-126)
    e = min(max(e, -126), 126);
    *inverse = __uint_as_float((unsigned)(127 - e) << 23);
    return __uint_as_float((unsigned)(127 + e) << 23);
}

// A workgroup takes LANES packs of columns and a chunk of rows, 256 / LANES rows at a time.
// Bound by the bytes: 8192 x 8192 bf16 40 us, 3.3 TB/s; narrow matrices by the loads' latency
// (whole gradients, bf16, 64 lanes / as many as have columns: 8192 x 9000 x 30 83 / 71 us, 8192 x 1100 x 250 47 / 40 us).
template <class T, bool WHOLE, int LANES>
__global__ void __launch_bounds__(kCT)
k_col_stats(const T *__restrict__ dz, int64_t ldz, const float *__restrict__ scales, int R, int N, int chunk_rows,
            unsigned *__restrict__ part_max, float *__restrict__ part_sum) {
    constexpr int n = Pack<T>::n, groups = kCT / LANES, width = LANES * n;
    __shared__ unsigned group_max[kCT * n];
    __shared__ float group_sum[kCT * n];
    const int t = threadIdx.x, chunk = blockIdx.y, c0 = blockIdx.x * width, c = c0 + t % LANES * n;
    unsigned m[n] = {};
    float s[n] = {};
    const int end = min(R, (chunk + 1) * chunk_rows);
    if (c < N)
#pragma unroll 8
        for (int r = chunk * chunk_rows + t / LANES; r < end; r += groups) {
            const Pack<T> p = load_pack<T, WHOLE>(dz + r * ldz, c, N);
            const float scale = scales[r];
#pragma unroll
            for (int e = 0; e < n; ++e) {
                const float g = (float)p.v[e];
                m[e] = max(m[e], abs_bits(g * scale));
                s[e] += g;
            }
        }
#pragma unroll
    for (int e = 0; e < n; ++e) group_max[t * n + e] = m[e], group_sum[t * n + e] = s[e];
    __syncthreads();
    for (int i = t; i < width; i += kCT)
        if (c0 + i < N) {
            unsigned top = 0;
            float sum = 0.0f;
            for (int q = 0; q < groups; ++q) top = max(top, group_max[q * width + i]), sum += group_sum[q * width + i];
            part_max[(int64_t)chunk * N + c0 + i] = top;
            part_sum[(int64_t)chunk * N + c0 + i] = sum;
        }
}

// 64 columns, every wave a quarter of the chunks.
template <class T>
__global__ void __launch_bounds__(kCT)
k_col_factors(const unsigned *__restrict__ part_max, const float *__restrict__ part_sum, int chunks, int N, float *__restrict__ factor,
              float *__restrict__ inverse, T *__restrict__ db) {
    __shared__ unsigned wave_max[4][64];
    __shared__ float wave_sum[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * 64 + lane;
    unsigned m = 0;
    float s = 0.0f;
    if (n < N)
#pragma unroll 8
        for (int c = wave; c < chunks; c += 4) {
            m = max(m, part_max[(int64_t)c * N + n]);
            s += part_sum[(int64_t)c * N + n];
        }
    wave_max[wave][lane] = m, wave_sum[wave][lane] = s;
    __syncthreads();
    if (wave > 0 || n >= N) return;
    for (int w = 1; w < 4; ++w) m = max(m, wave_max[w][lane]), s += wave_sum[w][lane];
    factor[n] = column_factor(m, inverse + n);
    if (db) db[n] = (T)s;
}

struct Prepared {  // what k_prepare reads of the statistics, and what it leaves
    const unsigned *part_max;
    const float *part_sum;
    int chunks;
    float *factor, *inverse;
    f16 *planes, *codes_t;
};

constexpr int kSplitCols = 64, kCodeCols = 128;

// dz -> planes for 64 columns and 64 rows, the columns' factors first.  v = dz s c is formed in float32 and split before it
// goes to LDS; a lane then collects 8 rows of one column, 16 bytes of each plane.
template <class T, int PLANES, bool WHOLE, Stats STATS>
__device__ void split_block(const T *__restrict__ dz, int64_t ldz, const float *__restrict__ scales, int R, int N, int64_t Rp, int n0,
                            int r0, const Prepared &out, T *__restrict__ db, uint8_t *lds) {
    constexpr int n = Pack<T>::n, packs = kSplitCols / n, ld = kSplitCols + 1;
    unsigned(*tile)[ld] = (unsigned(*)[ld])lds;              // [64 rows]: hi | lo << 16
    float *factor = (float *)(lds + 64 * ld * 4);
    const int t = threadIdx.x;
    if constexpr (STATS == kOwn) {
        unsigned *top = (unsigned *)lds;                     // [16 row groups][64 columns]
        float *sum = (float *)lds + 16 * kSplitCols;
        static_assert(2 * 16 * kSplitCols <= 64 * ld, "the statistics fit the tile");
        const int g = t >> 4, c = (t & 15) * 4;              // 4 columns, every 16th row
        unsigned m[4] = {};
        float s[4] = {};
#pragma unroll 4
        for (int r = g; r < R; r += 16) {
            const float scale = scales[r];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = n0 + c + e < N ? (float)dz[r * ldz + n0 + c + e] : 0.0f;
                m[e] = max(m[e], abs_bits(x * scale));
                s[e] += x;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) top[g * kSplitCols + c + e] = m[e], sum[g * kSplitCols + c + e] = s[e];
        __syncthreads();
        if (t < kSplitCols) {
            unsigned mm = 0;
            float ss = 0.0f;
            for (int q = 0; q < 16; ++q) mm = max(mm, top[q * kSplitCols + t]), ss += sum[q * kSplitCols + t];
            float inv;
            factor[t] = column_factor(mm, &inv);
            if (r0 == 0 && n0 + t < N) {
                out.inverse[n0 + t] = inv;
                if (db) db[n0 + t] = (T)ss;
            }
        }
    } else if (STATS == kChunks && t < kSplitCols) {
        unsigned m = 0;
        float s = 0.0f, inv;
        if (n0 + t < N)
#pragma unroll
            for (int c = 0; c < kFewChunks; ++c)
                if (c < out.chunks) m = max(m, out.part_max[(int64_t)c * N + n0 + t]), s += out.part_sum[(int64_t)c * N + n0 + t];
        factor[t] = column_factor(m, &inv);
        if (r0 == 0 && n0 + t < N) {
            out.inverse[n0 + t] = inv;
            if (db) db[n0 + t] = (T)s;
        }
    } else if (t < kSplitCols) {
        factor[t] = n0 + t < N ? out.factor[n0 + t] : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int i = t; i < 64 * packs; i += kCT) {
        const int r = i / packs, c = i % packs * n;
        Pack<T> p{};
        float scale = 0.0f;
        if (r0 + r < R && n0 + c < N) {
            p = load_pack<T, WHOLE, STATS != kOwn>(dz + (r0 + r) * ldz, n0 + c, N);
            scale = scales[r0 + r];
        }
#pragma unroll
        for (int e = 0; e < n; ++e) {
            const float v = r0 + r < R ? ((float)p.v[e] * scale) * factor[c + e] : 0.0f;
            const f16 hi = (f16)v, lo = (f16)(v - (float)hi);
            tile[r][c + e] = (unsigned)__builtin_bit_cast(unsigned short, hi) | (unsigned)__builtin_bit_cast(unsigned short, lo) << 16;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = t; i < kSplitCols * 8; i += kCT) {
        const int c = i >> 3, r = (i & 7) * 8;
        if (n0 + c >= N) continue;
        u32x4 hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const unsigned x = tile[r + 2 * e][c], y = tile[r + 2 * e + 1][c];
            hi[e] = (x & 0xFFFFu) | y << 16;
            lo[e] = x >> 16 | (y & 0xFFFF0000u);
        }
        f16 *row = out.planes + (int64_t)(n0 + c) * PLANES * Rp + r0 + r;
        *(u32x4 *)row = hi;
        if (PLANES == 2) *(u32x4 *)(row + Rp) = lo;
    }
}

// codes -> fp16 for 128 columns and 64 rows: a lane collects 8 rows of 4 columns from 8 words.
__device__ void codes_block(const int8_t *__restrict__ codes, int64_t ldc, int R, int K, int64_t Rp, int k0, int r0,
                            f16 *__restrict__ codes_t, uint8_t *lds) {
    constexpr int ld = kCodeCols + 4;
    const int t = threadIdx.x;
#pragma unroll
    for (int i = t; i < 64 * kCodeCols / 16; i += kCT) {
        const int r = i / (kCodeCols / 16), c = i % (kCodeCols / 16) * 16;
        u32x4 v = {};
        if (r0 + r < R && k0 + c < K) v = *(const u32x4 *)(codes + (r0 + r) * ldc + k0 + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) *(unsigned *)(lds + r * ld + c + 4 * e) = v[e];
    }
    __syncthreads();
#pragma unroll
    for (int i = t; i < kCodeCols / 4 * 8; i += kCT) {
        const int c = (i >> 3) * 4, r = (i & 7) * 8;
        unsigned w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = *(const unsigned *)(lds + (r + e) * ld + c);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            h16x8 h;
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = (f16)(float)(int8_t)(w[e] >> 8 * q);
            if (k0 + c + q < K) *(h16x8 *)(codes_t + (int64_t)(k0 + c + q) * Rp + r0 + r) = h;
        }
    }
}

// Bound by the bytes: 8192 rows of 8192 bf16 and of 4096 codes 69 us, 370 MB, 5.4 TB/s.
// Workgroups 0 .. split_blocks - 1: 64 columns of dz each; the others 128 columns of codes; all of them 64 rows.
template <class T, int PLANES, bool WHOLE, Stats STATS>
__global__ void __launch_bounds__(kCT)
k_prepare(const T *__restrict__ dz, int64_t ldz, const float *__restrict__ scales, int R, int N, const int8_t *__restrict__ codes,
          int64_t ldc, int K, int64_t Rp, int split_blocks, Prepared out, T *__restrict__ db) {
    __shared__ __align__(16) uint8_t lds[64 * (kSplitCols + 1) * 4 + kSplitCols * 4];
    const int r0 = blockIdx.y * 64;
    if ((int)blockIdx.x < split_blocks)
        split_block<T, PLANES, WHOLE, STATS>(dz, ldz, scales, R, N, Rp, blockIdx.x * kSplitCols, r0, out, db, lds);
    else
        codes_block(codes, ldc, R, K, Rp, (blockIdx.x - split_blocks) * kCodeCols, r0, out.codes_t, lds);
}

// Bound by the matrix cores: 8192 x 4096 x 8192 with one plane 373 to 450 us (the clock follows the load), 1.2 to 1.5 PFLOP/s
// (a library's fp16 product of 8192^3 1.50); two planes (whole calls, float32
// 1030 us, float16 920, against 500 to 530) take twice that.
template <class T, class Tl>
__global__ void __launch_bounds__(Tl::threads)
k_weight_grad(const f16 *__restrict__ codes_t, const f16 *__restrict__ planes, const float *__restrict__ inverse, int K, int N,
              int64_t Rp, int n_planes, T *__restrict__ dw, int64_t ldw, bool aligned, int tiles_k, int tiles_n, int splits,
              float *__restrict__ partial) {
    __shared__ __align__(16) uint8_t lds[Tl::lds_bytes];
    const int split = blockIdx.x % splits;
    const TileAt at = tile_at(blockIdx.x / splits, tiles_k, tiles_n, 8);
    const int k0 = at.inner * Tl::TI, n0 = at.outer * Tl::TO;
    const Operand inner{(const uint8_t *)codes_t, 2 * Rp, K, (int)(2 * Rp)};
    const Operand outer{(const uint8_t *)planes, 2 * Rp * n_planes, N, (int)(2 * Rp * n_planes)};
    const int steps = outer.wrap / kStep;
    typename Tl::Acc acc;
    Tl::product(inner, k0, outer, n0, (int)((int64_t)steps * split / splits), (int)((int64_t)steps * (split + 1) / splits), lds, acc);
    const int k = k0 + Tl::inner_of();
    if (splits > 1) {
        const int Kq = (K + 3) / 4 * 4;
        float *out = partial + (int64_t)split * N * Kq;
        Tl::template drain<true>(lds, acc, [](int, const f32x4 &v) { return v; }, [&](int n, const f32x4 &v) {
            if (n0 + n < N && k < K) *(f32x4 *)(out + (int64_t)(n0 + n) * Kq + k) = v;
        });
        return;
    }
    float inv[Tl::NO];
#pragma unroll
    for (int b = 0; b < Tl::NO; ++b) inv[b] = inverse[min(n0 + Tl::outer_of(b), N - 1)];
    Tl::template drain<true>(lds, acc, [&](int b, const f32x4 &v) { return v * inv[b]; }, [&](int n, const f32x4 &v) {
        if (n0 + n >= N) return;
        const float o[4] = {v[0], v[1], v[2], v[3]};
        store_quad<false>(dw + (n0 + n) * ldw, k, K, aligned, o);
    });
}

// Sums of the parts of a split reduction, in a fixed order: one thread per four values of a row of dW; bound by the bytes.
// `inverse` undoes the columns' factors; part_sum holds the parts of db where the parts' kernel formed them.
template <class T>
__global__ void __launch_bounds__(256)
k_weight_join(const float *__restrict__ partial, int splits, const float *__restrict__ inverse, int K, int N, T *__restrict__ dw,
              int64_t ldw, bool aligned, const float *__restrict__ part_sum, T *__restrict__ db) {
    const int quads = (K + 3) / 4, n = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x, k = 4 * c;
    if (c < quads) {
        f32x4 sum = sum_parts<f32x4>(partial, splits, (int64_t)N * quads, (int64_t)n * quads + c);
        if (inverse) sum *= inverse[n];
        const float o[4] = {sum[0], sum[1], sum[2], sum[3]};
        store_quad<false>(dw + n * ldw, k, K, aligned, o);
    }
    if (db && part_sum && c == 0) {
        float sum = 0.0f;
#pragma unroll 8
        for (int p = 0; p < splits; ++p) sum += part_sum[(int64_t)p * N + n];
        db[n] = (T)sum;
    }
}

// ---------------------------------------------------------------- few rows or a small dW: one launch, or two
// A workgroup forms 32 x 64 values of dW, its eight waves every eighth 32 rows; a lane reads 2 columns of dz and 4 of the
// codes from 8 rows, which is a fragment of the instruction already, so nothing is transposed and nothing waits for the
// columns' factors: v = dz s is held in bfloat16 planes, which have float32's range,
//     two    hi = bf16(v), mid = bf16(v - hi)         16 bits: 16-bit dz with scales of 3 significant bits, exact
//     three  and lo = bf16(v - hi - mid)              24 bits, as v itself
// (below 2^-110 the last one loses bits to its smallest value, 2^-133).
constexpr int kFewN = 32, kFewK = 64, kFewWaves = 8, kFewSplit = 2048;

using b16x8 = __attribute__((ext_vector_type(8))) __bf16;

template <class T, int PLANES, bool PAIRS>
__global__ void __launch_bounds__(64 * kFewWaves, 4)
k_weight_grad_few(const T *__restrict__ dz, int64_t ldz, const float *__restrict__ scales, int R, int N,
                  const int8_t *__restrict__ codes, int64_t ldc, int K, T *__restrict__ dw, int64_t ldw, bool aligned,
                  T *__restrict__ db, int tiles_k, int part_rows, float *__restrict__ partial, float *__restrict__ part_sum) {
    constexpr int ld = kFewK + 4;
    __shared__ __align__(16) float sums[kFewWaves][kFewN * ld];
    __shared__ float db_sums[kFewWaves][kFewN];
    struct alignas(2 * sizeof(T)) Pair {
        T v[2];
    };
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const int k0 = (int)(blockIdx.x % tiles_k) * kFewK, n0 = (int)(blockIdx.x / tiles_k) * kFewN;
    // rows and columns behind the last one are read as the last one: the rows count as zero, the columns are not stored
    const int8_t *q0 = codes + min(k0 / 4 + c, (K - 1) / 4) * 4;
    const T *d0 = dz + min(n0 + 2 * c, PAIRS ? N - 2 : N - 1), *d1 = dz + min(n0 + 2 * c + 1, N - 1);
    struct Rows {
        unsigned q[8];
        Pair d[8];
        float s[8];
    };
    const auto load = [&](int r0) {
        Rows x;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int64_t r = min(r0 + 8 * g + j, R - 1);
            x.s[j] = scales[r];
            x.q[j] = *(const unsigned *)(q0 + r * ldc);
            if (PAIRS) x.d[j] = *(const Pair *)(d0 + r * ldz);
            else x.d[j] = {d0[r * ldz], d1[r * ldz]};
        }
        return x;
    };
    f32x4 acc[2][4] = {};
    float col[2] = {};
    const int begin = blockIdx.y * part_rows, end = min(R, begin + part_rows);
    const int waves = min(kFewWaves, (end - begin + 31) / 32);  // with rows to take
    if (wave < waves) {
        Rows next = load(begin + wave * 32);
        for (int r0 = begin + wave * 32; r0 < end; r0 += kFewWaves * 32) {
            const Rows x = next;
            next = load(r0 + kFewWaves * 32);
            b16x8 plane[2][PLANES], code[4];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool live = r0 + 8 * g + j < end;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float d = live ? (float)x.d[j].v[e] : 0.0f;
                    float v = live ? d * x.s[j] : 0.0f;
                    col[e] += d;
#pragma unroll
                    for (int p = 0; p < PLANES; ++p) {
                        plane[e][p][j] = (__bf16)v;
                        v -= (float)plane[e][p][j];
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) code[e][j] = (__bf16)(float)(int8_t)(x.q[j] >> 8 * e);
            }
#pragma unroll
            for (int p = PLANES - 1; p >= 0; --p)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int h = 0; h < 4; ++h)
                        acc[e][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(code[h], plane[e][p], acc[e][h], 0, 0, 0);
        }
    }
    // acc[e][h][i] of a lane: dW of column n0 + 2 c + e, input k0 + 4 (4 g + i) + h
    if (wave < waves) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(f32x4 *)&sums[wave][(2 * c + e) * ld + 4 * (4 * g + i)] = f32x4{acc[e][0][i], acc[e][1][i], acc[e][2][i], acc[e][3][i]};
            col[e] += __shfl_xor(col[e], 16);
            col[e] += __shfl_xor(col[e], 32);
            if (g == 0) db_sums[wave][2 * c + e] = col[e];
        }
    }
    __syncthreads();
    const int row = threadIdx.x >> 4, kq = (threadIdx.x & 15) * 4;
    f32x4 sum = {};
#pragma unroll
    for (int w = 0; w < kFewWaves; ++w)
        if (w < waves) sum += *(const f32x4 *)&sums[w][row * ld + kq];
    if (n0 + row < N) {
        const float o[4] = {sum[0], sum[1], sum[2], sum[3]};
        const int Kq = (K + 3) / 4 * 4;
        if (!partial) store_quad<false>(dw + (n0 + row) * ldw, k0 + kq, K, aligned, o);
        else if (k0 + kq < K) *(f32x4 *)(partial + ((int64_t)blockIdx.y * N + n0 + row) * Kq + k0 + kq) = sum;
    }
    if (db && k0 == 0 && threadIdx.x < kFewN && n0 + (int)threadIdx.x < N) {
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWaves; ++w)
            if (w < waves) total += db_sums[w][threadIdx.x];
        if (!partial) db[n0 + threadIdx.x] = (T)total;
        else part_sum[(int64_t)blockIdx.y * N + n0 + threadIdx.x] = total;
    }
}

// Up to here the one launch wins (us, this / the kernels above; float32): 256 x 168 x 256 (rows, K, N) 5.1 / 15.0,
// 1024 x 512 x 512 10 / 29, 2048 x 1024 x 1024 33 / 41, 512 x 2048 x 2048 35 / 35; behind it not: 256 x 4096 x 4096 83 / 43,
// 64 x 4096 x 4096 46 / 24.  Its time is the latency of the rows' loads, 1.5 us for every 256 rows, or with many tiles the
// conversions, which every workgroup does for itself.
// Any number of rows of a layer of up to 2^18 weights goes in parts of at least 512 rows, joined by a second launch, up to
// two workgroups per compute unit: 16384 x 64 x 64 12 / 25, 16384 x 168 x 256 23 / 34, 8192 x 512 x 512 35 / 47, 10^6 x 64 x 64
// 127 / 1116, but 65536 x 512 x 512 216 / 207 and, with 2^20 weights, 8192 x 1024 x 1024 111 / 77.  Up to kFewSplit rows the
// second launch costs more than it gives (1536 x 168 x 64 undivided 14).
bool few_rows(int64_t R, int64_t N, int64_t K) {
    return (R <= 4096 && N * K <= 1LL << 22 && R * N * K <= 1LL << 31) || (N * K <= 1LL << 18 && N <= 32768);
}

struct Few {
    int tiles_k, tiles_n, parts, part_rows;
    int64_t off_sum, bytes;
};

Few few_layout(int64_t R, int64_t N, int64_t K) {
    Few f;
    f.tiles_k = (int)((K + kFewK - 1) / kFewK), f.tiles_n = (int)((N + kFewN - 1) / kFewN);
    const int64_t tiles = (int64_t)f.tiles_k * f.tiles_n;
    const int64_t parts = R <= kFewSplit ? 1 : std::max<int64_t>(1, std::min({R / 512, 512 / tiles, (int64_t)64}));
    f.part_rows = (int)round_up((R + parts - 1) / parts, kFewWaves * 32);
    f.parts = (int)((R + f.part_rows - 1) / f.part_rows);
    f.off_sum = f.parts > 1 ? f.parts * N * round_up(K, 4) * 4 : 0;
    f.bytes = f.parts > 1 ? f.off_sum + f.parts * N * 4 : 0;
    return f;
}

struct Layout {
    int planes, chunks, chunk_rows;
    Shape shape;
    int64_t Rp, off_sum, off_factor, off_inverse, off_planes, off_codes, off_partial, bytes;
};

Layout layout(int32_t type, int32_t scale_bits, int64_t R, int64_t N, int64_t K) {
    Layout l;
    l.planes = type == MZ_TYPE_BF16 && scale_bits == 3 ? 1 : 2;
    l.Rp = round_up(R, 64);
    // few rows: every workgroup of k_prepare forms its columns' statistics itself, no launches of their own
    l.chunks = R <= kFewRows ? 0 : (int)(R < 64 * kMaxChunks ? (R + 63) / 64 : kMaxChunks);
    l.chunk_rows = l.chunks ? (int)((R + l.chunks - 1) / l.chunks) : 0;
    const int64_t stat = round_up((int64_t)l.chunks * N * 4, 128);
    l.off_sum = stat;
    l.off_factor = 2 * stat;
    l.off_inverse = l.off_factor + round_up(N * 4, 128);
    l.off_planes = l.off_inverse + round_up(N * 4, 128);
    l.off_codes = l.off_planes + N * l.planes * l.Rp * 2;
    l.off_partial = l.off_codes + round_up(K * l.Rp * 2, 128);
    l.shape = shape_of(N, K, l.Rp * 2 * l.planes / kStep);
    l.bytes = l.off_partial + (l.shape.splits > 1 ? l.shape.splits * N * round_up(K, 4) * 4 : 0);
    return l;
}

constexpr int64_t kMaxRows = 1 << 20;  // a row of two fp16 planes is then at most 2^22 bytes (mz_tile.h: Operand)

}  // namespace

extern "C" {

int64_t mz_ckpt8_workspace(int32_t type, int32_t scale_bits, int32_t rows, int32_t N, int32_t K) {
    if (rows <= 0 || N <= 0 || K <= 0 || rows > kMaxRows) return 0;
    if (few_rows(rows, N, K)) return few_layout(rows, N, K).bytes;
    return layout(type, scale_bits, rows, N, K).bytes;
}

int mz_ckpt8_weight_grad(const void *dz, int32_t type, int64_t ldz, int32_t rows, int32_t N, const int8_t *codes, int64_t ldc,
                         const float *scales, int32_t scale_bits, int32_t K, void *dw, int64_t ldw, void *db, void *workspace,
                         int64_t workspace_bytes, void *stream) {
    if (rows <= 0 || N <= 0 || K <= 0 || rows > kMaxRows)
        return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: bad dimensions rows=%d N=%d K=%d", rows, N, K);
    if (!type_ok(type)) return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: unknown element type %d", type);
    if (scale_bits != 24 && scale_bits != 3)
        return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: scale_bits must be 24 or 3, not %d", scale_bits);
    if (!dz || !codes || !scales || !dw) return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: NULL argument");
    if (ldz < N || ldw < K || ldc < K || ldc % 16 != 0 || ((uintptr_t)codes & 15) != 0 ||
        (((uintptr_t)dz | (uintptr_t)dw | (uintptr_t)db) & (type_bytes(type) - 1)) != 0)
        return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: bad stride or alignment (ldz=%lld ldw=%lld ldc=%lld)", (long long)ldz,
                        (long long)ldw, (long long)ldc);
    const int64_t need = mz_ckpt8_workspace(type, scale_bits, rows, N, K);
    if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0))
        return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
                        (long long)workspace_bytes);
    if (few_rows(rows, N, K)) {
        const Few f = few_layout(rows, N, K);
        float *partial = f.parts > 1 ? (float *)workspace : nullptr, *part_sum = (float *)((uint8_t *)workspace + f.off_sum);
        with_type(type, [&](auto t) {
            using T = decltype(t);
            const bool pairs = (uintptr_t)dz % (2 * sizeof(T)) == 0 && ldz % 2 == 0 && N % 2 == 0, aligned = quads_aligned((T *)dw, ldw);
            const auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3((unsigned)(f.tiles_k * f.tiles_n), (unsigned)f.parts), dim3(64 * kFewWaves), 0,
                                   (hipStream_t)stream, (const T *)dz, ldz, scales, rows, N, codes, ldc, K, (T *)dw, ldw, aligned, (T *)db,
                                   f.tiles_k, f.part_rows, partial, part_sum);
            };
            const auto planes = [&](auto planes_tag) {
                constexpr int P = decltype(planes_tag)::value;
                pairs ? go(k_weight_grad_few<T, P, true>) : go(k_weight_grad_few<T, P, false>);
            };
            if constexpr (sizeof(T) == 2) {
                if (scale_bits == 3) planes(std::integral_constant<int, 2>{});
                else planes(std::integral_constant<int, 3>{});
            } else {
                planes(std::integral_constant<int, 3>{});
            }
            if (f.parts > 1)
                hipLaunchKernelGGL(k_weight_join<T>, dim3((unsigned)tiles_of(K, 1024), (unsigned)N), dim3(256), 0, (hipStream_t)stream,
                                   (const float *)partial, f.parts, (const float *)nullptr, K, N, (T *)dw, ldw, aligned,
                                   (const float *)part_sum, (T *)db);
        });
        return mz::check_launch("mz_ckpt8_weight_grad");
    }
    const Layout l = layout(type, scale_bits, rows, N, K);
    const int64_t tiles = (round_up(N, 64) / 64) * (round_up(K, 64) / 64);
    if (tiles > (1 << 23) || l.Rp / 64 > 65535)
        return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: rows=%d N=%d K=%d is too large for one call", rows, N, K);
    uint8_t *ws = (uint8_t *)workspace;
    unsigned *part_max = (unsigned *)ws;
    float *part_sum = (float *)(ws + l.off_sum), *inverse = (float *)(ws + l.off_inverse);
    f16 *planes = (f16 *)(ws + l.off_planes), *codes_t = (f16 *)(ws + l.off_codes);
    float *partial = (float *)(ws + l.off_partial);
    hipStream_t st = (hipStream_t)stream;
    const Prepared prepared{part_max, part_sum, l.chunks, (float *)(ws + l.off_factor), inverse, planes, codes_t};
    const int split_blocks = (N + kSplitCols - 1) / kSplitCols;
    const dim3 grid((unsigned)(split_blocks + (K + kCodeCols - 1) / kCodeCols), (unsigned)(l.Rp / 64));
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_flag(rows_aligned<T>(dz, ldz), [&](auto whole) {
            constexpr bool W = decltype(whole)::value;
            if (l.chunks > 0) {
                const auto stats = [&](auto lanes) {
                    constexpr int L = decltype(lanes)::value;
                    hipLaunchKernelGGL((k_col_stats<T, W, L>), dim3((unsigned)tiles_of(N, L * Pack<T>::n), (unsigned)l.chunks), dim3(kCT), 0, st,
                                       (const T *)dz, ldz, scales, rows, N, l.chunk_rows, part_max, part_sum);
                };
                if (N <= 8 * Pack<T>::n) stats(std::integral_constant<int, 8>{});
                else if (N <= 32 * Pack<T>::n) stats(std::integral_constant<int, 32>{});
                else stats(std::integral_constant<int, 64>{});
            }
            if (l.chunks > kFewChunks)
                hipLaunchKernelGGL(k_col_factors<T>, dim3((unsigned)tiles_of(N, 64)), dim3(kCT), 0, st, part_max, part_sum, l.chunks, N,
                                   prepared.factor, inverse, (T *)db);
            const auto prepare = [&](auto planes_tag) {
                constexpr int P = decltype(planes_tag)::value;
                const auto go = [&](auto kernel) {
                    hipLaunchKernelGGL(kernel, grid, dim3(kCT), 0, st, (const T *)dz, ldz, scales, rows, N, codes, ldc, K, l.Rp, split_blocks,
                                       prepared, (T *)db);
                };
                if (l.chunks == 0) go(k_prepare<T, P, W, kOwn>);
                else if (l.chunks <= kFewChunks) go(k_prepare<T, P, W, kChunks>);
                else go(k_prepare<T, P, W, kReady>);
            };
            if constexpr (std::is_same_v<T, bf16>) {
                if (l.planes == 1) return prepare(std::integral_constant<int, 1>{});
            }
            prepare(std::integral_constant<int, 2>{});
        });
        const auto launch = [&](auto tile) {
            using Tl = decltype(tile);
            const int tiles_k = (K + Tl::TI - 1) / Tl::TI, tiles_n = (N + Tl::TO - 1) / Tl::TO;
            const bool aligned = quads_aligned((T *)dw, ldw);
            hipLaunchKernelGGL((k_weight_grad<T, Tl>), dim3((unsigned)(tiles_k * tiles_n * l.shape.splits)), dim3(Tl::threads), 0, st,
                               codes_t, planes, inverse, K, N, l.Rp, l.planes, (T *)dw, ldw, aligned, tiles_k, tiles_n, l.shape.splits,
                               partial);
            if (l.shape.splits > 1) {
                hipLaunchKernelGGL(k_weight_join<T>, dim3((unsigned)tiles_of(K, 1024), (unsigned)N), dim3(256), 0, st, partial,
                                   l.shape.splits, inverse, K, N, (T *)dw, ldw, aligned, (const float *)nullptr, (T *)nullptr);
            }
        };
        if (l.shape.tile == 256) launch(Tile<OpF16, 256, 256, 4, 2>{});
        else if (l.shape.tile == 128) launch(Tile<OpF16, 128, 256, 2, 4>{});
        else launch(Tile<OpF16, 64, 64, 2, 2>{});
    });
    return mz::check_launch("mz_ckpt8_weight_grad");
}

}  // extern "C"
