// Weight gradients from 8-bit activation checkpoints (gfx950): a dense layer z = x W^T + b keeps its input as row codes
// (mz_quant8_rows: x_rk about s_r q_rk), and its backward pass forms
//     dW_nk = sum_r dz_rn s_r q_rk,     db_n = sum_r dz_rn
// without writing x out again.
//
// The product runs on the fp16 matrix instruction.  Codes are whole numbers up to 127: exact in fp16.  The row scale lies
// along the reduction, so it goes to the other side: v_rn = dz_rn s_r, which fp16 cannot hold as it is.  Each output row n
// is first brought into range by a power of two c_n (the largest |v_rn c_n| lies in 2^14 .. 2^15) and then held as
//     one plane   hi = fp16(v c)                       bfloat16 dz with scales of 3 significant bits: 8 + 3 = 11 bits,
//                                                      which is what fp16 has -- exact
//     two planes  hi = fp16(v c), lo = fp16(v c - hi)  everything else: 22 bits
// (values below 2^-16 of their row's largest lose bits of the second plane, values below 2^-28 of the first one: an
// absolute error of at most 2^-25 c_n^-1 then, 2^-39 of the largest).  The two planes' products go to one float32
// accumulator, and 1 / c_n is applied at the end, exact.
//   k_col_stats   per column of dz: largest |v| and sum of dz, for chunks of rows
//   k_split       dz -> planes, transposed to [n][plane][r]; db and 1 / c_n from the chunks
//   k_codes_t     codes -> fp16, transposed to [k][r]
//   k_weight_grad the product; k_weight_join the sum of its parts where the reduction is split
#include "mz_tile.h"

namespace {

using namespace mze;
using namespace mzt8;

constexpr int kCT = 256;
constexpr int kMaxChunks = 64;

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

template <class T>
__global__ void __launch_bounds__(kCT)
k_col_stats(const T *__restrict__ dz, int64_t ldz, const float *__restrict__ scales, int R, int N, int chunk_rows,
            unsigned *__restrict__ part_max, float *__restrict__ part_sum) {
    const int n = blockIdx.x * kCT + threadIdx.x, chunk = blockIdx.y;
    if (n >= N) return;
    unsigned m = 0;
    float s = 0.0f;
    for (int r = chunk * chunk_rows; r < min(R, (chunk + 1) * chunk_rows); ++r) {
        const float g = (float)dz[r * ldz + n];
        m = max(m, __float_as_uint(g * scales[r]) & 0x7FFFFFFFu);
        s += g;
    }
    part_max[(int64_t)chunk * N + n] = m;
    part_sum[(int64_t)chunk * N + n] = s;
}

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

// 64 x 64 values per workgroup, transposed through LDS; rows behind the last one become zeros.
template <class T, int PLANES>
__global__ void __launch_bounds__(kCT)
k_split(const T *__restrict__ dz, int64_t ldz, const float *__restrict__ scales, int R, int N, int64_t Rp, int chunks,
        const unsigned *__restrict__ part_max, const float *__restrict__ part_sum, f16 *__restrict__ planes,
        float *__restrict__ inverse, T *__restrict__ db) {
    __shared__ float tile[64][65];
    __shared__ float factor[64];
    const int n0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
    if (threadIdx.x < 64) {
        const int n = n0 + threadIdx.x;
        unsigned m = 0;
        float s = 0.0f;
        if (n < N)
            for (int c = 0; c < chunks; ++c) {
                m = max(m, part_max[(int64_t)c * N + n]);
                s += part_sum[(int64_t)c * N + n];
            }
        float inv;
        factor[threadIdx.x] = column_factor(m, &inv);
        if (n < N && blockIdx.y == 0) {
            inverse[n] = inv;
            if (db) db[n] = (T)s;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += kCT) {
        const int r = i >> 6, n = i & 63;
        float v = 0.0f;
        if (r0 + r < R && n0 + n < N) v = ((float)dz[(r0 + r) * ldz + n0 + n] * scales[r0 + r]) * factor[n];
        tile[r][n] = v;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += kCT) {
        const int n = i >> 6, r = i & 63;
        if (n0 + n >= N) continue;
        const float v = tile[r][n];
        const f16 hi = (f16)v;
        f16 *row = planes + (int64_t)(n0 + n) * PLANES * Rp;
        row[r0 + r] = hi;
        if (PLANES == 2) row[Rp + r0 + r] = (f16)(v - (float)hi);
    }
}

__global__ void __launch_bounds__(kCT)
k_codes_t(const int8_t *__restrict__ codes, int64_t ldc, int R, int K, int64_t Rp, f16 *__restrict__ out) {
    __shared__ int8_t tile[64][68];
    const int k0 = blockIdx.x * 64, r0 = blockIdx.y * 64;
    for (int i = threadIdx.x; i < 64 * 64; i += kCT) {
        const int r = i >> 6, k = i & 63;
        tile[r][k] = r0 + r < R && k0 + k < K ? codes[(r0 + r) * ldc + k0 + k] : (int8_t)0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * 64; i += kCT) {
        const int k = i >> 6, r = i & 63;
        if (k0 + k < K) out[(k0 + k) * Rp + r0 + r] = (f16)(float)tile[r][k];
    }
}

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
        store_quad(dw + (n0 + n) * ldw, k, K, aligned, o);
    });
}

// Sums of the parts of a split reduction, in a fixed order: one thread per four values of a row of dW.
template <class T>
__global__ void __launch_bounds__(256)
k_weight_join(const float *__restrict__ partial, int splits, const float *__restrict__ inverse, int K, int N, T *__restrict__ dw,
              int64_t ldw, bool aligned) {
    const int quads = (K + 3) / 4;
    const int64_t jobs = (int64_t)N * quads;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < jobs; q += (int64_t)gridDim.x * 256) {
        const int n = (int)(q / quads), k = 4 * (int)(q - (int64_t)n * quads);
        f32x4 sum = *(const f32x4 *)(partial + q * 4);
        for (int p = 1; p < splits; ++p) sum += *(const f32x4 *)(partial + (p * jobs + q) * 4);
        sum *= inverse[n];
        const float o[4] = {sum[0], sum[1], sum[2], sum[3]};
        store_quad(dw + n * ldw, k, K, aligned, o);
    }
}

struct Layout {
    int planes, chunks, chunk_rows;
    Shape shape;
    int64_t Rp, off_sum, off_inverse, off_planes, off_codes, off_partial, bytes;
};

Layout layout(int32_t type, int32_t scale_bits, int64_t R, int64_t N, int64_t K) {
    Layout l;
    l.planes = type == MZ_TYPE_BF16 && scale_bits == 3 ? 1 : 2;
    l.Rp = round_up(R, 64);
    l.chunks = (int)(R < 32 * kMaxChunks ? (R + 31) / 32 : kMaxChunks);
    l.chunk_rows = (int)((R + l.chunks - 1) / l.chunks);
    const int64_t stat = round_up((int64_t)l.chunks * N * 4, 128);
    l.off_sum = stat;
    l.off_inverse = 2 * stat;
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
    const Layout l = layout(type, scale_bits, rows, N, K);
    if (!workspace || workspace_bytes < l.bytes || ((uintptr_t)workspace & 15) != 0)
        return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: needs a 16-byte aligned workspace of %lld bytes (got %lld)",
                        (long long)l.bytes, (long long)workspace_bytes);
    const int64_t tiles = (round_up(N, 64) / 64) * (round_up(K, 64) / 64);
    if (tiles > (1 << 23) || l.Rp / 64 > 65535)
        return mz::fail(MZ_ERR_ARG, "mz_ckpt8_weight_grad: rows=%d N=%d K=%d is too large for one call", rows, N, K);
    uint8_t *ws = (uint8_t *)workspace;
    unsigned *part_max = (unsigned *)ws;
    float *part_sum = (float *)(ws + l.off_sum), *inverse = (float *)(ws + l.off_inverse);
    f16 *planes = (f16 *)(ws + l.off_planes), *codes_t = (f16 *)(ws + l.off_codes);
    float *partial = (float *)(ws + l.off_partial);
    hipStream_t st = (hipStream_t)stream;
    const dim3 split_grid((unsigned)((N + 63) / 64), (unsigned)(l.Rp / 64)), codes_grid((unsigned)((K + 63) / 64), (unsigned)(l.Rp / 64));
    with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL(k_col_stats<T>, dim3((unsigned)((N + kCT - 1) / kCT), (unsigned)l.chunks), dim3(kCT), 0, st, (const T *)dz,
                           ldz, scales, rows, N, l.chunk_rows, part_max, part_sum);
        if (l.planes == 1)
            hipLaunchKernelGGL((k_split<T, 1>), split_grid, dim3(kCT), 0, st, (const T *)dz, ldz, scales, rows, N, l.Rp, l.chunks,
                               part_max, part_sum, planes, inverse, (T *)db);
        else
            hipLaunchKernelGGL((k_split<T, 2>), split_grid, dim3(kCT), 0, st, (const T *)dz, ldz, scales, rows, N, l.Rp, l.chunks,
                               part_max, part_sum, planes, inverse, (T *)db);
        hipLaunchKernelGGL(k_codes_t, codes_grid, dim3(kCT), 0, st, codes, ldc, rows, K, l.Rp, codes_t);
        const auto launch = [&](auto tile) {
            using Tl = decltype(tile);
            const int tiles_k = (K + Tl::TI - 1) / Tl::TI, tiles_n = (N + Tl::TO - 1) / Tl::TO;
            const bool aligned = quads_aligned((T *)dw, ldw);
            hipLaunchKernelGGL((k_weight_grad<T, Tl>), dim3((unsigned)(tiles_k * tiles_n * l.shape.splits)), dim3(Tl::threads), 0, st,
                               codes_t, planes, inverse, K, N, l.Rp, l.planes, (T *)dw, ldw, aligned, tiles_k, tiles_n, l.shape.splits,
                               partial);
            if (l.shape.splits > 1) {
                const int64_t groups = ((int64_t)N * ((K + 3) / 4) + 255) / 256;
                hipLaunchKernelGGL(k_weight_join<T>, dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, st, partial,
                                   l.shape.splits, inverse, K, N, (T *)dw, ldw, aligned);
            }
        };
        if (l.shape.tile == 256) launch(Tile<OpF16, 256, 256, 4, 2>{});
        else if (l.shape.tile == 128) launch(Tile<OpF16, 128, 256, 2, 4>{});
        else launch(Tile<OpF16, 64, 64, 2, 2>{});
    });
    return mz::check_launch("mz_ckpt8_weight_grad");
}

}  // extern "C"
