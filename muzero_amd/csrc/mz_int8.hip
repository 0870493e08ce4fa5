// Dense layers in 8-bit integers (gfx950): y = act(x W^T + b) with a scale for each row of x and each row of W
// (mz_quant8_rows with full scales),
//     y_rn = act((fl(sum_k q_rk w_nk) s_r) t_n + b_n),
// the sum in 32-bit integers, which K <= 131072 keeps exact.
#include <cmath>

#include "mz_codes.h"
#include "mz_tile.h"

namespace {

using namespace mze;
using namespace mzt8;

constexpr int kMaxK = 131072;

__device__ __forceinline__ float activate(float v, int act) {
    switch (act) {
        case MZ_ACT_RELU: return v > 0.0f || v != v ? v : 0.0f;
        case MZ_ACT_TANH: return tanhf(v);
        case MZ_ACT_SIGMOID: return 1.0f / (1.0f + expf(-v));
        default: return v;
    }
}

// The tiled product, its epilogue on the accumulators: 8192 x 4096 x 8192 bf16 224 us, 2.45 POP/s (a library's int8 product of
// 8192^3 2.43), bound by the matrix cores; 256 x 18432 x 9216 in seven parts 45 us, 3.8 TB/s of weights.
template <class T, class Tl, bool PAST>
__global__ void __launch_bounds__(Tl::threads)
k_int8(const int8_t *__restrict__ xc, int64_t ldxc, const float *__restrict__ xs, int rows, const int8_t *__restrict__ wc,
       int64_t ldw, const float *__restrict__ ws, int N, int kbytes, const float *__restrict__ bias, int act, T *__restrict__ y,
       int64_t ldy, bool aligned, int tiles_n, int tiles_r, int splits, int *__restrict__ partial) {
    __shared__ __align__(16) uint8_t lds[Tl::lds_bytes];
    const int split = blockIdx.x % splits;
    const TileAt at = tile_at(blockIdx.x / splits, tiles_n, tiles_r, 8);
    const int n0 = at.inner * Tl::TI, r0 = at.outer * Tl::TO;
    const Operand inner{(const uint8_t *)wc, ldw, N, kbytes}, outer{(const uint8_t *)xc, ldxc, rows, kbytes};
    const int steps = kbytes / kStep;
    typename Tl::Acc acc;
    Tl::product(inner, n0, outer, r0, steps * split / splits, steps * (split + 1) / splits, lds, acc);
    const int n = n0 + Tl::inner_of();
    if (splits > 1) {
        const int Nq = (N + 3) / 4 * 4;
        int *out = partial + (int64_t)split * rows * Nq;
        Tl::template drain<true>(lds, acc, [](int, const i32x4 &v) { return v; }, [&](int r, const i32x4 &v) {
            if (r0 + r < rows && n < N) *(i32x4 *)(out + (int64_t)(r0 + r) * Nq + n) = v;
        });
        return;
    }
    float t[4], c[4], s[Tl::NO];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        t[e] = n + e < N ? ws[n + e] : 0.0f;
        c[e] = bias && n + e < N ? bias[n + e] : 0.0f;
    }
#pragma unroll
    for (int b = 0; b < Tl::NO; ++b) s[b] = xs[min(r0 + Tl::outer_of(b), rows - 1)];
    const auto scaled = [&](int b, const i32x4 &v) { return f32x4{(float)v[0] * s[b], (float)v[1] * s[b], (float)v[2] * s[b], (float)v[3] * s[b]}; };
    const auto put = [&](int r, const f32x4 &v, auto &&f) {
        if (r0 + r >= rows) return;
        const float o[4] = {f(v[0] * t[0] + c[0]), f(v[1] * t[1] + c[1]), f(v[2] * t[2] + c[2]), f(v[3] * t[3] + c[3])};
        store_quad<PAST>(y + (r0 + r) * ldy, n, N, aligned, o);
    };
    if (act == MZ_ACT_NONE || act == MZ_ACT_RELU) {
        const float least = act == MZ_ACT_RELU ? 0.0f : -INFINITY;  // a NaN is not less: it passes
        Tl::template drain<true>(lds, acc, scaled, [&](int r, const f32x4 &v) { put(r, v, [&](float x) { return x < least ? least : x; }); });
    } else {
        Tl::template drain<false>(lds, acc, scaled, [&](int r, const f32x4 &v) { put(r, v, [&](float x) { return activate(x, act); }); });
    }
}

// Sums of the parts of a split reduction, scales, bias, activation: one thread per four values of an output row.  Bound by
// the bytes: 256 x 9216 from seven parts 13.4 us, 5.6 TB/s.
template <class T>
__global__ void __launch_bounds__(256)
k_int8_join(const int *__restrict__ partial, int splits, const float *__restrict__ xs, int rows, const float *__restrict__ ws, int N,
            const float *__restrict__ bias, int act, T *__restrict__ y, int64_t ldy, bool aligned) {
    const int quads = (N + 3) / 4, r = blockIdx.y, c = blockIdx.x * 256 + threadIdx.x, n = 4 * c;
    if (c >= quads) return;
    const i32x4 sum = sum_parts<i32x4>(partial, splits, (int64_t)rows * quads, (int64_t)r * quads + c);
    const float s = xs[r];
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = n + e < N ? activate((float)sum[e] * s * ws[n + e] + (bias ? bias[n + e] : 0.0f), act) : 0.0f;
    store_quad<false>(y + r * ldy, n, N, aligned, o);
}

// A few rows (at most 16 NB): bound by reading the weights once.  A workgroup takes 16 output channels and all rows, its
// eight waves every eighth 128 bytes of the reduction; a lane reads 32 consecutive bytes of one channel and of NB rows of x
// and feeds them to the instructions straight from registers: weights are used once, so LDS would only add a barrier.
// The waves' sums meet in LDS.  1 x 9216 x 9216: 18 us, 4.7 TB/s, where the last level still holds the weights of the
// call before; 22 us, 3.8 TB/s, for twelve weights in turn (64 x 64 tiles, the reduction in four: 18 + the quantiser;
// 1 x 4096 x 4096: 4.5 against 8.6).  32 channels per workgroup: 23 us.
constexpr int kFewWaves = 8;

template <class T, int NB>
__global__ void __launch_bounds__(64 * kFewWaves)
k_int8_few(const int8_t *__restrict__ xc, int64_t ldxc, const float *__restrict__ xs, int rows, const int8_t *__restrict__ wc,
           int64_t ldw, const float *__restrict__ ws, int N, int kbytes, const float *__restrict__ bias, int act, T *__restrict__ y,
           int64_t ldy) {
    __shared__ __align__(16) int sums[kFewWaves][256 * NB];  // [row][channel]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, n0 = blockIdx.x * 16;
    const int8_t *w = wc + (int64_t)min(n0 + c, N - 1) * ldw + (lane >> 4) * 32, *x[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) x[b] = xc + (int64_t)min(16 * b + c, rows - 1) * ldxc + (lane >> 4) * 32;
    i32x4 acc[NB] = {};
    int k = wave * kStep;
    const auto steps = [&](auto count) {  // the loads of `count` steps in flight
        constexpr int C = decltype(count)::value;
        u32x4 p[C][2], q[C][NB][2];
#pragma unroll
        for (int u = 0; u < C; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) p[u][h] = *(const u32x4 *)(w + k + u * kFewWaves * kStep + h * 16);
#pragma unroll
        for (int u = 0; u < C; ++u)
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) q[u][b][h] = *(const u32x4 *)(x[b] + k + u * kFewWaves * kStep + h * 16);
#pragma unroll
        for (int u = 0; u < C; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int b = 0; b < NB; ++b) acc[b] = OpI8::mfma(p[u][h], q[u][b][h], acc[b]);
        k += C * kFewWaves * kStep;
    };
    while (k + 3 * kFewWaves * kStep < kbytes) steps(std::integral_constant<int, 4>{});
    while (k < kbytes) steps(std::integral_constant<int, 1>{});
#pragma unroll
    for (int b = 0; b < NB; ++b) *(i32x4 *)&sums[wave][(16 * b + c) * 16 + 4 * (lane >> 4)] = acc[b];
    __syncthreads();
    for (int i = threadIdx.x; i < 256 * NB; i += 64 * kFewWaves) {
        const int r = i >> 4, n = n0 + (i & 15);
        if (r >= rows || n >= N) continue;
        int sum = 0;
#pragma unroll
        for (int q = 0; q < kFewWaves; ++q) sum += sums[q][i];
        y[r * ldy + n] = (T)activate((float)sum * xs[r] * ws[n] + (bias ? bias[n] : 0.0f), act);
    }
}

// The same for up to kFusedRows rows that are not coded yet, in one launch: every workgroup codes them for itself, into
// LDS, while its first weights are on their way (a row of 9216 float32 comes from L2; a launch of the quantiser of its own
// costs more than that).  Up to kSharedRows rows all waves work on one after the other; beyond, every wave has its own rows,
// up to kOwnValues values in all (SHARED, a constant: with both in one kernel 1 x 9216 x 9216 takes 20.4 us, not 17.8).  us
// per layer in a chain, one launch / two (which also cost 3 us more of the host): 5 x 512 4.2 / 5.0, 5 x 2048 5.9 / 6.4,
// 16 x 168 4.8 / 5.1, 16 x 1024 6.3 / 6.1; behind it 16 x 2048 8.7 / 7.0.
constexpr int kFusedRows = 16, kSharedRows = 4, kOwnValues = 16384, kFusedBytes = 40960;

int64_t fused_stride(int64_t K) { return (K + 127) / 128 * 128 + 16; }  // rows of codes in different banks

template <class T, bool WHOLE, bool SHARED>
__global__ void __launch_bounds__(64 * kFewWaves)
k_int8_fused(const T *__restrict__ xp, int64_t ldx, int rows, int K, const int8_t *__restrict__ wc, int64_t ldw,
             const float *__restrict__ ws, int N, const float *__restrict__ bias, int act, T *__restrict__ y, int64_t ldy) {
    extern __shared__ __align__(16) uint8_t codes[];
    __shared__ __align__(16) int sums[kFewWaves][16 * 16];
    __shared__ unsigned top[kFusedRows][kFewWaves];
    constexpr int n = Pack<T>::n, threads = 64 * kFewWaves, U = 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, n0 = blockIdx.x * 16, kbytes = (K + 127) / 128 * 128,
              stride = kbytes + 16;
    const int8_t *w = wc + (int64_t)min(n0 + c, N - 1) * ldw + (lane >> 4) * 32;
    u32x4 first[U][2];  // the first weights, before anything is waited for
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k = (wave + u * kFewWaves) * kStep;
#pragma unroll
        for (int h = 0; h < 2; ++h) first[u][h] = k < kbytes ? *(const u32x4 *)(w + k + h * 16) : u32x4{};
    }
    if constexpr (SHARED) {  // all waves on one row after the other
        for (int r = 0; r < rows; ++r) {
            unsigned m = 0;
#pragma unroll 4
            for (int j = threadIdx.x * n; j < K; j += threads * n) {
                const Pack<T> p = load_pack<T, WHOLE>(xp + r * ldx, j, K);
#pragma unroll
                for (int e = 0; e < n; ++e) m = max(m, abs_bits((float)p.v[e]));
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o));
            if (lane == 0) top[r][wave] = m;
        }
        __syncthreads();
        for (int r = 0; r < rows; ++r) {
            unsigned m = 0;
#pragma unroll
            for (int q = 0; q < kFewWaves; ++q) m = max(m, top[r][q]);
            const RowScale rs = row_scale(m, 24);
#pragma unroll 4
            for (int j = threadIdx.x * n; j < kbytes; j += threads * n)
                store_codes((int8_t *)codes + r * stride + j, load_pack<T, WHOLE>(xp + r * ldx, j, K), rs.inverse);
        }
    } else {  // every wave its own rows
        for (int r = wave; r < rows; r += kFewWaves) {
            unsigned m = 0;
#pragma unroll 4
            for (int j = lane * n; j < K; j += 64 * n) {
                const Pack<T> p = load_pack<T, WHOLE>(xp + r * ldx, j, K);
#pragma unroll
                for (int e = 0; e < n; ++e) m = max(m, abs_bits((float)p.v[e]));
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o));
            if (lane < kFewWaves) top[r][lane] = m;
            const RowScale rs = row_scale(m, 24);
#pragma unroll 4
            for (int j = lane * n; j < kbytes; j += 64 * n)
                store_codes((int8_t *)codes + r * stride + j, load_pack<T, WHOLE>(xp + r * ldx, j, K), rs.inverse);
        }
    }
    __syncthreads();
    const uint8_t *x = codes + min(c, rows - 1) * stride + (lane >> 4) * 32;
    i32x4 acc = {};
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k = (wave + u * kFewWaves) * kStep;
        if (k < kbytes)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = OpI8::mfma(first[u][h], *(const u32x4 *)(x + k + h * 16), acc);
    }
    int k = (wave + U * kFewWaves) * kStep;
    const auto steps = [&](auto count) {
        constexpr int C = decltype(count)::value;
        u32x4 p[C][2];
#pragma unroll
        for (int u = 0; u < C; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) p[u][h] = *(const u32x4 *)(w + k + u * kFewWaves * kStep + h * 16);
#pragma unroll
        for (int u = 0; u < C; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc = OpI8::mfma(p[u][h], *(const u32x4 *)(x + k + u * kFewWaves * kStep + h * 16), acc);
        k += C * kFewWaves * kStep;
    };
    while (k + (U - 1) * kFewWaves * kStep < kbytes) steps(std::integral_constant<int, U>{});
    while (k < kbytes) steps(std::integral_constant<int, 1>{});
    *(i32x4 *)&sums[wave][c * 16 + 4 * (lane >> 4)] = acc;
    __syncthreads();
    if (threadIdx.x < 256) {
        const int r = threadIdx.x >> 4, o = n0 + (threadIdx.x & 15);
        if (r < rows && o < N) {
            unsigned m = 0;
            int sum = 0;
#pragma unroll
            for (int q = 0; q < kFewWaves; ++q) m = max(m, top[r][q]), sum += sums[q][threadIdx.x];
            y[r * ldy + o] = (T)activate((float)sum * row_scale(m, 24).scale * ws[o] + (bias ? bias[o] : 0.0f), act);
        }
    }
}

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

int check_code_rows(const char *what, const int8_t *codes, int64_t ldc, const float *scales, int32_t K) {
    if (!codes || !scales) return mz::fail(MZ_ERR_ARG, "%s: NULL argument", what);
    if (ldc < K || ldc % 128 != 0 || ldc > (1 << 22) || ((uintptr_t)codes & 15) != 0)
        return mz::fail(MZ_ERR_ARG, "%s: codes need 16-byte aligned rows of a multiple of 128 bytes (at most 2^22), zero behind K=%d (row stride %lld)",
                        what, K, (long long)ldc);
    return MZ_OK;
}

int check_int8(int32_t rows, int32_t K, const int8_t *w_codes, int64_t ldw, const float *w_scales, int32_t N, int32_t activation,
               const void *y, int32_t type, int64_t ldy) {
    if (rows < 0 || K <= 0 || N <= 0 || N > (1 << 26)) return mz::fail(MZ_ERR_ARG, "mz_int8_forward: bad dimensions rows=%d K=%d N=%d", rows, K, N);
    if (K > kMaxK) return mz::fail(MZ_ERR_ARG, "mz_int8_forward: K=%d above %d would overflow the 32-bit sums", K, kMaxK);
    if (!type_ok(type)) return mz::fail(MZ_ERR_ARG, "mz_int8_forward: unknown element type %d", type);
    if (activation < MZ_ACT_NONE || activation > MZ_ACT_SIGMOID)
        return mz::fail(MZ_ERR_ARG, "mz_int8_forward: activation %d is not element-wise", activation);
    MZ_TRY(check_code_rows("mz_int8_forward", w_codes, ldw, w_scales, K));
    if (rows > 0 && !y) return mz::fail(MZ_ERR_ARG, "mz_int8_forward: NULL argument");
    if (ldy < N || ((uintptr_t)y & (type_bytes(type) - 1)) != 0)
        return mz::fail(MZ_ERR_ARG, "mz_int8_forward: bad output stride %lld or alignment for N=%d", (long long)ldy, N);
    if ((round_up(N, 64) / 64) * (round_up(rows, 64) / 64) > (1 << 23))
        return mz::fail(MZ_ERR_ARG, "mz_int8_forward: output of %d x %d is too large for one call", rows, N);
    return MZ_OK;
}

int check_workspace(const void *workspace, int64_t bytes, int64_t need) {
    if (need > 0 && (!workspace || bytes < need || ((uintptr_t)workspace & 15) != 0))
        return mz::fail(MZ_ERR_ARG, "mz_int8_forward: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
                        (long long)bytes);
    return MZ_OK;
}

struct Int8Args {
    const int8_t *xc;
    int64_t ldxc;
    const float *xs;
    int rows;
    const int8_t *wc;
    int64_t ldw;
    const float *ws;
    int N, K;
    const float *bias;
    int act;
    void *y;
    int64_t ldy;
    int *partial;
};

template <class T, class Tl, bool PAST = false>
void launch_tiles(const Int8Args &a, int splits, hipStream_t st) {
    const int tiles_n = (a.N + Tl::TI - 1) / Tl::TI, tiles_r = (a.rows + Tl::TO - 1) / Tl::TO;
    const bool aligned = quads_aligned((T *)a.y, a.ldy);
    hipLaunchKernelGGL((k_int8<T, Tl, PAST>), dim3((unsigned)(tiles_n * tiles_r * splits)), dim3(Tl::threads), 0, st, a.xc, a.ldxc, a.xs, a.rows,
                       a.wc, a.ldw, a.ws, a.N, (int)round_up(a.K, kStep), a.bias, a.act, (T *)a.y, a.ldy, aligned, tiles_n, tiles_r, splits,
                       a.partial);
    if (splits > 1) {
        hipLaunchKernelGGL(k_int8_join<T>, dim3((unsigned)tiles_of(a.N, 1024), (unsigned)a.rows), dim3(256), 0, st, a.partial, splits, a.xs,
                           a.rows, a.ws, a.N, a.bias, a.act, (T *)a.y, a.ldy, aligned);
    }
}

Shape shape_of_int8(int64_t rows, int64_t N, int64_t K) { return shape_of(rows, N, round_up(K, kStep) / kStep); }

template <class T, int NB>
void launch_few(const Int8Args &a, hipStream_t st) {
    hipLaunchKernelGGL((k_int8_few<T, NB>), dim3((unsigned)tiles_of(a.N, 16)), dim3(64 * kFewWaves), 0, st, a.xc, a.ldxc, a.xs, a.rows, a.wc,
                       a.ldw, a.ws, a.N, (int)round_up(a.K, kStep), a.bias, a.act, (T *)a.y, a.ldy);
}

// Few rows go by k_int8_few: up to 4 always, up to 32 where the weights are small (us, k_int8_few / tiles: 16 x 4096 x 4096
// 5.8 / 9.1, 32 x 4096 x 4096 7.8 / 10; but 16 x 9216 x 9216 26 / 19, 32 x 9216 x 18432 73 / 31, as every workgroup reads
// all rows of x again); not where a few channels have long rows, which tiles in parts share among more compute units
// (1 x 65536 x 256 37 / 11, 16 x 18432 x 16 17 / 9.7, 32 x 18432 x 256 26 / 10; but 16 x 8192 x 16 8.8 / 9.6).
bool few_rows(int64_t rows, int64_t N, int64_t K) {
    if (K > 12288 && N <= 1024) return false;
    return rows <= 4 || (rows <= 32 && N * K <= 24LL * 1000 * 1000);
}

// One launch where x has the result's type and its codes fit a workgroup's share of LDS; asked before few_rows, for long rows
// of a few channels too (whole calls, us, one launch / rows coded by a call of their own and tiles: 1 x 12288 x 256 12.3 / 20,
// 1 x 20480 x 256 14.5 / 24, 1 x 32768 x 1024 22.3 / 23.8; at the end of its range, 1 x 40832 x 256, 26.3 / 23.8).
bool fused(int32_t x_type, int32_t type, int64_t rows, int64_t K) {
    return x_type == type && (rows <= kSharedRows || (rows <= kFusedRows && rows * K <= kOwnValues)) && rows * fused_stride(K) <= kFusedBytes;
}

template <class T>
void launch_shape(const Int8Args &a, hipStream_t st) {
    if (few_rows(a.rows, a.N, a.K)) {
        if (a.rows <= 16) launch_few<T, 1>(a, st);
        else launch_few<T, 2>(a, st);
        return;
    }
    const Shape s = shape_of_int8(a.rows, a.N, a.K);
    const bool past = past_caches((int64_t)a.rows * a.N * (int64_t)sizeof(T));  // 256 x 256 tiles, but for up to 64 rows
    if (s.tile == 256 && past) launch_tiles<T, Tile<OpI8, 256, 256, 4, 2>, true>(a, s.splits, st);
    else if (s.tile == 256) launch_tiles<T, Tile<OpI8, 256, 256, 4, 2>>(a, s.splits, st);
    else if (s.tile == 128) launch_tiles<T, Tile<OpI8, 128, 256, 2, 4>>(a, s.splits, st);
    else launch_tiles<T, Tile<OpI8, 64, 64, 2, 2>>(a, s.splits, st);
}

int64_t partial_bytes(int64_t rows, int64_t N, int64_t K) {
    const Shape s = shape_of_int8(rows, N, K);
    return !few_rows(rows, N, K) && s.splits > 1 ? s.splits * rows * round_up(N, 4) * 4 : 0;
}

}  // namespace

extern "C" {

int64_t mz_int8_codes_workspace(int32_t rows, int32_t K, int32_t N) {
    return rows <= 0 || K <= 0 || N <= 0 ? 0 : partial_bytes(rows, N, K);
}

int mz_int8_forward_codes(const int8_t *x_codes, int64_t ldxc, const float *x_scales, int32_t rows, int32_t K,
                          const int8_t *w_codes, int64_t ldw, const float *w_scales, int32_t N, const float *bias,
                          int32_t activation, void *y, int32_t type, int64_t ldy, void *workspace, int64_t workspace_bytes,
                          void *stream) {
    MZ_TRY(check_int8(rows, K, w_codes, ldw, w_scales, N, activation, y, type, ldy));
    if (rows == 0) return MZ_OK;
    MZ_TRY(check_code_rows("mz_int8_forward", x_codes, ldxc, x_scales, K));
    MZ_TRY(check_workspace(workspace, workspace_bytes, mz_int8_codes_workspace(rows, K, N)));
    const Int8Args a{x_codes, ldxc, x_scales, rows, w_codes, ldw, w_scales, N, K, bias, activation, y, ldy, (int *)workspace};
    with_type(type, [&](auto t) { launch_shape<decltype(t)>(a, (hipStream_t)stream); });
    return mz::check_launch("k_int8");
}

int64_t mz_int8_workspace(int32_t rows, int32_t K, int32_t N) {
    if (rows <= 0 || K <= 0 || N <= 0) return 0;
    return round_up(partial_bytes(rows, N, K), 128) + round_up((int64_t)rows * 4, 128) + (int64_t)rows * round_up(K, kStep);
}

int mz_int8_forward(const void *x, int32_t x_type, int64_t ldx, int32_t rows, int32_t K, const int8_t *w_codes, int64_t ldw,
                    const float *w_scales, int32_t N, const float *bias, int32_t activation, void *y, int32_t type, int64_t ldy,
                    void *workspace, int64_t workspace_bytes, void *stream) {
    MZ_TRY(check_int8(rows, K, w_codes, ldw, w_scales, N, activation, y, type, ldy));
    if (rows == 0) return MZ_OK;
    MZ_TRY(check_workspace(workspace, workspace_bytes, mz_int8_workspace(rows, K, N)));
    if (fused(x_type, type, rows, K)) {
        MZ_TRY(check_rows("mz_int8_forward", x, x_type, ldx, rows, K));
        with_type(type, [&](auto t) {
            using T = decltype(t);
            with_flag(rows_aligned<T>(x, ldx), [&](auto whole) {
                constexpr bool W = decltype(whole)::value;
                const auto launch = [&](auto kernel) {
                    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles_of(N, 16)), dim3(64 * kFewWaves), (size_t)(rows * fused_stride(K)),
                                       (hipStream_t)stream, (const T *)x, ldx, rows, K, w_codes, ldw, w_scales, N, bias, activation, (T *)y, ldy);
                };
                rows <= kSharedRows ? launch(k_int8_fused<T, W, true>) : launch(k_int8_fused<T, W, false>);
            });
        });
        return mz::check_launch("k_int8_fused");
    }
    const int64_t partial = round_up(partial_bytes(rows, N, K), 128), ldc = round_up(K, kStep);
    float *scales = (float *)((uint8_t *)workspace + partial);
    int8_t *codes = (int8_t *)workspace + partial + round_up((int64_t)rows * 4, 128);
    MZ_TRY(mz_quant8_rows(x, x_type, ldx, rows, K, 24, codes, ldc, scales, stream));
    const Int8Args a{codes, ldc, scales, rows, w_codes, ldw, w_scales, N, K, bias, activation, y, ldy, (int *)workspace};
    with_type(type, [&](auto t) { launch_shape<decltype(t)>(a, (hipStream_t)stream); });
    return mz::check_launch("k_int8");
}

}  // extern "C"
