// Rows of activations or weights in 8 bits (gfx950): the codes an int8 product multiplies (mz_int8.hip) and the form
// an activation is kept in for the backward pass (mz_ckpt8.hip).
//
// One scale per row.  a = max |x| of the row;
//     full scale (24 bits)    s = fl(a / 127),                        i = fl(127 / a)
//     short scale (3 bits)    s = fl(a / 127) rounded UP to 3 bits,   i = fl(1 / s)
//     q = rne(fl(x i)) in -127 .. 127,   x is about q s   (error at most s / 2 and two roundings)
// fl is one float32 rounding, rne rounds half to even.  A row whose a is below 2^-119 (1 / s would leave the range of
// float32) is held as zeros with s = 0; a row with an infinity or a NaN as zeros with s = NaN, so that whatever is
// formed from it is NaN and not silently finite.
#include "mz_codes.h"

namespace {

using namespace mze;

constexpr int kQT = 256;
// THREADS threads per row (64: four rows per workgroup).  The first HELD packs of a thread stay in registers between the
// maximum and the codes; the rest of a longer row is read again, from cache.  Bound by the memory: 1536 x 18432 float32,
// 142 MB with the codes, 28 us, 5.0 TB/s.
template <class T, int THREADS, int HELD, bool WHOLE>
__global__ void __launch_bounds__(THREADS < kQT ? kQT : THREADS)
k_quant8(const T *__restrict__ x, int64_t ldx, int64_t rows, int K, int scale_bits, int8_t *__restrict__ codes, int64_t ldc,
         float *__restrict__ scales) {
    constexpr int n = Pack<T>::n, per = THREADS < kQT ? kQT / THREADS : 1;
    __shared__ unsigned part[THREADS / 64];
    const int t = threadIdx.x % THREADS, packs = (int)(ldc / n);
    for (int64_t row0 = (int64_t)blockIdx.x * per; row0 < rows; row0 += (int64_t)gridDim.x * per) {
        const int64_t row = row0 + threadIdx.x / THREADS;
        if (THREADS == 64 && row >= rows) break;
        const T *xr = x + row * ldx;
        Pack<T> held[HELD];
        unsigned m = 0;
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if ((t + h * THREADS) * n < K) held[h] = load_pack<T, WHOLE, true>(xr, (t + h * THREADS) * n, K);
            else held[h] = Pack<T>{};
#pragma unroll
        for (int h = 0; h < HELD; ++h)
#pragma unroll
            for (int e = 0; e < n; ++e) m = max(m, abs_bits((float)held[h].v[e]));
        for (int i = t + HELD * THREADS; i < packs; i += THREADS) {
            const Pack<T> p = load_pack<T, WHOLE>(xr, i * n, K);
#pragma unroll
            for (int e = 0; e < n; ++e) m = max(m, abs_bits((float)p.v[e]));
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o));
        if (THREADS > 64) {
            __syncthreads();  // the last row's maxima have been read
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < THREADS / 64; ++w) m = max(m, part[w]);
        }
        const RowScale rs = row_scale(m, scale_bits);
        if (t == 0) scales[row] = rs.scale;
        int8_t *cr = codes + row * ldc;
#pragma unroll
        for (int h = 0; h < HELD; ++h)
            if (t + h * THREADS < packs) store_codes(cr + (t + h * THREADS) * n, held[h], rs.inverse);
        for (int i = t + HELD * THREADS; i < packs; i += THREADS) store_codes(cr + i * n, load_pack<T, WHOLE>(xr, i * n, K), rs.inverse);
    }
}

// Bound by the memory: 1536 x 18432 to float32, 113 MB from 28 MB of codes in cache, 22 us.
template <class T, int THREADS, bool WHOLE, bool PAST>
__global__ void __launch_bounds__(kQT)
k_dequant8(const int8_t *__restrict__ codes, int64_t ldc, const float *__restrict__ scales, int64_t rows, int K,
           T *__restrict__ x, int64_t ldx) {
    constexpr int n = Pack<T>::n, per = kQT / THREADS;
    const int t = threadIdx.x % THREADS;
    for (int64_t row = (int64_t)blockIdx.x * per + threadIdx.x / THREADS; row < rows; row += (int64_t)gridDim.x * per) {
        const float s = scales[row];
        const int8_t *cr = codes + row * ldc;
#pragma unroll 4
        for (int j = t * n; j < K; j += THREADS * n) {
            alignas(8) int8_t q[n];  // the padding of a row covers a pack
            if constexpr (n == 4) *(unsigned *)q = *(const unsigned *)(cr + j);
            else *(uint2 *)q = *(const uint2 *)(cr + j);
            Pack<T> p;
#pragma unroll
            for (int e = 0; e < n; ++e) p.v[e] = (T)((float)q[e] * s);
            store_pack<T, WHOLE, PAST>(x + row * ldx, j, K, p);
        }
    }
}

// Eight consecutive values of a row, zeros behind its end.
template <class T, bool WHOLE>
__device__ __forceinline__ void load8(const T *row, int j, int N, float (&v)[8]) {
    constexpr int n = Pack<T>::n;
#pragma unroll
    for (int h = 0; h < 8 / n; ++h) {
        const Pack<T> p = load_pack<T, WHOLE>(row, j + h * n, N);
#pragma unroll
        for (int e = 0; e < n; ++e) v[h * n + e] = (float)p.v[e];
    }
}

// Both passes over an activation are one read and one write of it, bound by the memory.
// What the backward pass needs of y = act(z): relu one bit, [not y <= 0]; tanh and sigmoid a code of 8 bits on a fixed
// scale, -128 for a NaN.  A thread takes 8 values: a byte of bits, or 8 codes.
template <class T, bool WHOLE>
__global__ void __launch_bounds__(kQT)
k_act_save(const T *__restrict__ y, int64_t ldy, int64_t rows, int N, int act, uint8_t *__restrict__ saved, int64_t lds) {
    const int t = threadIdx.x % 64;
    for (int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; row < rows; row += (int64_t)gridDim.x * 4)
#pragma unroll 2
        for (int j = t * 8; j < N; j += 64 * 8) {
            float v[8];
            load8<T, WHOLE>(y + row * ldy, j, N, v);
            if (act == MZ_ACT_RELU) {
                unsigned bits = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) bits |= (unsigned)(j + e < N && !(v[e] <= 0.0f)) << e;
                saved[row * lds + (j >> 3)] = (uint8_t)bits;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float c = rintf(act == MZ_ACT_TANH ? v[e] * 127.0f : v[e] * 254.0f - 127.0f);
                    const unsigned code = v[e] == v[e] ? (unsigned)(int)fminf(fmaxf(c, -127.0f), 127.0f) : 0x80u;
                    if (j + e < N) saved[row * lds + j + e] = (uint8_t)code;
                }
            }
        }
}

// dz = dy act'(y): relu [y > 0]; tanh 1 - t^2 with t = q / 127; sigmoid s (1 - s) = (1 - t^2) / 4 with t = 2 s - 1.
template <class T, bool WHOLE>
__global__ void __launch_bounds__(kQT)
k_act_grad(const T *dy, int64_t ldy, const uint8_t *__restrict__ saved, int64_t lds, int64_t rows, int N, int act, T *dz,
           int64_t ldz) {
    constexpr int n = Pack<T>::n;
    const int t = threadIdx.x % 64;
    for (int64_t row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64; row < rows; row += (int64_t)gridDim.x * 4)
#pragma unroll 2
        for (int j = t * 8; j < N; j += 64 * 8) {
            float v[8];
            load8<T, WHOLE>(dy + row * ldy, j, N, v);
            if (act == MZ_ACT_RELU) {
                const unsigned bits = saved[row * lds + (j >> 3)];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = bits >> e & 1 ? v[e] : 0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int q = j + e < N ? (int8_t)saved[row * lds + j + e] : 0;
                    const float u = q == -128 ? __uint_as_float(0x7FC00000u) : (float)q / 127.0f;
                    v[e] *= (1.0f - u * u) * (act == MZ_ACT_TANH ? 1.0f : 0.25f);
                }
            }
#pragma unroll
            for (int h = 0; h < 8 / n; ++h) {
                Pack<T> p;
#pragma unroll
                for (int e = 0; e < n; ++e) p.v[e] = (T)v[h * n + e];
                store_pack<T, WHOLE>(dz + row * ldz, j + h * n, N, p);
            }
        }
}

// Workgroups for `rows` rows, `per` of them each, up to this many (a grid holds fewer than 2^32 threads); more rows are
// taken in turns.
dim3 row_grid(int64_t rows, int per) {
    const int64_t groups = (rows + per - 1) / per;
    return dim3((unsigned)(groups < (1 << 20) ? groups : (1 << 20)));
}

int check_codes(const char *what, const int8_t *codes, int64_t ldc, const float *scales, int64_t rows, int32_t K) {
    if (rows > 0 && (!codes || !scales)) return mz::fail(MZ_ERR_ARG, "%s: NULL argument", what);
    if (ldc < K || ldc % 16 != 0 || ldc > 0x7FFFFFFF || ((uintptr_t)codes & 15) != 0)
        return mz::fail(MZ_ERR_ARG, "%s: codes need 16-byte aligned rows of at least K=%d bytes (row stride %lld)", what, K, (long long)ldc);
    return MZ_OK;
}

bool act_saved_ok(int act) { return act == MZ_ACT_RELU || act == MZ_ACT_TANH || act == MZ_ACT_SIGMOID; }

}  // namespace

extern "C" {

int mz_quant8_rows(const void *x, int32_t type, int64_t ldx, int64_t rows, int32_t K, int32_t scale_bits, int8_t *codes,
                   int64_t ldc, float *scales, void *stream) {
    MZ_TRY(check_rows("mz_quant8_rows", x, type, ldx, rows, K));
    MZ_TRY(check_codes("mz_quant8_rows", codes, ldc, scales, rows, K));
    if (scale_bits != 24 && scale_bits != 3)
        return mz::fail(MZ_ERR_ARG, "mz_quant8_rows: scale_bits must be 24 or 3, not %d", scale_bits);
    if (rows == 0) return MZ_OK;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_flag(rows_aligned<T>(x, ldx), [&](auto whole) {
            constexpr bool W = decltype(whole)::value;
            const auto launch = [&](auto kernel, int per, int threads = kQT) {
                hipLaunchKernelGGL(kernel, row_grid(rows, per), dim3(threads), 0, (hipStream_t)stream, (const T *)x, ldx, rows, K, scale_bits,
                                   codes, ldc, scales);
            };
            // A wave per row up to 4 packs a lane, else a workgroup of 256 or 1024 threads, with as few registers for packs
            // as hold the row (1536 x 18432 float32: 1024 threads 26 us, 512 29 us, 256 37 us).
            const int64_t packs = ldc / Pack<T>::n;
            if (packs <= 2 * 64) launch(k_quant8<T, 64, 2, W>, 4);
            else if (packs <= 4 * 64) launch(k_quant8<T, 64, 4, W>, 4);
            else if (packs <= 2 * 256) launch(k_quant8<T, 256, 2, W>, 1);
            else if (packs <= 4 * 256) launch(k_quant8<T, 256, 4, W>, 1);
            else if (packs <= 2 * 1024) launch(k_quant8<T, 1024, 2, W>, 1, 1024);
            else launch(k_quant8<T, 1024, 5, W>, 1, 1024);
        });
    });
    return mz::check_launch("k_quant8");
}

int mz_dequant8_rows(const int8_t *codes, int64_t ldc, const float *scales, int64_t rows, int32_t K, void *x, int32_t type,
                     int64_t ldx, void *stream) {
    MZ_TRY(check_rows("mz_dequant8_rows", x, type, ldx, rows, K));
    MZ_TRY(check_codes("mz_dequant8_rows", codes, ldc, scales, rows, K));
    if (rows == 0) return MZ_OK;
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_flag(rows_aligned<T>(x, ldx), [&](auto whole) {
            constexpr bool W = decltype(whole)::value;
            const auto launch = [&](auto kernel, int per) {
                hipLaunchKernelGGL(kernel, row_grid(rows, per), dim3(kQT), 0, (hipStream_t)stream, codes, ldc, scales, rows, K, (T *)x, ldx);
            };
            with_flag(past_caches(rows * K * (int64_t)sizeof(T)), [&](auto past) {
                constexpr bool P = decltype(past)::value;
                if (K <= 4 * 64 * Pack<T>::n) launch(k_dequant8<T, 64, W, P>, 4);
                else launch(k_dequant8<T, 256, W, P>, 1);
            });
        });
    });
    return mz::check_launch("k_dequant8");
}

int64_t mz_ckpt8_act_bytes(int32_t N, int32_t activation) {
    if (N <= 0 || !act_saved_ok(activation)) return 0;
    return activation == MZ_ACT_RELU ? ((int64_t)N + 7) / 8 : N;
}

int mz_ckpt8_act_save(const void *y, int32_t type, int64_t ldy, int64_t rows, int32_t N, int32_t activation, uint8_t *saved,
                      void *stream) {
    MZ_TRY(check_rows("mz_ckpt8_act_save", y, type, ldy, rows, N));
    if (!act_saved_ok(activation)) return mz::fail(MZ_ERR_ARG, "mz_ckpt8_act_save: activation %d keeps nothing", activation);
    if (rows == 0) return MZ_OK;
    if (!saved) return mz::fail(MZ_ERR_ARG, "mz_ckpt8_act_save: NULL argument");
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_flag(rows_aligned<T>(y, ldy), [&](auto whole) {
            hipLaunchKernelGGL((k_act_save<T, decltype(whole)::value>), row_grid(rows, 4), dim3(kQT), 0, (hipStream_t)stream, (const T *)y,
                               ldy, rows, N, activation, saved, mz_ckpt8_act_bytes(N, activation));
        });
    });
    return mz::check_launch("k_act_save");
}

int mz_ckpt8_act_grad(const void *dy, int32_t type, int64_t ldy, const uint8_t *saved, int64_t rows, int32_t N,
                      int32_t activation, void *dz, int64_t ldz, void *stream) {
    MZ_TRY(check_rows("mz_ckpt8_act_grad", dy, type, ldy, rows, N));
    MZ_TRY(check_rows("mz_ckpt8_act_grad", dz, type, ldz, rows, N));
    if (!act_saved_ok(activation)) return mz::fail(MZ_ERR_ARG, "mz_ckpt8_act_grad: activation %d keeps nothing", activation);
    if (rows == 0) return MZ_OK;
    if (!saved) return mz::fail(MZ_ERR_ARG, "mz_ckpt8_act_grad: NULL argument");
    with_type(type, [&](auto t) {
        using T = decltype(t);
        with_flag(rows_aligned<T>(dy, ldy) && rows_aligned<T>(dz, ldz), [&](auto whole) {
            hipLaunchKernelGGL((k_act_grad<T, decltype(whole)::value>), row_grid(rows, 4), dim3(kQT), 0, (hipStream_t)stream, (const T *)dy,
                               ldy, saved, mz_ckpt8_act_bytes(N, activation), rows, N, activation, (T *)dz, ldz);
        });
    });
    return mz::check_launch("k_act_grad");
}

}  // extern "C"
