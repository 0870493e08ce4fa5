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
#include "mz_elem.h"

namespace {

using namespace mze;

constexpr int kQT = 256;
constexpr float kTiny = 0x1p-119f;

__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Maximum over the workgroup of unsigned values (NaN bit patterns order above infinity, so they win).
__device__ __forceinline__ unsigned block_max(unsigned v) {
    __shared__ unsigned part[kQT / 64];
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
    __syncthreads();  // the last row's values have been read
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < kQT / 64; ++w) v = max(v, part[w]);
    return v;
}

struct RowScale {
    float scale, inverse;
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

// One workgroup per row: the row is read twice (the second time from cache).
template <class T>
__global__ void __launch_bounds__(kQT)
k_quant8(const T *__restrict__ x, int64_t ldx, int64_t rows, int K, int scale_bits, int8_t *__restrict__ codes, int64_t ldc,
         float *__restrict__ scales) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * ldx;
    unsigned m = 0;
    for (int k = threadIdx.x; k < K; k += kQT) m = max(m, abs_bits((float)xr[k]));
    m = block_max(m);
    const RowScale rs = row_scale(m, scale_bits);
    if (threadIdx.x == 0) scales[row] = rs.scale;
    const bool live = rs.inverse != 0.0f;
    for (int k = threadIdx.x; k < ldc; k += kQT)
        codes[row * ldc + k] = (k < K && live) ? (int8_t)(int)rintf((float)xr[k] * rs.inverse) : (int8_t)0;
    }
}

template <class T>
__global__ void __launch_bounds__(kQT)
k_dequant8(const int8_t *__restrict__ codes, int64_t ldc, const float *__restrict__ scales, int64_t rows, int K,
           T *__restrict__ x, int64_t ldx) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float s = scales[row];
        for (int k = threadIdx.x; k < K; k += kQT) x[row * ldx + k] = (T)((float)codes[row * ldc + k] * s);
    }
}

// What the backward pass needs of y = act(z): relu one bit, [not y <= 0]; tanh and sigmoid a code of 8 bits on a fixed
// scale, -128 for a NaN.
template <class T>
__global__ void __launch_bounds__(kQT)
k_act_save(const T *__restrict__ y, int64_t ldy, int64_t rows, int N, int act, uint8_t *__restrict__ saved, int64_t lds) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
        for (int j = threadIdx.x; j < lds; j += kQT) {
            unsigned out = 0;
            if (act == MZ_ACT_RELU) {
                for (int b = 0; b < 8; ++b)
                    if (8 * j + b < N && !((float)y[row * ldy + 8 * j + b] <= 0.0f)) out |= 1u << b;
            } else {
                const float v = (float)y[row * ldy + j];
                const float c = rintf(act == MZ_ACT_TANH ? v * 127.0f : v * 254.0f - 127.0f);
                out = v == v ? (unsigned)(int)fminf(fmaxf(c, -127.0f), 127.0f) : 0x80u;
            }
            saved[row * lds + j] = (uint8_t)out;
        }
}

// dz = dy act'(y): relu [y > 0]; tanh 1 - t^2 with t = q / 127; sigmoid s (1 - s) = (1 - t^2) / 4 with t = 2 s - 1.
template <class T>
__global__ void __launch_bounds__(kQT)
k_act_grad(const T *dy, int64_t ldy, const uint8_t *__restrict__ saved, int64_t lds, int64_t rows, int N, int act, T *dz,
           int64_t ldz) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
    for (int j = threadIdx.x; j < N; j += kQT) {
        const float g = (float)dy[row * ldy + j];
        float d;
        if (act == MZ_ACT_RELU) {
            d = (saved[row * lds + (j >> 3)] >> (j & 7)) & 1 ? g : 0.0f;
        } else {
            const int q = (int8_t)saved[row * lds + j];
            const float t = q == -128 ? __uint_as_float(0x7FC00000u) : (float)q / 127.0f;
            d = g * ((1.0f - t * t) * (act == MZ_ACT_TANH ? 1.0f : 0.25f));
        }
        dz[row * ldz + j] = (T)d;
    }
}

// One workgroup per row up to this many (a grid holds fewer than 2^32 threads); more rows are taken in turns.
dim3 row_grid(int64_t rows) { return dim3((unsigned)(rows < (1 << 20) ? rows : (1 << 20))); }

int check_rows(const char *what, const void *x, int type, int64_t ld, int64_t rows, int64_t K) {
    if (!type_ok(type)) return mz::fail(MZ_ERR_ARG, "%s: unknown element type %d", what, type);
    if (rows < 0 || rows > 0x7FFFFFFF || K <= 0 || K > 0x7FFFFF00)
        return mz::fail(MZ_ERR_ARG, "%s: bad dimensions rows=%lld K=%lld", what, (long long)rows, (long long)K);
    if (rows > 0 && !x) return mz::fail(MZ_ERR_ARG, "%s: NULL argument", what);
    if (ld < K) return mz::fail(MZ_ERR_ARG, "%s: row stride %lld below the %lld values of a row", what, (long long)ld, (long long)K);
    if (((uintptr_t)x & (type_bytes(type) - 1)) != 0) return mz::fail(MZ_ERR_ARG, "%s: misaligned elements", what);
    return MZ_OK;
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
        hipLaunchKernelGGL(k_quant8<T>, row_grid(rows), dim3(kQT), 0, (hipStream_t)stream, (const T *)x, ldx, rows, K, scale_bits,
                           codes, ldc, scales);
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
        hipLaunchKernelGGL(k_dequant8<T>, row_grid(rows), dim3(kQT), 0, (hipStream_t)stream, codes, ldc, scales, rows, K,
                           (T *)x, ldx);
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
        hipLaunchKernelGGL(k_act_save<T>, row_grid(rows), dim3(kQT), 0, (hipStream_t)stream, (const T *)y, ldy, rows, N,
                           activation, saved, mz_ckpt8_act_bytes(N, activation));
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
        hipLaunchKernelGGL(k_act_grad<T>, row_grid(rows), dim3(kQT), 0, (hipStream_t)stream, (const T *)dy, ldy, saved,
                           mz_ckpt8_act_bytes(N, activation), rows, N, activation, (T *)dz, ldz);
    });
    return mz::check_launch("k_act_grad");
}

}  // extern "C"
