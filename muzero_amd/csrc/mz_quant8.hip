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
// THREADS threads per row (up to 64: several rows per workgroup).  The first HELD packs of a thread stay in registers between the
// maximum and the codes; the rest of a longer row is read again, from cache.  Bound by the memory: 1536 x 18432 float32,
// 142 MB with the codes, 28 us, 5.0 TB/s.
template <class T, int THREADS, int HELD, bool WHOLE>
__global__ void __launch_bounds__(THREADS < kQT ? kQT : THREADS)
k_quant8(const T *__restrict__ x, int64_t ldx, int64_t rows, int K, int scale_bits, int8_t *__restrict__ codes, int64_t ldc,
         float *__restrict__ scales) {
    constexpr int n = Pack<T>::n, per = THREADS < kQT ? kQT / THREADS : 1;
    __shared__ unsigned part[THREADS < 64 ? 1 : THREADS / 64];
    const int t = threadIdx.x % THREADS, packs = (int)(ldc / n);
    for (int64_t row0 = (int64_t)blockIdx.x * per; row0 < rows; row0 += (int64_t)gridDim.x * per) {
        const int64_t row = row0 + threadIdx.x / THREADS;
        if (THREADS <= 64 && row >= rows) break;
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
        for (int o = THREADS < 64 ? THREADS / 2 : 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o));
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

// The kernels below go through a matrix without crossing rows: a team of LANES lanes takes a piece of a row, kHold packs
// of columns per lane, all of its loads in flight together.  Narrow rows have 8 lanes, long ones several pieces (tanh
// derivative of 10^6 x 8 float32, 8 lanes / a wave per row: 51 / 394 us; of 64 x 131072, pieces / a wave per row: 14 / 414).
constexpr int kHold = 4;

struct Pieces {
    int lanes;
    int64_t per_row;
    dim3 grid;
};

Pieces pieces_of(int64_t rows, int64_t packs) {
    Pieces p;
    p.lanes = packs <= 8 * kHold ? 8 : 64;
    p.per_row = (packs + p.lanes * kHold - 1) / (p.lanes * kHold);
    const int64_t teams = kQT / p.lanes, groups = (rows * p.per_row + teams - 1) / teams;
    p.grid = dim3((unsigned)(groups < (1 << 20) ? groups : (1 << 20)));
    return p;
}

// f(row, this lane's first pack; the others are LANES apart) for every piece
template <int LANES, class F>
__device__ __forceinline__ void each_piece(int64_t rows, int64_t per_row, F &&f) {
    constexpr int teams = kQT / LANES;
    for (int64_t job = (int64_t)blockIdx.x * teams + threadIdx.x / LANES; job < rows * per_row; job += (int64_t)gridDim.x * teams) {
        const int64_t row = per_row == 1 ? job : job / per_row;
        f(row, (int)(job - row * per_row) * LANES * kHold + threadIdx.x % LANES);
    }
}

// Bound by the memory: 1536 x 18432 to float32, 113 MB from 28 MB of codes in cache, 22 us.
template <class T, int LANES, bool WHOLE, bool PAST>
__global__ void __launch_bounds__(kQT)
k_dequant8(const int8_t *__restrict__ codes, int64_t ldc, const float *__restrict__ scales, int64_t rows, int64_t per_row, int K,
           T *__restrict__ x, int64_t ldx) {
    constexpr int n = Pack<T>::n;
    using word = std::conditional_t<n == 4, unsigned, uint2>;
    each_piece<LANES>(rows, per_row, [&](int64_t row, int at) {
        const float s = scales[row];
        word w[kHold];
#pragma unroll
        for (int h = 0; h < kHold; ++h)  // a row of codes is padded to whole packs; behind K the last one is read again
            w[h] = *(const word *)(codes + row * ldc + min(at + h * LANES, (K - 1) / n) * n);
#pragma unroll
        for (int h = 0; h < kHold; ++h) {
            const int j = (at + h * LANES) * n;
            const int8_t *q = (const int8_t *)&w[h];
            Pack<T> p;
#pragma unroll
            for (int e = 0; e < n; ++e) p.v[e] = (T)((float)q[e] * s);
            if (j < K) store_pack<T, WHOLE, PAST>(x + row * ldx, j, K, p);
        }
    });
}

// Eight consecutive values of a row, zeros behind its end.  EIGHTS: N is a multiple of 8, the caller keeps j below it.
template <class T, bool WHOLE, bool EIGHTS>
__device__ __forceinline__ void load8(const T *row, int j, int N, float (&v)[8]) {
    constexpr int n = Pack<T>::n;
#pragma unroll
    for (int h = 0; h < 8 / n; ++h) {
        const Pack<T> p = WHOLE && EIGHTS ? *(const Pack<T> *)(row + j + h * n) : load_pack<T, WHOLE>(row, j + h * n, N);
#pragma unroll
        for (int e = 0; e < n; ++e) v[h * n + e] = (float)p.v[e];
    }
}

// Eight consecutive bytes of a row of N; EIGHTS: rows start on multiples of 8 and have whole ones.
template <bool EIGHTS>
__device__ __forceinline__ uint64_t load_bytes(const uint8_t *row, int j, int N) {
    if (EIGHTS) return *(const uint64_t *)(row + j);
    uint64_t v = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (j + e < N) v |= (uint64_t)row[j + e] << 8 * e;
    return v;
}

// What the backward pass needs of y = act(z): relu one bit, [not y <= 0]; tanh and sigmoid a code of 8 bits on a fixed
// scale, -128 for a NaN.  A lane takes 8 values at a time: a byte of bits, or 8 codes.  Bound by the memory: 65536 x 1000
// float32 relu 40 us, 6.7 TB/s, tanh 59 us.
template <class T, int LANES, bool WHOLE, bool EIGHTS>
__global__ void __launch_bounds__(kQT)
k_act_save(const T *__restrict__ y, int64_t ldy, int64_t rows, int64_t per_row, int N, int act, uint8_t *__restrict__ saved,
           int64_t lds) {
    each_piece<LANES>(rows, per_row, [&](int64_t row, int at) {
        float v[kHold][8];
#pragma unroll
        for (int h = 0; h < kHold; ++h)  // behind the row the last values are read again: no branch between the loads
            load8<T, WHOLE, EIGHTS>(y + row * ldy, min((at + h * LANES) * 8, EIGHTS ? N - 8 : N), N, v[h]);
#pragma unroll
        for (int h = 0; h < kHold; ++h) {
            const int j = (at + h * LANES) * 8;
            if (j >= N) continue;
            uint8_t *out = saved + row * lds;
            if (act == MZ_ACT_RELU) {
                unsigned bits = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) bits |= (unsigned)(j + e < N && !(v[h][e] <= 0.0f)) << e;
                out[j >> 3] = (uint8_t)bits;
                continue;
            }
            uint64_t word = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = v[h][e], c = rintf(act == MZ_ACT_TANH ? x * 127.0f : x * 254.0f - 127.0f);
                const unsigned code = x == x ? (unsigned)(int)fminf(fmaxf(c, -127.0f), 127.0f) & 0xFFu : 0x80u;
                word |= (uint64_t)code << 8 * e;
            }
            if (EIGHTS) *(uint64_t *)(out + j) = word;
            else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (j + e < N) out[j + e] = (uint8_t)(word >> 8 * e);
        }
    });
}

// dz = dy act'(y): relu [y > 0]; tanh 1 - t^2 with t = q / 127; sigmoid s (1 - s) = (1 - t^2) / 4 with t = 2 s - 1.
// Bound by the memory: 65536 x 1000 float32 relu 102 us, 5.2 TB/s, tanh 109 us.
template <class T, int LANES, bool WHOLE, bool EIGHTS>
__global__ void __launch_bounds__(kQT)
k_act_grad(const T *dy, int64_t ldy, const uint8_t *__restrict__ saved, int64_t lds, int64_t rows, int64_t per_row, int N, int act,
           T *dz, int64_t ldz) {
    constexpr int n = Pack<T>::n;
    each_piece<LANES>(rows, per_row, [&](int64_t row, int at) {
        float v[kHold][8];
        uint64_t q[kHold];
#pragma unroll
        for (int h = 0; h < kHold; ++h) {
            const int j = min((at + h * LANES) * 8, EIGHTS ? N - 8 : N);
            load8<T, WHOLE, EIGHTS>(dy + row * ldy, j, N, v[h]);
            if (act == MZ_ACT_RELU) q[h] = saved[row * lds + min(j >> 3, (int)lds - 1)];
            else q[h] = load_bytes<EIGHTS>(saved + row * lds, j, N);
        }
#pragma unroll
        for (int h = 0; h < kHold; ++h) {
            const int j = (at + h * LANES) * 8;
            if (j >= N) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int code = (int8_t)(q[h] >> 8 * e);
                const float t = (float)code * (1.0f / 127.0f), slope = (1.0f - t * t) * (act == MZ_ACT_TANH ? 1.0f : 0.25f);
                if (act == MZ_ACT_RELU) v[h][e] = q[h] >> e & 1 ? v[h][e] : 0.0f;
                else v[h][e] *= code == -128 ? __uint_as_float(0x7FC00000u) : slope;
            }
#pragma unroll
            for (int k = 0; k < 8 / n; ++k) {
                Pack<T> p;
#pragma unroll
                for (int e = 0; e < n; ++e) p.v[e] = (T)v[h][k * n + e];
                store_pack<T, WHOLE>(dz + row * ldz, j + k * n, N, p);
            }
        }
    });
}

// Rows to where they belong, one wave each.
__global__ void __launch_bounds__(kQT)
k_scatter_rows(const float *__restrict__ x, int64_t ldx, const int32_t *__restrict__ rows, int64_t B, int D, float *__restrict__ y,
               int64_t ldy, int64_t y_rows) {
    for (int64_t r = (int64_t)blockIdx.x * (kQT / 64) + (threadIdx.x >> 6); r < B; r += (int64_t)gridDim.x * (kQT / 64)) {
        const int64_t to = rows[r];
        if (to < 0 || to >= y_rows) continue;
        for (int c = threadIdx.x & 63; c < D; c += 64) y[to * ldy + c] = x[r * ldx + c];
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
            // A quarter, half or whole wave per row up to 4 packs a lane, else a workgroup of 256 or 1024 threads, with as few
            // registers for packs as hold the row (1536 x 18432 float32: 1024 threads 26 us, 512 29 us, 256 37 us; 200000 x 168
            // bfloat16: 16 threads 30 us, 64 71 us).
            const int64_t packs = ldc / Pack<T>::n;
            if (packs <= 2 * 16) launch(k_quant8<T, 16, 2, W>, 16);
            else if (packs <= 2 * 32) launch(k_quant8<T, 32, 2, W>, 8);
            else if (packs <= 2 * 64) launch(k_quant8<T, 64, 2, W>, 4);
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
            const Pieces p = pieces_of(rows, (K + Pack<T>::n - 1) / Pack<T>::n);
            const auto launch = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, p.grid, dim3(kQT), 0, (hipStream_t)stream, codes, ldc, scales, rows, p.per_row, K, (T *)x, ldx);
            };
            with_flag(past_caches(rows * K * (int64_t)sizeof(T)), [&](auto past) {
                constexpr bool P = decltype(past)::value;
                p.lanes == 8 ? launch(k_dequant8<T, 8, W, P>) : launch(k_dequant8<T, 64, W, P>);
            });
        });
    });
    return mz::check_launch("k_dequant8");
}

int mz_scatter_rows(const float *x, int64_t ldx, const int32_t *rows, int32_t B, int32_t D, float *y, int64_t ldy, int64_t y_rows,
                    void *stream) {
    MZ_TRY(check_rows("mz_scatter_rows", x, MZ_TYPE_F32, ldx, B, D));
    MZ_TRY(check_rows("mz_scatter_rows", y, MZ_TYPE_F32, ldy, B, D));
    if (B == 0) return MZ_OK;
    if (!rows) return mz::fail(MZ_ERR_ARG, "mz_scatter_rows: NULL argument");
    hipLaunchKernelGGL(k_scatter_rows, row_grid(B, kQT / 64), dim3(kQT), 0, (hipStream_t)stream, x, ldx, rows, (int64_t)B, D, y, ldy,
                       y_rows);
    return mz::check_launch("k_scatter_rows");
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
            constexpr bool W = decltype(whole)::value;
            const int64_t lds = mz_ckpt8_act_bytes(N, activation);
            const Pieces p = pieces_of(rows, (N + 7) / 8);
            const auto launch = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, p.grid, dim3(kQT), 0, (hipStream_t)stream, (const T *)y, ldy, rows, p.per_row, N, activation, saved, lds);
            };
            with_flag(N % 8 == 0 && (uintptr_t)saved % 8 == 0, [&](auto eights) {
                constexpr bool E = decltype(eights)::value;
                p.lanes == 8 ? launch(k_act_save<T, 8, W, E>) : launch(k_act_save<T, 64, W, E>);
            });
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
            constexpr bool W = decltype(whole)::value;
            const int64_t lds = mz_ckpt8_act_bytes(N, activation);
            const Pieces p = pieces_of(rows, (N + 7) / 8);
            const auto launch = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, p.grid, dim3(kQT), 0, (hipStream_t)stream, (const T *)dy, ldy, saved, lds, rows, p.per_row, N, activation,
                                   (T *)dz, ldz);
            };
            with_flag(N % 8 == 0 && (uintptr_t)saved % 8 == 0, [&](auto eights) {
                constexpr bool E = decltype(eights)::value;
                p.lanes == 8 ? launch(k_act_grad<T, 8, W, E>) : launch(k_act_grad<T, 64, W, E>);
            });
        });
    });
    return mz::check_launch("k_act_grad");
}

}  // extern "C"
