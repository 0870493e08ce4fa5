// Scores of given actions under a policy head's logits (gfx950): log probability, entropy and the best alternatives of
// every row, and their gradient with respect to the logits.
//
//     m = max_j z_j,  S = sum_j e^(z_j - m),  U = sum_j e^(z_j - m) (z_j - m)
//     log p_j = (z_j - m) - log S,     entropy H = -sum_j p_j log p_j = log S - U / S
//     d log p_a / d z_j = [j = a] - p_j,     d H / d z_j = -p_j (log p_j + H)
// The differences z_j - m keep S and U exact in magnitude whatever the size of the logits; m and log S stay apart (two
// float32 values), as their sum would round the log probabilities of large logits.  A row without any finite or infinite
// value left (every logit -inf) has log p = -inf, H = 0 and no gradient.  NaN and +inf make the row's results NaN.
// Alternatives are ordered by (logit, lowest index first); NaN counts as the largest value, -0 equals 0.
#include "mz_elem.h"

namespace {

using namespace mze;

constexpr int kST = 256;
constexpr int kMaxTop = 32;

struct Sums {  // running maximum, sum of e^(z - m) and of e^(z - m) (z - m)
    float m, s, u;
};

__device__ __forceinline__ Sums none() { return {-INFINITY, 0.0f, 0.0f}; }

// The sums of two disjoint sets of logits relative to the larger maximum: with d = m_old - m_new <= 0,
// S' = S e^d and U' = e^d (U + d S).  An empty (or fully masked) side has m = -inf and S = 0.
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.s + b.s, a.u + b.u};  // nothing but masked logits, or NaN sums
    const float da = a.m == -INFINITY ? -INFINITY : a.m - m, db = b.m == -INFINITY ? -INFINITY : b.m - m;
    const float ea = expf(da), eb = expf(db);
    // 0 * -inf would be NaN: an empty side adds nothing
    const float ua = a.s == 0.0f ? 0.0f : ea * (a.u + fmaxf(da, -1e30f) * a.s);
    const float ub = b.s == 0.0f ? 0.0f : eb * (b.u + fmaxf(db, -1e30f) * b.s);
    return {m, (a.s == 0.0f ? 0.0f : a.s * ea) + (b.s == 0.0f ? 0.0f : b.s * eb), ua + ub};
}

__device__ __forceinline__ Sums one(float z) {
    if (z != z) return {-INFINITY, z, z};
    if (z == -INFINITY) return none();
    if (z == INFINITY) return {z, NAN, NAN};
    return {z, 1.0f, 0.0f};
}

// Order of the alternatives as one unsigned 64-bit key: the larger key comes first.
__device__ __forceinline__ unsigned long long order_key(float z, unsigned j) {
    z = z + 0.0f;  // -0 -> 0
    unsigned b = z != z ? 0x7FC00000u : __float_as_uint(z);
    b ^= (b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u;
    return ((unsigned long long)b << 32) | (unsigned)~j;
}

__device__ __forceinline__ float key_value(unsigned long long k) {
    unsigned b = (unsigned)(k >> 32);
    b ^= (b & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu;
    return __uint_as_float(b);
}

// One workgroup per row; the alternatives are found one after the other, each in a pass over the row.
template <class T>
__global__ void __launch_bounds__(kST)
k_scores(const T *__restrict__ logits, int64_t ld, const int64_t *__restrict__ actions, int64_t rows, int V, int top,
         float *__restrict__ log_prob, float *__restrict__ entropy, float *__restrict__ stats,
         int64_t *__restrict__ top_actions, float *__restrict__ top_log_probs) {
    __shared__ Sums part[kST];
    __shared__ unsigned long long keys[kST];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *z = logits + row * ld;
        Sums acc = none();
        for (int j = threadIdx.x; j < V; j += kST) acc = join(acc, one((float)z[j]));
        __syncthreads();
        part[threadIdx.x] = acc;
        __syncthreads();
        for (int k = kST / 2; k > 0; k >>= 1) {
            if ((int)threadIdx.x < k) part[threadIdx.x] = join(part[threadIdx.x], part[threadIdx.x + k]);
            __syncthreads();
        }
        acc = part[0];
        const bool empty = acc.m == -INFINITY && acc.s == 0.0f;
        const float log_s = logf(acc.s);
        if (threadIdx.x == 0) {
            stats[2 * row] = empty ? -INFINITY : acc.m;
            stats[2 * row + 1] = empty ? 0.0f : log_s;
            entropy[row] = empty ? 0.0f : log_s - acc.u / acc.s;
            if (actions) {
                const int64_t a = actions[row];
                float lp = 0.0f;
                if (a >= V) lp = NAN;
                else if (a >= 0) lp = empty ? -INFINITY : ((float)z[a] - acc.m) - log_s;
                log_prob[row] = lp;
            }
        }
        unsigned long long last = ~0ull;
        for (int i = 0; i < top; ++i) {
            unsigned long long best = 0;
            for (int j = threadIdx.x; j < V; j += kST) {
                const unsigned long long key = order_key((float)z[j], (unsigned)j);
                if (key < last && key > best) best = key;
            }
            keys[threadIdx.x] = best;
            __syncthreads();
            for (int k = kST / 2; k > 0; k >>= 1) {
                if ((int)threadIdx.x < k && keys[threadIdx.x + k] > keys[threadIdx.x]) keys[threadIdx.x] = keys[threadIdx.x + k];
                __syncthreads();
            }
            last = keys[0];
            if (threadIdx.x == 0) {
                top_actions[row * top + i] = (int64_t)(unsigned)~(unsigned)last;
                top_log_probs[row * top + i] = empty ? -INFINITY : (key_value(last) - acc.m) - log_s;
            }
            __syncthreads();
        }
    }
}

struct RowGrad {
    float m, log_s, h, g_lp, g_ent, g_sum;
    int64_t a;
    bool empty;
};

// The gradient of one logit without the [j = alternative] terms of the top list.
__device__ __forceinline__ float grad_one(const RowGrad &r, float z, int64_t j) {
    if (r.empty) return 0.0f;
    const float lp = (z - r.m) - r.log_s;
    const float p = expf(lp);
    // p (log p + H) is 0 in the limit of p = 0; NaN stays NaN
    const float ent = p == 0.0f ? 0.0f : p * (lp + r.h);
    return (j == r.a ? r.g_lp : 0.0f) - p * r.g_sum - r.g_ent * ent;
}

__device__ __forceinline__ RowGrad row_grad(const int64_t *actions, int64_t row, int V, int top, const float *stats,
                                            const float *entropy, const float *g_lp, const float *g_ent, const float *g_top) {
    RowGrad r;
    r.m = stats[2 * row], r.log_s = stats[2 * row + 1], r.h = entropy[row];
    r.empty = r.m == -INFINITY && r.log_s == 0.0f;
    r.a = actions ? actions[row] : -1;
    r.g_lp = g_lp && r.a >= 0 ? g_lp[row] : 0.0f;
    if (r.a >= V) r.g_lp *= NAN;  // an action that does not exist: its score was NaN
    r.g_ent = g_ent ? g_ent[row] : 0.0f;
    r.g_sum = r.g_lp;
    if (g_top)
        for (int i = 0; i < top; ++i) r.g_sum += g_top[row * top + i];
    return r;
}

template <class T>
__global__ void __launch_bounds__(kST)
k_scores_grad(const T *__restrict__ logits, int64_t ld, const int64_t *__restrict__ actions, int64_t rows, int V, int top,
              const float *__restrict__ stats, const float *__restrict__ entropy, const int64_t *__restrict__ top_actions,
              const float *__restrict__ g_lp, const float *__restrict__ g_ent, const float *__restrict__ g_top,
              T *__restrict__ grad, int64_t ldg) {
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const RowGrad r = row_grad(actions, row, V, top, stats, entropy, g_lp, g_ent, g_top);
        for (int j = threadIdx.x; j < V; j += kST) {
            float g = grad_one(r, (float)logits[row * ld + j], j);
            if (g_top && !r.empty)
                for (int i = 0; i < top; ++i)
                    if (top_actions[row * top + i] == j) g += g_top[row * top + i];
            grad[row * ldg + j] = (T)g;
        }
    }
}

dim3 row_grid(int64_t rows) { return dim3((unsigned)(rows < (1 << 20) ? rows : (1 << 20))); }

int check_logits(const char *what, const void *p, int32_t type, int64_t ld, int64_t T, int32_t V, int32_t top) {
    if (!type_ok(type)) return mz::fail(MZ_ERR_ARG, "%s: unknown element type %d", what, type);
    if (T < 0 || T > 0x7FFFFFFF || V <= 0) return mz::fail(MZ_ERR_ARG, "%s: bad dimensions T=%lld V=%d", what, (long long)T, V);
    if (top < 0 || top > kMaxTop || top > V)
        return mz::fail(MZ_ERR_ARG, "%s: top=%d must lie in 0..%d and not exceed V=%d", what, top, kMaxTop, V);
    if (ld < V) return mz::fail(MZ_ERR_ARG, "%s: row stride %lld below V=%d", what, (long long)ld, V);
    if (T > 0 && !p) return mz::fail(MZ_ERR_ARG, "%s: NULL argument", what);
    if (((uintptr_t)p & (type_bytes(type) - 1)) != 0) return mz::fail(MZ_ERR_ARG, "%s: misaligned elements", what);
    return MZ_OK;
}

}  // namespace

extern "C" {

int64_t mz_policy_scores_workspace(int32_t type, int64_t T, int32_t V, int32_t top) {
    (void)type, (void)T, (void)V, (void)top;
    return 0;
}

int mz_policy_scores(const void *logits, int32_t type, int64_t ld, const int64_t *actions, int64_t T, int32_t V, int32_t top,
                     float *log_prob, float *entropy, float *stats, int64_t *top_actions, float *top_log_probs,
                     void *workspace, int64_t workspace_bytes, void *stream) {
    MZ_TRY(check_logits("mz_policy_scores", logits, type, ld, T, V, top));
    if (T == 0) return MZ_OK;
    if (!entropy || !stats || (actions && !log_prob) || (top > 0 && (!top_actions || !top_log_probs)))
        return mz::fail(MZ_ERR_ARG, "mz_policy_scores: NULL argument");
    const int64_t need = mz_policy_scores_workspace(type, T, V, top);
    if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0))
        return mz::fail(MZ_ERR_ARG, "mz_policy_scores: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
                        (long long)workspace_bytes);
    with_type(type, [&](auto t) {
        using E = decltype(t);
        hipLaunchKernelGGL(k_scores<E>, row_grid(T), dim3(kST), 0, (hipStream_t)stream, (const E *)logits, ld, actions, T, V, top,
                           log_prob, entropy, stats, top_actions, top_log_probs);
    });
    return mz::check_launch("k_scores");
}

int mz_policy_scores_backward(const void *logits, int32_t type, int64_t ld, const int64_t *actions, int64_t T, int32_t V,
                              int32_t top, const float *stats, const float *entropy, const int64_t *top_actions,
                              const float *g_log_prob, const float *g_entropy, const float *g_top, void *grad, int64_t ld_grad,
                              void *stream) {
    MZ_TRY(check_logits("mz_policy_scores_backward", logits, type, ld, T, V, top));
    MZ_TRY(check_logits("mz_policy_scores_backward", grad, type, ld_grad, T, V, top));
    if (T == 0) return MZ_OK;
    if (!stats || !entropy || (g_top && top > 0 && !top_actions) || (g_log_prob && !actions))
        return mz::fail(MZ_ERR_ARG, "mz_policy_scores_backward: NULL argument");
    if (top == 0) g_top = nullptr;
    with_type(type, [&](auto t) {
        using E = decltype(t);
        hipLaunchKernelGGL(k_scores_grad<E>, row_grid(T), dim3(kST), 0, (hipStream_t)stream, (const E *)logits, ld, actions, T, V,
                           top, stats, entropy, top_actions, g_log_prob, g_entropy, g_top, (E *)grad, ld_grad);
    });
    return mz::check_launch("k_scores_grad");
}

}  // extern "C"
