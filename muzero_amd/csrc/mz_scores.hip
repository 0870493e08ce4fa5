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
#include <algorithm>

#include "mz_elem.h"

namespace {

using namespace mze;

constexpr int kMaxTop = 32;
constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLowest = -3.402823466e38f;

// e^d for d <= 0 (or NaN): the exponent is rounded once, so the result is off by |d| u and one unit.
__device__ __forceinline__ float exp_le0(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// Running maximum and sums of a set of logits.  m starts at the lowest finite value, not at -inf: z - m is then -inf for
// a masked logit (e = 0) and never inf - inf.  s == 0 says that nothing but masked logits was met, since the largest
// live one contributes e^0 = 1.
struct Sums {
    float m, s, u;
};

__device__ __forceinline__ Sums none() { return {kLowest, 0.0f, 0.0f}; }

// u's share of one logit: e (z - m), with 0 * -inf read as 0 (a NaN is in s already)
__device__ __forceinline__ float share(float e, float d) { return e * fmaxf(d, -1e30f); }

// The sums of two disjoint sets relative to the larger maximum: with d = m_old - m_new <= 0,
// S' = S e^d and U' = e^d (U + d S).
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    const float m = fmaxf(a.m, b.m), da = a.m - m, db = b.m - m;
    const float ea = exp_le0(da), eb = exp_le0(db);
    return {m, a.s * ea + b.s * eb, ea * a.u + share(ea, da) * a.s + eb * b.u + share(eb, db) * b.s};
}

struct Row {  // what follows from the sums of a whole row
    float m, log_s, h;
    bool empty, loud;  // nothing but masked logits; a NaN or +inf among them
};

__device__ __forceinline__ Row row_of(const Sums &a) {
    Row r;
    r.empty = a.s == 0.0f;
    r.loud = a.s != a.s;
    r.m = r.empty ? -INFINITY : a.m;
    r.log_s = r.empty ? 0.0f : logf(a.s);
    r.h = r.empty ? 0.0f : r.log_s - a.u / a.s;
    return r;
}

__device__ __forceinline__ float log_p(const Row &r, float z) { return r.empty ? -INFINITY : (z - r.m) - r.log_s; }

// Order of the alternatives as one unsigned 64-bit key (value, then lowest index): the larger key comes first, 0 is none.
__device__ __forceinline__ unsigned order_bits(float z) {
    z = z + 0.0f;  // -0 -> 0
    const unsigned b = z != z ? 0x7FC00000u : __float_as_uint(z);
    return b ^ ((b & 0x80000000u) ? 0xFFFFFFFFu : 0x80000000u);
}

using Key = unsigned long long;

__device__ __forceinline__ Key order_key(float z, int j) { return ((Key)order_bits(z) << 32) | (unsigned)~j; }

__device__ __forceinline__ float bits_value(unsigned b) { return __uint_as_float(b ^ ((b & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu)); }
__device__ __forceinline__ float key_value(Key k) { return bits_value((unsigned)(k >> 32)); }
__device__ __forceinline__ int key_index(Key k) { return (int)~(unsigned)k; }

// Maximum over the 64 lanes (every lane gets it), by lane moves inside the vector unit.
__device__ __forceinline__ unsigned wave_max(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true));   // row_shr:1
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true));   // row_shr:2
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true));   // row_shr:4
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true));   // row_shr:8
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));  // row_bcast:15
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));  // row_bcast:31
    return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ Key wave_max(Key k) {
    const unsigned hi = wave_max((unsigned)(k >> 32));
    const unsigned lo = wave_max((unsigned)(k >> 32) == hi ? (unsigned)k : 0u);
    return ((Key)hi << 32) | lo;
}

__device__ __forceinline__ Key lane_key(Key k, int lane) {
    return ((Key)(unsigned)__builtin_amdgcn_readlane((int)(k >> 32), lane) << 32) | (unsigned)__builtin_amdgcn_readlane((int)k, lane);
}

struct Out {  // the result arrays of a call
    const int64_t *actions;
    float *log_prob, *entropy, *stats;
    int64_t *top_actions;
    float *top_log_probs;
    int V, top;

    template <class T>
    __device__ void row(int64_t row, const Row &r, const T *z) const {
        entropy[row] = r.h;
        if (stats) stats[3 * row] = r.m, stats[3 * row + 1] = r.log_s, stats[3 * row + 2] = r.h;
        if (!actions) return;
        const int64_t a = actions[row];
        log_prob[row] = a < 0 ? 0.0f : a >= V ? NAN : log_p(r, (float)z[a]);
    }
    __device__ void alternative(int64_t row, int i, const Row &r, Key k) const {
        top_actions[row * top + i] = key_index(k);
        top_log_probs[row * top + i] = log_p(r, key_value(k));
    }
};

// ---------------------------------------------------------------- rows of up to 64 logits
// LANES lanes per row, one logit each, 256 / LANES rows per workgroup.  An alternative costs log2(LANES) exchanges, against
// a list built in shared memory for longer rows.  Bound by the launch: 1536 x 7 (bf16, 3 alternatives) is one wave's chain.
template <class T, int LANES>
__global__ void __launch_bounds__(256)
k_scores_small(const T *__restrict__ logits, int64_t ld, int64_t rows, Out out) {
    const int lane = threadIdx.x % LANES, V = out.V;
    for (int64_t row0 = (int64_t)blockIdx.x * (256 / LANES); row0 < rows; row0 += (int64_t)gridDim.x * (256 / LANES)) {
        const int64_t row = row0 + threadIdx.x / LANES;
        const bool live = row < rows;
        const T *z = logits + (live ? row : 0) * ld;
        const float v = lane < V ? (float)z[lane] : -INFINITY;
        Sums acc = {fmaxf(v, kLowest), 0.0f, 0.0f};
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) acc.m = fmaxf(acc.m, __shfl_xor(acc.m, o));
        const float d = v - acc.m;
        acc.s = exp_le0(d);
        acc.u = share(acc.s, d);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
            acc.s += __shfl_xor(acc.s, o);
            acc.u += __shfl_xor(acc.u, o);
        }
        const Row r = row_of(acc);
        if (live && lane == 0) out.row(row, r, z);
        Key mine = lane < V ? order_key(v, lane) : 0;
        for (int i = 0; i < out.top; ++i) {
            Key best = mine;
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) {
                const Key k = __shfl_xor(best, o);
                if (k > best) best = k;
            }
            if (mine == best) mine = 0;  // keys are unique
            if (live && lane == 0) out.alternative(row, i, r, best);
        }
    }
}

// The logits [lo, hi) of a row as 16-byte packs that lie on 16-byte addresses, whatever the row's own alignment: pack i
// holds the logits first + i n .. + n - 1.  Packs whole_lo .. whole_hi - 1 are owned whole; the first and the last pack may
// only be owned in part.
template <class T>
struct Span {
    static constexpr int n = Pack<T>::n;
    const T *z;
    int lo, hi, first, packs, whole_lo, whole_hi;

    __device__ Span(const T *row, int lo_, int hi_) : z(row), lo(lo_), hi(hi_) {
        first = lo - (int)(((uintptr_t)(row + lo) & 15) / sizeof(T));
        packs = (hi - first + n - 1) / n;
        whole_lo = first < lo ? 1 : 0;
        whole_hi = first + packs * n > hi ? packs - 1 : packs;
    }
    __device__ __forceinline__ int at(int i) const { return first + i * n; }
    __device__ __forceinline__ bool owns(int j) const { return j >= lo && j < hi; }
    __device__ __forceinline__ Pack<T> whole(int i) const { return *(const Pack<T> *)(z + at(i)); }
    __device__ __forceinline__ Pack<T> part(int i) const {  // -inf where the pack is not owned
        Pack<T> p;
#pragma unroll
        for (int e = 0; e < n; ++e) p.v[e] = owns(at(i) + e) ? z[at(i) + e] : (T)-INFINITY;
        return p;
    }
    __device__ __forceinline__ Pack<T> load(int i) const { return i >= whole_lo && i < whole_hi ? whole(i) : part(i); }
    // f(pack) for packs t, t + THREADS, ...: four whole ones in flight, without a branch between the loads
    template <int THREADS, class F>
    __device__ __forceinline__ void each(int t, F &&f) const {
        int i = t;
        if (i < whole_lo && i < packs) {
            f(part(i), i);
            i += THREADS;
        }
        for (; i + 3 * THREADS < whole_hi; i += 4 * THREADS) {
            Pack<T> p[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) p[q] = whole(i + q * THREADS);
#pragma unroll
            for (int q = 0; q < 4; ++q) f(p[q], i + q * THREADS);
        }
        for (; i < whole_hi; i += THREADS) f(whole(i), i);
        if (i < packs) f(part(i), i);
    }
};

// ---------------------------------------------------------------- rows of up to about 4096 logits: one wave per row
// The row stays in registers (P packs a lane).  The alternatives: every lane's largest logit gives a lower bound of the
// `top`-th largest one (as many lanes reach it); the few logits that reach the bound are collected and ranked by counting.
// Rows with more than 64 of those (equal values, everything masked, a NaN) find one alternative per pass.
// No barrier and no second read; bound by the bytes with many rows and by the load's latency with few.  us for 20000 rows
// (fp16, without / with 5 alternatives), and in brackets for a workgroup per row: 1000 logits 12.7 / 18.9, 2048 21.6 / 32.6
// (58.9 / 109), 3000 34 / 53 (68 / 119), 4000 68 / 113 (72 / 122); 256 rows of 2048 3.9 / 5.6 (4.3 / 6.8), of 4000 4.7 / 6.9
// (4.6 / 7.2).  2048 half-precision logits without alternatives are 3.8 TB/s, against
// 5.1 to 5.6 of a kernel that only reads: from 4 packs a lane on, the packs' registers leave 3 waves per SIMD, 1 or 2 for 8.
template <class T, int P>
__global__ void __launch_bounds__(256)
k_scores_wave(const T *__restrict__ logits, int64_t ld, int64_t rows, Out out) {
    constexpr int n = Span<T>::n;
    __shared__ Key cand[4][64];
    const int lane = threadIdx.x & 63, top = out.top;
    Key *list = cand[threadIdx.x >> 6];
    for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (int64_t)gridDim.x * 4) {
        const T *z = logits + row * ld;
        const Span<T> span(z, 0, out.V);
        Pack<T> p[P];
#pragma unroll
        for (int q = 0; q < P; ++q)  // no branch between the loads: other lanes read a pack that exists, and correct it
            p[q] = span.whole(min(max(lane + 64 * q, span.whole_lo), span.whole_hi - 1));
        float m = -INFINITY;
#pragma unroll
        for (int q = 0; q < P; ++q) {
            const int i = lane + 64 * q;
            if (i >= span.packs) {
#pragma unroll
                for (int e = 0; e < n; ++e) p[q].v[e] = (T)-INFINITY;
            } else if (i < span.whole_lo || i >= span.whole_hi) {
                p[q] = span.part(i);
            }
#pragma unroll
            for (int e = 0; e < n; ++e) m = fmaxf(m, (float)p[q].v[e]);
        }
        const unsigned mine = order_bits(m);
        Sums acc = {fmaxf(bits_value(wave_max(mine)), kLowest), 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < P; ++q)
#pragma unroll
            for (int e = 0; e < n; ++e) {
                const float d = (float)p[q].v[e] - acc.m, x = exp_le0(d);
                acc.s += x;
                acc.u += share(x, d);
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            acc.s += __shfl_xor(acc.s, o);
            acc.u += __shfl_xor(acc.u, o);
        }
        const Row r = row_of(acc);
        if (lane == 0) out.row(row, r, z);
        if (top == 0) continue;
        unsigned bound = 0;
        for (int bit = 31; bit >= 16; --bit) {
            const unsigned probe = bound | (1u << bit);
            if (__popcll(__ballot(mine >= probe)) >= top) bound = probe;
        }
        int count = 65;
        if (!r.loud && bound > order_bits(-INFINITY)) {
            const float t = bits_value(bound);
            count = 0;
            __builtin_amdgcn_wave_barrier();  // the list is the wave's own: LDS keeps a wave's order, the compiler has to as well
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int e = 0; e < n; ++e) {
                    const float x = (float)p[q].v[e];
                    const unsigned long long hits = __ballot(x >= t);
                    if (hits) {
                        const int at = count + __builtin_amdgcn_mbcnt_hi((unsigned)(hits >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)hits, 0));
                        if (x >= t && at < 64) list[at] = order_key(x, span.at(lane + 64 * q) + e);
                        count += __popcll(hits);
                    }
                }
        }
        if (count <= 64) {
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            const Key k = lane < count ? list[lane] : 0;
            int rank = 0;
            for (int o = 0; o < count; ++o) rank += lane_key(k, o) > k;
            if (rank < top && k != 0) out.alternative(row, rank, r, k);
            continue;
        }
        Key last = ~0ull;
        for (int a = 0; a < top; ++a) {
            Key best = 0;
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
                for (int e = 0; e < n; ++e) {
                    const int j = span.at(lane + 64 * q) + e;
                    const Key k = span.owns(j) ? order_key((float)p[q].v[e], j) : 0;
                    if (k < last && k > best) best = k;
                }
            last = wave_max(best);
            if (lane == 0) out.alternative(row, a, r, last);
        }
    }
}

// ---------------------------------------------------------------- long rows: a workgroup streams a row, or a part of it
// One pass with a running maximum per thread; bound by the bytes: 3001 x 50001 float32 with 8 alternatives 117 us, 5.1 TB/s,
// 4096 x 32768 bf16 without any 48 us, 5.6 TB/s (an instantiation of its own: the alternatives' registers halve the waves at
// work).  The alternatives read a few packs again, those of the threads whose largest logit reaches the bound.
constexpr int kCand = 1024;       // candidates for the alternatives that a workgroup can hold
constexpr int kMaxParts = 64;     // parts of one row (one lane of the joining wave each)

template <class T>
__device__ __forceinline__ void add(Sums &a, const Pack<T> &p) {
    constexpr int n = Pack<T>::n;
    float v[n];
#pragma unroll
    for (int e = 0; e < n; ++e) v[e] = (float)p.v[e];
    float m = v[0];
#pragma unroll
    for (int e = 1; e < n; ++e) m = fmaxf(m, v[e]);
    if (m > a.m) {
        const float d = a.m - m, x = exp_le0(d);
        a.u = x * a.u + share(x, d) * a.s;
        a.s *= x;
        a.m = m;
    }
#pragma unroll
    for (int e = 0; e < n; ++e) {
        const float d = v[e] - a.m, x = exp_le0(d);
        a.s += x;
        a.u += share(x, d);
    }
}

template <int LT>
struct Shared {
    Sums part[LT / 64];
    Key cand[kCand];
    unsigned best[LT];
    Key thread_key[LT];
    int owner[LT];
    Key found[kMaxTop];
    Key threshold;
    int count, owners;
};

// Largest value t (its low 16 order bits dropped) that at least `top` of 64 groups of threads reach with their largest
// logit: at least `top` logits are >= t, so no smaller one is an alternative.  Every wave finds it by itself.
template <int LT>
__device__ __forceinline__ float value_threshold(const Shared<LT> &sh, int top) {
    const int lane = threadIdx.x & 63;
    unsigned b = 0, t = 0;
#pragma unroll
    for (int w = 0; w < LT / 64; ++w) b = max(b, sh.best[w * 64 + lane]);
    for (int bit = 31; bit >= 16; --bit) {
        const unsigned probe = t | (1u << bit);
        if (__popcll(__ballot(b >= probe)) >= top) t = probe;
    }
    return t <= order_bits(-INFINITY) ? -INFINITY : bits_value(t);
}

// The candidates in sh.cand, ranked by counting the larger ones: the `top` first go to sh.found in order.
template <int LT>
__device__ __forceinline__ void rank_candidates(Shared<LT> &sh, int count, int top) {
    if (count <= 64) {  // in the registers of one wave
        if (threadIdx.x < 64) {
            const Key k = (int)threadIdx.x < count ? sh.cand[threadIdx.x] : 0;
            int rank = 0;
            for (int o = 0; o < count; ++o) rank += lane_key(k, o) > k;
            if (rank < top && k != 0) sh.found[rank] = k;
        }
    } else {
        for (int c = threadIdx.x; c < count; c += LT) {
            const Key k = sh.cand[c];
            int rank = 0;
            for (int o = 0; o < count; ++o) rank += sh.cand[o] > k;
            if (rank < top) sh.found[rank] = k;
        }
    }
    __syncthreads();
}

// sh.found = the `top` first alternatives among the logits of `span` (at least `top` of them), which every thread has
// streamed in the order of add(): its own largest one is in sh.best.  `loud`: there is a NaN or an infinity.
//  1. candidates are the logits that reach value_threshold; only the packs of threads that reach it are read again, by
//     all threads together;
//  2. rows with too many equal values for that (all masked, all equal): the same with (value, index) keys;
//  3. whatever overflows that, too: one alternative per pass.
template <class T, int LT>
__device__ void find_alternatives(const Span<T> &span, Shared<LT> &sh, int top, bool loud) {
    constexpr int n = Span<T>::n;
    const int per_thread = (span.packs + LT - 1) / LT;
    // the logits of the threads with `mine` that are `wanted`; sh.count and sh.owners are 0 before
    const auto collect = [&](bool mine, auto &&wanted) {
        if (mine) sh.owner[atomicAdd(&sh.owners, 1)] = threadIdx.x;
        __syncthreads();
        const int items = sh.owners * per_thread;
        for (int q = threadIdx.x; q < items; q += LT) {
            const int o = q / per_thread, i = sh.owner[o] + (q - o * per_thread) * LT;
            if (i >= span.packs) continue;
            const Pack<T> p = span.load(i);
#pragma unroll
            for (int e = 0; e < n; ++e) {
                const int j = span.at(i) + e;
                const float z = (float)p.v[e];
                if (span.owns(j) && wanted(z, j)) {
                    const int c = atomicAdd(&sh.count, 1);
                    if (c < kCand) sh.cand[c] = order_key(z, j);
                }
            }
        }
        __syncthreads();
        return sh.count;
    };
    int count = kCand + 1;
    if (!loud) {
        const float t = value_threshold(sh, top);
        if (threadIdx.x == 0) sh.count = 0, sh.owners = 0;
        __syncthreads();
        count = collect(sh.best[threadIdx.x] >= order_bits(t), [&](float z, int) { return z >= t; });
        if (count > kCand) {
            Key mine = 0;
            span.template each<LT>(threadIdx.x, [&](const Pack<T> &p, int i) {
#pragma unroll
                for (int e = 0; e < n; ++e) {
                    const int j = span.at(i) + e;
                    const Key k = span.owns(j) ? order_key((float)p.v[e], j) : 0;
                    if (k > mine) mine = k;
                }
            });
            __syncthreads();  // everybody has read sh.count
            sh.thread_key[threadIdx.x] = mine;
            if (threadIdx.x == 0) sh.count = 0, sh.owners = 0, sh.threshold = 0;  // fewer owning threads than top: everything
            __syncthreads();
            int rank = 0;
            for (int o = 0; o < LT; ++o) rank += sh.thread_key[o] > mine;
            if (rank == top - 1 && mine != 0) sh.threshold = mine;
            __syncthreads();
            const Key t2 = sh.threshold;
            count = collect(mine >= t2 && mine != 0, [&](float z, int j) { return order_key(z, j) >= t2; });
        }
    }
    if (count <= kCand) {
        rank_candidates(sh, count, top);
        return;
    }
    Key last = ~0ull;
    for (int a = 0; a < top; ++a) {
        Key best = 0;
        span.template each<LT>(threadIdx.x, [&](const Pack<T> &p, int i) {
#pragma unroll
            for (int e = 0; e < n; ++e) {
                const int j = span.at(i) + e;
                const Key k = span.owns(j) ? order_key((float)p.v[e], j) : 0;
                if (k < last && k > best) best = k;
            }
        });
        best = wave_max(best);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.thread_key[threadIdx.x >> 6] = best;
        __syncthreads();
        last = sh.thread_key[0];
        for (int w = 1; w < LT / 64; ++w) last = max(last, sh.thread_key[w]);
        if (threadIdx.x == 0) sh.found[a] = last;
    }
    __syncthreads();
}

// Workgroup (row, part).  One part: the results.  Several: the part's sums and alternatives to the workspace.
template <class T, int LT, bool TOP>
__global__ void __launch_bounds__(LT)
k_scores_long(const T *__restrict__ logits, int64_t ld, int64_t rows, int parts, Out out, Sums *__restrict__ part_sums,
              Key *__restrict__ part_keys) {
    __shared__ Shared<LT> sh;
    const int top = TOP ? out.top : 0;
    for (int64_t job = blockIdx.x; job < rows * parts; job += gridDim.x) {
        const int64_t row = job / parts;
        const int part = (int)(job - row * parts);
        const T *z = logits + row * ld;
        const Span<T> span(z, (int)((int64_t)out.V * part / parts), (int)((int64_t)out.V * (part + 1) / parts));
        Sums acc = none();
        span.template each<LT>(threadIdx.x, [&](const Pack<T> &p, int) { add(acc, p); });
        __syncthreads();  // the last job's shared values have been read
        sh.best[threadIdx.x] = order_bits(acc.s == 0.0f ? -INFINITY : acc.m);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) acc = join(acc, {__shfl_xor(acc.m, o), __shfl_xor(acc.s, o), __shfl_xor(acc.u, o)});
        if ((threadIdx.x & 63) == 0) sh.part[threadIdx.x >> 6] = acc;
        __syncthreads();
        acc = sh.part[0];
        for (int w = 1; w < LT / 64; ++w) acc = join(acc, sh.part[w]);
        const Row r = row_of(acc);
        if constexpr (TOP) find_alternatives(span, sh, top, r.loud);
        if (parts == 1) {
            if (threadIdx.x == 0) out.row(row, r, z);
            if ((int)threadIdx.x < top) out.alternative(row, threadIdx.x, r, sh.found[threadIdx.x]);
        } else {
            if (threadIdx.x == 0) part_sums[job] = acc;
            if ((int)threadIdx.x < top) part_keys[job * top + threadIdx.x] = sh.found[threadIdx.x];
        }
    }
}

// One wave per row: joins the sums of its parts in a fixed order and merges their lists, one lane per part.  Bound by the
// latency of its steps: 16 lists of 5 3.7 us, 8 lists of 20 for 64 rows 7.1 us.
template <class T>
__global__ void __launch_bounds__(64)
k_scores_join(const T *__restrict__ logits, int64_t ld, int64_t rows, int parts, Out out, const Sums *__restrict__ part_sums,
              const Key *__restrict__ part_keys) {
    __shared__ Key lists[kMaxParts * kMaxTop], found[kMaxTop];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const int lane = threadIdx.x, top = out.top;
#pragma unroll 8
        for (int i = lane; i < parts * top; i += 64) lists[i] = part_keys[row * parts * top + i];
        Sums acc = lane < parts ? part_sums[row * parts + lane] : none();
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) acc = join(acc, {__shfl_xor(acc.m, o), __shfl_xor(acc.s, o), __shfl_xor(acc.u, o)});
        const Row r = row_of(acc);
        if (lane == 0) out.row(row, r, logits + row * ld);
        __syncthreads();
        int next = lane * top;
        const int end = lane < parts ? next + top : next;
        Key head = next < end ? lists[next] : 0;
        for (int i = 0; i < top; ++i) {
            const Key best = wave_max(head);
            if (lane == 0) found[i] = best;
            if (head == best) head = ++next < end ? lists[next] : 0;  // keys are unique: one lane moves on
        }
        __syncthreads();
        if (lane < top) out.alternative(row, lane, r, found[lane]);
        __syncthreads();
    }
}

// ---------------------------------------------------------------- gradient
struct RowGrad {
    float m, log_s, h, g_lp, g_ent, g_sum;
    int64_t a;
    bool empty;
};

// The gradient of one logit without the [j = alternative] terms of the top list.
__device__ __forceinline__ float grad_one(const RowGrad &r, float z, int j) {
    const float lp = (z - r.m) - r.log_s, p = exp_le0(lp);
    // p (log p + H) is 0 in the limit of p = 0
    const float ent = p == 0.0f ? 0.0f : p * (lp + r.h);
    const float g = (j == r.a ? r.g_lp : 0.0f) - p * r.g_sum - r.g_ent * ent;
    return r.empty ? 0.0f : g;
}

struct Grads {
    const int64_t *actions;
    const float *stats;
    const int64_t *top_actions;
    const float *g_lp, *g_ent, *g_top;
    int V, top;

    __device__ RowGrad row(int64_t row) const {
        RowGrad r;
        r.m = stats[3 * row], r.log_s = stats[3 * row + 1], r.h = stats[3 * row + 2];
        r.empty = r.m == -INFINITY && r.log_s == 0.0f;
        r.a = actions ? actions[row] : -1;
        r.g_lp = g_lp && r.a >= 0 ? g_lp[row] : 0.0f;
        if (g_lp && r.a >= V) r.g_lp = NAN;  // an action that does not exist: its score was NaN
        r.g_ent = g_ent ? g_ent[row] : 0.0f;
        r.g_sum = r.g_lp;
        if (g_top)
            for (int i = 0; i < top; ++i) r.g_sum += g_top[row * top + i];
        return r;
    }
};

// Rows of up to 64 logits, LANES lanes per row.
template <class T, int LANES>
__global__ void __launch_bounds__(256)
k_grad_small(const T *__restrict__ logits, int64_t ld, int64_t rows, Grads in, T *__restrict__ grad, int64_t ldg) {
    const int lane = threadIdx.x % LANES;
    const int64_t step = (int64_t)gridDim.x * (256 / LANES);
    for (int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; row < rows; row += step) {
        const RowGrad r = in.row(row);
        for (int j = lane; j < in.V; j += LANES) grad[row * ldg + j] = (T)grad_one(r, (float)logits[row * ld + j], j);
    }
}

// Longer rows in pieces of LANES lanes with kGradPacks packs each: a wave per piece while that covers a row, else a workgroup.
// From the last row to the first, as the forward pass left the last ones in cache (4096 x 32768 bf16, both passes: 170
// against 176 us), and past the caches on the way out (140).  Bound by the bytes: 20000 x 32768 fp16 5.5 TB/s.
constexpr int kGradPacks = 4;

template <class T, int LANES>
__global__ void __launch_bounds__(256)
k_grad_long(const T *__restrict__ logits, int64_t ld, int64_t rows, int pieces, Grads in, T *__restrict__ grad, int64_t ldg) {
    constexpr int n = Span<T>::n;
    constexpr int64_t kTeams = 256 / LANES;
    for (int64_t job = blockIdx.x * kTeams + threadIdx.x / LANES; job < rows * pieces; job += gridDim.x * kTeams) {
        const int64_t at = rows * pieces - 1 - job, row = at / pieces;
        const int piece = (int)(at - row * pieces);
        const Span<T> span(logits + row * ld, 0, in.V);
        T *out = grad + row * ldg;
        // packs of the logits' alignment: stores are whole when the gradient's row has the same one
        const bool whole = ((uintptr_t)(out + span.first) & 15) == 0;
        const RowGrad r = in.row(row);
        const int i0 = piece * kGradPacks * LANES + threadIdx.x % LANES;
        const auto put = [&](const Pack<T> &z, int i) {
            const int j = span.at(i);
            Pack<T> p;
#pragma unroll
            for (int e = 0; e < n; ++e) p.v[e] = (T)grad_one(r, (float)z.v[e], j + e);
            if (whole && i >= span.whole_lo && i < span.whole_hi) {
                store_past((Pack<T> *)(out + j), p);  // of any size: 67 MB 55 against 58 us, and not slower with a reader
            } else {
#pragma unroll
                for (int e = 0; e < n; ++e)
                    if (span.owns(j + e)) out[j + e] = p.v[e];
            }
        };
        if (i0 >= span.whole_lo && i0 + (kGradPacks - 1) * LANES < span.whole_hi) {  // all loads in flight
            Pack<T> z[kGradPacks];
#pragma unroll
            for (int q = 0; q < kGradPacks; ++q) z[q] = span.whole(i0 + q * LANES);
#pragma unroll
            for (int q = 0; q < kGradPacks; ++q) put(z[q], i0 + q * LANES);
        } else {
            for (int q = 0; q < kGradPacks && i0 + q * LANES < span.packs; ++q) put(span.load(i0 + q * LANES), i0 + q * LANES);
        }
    }
}

// The logits that are alternatives, once more and with all their terms (after the kernels above, which leave those out):
// one thread per (row, alternative).
template <class T>
__global__ void __launch_bounds__(256)
k_grad_top(const T *__restrict__ logits, int64_t ld, int64_t rows, Grads in, T *__restrict__ grad, int64_t ldg) {
    const int64_t n = rows * in.top;
    for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < n; t += (int64_t)gridDim.x * 256) {
        const int64_t row = t / in.top;
        const int64_t at = in.top_actions[t];
        if (at < 0 || at >= in.V) continue;
        const int j = (int)at;
        const RowGrad r = in.row(row);
        const float g = grad_one(r, (float)logits[row * ld + j], j);
        grad[row * ldg + j] = (T)(r.empty ? 0.0f : g + in.g_top[t]);
    }
}

constexpr int64_t kMaxGrid = 1 << 20;

dim3 grid_of(int64_t n) { return dim3((unsigned)(n < kMaxGrid ? n : kMaxGrid)); }

// Rows of up to kSmall logits take part of a wave, up to kWave a whole one (16 packs of 4 float32 a lane, wherever the row
// starts).  Longer ones are streamed by workgroups; a short batch of them has to reach all 256 compute units and still be
// few launches, as the one that joins the parts of rows costs 3 us and as much again on the host:
//   more than kRows rows      256 threads per row, below kFill workgroups in parts of at least kPartBytes
//   rows up to kShort bytes   256 threads
//   up to kWhole bytes, or    1024 threads
//     from kManyRows rows on
//   else                      256 threads, in parts as above
// GPU us (bf16; with 5 or 20 alternatives) for 256 threads / 1024 threads / parts: 1 x 5000 6.2 / 8.3 / -, 1 x 20000 7.7 /
// 9.5 / 10.3, 1 x 32768 - / 10.1 / 9.5 (16 against 20 for a call with its host's work), 1 x 65536 - / 12.4 / 9.7,
// 1 x 131072 - / 16.7 / 10.2, 64 x 131072 - / 18.4 / 16.8, 100 x 131072 - / 18.5 / 21.8, 200 x 131072 - / 20 / 27.8,
// 300 x 131072 - / 47 / 27; kFill 256 / 512 / 1024: 300 x 32768 (float32) 14.1 / 16.4 / 17.3, 64 x 131072 20.8 / 17.2 / 18.6;
// kPartBytes 8192 / 16384 / 32768: 1 x 131072 10.2 / 10.5 / 11.4.
constexpr int kSmall = 64, kWave = 4088, kRows = 256, kManyRows = 96, kShort = 48 << 10, kWhole = 96 << 10, kFill = 512,
              kPartBytes = 16 << 10;
static_assert((kWave + 2 * 7) / 8 <= 8 * 64 && (kWave + 2 * 3) / 4 <= 16 * 64, "8 or 16 packs a lane hold a row of kWave logits");

struct Split {
    int threads, parts;
};

Split split_of(int32_t type, int64_t T, int32_t V) {
    const int64_t bytes = (int64_t)V * type_bytes(type);
    if (V <= kWave || (T <= kRows && bytes <= kShort)) return {256, 1};
    if (T <= kRows && (bytes <= kWhole || T >= kManyRows)) return {1024, 1};
    const int64_t parts = std::min(bytes / kPartBytes, (kFill + T - 1) / T);
    return {256, (int)std::max<int64_t>(1, std::min<int64_t>(parts, kMaxParts))};
}

template <class T>
void launch_scores(const T *logits, int64_t ld, int64_t rows, Split split, const Out &out, void *workspace, hipStream_t st) {
    using std::integral_constant;
    const int V = out.V;
    const auto small = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        hipLaunchKernelGGL((k_scores_small<T, L>), grid_of((rows + 256 / L - 1) / (256 / L)), dim3(256), 0, st, logits, ld, rows, out);
    };
    if (V <= 8) return small(integral_constant<int, 8>{});
    if (V <= 16) return small(integral_constant<int, 16>{});
    if (V <= 32) return small(integral_constant<int, 32>{});
    if (V <= kSmall) return small(integral_constant<int, 64>{});
    if (V <= kWave) {
        const auto wave = [&](auto packs) {
            hipLaunchKernelGGL((k_scores_wave<T, decltype(packs)::value>), grid_of((rows + 3) / 4), dim3(256), 0, st, logits, ld, rows, out);
        };
        constexpr int n = Pack<T>::n;
        const bool aligned = (uintptr_t)logits % 16 == 0 && (ld % n == 0 || rows == 1);
        const int packs = (V + (aligned ? n - 1 : 2 * (n - 1))) / n;  // of a row that starts anywhere: up to one more
        if (packs <= 64) wave(integral_constant<int, 1>{});
        else if (packs <= 128) wave(integral_constant<int, 2>{});
        else if (packs <= 192) wave(integral_constant<int, 3>{});
        else if (packs <= 256) wave(integral_constant<int, 4>{});
        else if (packs <= 384) wave(integral_constant<int, 6>{});
        else if (n == 8 || packs <= 512) wave(integral_constant<int, 8>{});  // all that 16-bit logits need
        else if constexpr (n == 4) {
            if (packs <= 768) wave(integral_constant<int, 12>{});
            else wave(integral_constant<int, 16>{});
        }
        return;
    }
    const int parts = split.parts;
    Key *keys = (Key *)workspace;
    Sums *sums = (Sums *)(keys + (parts > 1 ? rows * parts * out.top : 0));
    const auto stream = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, grid_of(rows * parts), dim3(threads), 0, st, logits, ld, rows, parts, out, sums, keys);
    };
    if (split.threads == 1024) out.top > 0 ? stream(k_scores_long<T, 1024, true>, 1024) : stream(k_scores_long<T, 1024, false>, 1024);
    else out.top > 0 ? stream(k_scores_long<T, 256, true>, 256) : stream(k_scores_long<T, 256, false>, 256);
    if (parts > 1)
        hipLaunchKernelGGL(k_scores_join<T>, grid_of(rows), dim3(64), 0, st, logits, ld, rows, parts, out, (const Sums *)sums,
                           (const Key *)keys);
}

template <class T>
void launch_grad(const T *logits, int64_t ld, int64_t rows, const Grads &in, T *grad, int64_t ldg, hipStream_t st) {
    const auto small = [&](auto lanes) {
        constexpr int L = decltype(lanes)::value;
        const int64_t per_group = 256 / L;
        hipLaunchKernelGGL((k_grad_small<T, L>), grid_of((rows + per_group - 1) / per_group), dim3(256), 0, st, logits, ld, rows,
                           in, grad, ldg);
    };
    if (in.V <= 8) {
        small(std::integral_constant<int, 8>{});
    } else if (in.V <= 32) {
        small(std::integral_constant<int, 32>{});
    } else if (in.V <= 64) {
        small(std::integral_constant<int, 64>{});
    } else {
        const int packs = (in.V + Pack<T>::n - 1) / Pack<T>::n + 1;  // a row that starts off a 16-byte address has one more
        const auto large = [&](auto lanes) {
            constexpr int L = decltype(lanes)::value, teams = 256 / L;
            const int pieces = (packs + kGradPacks * L - 1) / (kGradPacks * L);
            hipLaunchKernelGGL((k_grad_long<T, L>), grid_of((rows * pieces + teams - 1) / teams), dim3(256), 0, st, logits, ld, rows,
                               pieces, in, grad, ldg);
        };
        if (packs <= kGradPacks * 64)
            large(std::integral_constant<int, 64>{});
        else
            large(std::integral_constant<int, 256>{});
    }
    if (in.g_top) {
        const int64_t groups = (rows * in.top + 255) / 256;
        hipLaunchKernelGGL(k_grad_top<T>, grid_of(groups), dim3(256), 0, st, logits, ld, rows, in, grad, ldg);
    }
}

int check_logits(const char *what, const void *p, int32_t type, int64_t ld, int64_t T, int32_t V, int32_t top) {
    if (!type_ok(type)) return mz::fail(MZ_ERR_ARG, "%s: unknown element type %d", what, type);
    if (T < 0 || T > 0x7FFFFFFF || V <= 0 || V > (1 << 30)) return mz::fail(MZ_ERR_ARG, "%s: bad dimensions T=%lld V=%d", what, (long long)T, V);
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
    if (!type_ok(type) || T <= 0 || V <= 0 || top < 0 || top > kMaxTop) return 0;
    const int parts = split_of(type, T, V).parts;
    return parts > 1 ? T * parts * ((int64_t)sizeof(Sums) + top * (int64_t)sizeof(Key)) : 0;
}

int mz_policy_scores(const void *logits, int32_t type, int64_t ld, const int64_t *actions, int64_t T, int32_t V, int32_t top,
                     float *log_prob, float *entropy, float *stats, int64_t *top_actions, float *top_log_probs,
                     void *workspace, int64_t workspace_bytes, void *stream) {
    MZ_TRY(check_logits("mz_policy_scores", logits, type, ld, T, V, top));
    if (T == 0) return MZ_OK;
    if (!entropy || (actions && !log_prob) || (top > 0 && (!top_actions || !top_log_probs)))
        return mz::fail(MZ_ERR_ARG, "mz_policy_scores: NULL argument");
    const int64_t need = mz_policy_scores_workspace(type, T, V, top);
    if (need > 0 && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0))
        return mz::fail(MZ_ERR_ARG, "mz_policy_scores: needs a 16-byte aligned workspace of %lld bytes (got %lld)", (long long)need,
                        (long long)workspace_bytes);
    const Out out{actions, log_prob, entropy, stats, top_actions, top_log_probs, V, top};
    with_type(type, [&](auto t) {
        using E = decltype(t);
        launch_scores((const E *)logits, ld, T, split_of(type, T, V), out, workspace, (hipStream_t)stream);
    });
    return mz::check_launch("k_scores");
}

int mz_policy_scores_backward(const void *logits, int32_t type, int64_t ld, const int64_t *actions, int64_t T, int32_t V,
                              int32_t top, const float *stats, const int64_t *top_actions,
                              const float *g_log_prob, const float *g_entropy, const float *g_top, void *grad, int64_t ld_grad,
                              void *stream) {
    MZ_TRY(check_logits("mz_policy_scores_backward", logits, type, ld, T, V, top));
    MZ_TRY(check_logits("mz_policy_scores_backward", grad, type, ld_grad, T, V, top));
    if (T == 0) return MZ_OK;
    if (!stats || (g_top && top > 0 && !top_actions) || (g_log_prob && !actions))
        return mz::fail(MZ_ERR_ARG, "mz_policy_scores_backward: NULL argument");
    if (top == 0) g_top = nullptr;
    const Grads in{actions, stats, top_actions, g_log_prob, g_entropy, g_top, V, top};
    with_type(type, [&](auto t) {
        using E = decltype(t);
        launch_grad((const E *)logits, ld, T, in, (E *)grad, ld_grad, (hipStream_t)stream);
    });
    return mz::check_launch("k_scores_grad");
}

}  // extern "C"
