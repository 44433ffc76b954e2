// logprobs.cu -- log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
// For a row x of V logits, with m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m):
//     log p_i = (x_i - m) - log s          entropy = log s - t / s
// One pass over the logits: a thread keeps a running (m, s, t) and rescales s and t when m grows
// (t' = f (t + s (m - m')), f = e^(m - m')). Sums are fp32; x - m is formed before it is scaled to
// log2 units, so large logits lose nothing. Pairs of logits share an instruction (fp32 pairs; the
// maximum of bf16 logits on bf16 pairs): 4.5 instructions a logit, of them one exponential, 16 a
// clock and SM.
//
// The K likeliest tokens come out of the same pass. A thread writes the maximum of each group of
// logits it reads (its cell) to shared memory. The K-th largest of the thread maxima is a bound that
// at least K logits reach, so only cells that reach it are read again (from L2, a few dozen of
// thousands): they are listed first and read all at once, since one after another, as each thread
// meets its own, they took 13 us of a block. The handful of logits at or above the bound are ranked
// by (logit, lower number). (The K-th largest of every warp's ceil(K / 8) best is a bound that is had
// sooner, but where a few warps hold nothing but -inf there are too few of those, and all the others'
// logits were ranked: 7 us.) The bound has the logit's upper 16 bits. Where more than LP_FEW
// cells or logits reach those (fp32 logits far from zero, bf16 logits with equal ones at the top), it is
// found again from the threads' best (logit, number) in 64 bits. Where even that leaves more than LP_CAND
// (thousands of likely tokens in fewer than K threads: a period of 1024 or 4096 fp32 logits), the block
// searches its segment K times. 512 x 163840 fp32, K = 20, by events: 77 us; 101 us with logits around
// 1030 and 95 us with equal ones (2205 us both when those were searched K times); 3.3 ms where the
// likely ones lie 1024 apart, K = 30.
//
// Rows are cut into segments of whole iterations when there are few of them: each block leaves
// (m, s, t) and its K best, and a second kernel joins a row's segments.
//
// Measured, the caches cold: 512 rows of 163840 fp32 logits with the 20 likeliest 69 us (4.9 TB/s, 74 %
// of a copy's rate; 59 us without the likeliest, whose work leaves a block's loads idle meanwhile); 2048
// rows of 163840 bf16 135 us (5.0 TB/s; back to back 124 us, the exponentials' unit 68 % busy); one such
// row 9.2 us. Blocks that begin their next segment's loads before they finish the last were slower
// (back to back 124 -> 149 us: segments are dealt out unevenly then), and so was one segment instead of
// two for 512 rows (72 us).
#include <algorithm>

#include "internal.cuh"
#include "sm100.cuh"

namespace k3 {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_MAX_IT = 32;      // iterations of a segment (cells per thread)
constexpr int LP_CAND = 1024;      // cells listed, candidates ranked at once
constexpr int LP_FEW = 256;        // of either that are taken without looking for a closer bound
constexpr int LP_MAX_SEG = 256;    // segments of a row
constexpr int LP_MAX_V = 1 << 24;
static_assert(K3CUDA_MAX_TOP * K3CUDA_MAX_TOP <= LP_CAND, "a join's candidates fit");
static_assert(LP_MAX_IT * LP_THREADS <= 65536, "a cell's number has 16 bits");
constexpr float LP_LOG2E = 1.4426950408889634f;

typedef unsigned long long u64;

// logits in ascending order as unsigned numbers (-0 as +0); 0 is below every logit
__device__ __forceinline__ unsigned ord(float x) {
    const unsigned u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unord(unsigned o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
constexpr unsigned LP_ORD_NINF = 0x007fffffu;  // ord(-inf)
// rank of token i with logit x: higher logits first, then lower numbers
__device__ __forceinline__ u64 key_of(float x, int i) {
    return ((u64)ord(x) << 32) | (0xffffffffu - (unsigned)i);
}

// running maximum and sums of a set of logits
struct Stat {
    float m, s, t;
};
// (s, t) of a maximum m taken to a maximum M >= m
__device__ __forceinline__ void move(Stat &a, float M) {
    if (a.s == 0.f) {  // an empty set: m = -inf (NaN sums stay NaN)
        a.t = 0.f;
    } else {
        const float d = a.m - M, f = sm100::ex2_approx(d * LP_LOG2E);
        a.t = f * (a.t + a.s * fmaxf(d, -1000.f));
        a.s *= f;
    }
    a.m = M;
}

struct LpArgs {
    const void *logits;
    long long stride;
    int T, V, S, n_it;  // segments per row, iterations per segment
    const int *tokens;
    int G;
    float *logprobs, *entropy;
    int K;
    int *top_ids;
    float *top_logprobs;
    Stat *stats;        // [T][S]
    u64 *keys;          // [T][S][K]
};

template <typename T> struct vec;
template <> struct vec<float> {
    static constexpr int N = 4;
    static constexpr unsigned NINF = 0xff800000u;  // a word of -inf
    static __device__ __forceinline__ void unpack(uint4 r, float *x) {
        x[0] = __uint_as_float(r.x); x[1] = __uint_as_float(r.y);
        x[2] = __uint_as_float(r.z); x[3] = __uint_as_float(r.w);
    }
    // of U vectors, as of fmaxf: NaN is no maximum
    template <int U> static __device__ __forceinline__ float max(const uint4 *r) {
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float x[N];
            unpack(r[u], x);
            m = sm100::max3(sm100::max3(m, x[0], x[1]), x[2], x[3]);
        }
        return m;
    }
};
template <> struct vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr unsigned NINF = 0xff80ff80u;
    static __device__ __forceinline__ void unpack(uint4 r, float *x) { sm100::unpack_bf8(r, x); }
    template <int U> static __device__ __forceinline__ float max(const uint4 *r) {
        __nv_bfloat162 m = reinterpret_cast<const __nv_bfloat162 &>(r[0].x);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const __nv_bfloat162 *x = reinterpret_cast<const __nv_bfloat162 *>(r + u);
#pragma unroll
            for (int i = u == 0; i < 4; i++) m = __hmax2(m, x[i]);
        }
        const float lo = __low2float(m), hi = __high2float(m);
        return fmaxf(fmaxf(lo, hi), -INFINITY);  // -inf where all are NaN
    }
};

// The vector of logits e .. of a row of V where some are outside of it: those are -inf.
template <typename T> __device__ __noinline__ uint4 edge_load(const T *x, int e, int V) {
    constexpr int N = vec<T>::N;
    unsigned w[4] = {vec<T>::NINF, vec<T>::NINF, vec<T>::NINF, vec<T>::NINF};
#pragma unroll
    for (int j = 0; j < N; j++)
        if (e + j >= 0 && e + j < V) {
            if (sizeof(T) == 4) {
                w[j & 3] = reinterpret_cast<const unsigned *>(x)[e + j];
            } else {
                const unsigned h = reinterpret_cast<const unsigned short *>(x)[e + j];
                const int sh = 16 * (j & 1);
                w[(j >> 1) & 3] = (w[(j >> 1) & 3] & ~(0xffffu << sh)) | (h << sh);
            }
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A row as 16-byte vectors from the vector boundary at or before its first logit: vector v holds
// logits v N - skew .. +N. The vectors at the row's ends are read logit by logit.
template <typename T> struct Row {
    const T *x;
    int V, skew;
    __device__ __forceinline__ Row(const LpArgs &a, int row) {
        x = static_cast<const T *>(a.logits) + (size_t)row * a.stride;
        V = a.V;
        skew = (int)(((uintptr_t)x / sizeof(T)) % vec<T>::N);
    }
    __device__ __forceinline__ int vectors() const { return (V + skew + vec<T>::N - 1) / vec<T>::N; }
    // vectors lo .. hi - 1 are whole
    __device__ __forceinline__ int lo() const { return skew > 0; }
    __device__ __forceinline__ int hi() const { return (V + skew) / vec<T>::N; }
    __device__ __forceinline__ uint4 whole(int v) const {
        uint4 r;
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                     : "l"(x + ((long long)v * vec<T>::N - skew)));
        return r;
    }
    __device__ __forceinline__ uint4 load(int v, int end) const {
        if (v >= lo() && v < min(hi(), end)) return whole(v);
        if (v < end) return edge_load<T>(x, v * vec<T>::N - skew, V);
        return make_uint4(vec<T>::NINF, vec<T>::NINF, vec<T>::NINF, vec<T>::NINF);
    }
};

// the logit of a row's g-th given token, -inf without one
template <typename T>
__device__ __forceinline__ float given(const LpArgs &a, int row, int g) {
    const int tok = g < a.G ? a.tokens[(size_t)row * a.G + g] : -1;
    if (tok < 0 || tok >= a.V) return -INFINITY;
    return io<T>::ld(static_cast<const T *>(a.logits) + (size_t)row * a.stride + tok);
}

// What a row's statistics and K best give: the outputs (block-wide; keys in shared memory, 0 for
// a place without a token; mine: this thread's first given token's logit).
template <typename T>
__device__ __forceinline__ void finish_row(const LpArgs &a, int row, Stat st, float mine,
                                           const u64 *best) {
    // no distribution: nothing but -inf (m = -inf), or a NaN or +inf (s is NaN then)
    const bool none = !(st.s > 0.f);
    const float ls = none ? NAN : logf(st.s);
    for (int g = threadIdx.x; g < a.G; g += LP_THREADS) {
        const float x = g == threadIdx.x ? mine : given<T>(a, row, g);
        a.logprobs[(size_t)row * a.G + g] = none ? NAN : (x - st.m) - ls;
    }
    if (threadIdx.x == 0 && a.entropy) a.entropy[row] = none ? NAN : ls - st.t / st.s;
    for (int k = threadIdx.x; k < a.K; k += LP_THREADS) {
        const u64 key = best[k];
        int id = -1;
        float lp = none ? NAN : -INFINITY;
        if (!none && key) {
            id = (int)(0xffffffffu - (unsigned)key);
            lp = (unord((unsigned)(key >> 32)) - st.m) - ls;
        }
        a.top_ids[(size_t)row * a.K + k] = id;
        a.top_logprobs[(size_t)row * a.K + k] = lp;
    }
}

// the block's joined statistics, in every thread
__device__ __forceinline__ Stat block_join(Stat st, Stat *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the maximum, as an ordered number; then plain sums
    const float m = unord(__reduce_max_sync(0xffffffffu, ord(st.m)));
    if (lane == 0) red[warp].m = m;
    __syncthreads();
    float M = red[0].m;
#pragma unroll
    for (int w = 1; w < LP_WARPS; w++) M = fmaxf(M, red[w].m);
    move(st, M);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
        st.t += __shfl_xor_sync(0xffffffffu, st.t, o);
    }
    if (lane == 0) {
        red[warp].s = st.s;
        red[warp].t = st.t;
    }
    __syncthreads();
    st.s = st.t = 0.f;
#pragma unroll
    for (int w = 0; w < LP_WARPS; w++) {
        st.s += red[w].s;
        st.t += red[w].t;
    }
    return st;
}

// rank n unique keys (n <= LP_CAND, in shared memory) and put the K largest into best, in order
__device__ __forceinline__ void rank_keys(const u64 *cand, int n, int K, u64 *best) {
    for (int k = threadIdx.x; k < K; k += LP_THREADS)
        if (k >= n) best[k] = 0;
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const u64 mine = cand[i];
        int r = 0;
#pragma unroll 4
        for (int j = 0; j < n; j++) r += cand[j] > mine;
        if (r < K) best[r] = mine;
    }
    __syncthreads();
}

struct LpShared {
    Stat red[LP_WARPS];
    int n, cells;
    unsigned short list[LP_CAND];  // cells that reach the bound
    u64 cand[LP_CAND], best[K3CUDA_MAX_TOP], wbest[LP_WARPS];
};

// The K-th largest of the threads' numbers (0 where fewer have one), bit by bit from `bit` on; `at`:
// the bits above that.
template <typename N> __device__ __forceinline__ N block_kth(N mine, int K, N at, N bit) {
#pragma unroll 1
    for (; bit; bit >>= 1)
        if (__syncthreads_count(mine >= (at | bit)) >= K) at |= bit;
    return at;
}

template <int U> __device__ __forceinline__ uint4 pick(const uint4 *r, int u) {
    uint4 x = r[0];
#pragma unroll
    for (int i = 1; i < U; i++)
        if (u == i) x = r[i];
    return x;
}

// This thread's best key: its largest logit m where that comes first (cells lie it, it + 1, .. one
// after another). 0 without a logit above -inf.
template <typename T, int U>
__device__ __noinline__ u64 best_key(const Row<T> r, const float *cell, int v0, int v1, int its,
                                     float m) {
    constexpr int N = vec<T>::N;
    if (m == -INFINITY) return 0;
    int it = 0;
    while (it < its - 1 && cell[it * LP_THREADS + threadIdx.x] != m) it++;
    for (int u = 0; u < U; u++) {
        const int v = v0 + (it * U + u) * LP_THREADS + threadIdx.x;
        float x[N];
        vec<T>::unpack(r.load(v, v1), x);
        for (int i = 0; i < N; i++)
            if (x[i] == m) return key_of(m, v * N - r.skew + i);
    }
    return 0;
}

// U: 16-byte vectors a thread reads per iteration
template <typename T, int U>
__global__ void __launch_bounds__(LP_THREADS, 4) token_logprobs_k(const LpArgs a) {
    constexpr int N = vec<T>::N;
    extern __shared__ float cell[];  // [n_it][LP_THREADS] maxima, where K > 0
    __shared__ LpShared sh;
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, row = blockIdx.x / a.S, seg = blockIdx.x % a.S;
    const Row<T> r(a, row);
    const int v0 = seg * a.n_it * U * LP_THREADS;
    const int v1 = min(r.vectors(), v0 + a.n_it * U * LP_THREADS);
    const int its = v1 > v0 ? (v1 - v0 + U * LP_THREADS - 1) / (U * LP_THREADS) : 0;
    Stat st{-INFINITY, 0.f, 0.f};
    const int lo = r.lo(), hi = min(r.hi(), v1);
    // iteration it's vectors (-inf behind the last)
    auto fetch = [&](uint4 *raw, int it) {
        const int v = v0 + it * U * LP_THREADS;
        if (v >= lo && v + U * LP_THREADS <= hi) {
#pragma unroll
            for (int u = 0; u < U; u++) raw[u] = r.whole(v + tid + u * LP_THREADS);
        } else {
#pragma unroll
            for (int u = 0; u < U; u++) raw[u] = r.load(v + tid + u * LP_THREADS, v1);
        }
    };
    auto add = [&](const uint4 *raw, int it) {
        const float cm = vec<T>::template max<U>(raw);
        if (a.K) cell[it * LP_THREADS + tid] = cm;
        if (cm > st.m) move(st, cm);
        const float m = st.m == -INFINITY ? 0.f : st.m;
        const float2 m2 = make_float2(-m, -m), k2 = make_float2(LP_LOG2E, LP_LOG2E);
        float2 s2 = make_float2(0.f, 0.f), t2 = s2;
#pragma unroll
        for (int u = 0; u < U; u++) {
            float x[N];
            vec<T>::unpack(raw[u], x);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const float2 d = sm100::add2(make_float2(x[i], x[i + 1]), m2);
                float2 e = sm100::mul2(d, k2);
                e.x = sm100::ex2_approx(e.x);
                e.y = sm100::ex2_approx(e.y);
                s2 = sm100::add2(s2, e);
                t2 = sm100::fma2(e, d, t2);
            }
        }
        float t = t2.x + t2.y;
        if (!(t == t)) {  // a forbidden token's 0 times -inf among them: without those
            t = 0.f;
#pragma unroll 1
            for (int u = 0; u < U; u++) {
                float x[N];
                vec<T>::unpack(pick<U>(raw, u), x);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const float d = x[i] - m;
                    t = fmaf(sm100::ex2_approx(d * LP_LOG2E), fmaxf(d, -1000.f), t);
                }
            }
        }
        st.s += s2.x + s2.y;
        st.t += t;
    };
    uint4 ra[U], rb[U];  // one iteration's loads are in flight while the other is summed
    fetch(ra, 0);
#pragma unroll 1
    for (int it = 0; it < its; it += 2) {
        fetch(rb, it + 1);
        add(ra, it);
        if (it + 1 >= its) break;
        fetch(ra, it + 2);
        add(rb, it + 1);
    }
    const float tm = st.m;
    const Stat all = block_join(st, sh.red);
    if (a.K) {
        // The bound: at least K logits of the block are at or above it (any above -inf where fewer
        // than K threads hold one). The K-th largest thread maximum to its upper 16 bits will do,
        // unless too many logits share those. Then it is the K-th largest of the threads' best keys,
        // which no two logits share.
        unsigned top = block_kth<unsigned>(tm == -INFINITY ? 0u : ord(tm) >> 16, a.K, 0u, 1u << 15);
        constexpr u64 least = (u64)(LP_ORD_NINF + 1) << 32;
        u64 bound = max((u64)top << 48, least);
        bool fits;
#pragma unroll 1
        for (bool exact = false;; exact = true) {
            if (tid == 0) sh.n = sh.cells = 0;
            __syncthreads();
            if (key_of(tm, 0) >= bound)
                for (int it = 0; it < its; it++) {
                    const int i = (v0 + it * U * LP_THREADS + tid) * N - r.skew;  // the cell's first
                    if (key_of(cell[it * LP_THREADS + tid], max(i, 0)) < bound) continue;
                    const int p = atomicAdd(&sh.cells, 1);
                    if (p < LP_CAND) sh.list[p] = (unsigned short)(it * LP_THREADS + tid);
                }
            __syncthreads();
            const int cells = sh.cells, limit = exact ? LP_CAND : LP_FEW;
#pragma unroll 1
            for (int e = tid; cells <= limit && e < cells * U * N; e += LP_THREADS) {
                const int c = sh.list[e / (U * N)];
                const int v = v0 + (c / LP_THREADS * U + e / N % U) * LP_THREADS + c % LP_THREADS;
                const int i = v * N - r.skew + e % N;
                if (v >= v1 || i < 0 || i >= r.V) continue;
                const float x = io<T>::ld(r.x + i);
                if (!(x <= INFINITY) || key_of(x, i) < bound) continue;
                const int p = atomicAdd(&sh.n, 1);
                if (p < LP_CAND) sh.cand[p] = key_of(x, i);
            }
            __syncthreads();
            fits = cells <= limit && sh.n <= limit;
            if (fits || exact) break;
            const u64 mine = best_key<T, U>(r, cell, v0, v1, its, tm);
            bound = max(block_kth<u64>(mine, a.K, (u64)top << 48, 1ull << 47), least);
        }
        if (fits) {
            rank_keys(sh.cand, sh.n, a.K, sh.best);
        } else {
            // the next best, K times
            u64 last = ~0ull;
            for (int k = 0; k < a.K; k++) {
                u64 top = 0;
                for (int v = v0 + tid; v < v1; v += LP_THREADS) {
                    float x[N];
                    vec<T>::unpack(r.load(v, v1), x);
                    for (int i = 0; i < N; i++) {
                        const u64 key = key_of(x[i], v * N - r.skew + i);
                        if (x[i] > -INFINITY && key < last && key > top) top = key;
                    }
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                if ((tid & 31) == 0) sh.wbest[tid >> 5] = top;
                __syncthreads();
                top = sh.wbest[0];
                for (int w = 1; w < LP_WARPS; w++) top = max(top, sh.wbest[w]);
                if (tid == 0) sh.best[k] = top;
                last = top;
                __syncthreads();
            }
        }
    }
    if (a.S == 1) {
        finish_row<T>(a, row, all, given<T>(a, row, tid), sh.best);
        return;
    }
    if (tid == 0) a.stats[blockIdx.x] = all;
    for (int k = tid; k < a.K; k += LP_THREADS) a.keys[(size_t)blockIdx.x * a.K + k] = sh.best[k];
}

// Join the segments of a row. The segments' best are in order, so the K-th largest of the first
// ceil(K / S) of each is a bound that K of them reach; at most K segments start at or above it.
template <typename T> __global__ void __launch_bounds__(LP_THREADS) token_logprobs_join(const LpArgs a) {
    __shared__ LpShared sh;
    __shared__ u64 bound;
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, row = blockIdx.x;
    const Stat *ss = a.stats + (size_t)row * a.S;
    const u64 *keys = a.keys + (size_t)row * a.S * a.K;
    Stat st{-INFINITY, 0.f, 0.f};
    if (tid < a.S) st = ss[tid];
    const float mine = given<T>(a, row, tid);  // on its way while the segments are joined
    const Stat all = block_join(st, sh.red);
    if (a.K) {
        const int per = (a.K + a.S - 1) / a.S, n = per * a.S;  // n < S + K <= LP_CAND
        for (int i = tid; i < n; i += LP_THREADS)
            sh.cand[i] = keys[(size_t)(i / per) * a.K + i % per];
        if (tid == 0) sh.n = 0;
        __syncthreads();
        for (int i = tid; i < n; i += LP_THREADS) {
            const u64 mine = sh.cand[i];
            int r = 0;
#pragma unroll 4
            for (int j = 0; j < n; j++) r += sh.cand[j] > mine || (sh.cand[j] == mine && j < i);
            if (r == a.K - 1) bound = mine;  // 0 where fewer than K places hold a token
        }
        __syncthreads();
        const u64 least = max(bound, 1ull);
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < a.S * a.K; i += LP_THREADS) {
            const u64 key = keys[i];
            if (key < least) continue;
            const int p = atomicAdd(&sh.n, 1);
            if (p < LP_CAND) sh.cand[p] = key;
        }
        __syncthreads();
        rank_keys(sh.cand, min(sh.n, LP_CAND), a.K, sh.best);
    }
    finish_row<T>(a, row, all, mine, sh.best);
}

// How rows are cut: U vectors per thread and iteration, n_it iterations per segment, S segments.
struct LpPlan {
    int U, n_it, S;
};

// Blocks to fill the GPU once (four an SM) where the rows allow it, on a B200's 148 SMs
// whatever the device, so that the workspace query needs no device.
constexpr int LP_BLOCKS = 148 * 4;
static LpPlan lp_plan(int T, int V, int io_dtype) {
    const int N = io_dtype == K3CUDA_F32 ? 4 : 8;
    const long long nv = ((long long)V + 2 * N - 2) / N;  // most vectors, whatever the skew
    constexpr long long want = LP_BLOCKS;
    LpPlan p;
    p.U = T * ((nv + 4 * LP_THREADS - 1) / (4 * LP_THREADS)) >= want ? 4 : 1;
    const long long its = (nv + p.U * LP_THREADS - 1) / (p.U * LP_THREADS);
    long long S = T > 0 && T < want ? want / T : 1;
    S = S < its ? S : its;
    S = S < LP_MAX_SEG ? S : LP_MAX_SEG;
    if ((its + S - 1) / S > LP_MAX_IT) S = (its + LP_MAX_IT - 1) / LP_MAX_IT;
    p.n_it = (int)((its + S - 1) / S);
    p.S = (int)((its + p.n_it - 1) / p.n_it);
    return p;
}

static size_t lp_align(size_t x) { return (x + 255) & ~(size_t)255; }

static int lp_shape(int T, int V, int K) {
    K3_ARG_CHECK(T >= 0 && V >= 1 && K >= 0 && K <= K3CUDA_MAX_TOP,
                 "token_logprobs: bad T=%d V=%d K=%d (K <= %d)", T, V, K, K3CUDA_MAX_TOP);
    if (V > LP_MAX_V)
        return set_error(K3CUDA_ERR_UNSUPPORTED, "token_logprobs: V=%d not built (<= %d)", V,
                         LP_MAX_V);
    return K3CUDA_OK;
}

static size_t lp_bytes(long long segments, int K) {
    return lp_align(segments * sizeof(Stat)) + lp_align(segments * K * sizeof(u64));
}
static size_t lp_need(const LpPlan &p, int T, int K) {
    return p.S == 1 || T == 0 ? 0 : lp_bytes((long long)T * p.S, K);
}
// What no call of up to T rows of up to V logits passes: LP_BLOCKS segments, or those that LP_MAX_IT
// cuts every row into.
static size_t lp_bound(int T, int V, int K, int io_dtype) {
    if (T == 0) return 0;
    const int N = io_dtype == K3CUDA_F32 ? 4 : 8;
    const long long nv = ((long long)V + 2 * N - 2) / N;
    const long long its = (nv + 4 * LP_THREADS - 1) / (4 * LP_THREADS);
    const long long cut = (its + LP_MAX_IT - 1) / LP_MAX_IT;
    return lp_bytes(std::max<long long>(LP_BLOCKS, cut > 1 ? T * cut : 0), K);
}

template <typename T> static int lp_run(k3cuda_ctx *ctx, const LpArgs &a, const LpPlan &p) {
    const size_t smem = a.K ? (size_t)p.n_it * LP_THREADS * sizeof(float) : 0;
    const dim3 grid((unsigned)a.T * p.S);
    const int rc = p.U == 4 ? launch_pdl(ctx, ctx->stream, "token_logprobs",
                                         token_logprobs_k<T, 4>, grid, dim3(LP_THREADS), smem, a)
                            : launch_pdl(ctx, ctx->stream, "token_logprobs",
                                         token_logprobs_k<T, 1>, grid, dim3(LP_THREADS), smem, a);
    if (rc || p.S == 1) return rc;
    return launch_pdl(ctx, ctx->stream, "token_logprobs_join", token_logprobs_join<T>, dim3(a.T),
                      dim3(LP_THREADS), 0, a);
}

}  // namespace k3

using namespace k3;

extern "C" int k3cuda_token_logprobs_workspace(int T, int V, int K, size_t *bytes) {
    K3_ARG_CHECK(bytes, "token_logprobs: null bytes");
    int rc = lp_shape(T, V, K);
    if (rc) return rc;
    *bytes = std::max(lp_bound(T, V, K, K3CUDA_F32), lp_bound(T, V, K, K3CUDA_BF16));
    return K3CUDA_OK;
}

extern "C" int k3cuda_token_logprobs(k3cuda_ctx *ctx, const void *logits, int io_dtype,
                                     long long row_stride, int T, int V, const int *tokens, int G,
                                     float *logprobs, float *entropy, int K, int *top_ids,
                                     float *top_logprobs, void *workspace,
                                     size_t workspace_bytes) {
    int rc = lp_shape(T, V, K);
    if (rc) return rc;
    K3_ARG_CHECK(io_dtype == K3CUDA_F32 || io_dtype == K3CUDA_BF16,
                 "token_logprobs: bad io_dtype %d", io_dtype);
    K3_ARG_CHECK(G >= 0 && (G == 0 || T == 0 || (tokens && logprobs)) &&
                     (K == 0 || T == 0 || (top_ids && top_logprobs)),
                 "token_logprobs: bad G=%d or null output", G);
    K3_ARG_CHECK(row_stride >= V, "token_logprobs: row_stride=%lld < V=%d", row_stride, V);
    const LpPlan p = lp_plan(T, V, io_dtype);
    const size_t need = lp_need(p, T, K);
    if (need && (!workspace || workspace_bytes < need))
        return set_error(K3CUDA_ERR_WORKSPACE, "token_logprobs: workspace %zu < %zu",
                         workspace_bytes, need);
    K3_ARG_CHECK(!need || aligned(workspace, 256),
                 "token_logprobs: workspace must be 256-byte aligned");
    K3_ARG_CHECK((long long)T * p.S < (1ll << 31), "token_logprobs: T=%d", T);
    K3_ARG_CHECK(aligned(logits, io_dtype == K3CUDA_F32 ? 4 : 2) && aligned(tokens, 4) &&
                     aligned(logprobs, 4) && aligned(entropy, 4) && aligned(top_ids, 4) &&
                     aligned(top_logprobs, 4),
                 "token_logprobs: pointers must be aligned to their elements");
    K3_ARG_CHECK(logits || T == 0, "token_logprobs: null logits");
    if ((rc = enter(ctx)) || T == 0) return rc;
    char *w = (char *)workspace;
    const LpArgs a{logits, row_stride, T, V, p.S, p.n_it, tokens, G, logprobs, entropy, K, top_ids,
                   top_logprobs, (Stat *)w,
                   (u64 *)(w ? w + lp_align((size_t)T * p.S * sizeof(Stat)) : w)};
    return io_dtype == K3CUDA_F32 ? lp_run<float>(ctx, a, p) : lp_run<__nv_bfloat16>(ctx, a, p);
}
