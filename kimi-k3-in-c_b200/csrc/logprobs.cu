// logprobs.cu -- log probabilities of given tokens, entropy and top alternatives of rows of logits.
//
// For a row x of V logits, with m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m):
//     log p_i = (x_i - m) - log s          entropy = log s - t / s
// One pass over the logits: a thread keeps a running (m, s, t) and rescales s and t when m grows
// (t' = f (t + s (m - m')), f = e^(m - m')). Sums are fp32; x - m is formed before it is scaled to
// log2 units, so large logits lose nothing.
//
// The K likeliest tokens come out of the same pass. A thread writes the maximum of each group of
// logits it reads (its cell) to shared memory. The K-th largest of some thread maxima is a bound
// that at least K logits reach, so only cells that reach it are read again (from L2, a few dozen
// of thousands), and the handful of logits at or above it are ranked by (logit, lower number).
// Where more of them reach it than the buffer holds (rows of equal logits), the block instead
// searches the row K times.
//
// Rows are cut into segments of whole iterations when there are few of them: each block leaves
// (m, s, t) and its K best, and a second kernel joins a row's segments.
#include "internal.cuh"
#include "sm100.cuh"

namespace k3 {

constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_MAX_IT = 32;      // iterations of a segment (cells per thread)
constexpr int LP_CAND = 1024;      // candidates ranked at once
constexpr int LP_MAX_SEG = 256;    // segments of a row
constexpr int LP_MAX_V = 1 << 24;
static_assert(K3CUDA_MAX_TOP * K3CUDA_MAX_TOP <= LP_CAND, "a join's candidates fit");
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
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    // an empty side (s = 0) has m = -inf; NaN sums stay NaN
    const float da = a.m - r.m, db = b.m - r.m;
    const float fa = a.s == 0.f ? 0.f : sm100::ex2_approx(da * LP_LOG2E);
    const float fb = b.s == 0.f ? 0.f : sm100::ex2_approx(db * LP_LOG2E);
    r.s = a.s * fa + b.s * fb;
    r.t = 0.f;
    if (a.s != 0.f) r.t += fa * (a.t + a.s * fmaxf(da, -1000.f));
    if (b.s != 0.f) r.t += fb * (b.t + b.s * fmaxf(db, -1000.f));
    return r;
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
};
template <> struct vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static constexpr unsigned NINF = 0xff80ff80u;
    static __device__ __forceinline__ void unpack(uint4 r, float *x) { sm100::unpack_bf8(r, x); }
};

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
    __device__ __forceinline__ uint4 load(int v, int end) const {
        constexpr int N = vec<T>::N;
        const int e = v * N - skew;
        uint4 r = make_uint4(vec<T>::NINF, vec<T>::NINF, vec<T>::NINF, vec<T>::NINF);
        if (v >= end) return r;
        if (e >= 0 && e + N <= V) {
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                         : "l"(x + e));
            return r;
        }
        unsigned w[4] = {r.x, r.y, r.z, r.w};
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
};

// What a row's statistics and K best give: the outputs (block-wide; keys in shared memory, 0 for
// a place without a token).
template <typename T>
__device__ __forceinline__ void finish_row(const LpArgs &a, int row, Stat st, const u64 *best) {
    const T *x = static_cast<const T *>(a.logits) + (size_t)row * a.stride;
    // no distribution: nothing but -inf (m = -inf), or a NaN or +inf (s is NaN then)
    const bool none = !(st.s > 0.f);
    const float ls = none ? NAN : logf(st.s);
    for (int g = threadIdx.x; g < a.G; g += LP_THREADS) {
        const int tok = a.tokens[(size_t)row * a.G + g];
        float lp = -INFINITY;
        if (none) lp = NAN;
        else if (tok >= 0 && tok < a.V) lp = (io<T>::ld(x + tok) - st.m) - ls;
        a.logprobs[(size_t)row * a.G + g] = lp;
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
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        Stat b;
        b.m = __shfl_xor_sync(0xffffffffu, st.m, o);
        b.s = __shfl_xor_sync(0xffffffffu, st.s, o);
        b.t = __shfl_xor_sync(0xffffffffu, st.t, o);
        // the same order on both lanes of a pair, so that they agree bit for bit
        st = (threadIdx.x & o) ? join(b, st) : join(st, b);
    }
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = st;
    __syncthreads();
    st = red[0];
    for (int w = 1; w < LP_WARPS; w++) st = join(st, red[w]);
    return st;
}

// rank n unique keys (n <= LP_CAND, in shared memory) and put the K largest into best, in order
__device__ __forceinline__ void rank_keys(const u64 *cand, int n, int K, u64 *best) {
    for (int k = threadIdx.x; k < K; k += LP_THREADS)
        if (k >= n) best[k] = 0;
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const u64 mine = cand[i];
        int r = 0;
        for (int j = 0; j < n; j++) r += cand[j] > mine;
        if (r < K) best[r] = mine;
    }
    __syncthreads();
}

struct LpShared {
    Stat red[LP_WARPS];
    unsigned head[32];        // thread maxima that set the bound
    unsigned bound;
    int n;
    u64 cand[LP_CAND], best[K3CUDA_MAX_TOP], wbest[LP_WARPS];
};

// The bound: at least K logits of the block are at or above it (LP_ORD_NINF + 1 where fewer than
// K are above -inf). Every warp gives its ceil(K / 8) largest thread maxima; the bound is the
// K-th largest of those.
__device__ __forceinline__ unsigned block_bound(float m, int K, LpShared &sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (K + LP_WARPS - 1) / LP_WARPS;
    unsigned mine = m == -INFINITY ? 0u : ord(m);
    for (int j = 0; j < per; j++) {
        const unsigned top = __reduce_max_sync(0xffffffffu, mine);
        const unsigned has = __ballot_sync(0xffffffffu, mine == top);
        if (lane == __ffs(has) - 1) mine = 0;
        if (lane == 0) sh.head[warp * per + j] = top;
    }
    __syncthreads();
    if (warp == 0) {
        const int n = per * LP_WARPS;
        const unsigned h = lane < n ? sh.head[lane] : 0u;
        int r = 0;
#pragma unroll
        for (int j = 0; j < 32; j++) {
            const unsigned o = __shfl_sync(0xffffffffu, h, j);
            r += o > h || (o == h && j < lane);
        }
        if (r == K - 1) sh.bound = max(h, LP_ORD_NINF + 1);
    }
    __syncthreads();
    return sh.bound;
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
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; u++) raw[u] = r.load(v0 + u * LP_THREADS + tid, v1);
    for (int it = 0; it < its; it++) {
        uint4 next[U];  // the next iteration's loads are in flight while this one is summed
        const int vn = v0 + (it + 1) * U * LP_THREADS + tid;
#pragma unroll
        for (int u = 0; u < U; u++) next[u] = r.load(vn + u * LP_THREADS, v1);
        float x[U * N];
#pragma unroll
        for (int u = 0; u < U; u++) vec<T>::unpack(raw[u], x + u * N);
        float cm = x[0];
#pragma unroll
        for (int i = 1; i < U * N; i++) cm = fmaxf(cm, x[i]);
        if (a.K) cell[it * LP_THREADS + tid] = cm;
        if (cm > st.m) {
            const float d = st.m - cm, f = sm100::ex2_approx(d * LP_LOG2E);
            st.t = st.s > 0.f ? f * (st.t + st.s * fmaxf(d, -1000.f)) : 0.f;
            st.s *= f;
            st.m = cm;
        }
        const float m = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
        for (int i = 0; i < U * N; i++) {
            const float d = x[i] - m;
            const float e = sm100::ex2_approx(d * LP_LOG2E);
            st.s += e;
            st.t = fmaf(e, fmaxf(d, -1000.f), st.t);
        }
#pragma unroll
        for (int u = 0; u < U; u++) raw[u] = next[u];
    }
    const float tm = st.m;
    const Stat all = block_join(st, sh.red);
    if (a.K) {
        const unsigned bound = block_bound(tm, a.K, sh);
        if (tid == 0) sh.n = 0;
        __syncthreads();
        if (ord(tm) >= bound)
            for (int it = 0; it < its; it++) {
                if (ord(cell[it * LP_THREADS + tid]) < bound) continue;
                for (int u = 0; u < U; u++) {
                    const int v = v0 + (it * U + u) * LP_THREADS + tid;
                    float x[N];
                    vec<T>::unpack(r.load(v, v1), x);
#pragma unroll
                    for (int i = 0; i < N; i++)
                        if (ord(x[i]) >= bound && x[i] <= INFINITY) {
                            const int p = atomicAdd(&sh.n, 1);
                            if (p < LP_CAND) sh.cand[p] = key_of(x[i], v * N - r.skew + i);
                        }
                }
            }
        __syncthreads();
        const int n = sh.n;
        if (n <= LP_CAND) {
            rank_keys(sh.cand, n, a.K, sh.best);
        } else {
            // the next best, K times
            u64 last = ~0ull;
            for (int k = 0; k < a.K; k++) {
                u64 top = 0;
                for (int v = v0 + tid; v < v1; v += LP_THREADS) {
                    float x[N];
                    vec<T>::unpack(r.load(v, v1), x);
#pragma unroll
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
        finish_row<T>(a, row, all, sh.best);
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
            for (int j = 0; j < n; j++) r += sh.cand[j] > mine || (sh.cand[j] == mine && j < i);
            if (r == a.K - 1) bound = mine;  // 0 where fewer than K places hold a token
        }
        __syncthreads();
        const u64 least = max(bound, 1ull);
        __syncthreads();
        if (tid < a.S)
            for (int k = 0; k < a.K; k++) {
                const u64 key = keys[(size_t)tid * a.K + k];
                if (key < least) break;
                const int p = atomicAdd(&sh.n, 1);
                if (p < LP_CAND) sh.cand[p] = key;
            }
        __syncthreads();
        rank_keys(sh.cand, min(sh.n, LP_CAND), a.K, sh.best);
    }
    finish_row<T>(a, row, all, sh.best);
}

// How rows are cut: U vectors per thread and iteration, n_it iterations per segment, S segments.
struct LpPlan {
    int U, n_it, S;
};

// Enough blocks to fill the GPU several times over where the rows allow it, on a B200's 148 SMs
// whatever the device, so that the workspace query needs no device.
static LpPlan lp_plan(int T, int V, int io_dtype) {
    const int N = io_dtype == K3CUDA_F32 ? 4 : 8;
    const long long nv = ((long long)V + 2 * N - 2) / N;  // most vectors, whatever the skew
    constexpr long long want = 148 * 8;
    LpPlan p;
    p.U = T * ((nv + 4 * LP_THREADS - 1) / (4 * LP_THREADS)) >= want ? 4 : 1;
    const long long its = (nv + p.U * LP_THREADS - 1) / (p.U * LP_THREADS);
    long long S = (want + T - 1) / (T > 0 ? T : 1);
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

static size_t lp_bytes(const LpPlan &p, int T, int K) {
    if (p.S == 1 || T == 0) return 0;
    return lp_align((size_t)T * p.S * sizeof(Stat)) + lp_align((size_t)T * p.S * K * sizeof(u64));
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
    const size_t a = lp_bytes(lp_plan(T, V, K3CUDA_F32), T, K);
    const size_t b = lp_bytes(lp_plan(T, V, K3CUDA_BF16), T, K);
    *bytes = a > b ? a : b;
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
    const size_t need = lp_bytes(p, T, K);
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
