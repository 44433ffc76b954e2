// mla_paged.cu -- new tokens into a paged latent cache, position rotation on the way.
//
// For token t of sequence b (row cu[b] + i, at cache position len_b + i, rotated by position p):
//     latent[row] = bf16(w * c / sqrt(mean(c^2) + eps)),  c = ct[t][0:512]
//     rope[row]   = bf16(R_p ct[t][512:576])
//     q_nope[t][h] = bf16(q[t][h][0:128]),  q_rope[t][h] = bf16(R_p q[t][h][128:192])
// R_p turns pair i of the 64 rope values by the angle p * inv_freq[i]; pair i is (i, i + 32) or
// (2 i, 2 i + 1). The angle is formed and reduced in 64 bits: at position 10^6 an fp32 angle is
// off by 0.06 rad. Norm statistics are summed in 64 bits, as k3cuda_mla_cache_append does.
//
// Memory-bound: every value is read once and written once. One block per (token, 16 heads) and
// one per token for the cache row, 128 threads with all loads of a thread issued before any
// use; a token's 32 angles are formed once per block. Measured with cold caches: 5058 tokens of 128
// heads in fp32 129 us, 5.9 TB/s of what has to be read and written (90 % of a copy's rate); 64 tokens of
// 16 heads 7.2 us, of which the host's part of the call is most.
#include "internal.cuh"
#include "paged.cuh"

namespace k3 {

constexpr int PA_DN = 128, PA_DR = 64, PA_DL = 512;
constexpr int PA_THREADS = 128;
constexpr int PA_HEADS = 16;   // query heads of one block
constexpr int PA_ITEMS = 24;   // 8-value items of one head: 16 of q_nope, 8 of q_rope
constexpr int PA_PER = PA_HEADS * PA_ITEMS / PA_THREADS;
static_assert(PA_HEADS * PA_ITEMS % PA_THREADS == 0, "items divide over the threads");

struct AppendArgs {
    PagedView v;
    __nv_bfloat16 *latent, *rope;
    const void *ct, *q;
    long long ct_stride, q_stride;  // elements between tokens
    __nv_bfloat16 *q_nope, *q_rope;
    const float *w;
    const float *inv_freq;          // nullptr: no rotation
    const int *positions;           // nullptr: the cache position
    float eps;
    int H, interleaved;
    unsigned *err;
};

__device__ __forceinline__ void load4(const float *p, float *v) {
    const float4 x = __ldcs(reinterpret_cast<const float4 *>(p));
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float *v) {
    const uint2 x = __ldcs(reinterpret_cast<const uint2 *>(p));
    v[0] = bf16lo(x.x); v[1] = bf16hi(x.x); v[2] = bf16lo(x.y); v[3] = bf16hi(x.y);
}
__device__ __forceinline__ void load8(const float *p, float *v) {
    load4(p, v);
    load4(p + 4, v + 4);
}
__device__ __forceinline__ void load8(const __nv_bfloat16 *p, float *v) {
    const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(p));
    const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = bf16lo(u[i]);
        v[2 * i + 1] = bf16hi(u[i]);
    }
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&p);
}

// The sequence of token t, in every thread; -1 for a row of none, or of one that its offsets leave
// out. The block looks all offsets over, since those before a sequence decide whether it counts. That
// is one memory latency for 512 sequences, where a search takes two (16 heads, back to back: 64 x 1 tokens
// 4.2 us instead of 4.3, 64 x 16 6.8 instead of 7.2, 1024 x 1 7.9 instead of 8.1; 5058 tokens of 3
// prompts 129 instead of 138). Many thousands pay for it (4096 x 1 34 us instead of 22, 16384 x 1 338
// instead of 92).
__device__ __forceinline__ int token_seq(const PagedView &v, int t, int2 *red) {
    int hit = v.B, bad = v.B;  // the first sequence with row t, the first that is out of order
    auto look = [&](int lo, int hi, int b) {
        // as paged_in_order; negative offsets are large ones
        if ((unsigned)lo > (unsigned)hi || (unsigned)hi > (unsigned)v.T) bad = min(bad, b);
        else if (lo <= t && t < hi) hit = min(hit, b);
    };
    const int skew = (int)((uintptr_t)v.cu / 4 % 4);
#pragma unroll 1
    for (int b = 4 * threadIdx.x - skew; b < v.B; b += 4 * PA_THREADS) {
        if (b >= 0 && b + 4 <= v.B) {
            const int4 c = *reinterpret_cast<const int4 *>(v.cu + b);
            const int end = v.cu[b + 4];
            look(c.x, c.y, b);
            look(c.y, c.z, b + 1);
            look(c.z, c.w, b + 2);
            look(c.w, end, b + 3);
        } else {
            for (int k = max(b, 0); k < min(b + 4, v.B); k++) look(v.cu[k], v.cu[k + 1], k);
        }
    }
    hit = __reduce_min_sync(0xffffffffu, hit);
    bad = __reduce_min_sync(0xffffffffu, bad);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_int2(hit, bad);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PA_THREADS / 32; w++) {
        hit = min(hit, red[w].x);
        bad = min(bad, red[w].y);
    }
    return hit < bad ? hit : -1;
}

template <typename T>
__global__ void __launch_bounds__(PA_THREADS) mla_paged_append_k(const AppendArgs a) {
    __shared__ float2 turn[PA_DR / 2];  // (cos, sin) of the token's angles
    __shared__ double red[PA_THREADS / 32];
    __shared__ int2 seq[PA_THREADS / 32];
    pdl_trigger();
    pdl_wait();
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const int b = token_seq(a.v, t, seq);
    if (t == 0 && blockIdx.y == 0)  // one block looks every sequence over
        for (int c = tid; c < a.v.B; c += PA_THREADS) {
            const int code = paged_seq(a.v, c, a.v.T).code;
            if (code) atomicCAS(a.err + 1, 0u, (unsigned)code);
        }
    if (b < 0) return;  // a padding row, or a sequence that was left out
    const PagedSeq s = paged_seq(a.v, b, a.v.T);
    const int i = t - s.first;
    if (i >= s.n) return;
    if (tid < PA_DR / 2) turn[tid] = make_float2(1.f, 0.f);
    if (a.inv_freq && tid < PA_DR / 2) {
        const int pos = a.positions ? a.positions[t] : s.len + i;
        const double angle = (double)pos * (double)a.inv_freq[tid];
        constexpr double two_pi = 6.283185307179586476925;
        const float r = (float)fma(-rint(angle / two_pi), two_pi, angle);  // in [-pi, pi]
        float sn, cs;
        sincosf(r, &sn, &cs);
        turn[tid] = make_float2(cs, sn);
    }
    if (blockIdx.y == 0) {
        // the cache row
        const T *src = static_cast<const T *>(a.ct) + (size_t)t * a.ct_stride;
        float x[4], y[2];
        load4(src + 4 * tid, x);
        const int r0 = a.interleaved ? 2 * tid : tid, r1 = a.interleaved ? 2 * tid + 1 : tid + 32;
        if (tid < PA_DR / 2) {
            y[0] = io<T>::ld(src + PA_DL + r0);
            y[1] = io<T>::ld(src + PA_DL + r1);
        }
        const float4 w = reinterpret_cast<const float4 *>(a.w)[tid];
        double ss = (double)x[0] * x[0] + (double)x[1] * x[1] + (double)x[2] * x[2] +
                    (double)x[3] * x[3];
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (lane == 0) red[tid >> 5] = ss;
        __syncthreads();
        ss = (red[0] + red[1]) + (red[2] + red[3]);
        const float inv = (float)(1.0 / sqrt(ss / (double)PA_DL + (double)a.eps));
        const long long row = paged_row(a.v, b, s.len + i);
        if (row < 0) {
            if (tid == 0) atomicCAS(a.err + 1, 0u, (unsigned)PAGED_PAGE);
            return;
        }
        reinterpret_cast<uint2 *>(a.latent + (size_t)row * PA_DL)[tid] =
            make_uint2(pack2(w.x * x[0] * inv, w.y * x[1] * inv),
                       pack2(w.z * x[2] * inv, w.w * x[3] * inv));
        if (tid < PA_DR / 2) {
            const float2 cs = turn[tid];
            __nv_bfloat16 *dst = a.rope + (size_t)row * PA_DR;
            dst[r0] = __float2bfloat16_rn(y[0] * cs.x - y[1] * cs.y);
            dst[r1] = __float2bfloat16_rn(y[0] * cs.y + y[1] * cs.x);
        }
        return;
    }
    // sixteen heads of queries
    const int h0 = (blockIdx.y - 1) * PA_HEADS;
    const T *q = static_cast<const T *>(a.q) + (size_t)t * a.q_stride;
    float v[PA_PER][8];
#pragma unroll
    for (int k = 0; k < PA_PER; k++) {
        const int e = tid + k * PA_THREADS, h = h0 + e / PA_ITEMS, c = e % PA_ITEMS;
        if (h >= a.H) continue;
        const T *src = q + (size_t)h * (PA_DN + PA_DR);
        if (c < 16 || a.interleaved) load8(src + 8 * c, v[k]);
        else {  // four pairs (j, j + 32)
            load4(src + PA_DN + 4 * (c - 16), v[k]);
            load4(src + PA_DN + 32 + 4 * (c - 16), v[k] + 4);
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PA_PER; k++) {
        const int e = tid + k * PA_THREADS, h = h0 + e / PA_ITEMS, c = e % PA_ITEMS;
        if (h >= a.H) continue;
        const size_t th = (size_t)t * a.H + h;
        float *x = v[k];
        if (c < 16) {
            reinterpret_cast<uint4 *>(a.q_nope + th * PA_DN)[c] =
                make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]),
                           pack2(x[6], x[7]));
            continue;
        }
        float o[8];
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const float2 cs = turn[4 * (c - 16) + p];
            const float x0 = a.interleaved ? x[2 * p] : x[p];
            const float x1 = a.interleaved ? x[2 * p + 1] : x[p + 4];
            const float y0 = x0 * cs.x - x1 * cs.y, y1 = x0 * cs.y + x1 * cs.x;
            if (a.interleaved) o[2 * p] = y0, o[2 * p + 1] = y1;
            else o[p] = y0, o[p + 4] = y1;
        }
        __nv_bfloat16 *dst = a.q_rope + th * PA_DR;
        const uint32_t w0 = pack2(o[0], o[1]), w1 = pack2(o[2], o[3]), w2 = pack2(o[4], o[5]),
                       w3 = pack2(o[6], o[7]);
        if (a.interleaved) reinterpret_cast<uint4 *>(dst)[c - 16] = make_uint4(w0, w1, w2, w3);
        else {
            reinterpret_cast<uint2 *>(dst)[c - 16] = make_uint2(w0, w1);
            reinterpret_cast<uint2 *>(dst + 32)[c - 16] = make_uint2(w2, w3);
        }
    }
}

int paged_args_ok(const char *what, const k3cuda_paged_cache *c, const k3cuda_token_batch *b) {
    K3_ARG_CHECK(c && b, "%s: null cache or batch", what);
    K3_ARG_CHECK(b->B >= 0 && b->T >= 0, "%s: bad B=%d T=%d", what, b->B, b->T);
    if (b->B == 0 || b->T == 0) return K3CUDA_OK;
    K3_ARG_CHECK(b->B < (1 << 24), "%s: B=%d", what, b->B);
    const int p = c->page_size;
    K3_ARG_CHECK(c->n_pages >= 1 && c->max_pages >= 1 && p >= 1,
                 "%s: bad n_pages=%d page_size=%d max_pages=%d", what, c->n_pages, p,
                 c->max_pages);
    if (p < 8 || (p & (p - 1)))
        return set_error(K3CUDA_ERR_UNSUPPORTED,
                         "%s: page_size=%d not built (a power of two, 8 or more)", what, p);
    K3_ARG_CHECK((long long)c->n_pages * p < (1ll << 31) &&
                     (long long)c->max_pages * p < (1ll << 31) - 128,
                 "%s: %d (table: %d) pages of %d rows pass 32-bit row numbers", what, c->n_pages,
                 c->max_pages, p);
    K3_ARG_CHECK(c->latent && c->rope && c->page_table && b->ctx_lens && b->cu_tokens,
                 "%s: null pointer in the cache or batch", what);
    K3_ARG_CHECK(aligned(c->latent, 16) && aligned(c->rope, 16),
                 "%s: caches must be 16-byte aligned", what);
    K3_ARG_CHECK(aligned(c->page_table, 4) && aligned(b->ctx_lens, 4) && aligned(b->cu_tokens, 4),
                 "%s: tables must be 4-byte aligned", what);
    return K3CUDA_OK;
}

PagedView paged_view(const k3cuda_paged_cache *c, const k3cuda_token_batch *b) {
    int shift = 0;
    while ((1 << shift) < c->page_size) shift++;
    return PagedView{c->page_table, c->n_pages,   c->page_size, c->max_pages, b->ctx_lens,
                     b->cu_tokens,  b->B,         b->T,         shift};
}

}  // namespace k3

using namespace k3;

extern "C" int k3cuda_mla_paged_append(k3cuda_ctx *ctx, const k3cuda_paged_cache *cache,
                                       const k3cuda_token_batch *batch, const void *ct,
                                       long long ct_stride, const void *q, long long q_stride,
                                       void *q_nope, void *q_rope, int io_dtype, int H,
                                       const float *kv_a_norm, float eps, const float *inv_freq,
                                       const int *positions, int rope_style, int dn, int dr,
                                       int dl) {
    const char *what = "mla_paged_append";
    int rc = paged_args_ok(what, cache, batch);
    if (rc) return rc;
    K3_ARG_CHECK(io_dtype == K3CUDA_F32 || io_dtype == K3CUDA_BF16, "%s: bad io_dtype %d", what,
                 io_dtype);
    K3_ARG_CHECK(rope_style == K3CUDA_ROPE_HALF || rope_style == K3CUDA_ROPE_INTERLEAVED,
                 "%s: bad rope_style %d", what, rope_style);
    if (dn != PA_DN || dr != PA_DR || dl != PA_DL)
        return set_error(K3CUDA_ERR_UNSUPPORTED, "%s: dn=%d dr=%d dl=%d not built", what, dn, dr,
                         dl);
    K3_ARG_CHECK(H >= 0 && H <= 128 && (q || H == 0), "%s: bad H=%d", what, H);
    if (batch->B == 0 || batch->T == 0) return enter(ctx);
    K3_ARG_CHECK(ct && kv_a_norm && (H == 0 || (q_nope && q_rope)), "%s: null pointer", what);
    const int unit = io_dtype == K3CUDA_F32 ? 4 : 8;  // elements of 16 bytes
    K3_ARG_CHECK(ct_stride >= PA_DL + PA_DR && ct_stride % unit == 0 &&
                     (H == 0 || (q_stride >= (long long)H * (PA_DN + PA_DR) &&
                                 q_stride % unit == 0)),
                 "%s: row strides ct=%lld q=%lld must cover a row and be multiples of 16 bytes",
                 what, ct_stride, q_stride);
    const void *al[] = {ct, kv_a_norm, q, q_nope, q_rope};
    for (const void *p : al)
        K3_ARG_CHECK(aligned(p, 16), "%s: pointers must be 16-byte aligned", what);
    K3_ARG_CHECK(aligned(inv_freq, 4) && aligned(positions, 4),
                 "%s: tables must be 4-byte aligned", what);
    if ((rc = enter(ctx))) return rc;
    const AppendArgs a{paged_view(cache, batch),
                       (__nv_bfloat16 *)cache->latent,
                       (__nv_bfloat16 *)cache->rope,
                       ct,
                       q,
                       ct_stride,
                       q_stride,
                       (__nv_bfloat16 *)q_nope,
                       (__nv_bfloat16 *)q_rope,
                       kv_a_norm,
                       inv_freq,
                       positions,
                       eps,
                       H,
                       rope_style == K3CUDA_ROPE_INTERLEAVED,
                       ctx->err_word};
    const dim3 grid(batch->T, 1 + (H + PA_HEADS - 1) / PA_HEADS);
    if (io_dtype == K3CUDA_F32)
        return launch_pdl(ctx, ctx->stream, what, mla_paged_append_k<float>, grid,
                          dim3(PA_THREADS), 0, a);
    return launch_pdl(ctx, ctx->stream, what, mla_paged_append_k<__nv_bfloat16>, grid,
                      dim3(PA_THREADS), 0, a);
}
