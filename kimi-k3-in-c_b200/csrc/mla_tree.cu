// mla_tree.cu -- absorbed MLA attention of drafted tokens over a paged latent cache.
//
// Token i of sequence b, head h (W_UK, W_UV: the head's blocks of kv_b):
//     qa    = W_UK^T q_nope
//     s_r   = (qa . c_r + q_rope . r_r) scale        over the cache rows r that i sees
//     out   = W_UV (sum_r e^(s_r - m) c_r / sum_r e^(s_r - m)),  m = max s_r
// i sees the sequence's cached rows and the drafts whose bits are set in its word.
#include "internal.cuh"
#include "paged.cuh"

namespace k3 {

constexpr int TR_DN = 128, TR_DR = 64, TR_DL = 512, TR_DV = 128, TR_H = 128;
constexpr int TR_WARPS = 8;

struct TreeArgs {
    PagedView v;
    const __nv_bfloat16 *latent, *rope, *q_nope, *q_rope, *w_uk, *w_uv;
    const unsigned long long *mask;
    int H;
    float scale;
    unsigned *err;
};

// One block per (token, head); a warp takes every eighth row with its own running maximum, sum
// and o, and the warps' parts are joined at the end.
template <typename OUT>
__global__ void __launch_bounds__(32 * TR_WARPS) mla_tree_attend_k(const TreeArgs a, OUT *out) {
    __shared__ float q[TR_DL + TR_DR], qn[TR_DN], o[TR_WARPS][TR_DL], ml[TR_WARPS][2];
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = last_at_most(a.v.cu, a.v.B, t);
    const PagedSeq s = paged_seq(a.v, b, K3CUDA_MAX_DRAFTS);
    if (t == 0 && h == 0)
        for (int c = tid; c < a.v.B; c += 32 * TR_WARPS) {
            const int code = paged_seq(a.v, c, K3CUDA_MAX_DRAFTS).code;
            if (code) atomicCAS(a.err + 1, 0u, (unsigned)code);
        }
    const int i = t - s.first;
    if (i < 0 || i >= s.n) return;
    const size_t th = (size_t)t * a.H + h;
    const uint64_t word = a.mask ? a.mask[t] : (i == 63 ? ~0ull : (1ull << (i + 1)) - 1);
    if (tid < TR_DN) qn[tid] = __bfloat162float(a.q_nope[th * TR_DN + tid]);
    if (tid < TR_DR) q[TR_DL + tid] = __bfloat162float(a.q_rope[th * TR_DR + tid]);
    __syncthreads();
    for (int c = tid; c < TR_DL; c += 32 * TR_WARPS) {
        float v = 0.f;
        for (int d = 0; d < TR_DN; d++)
            v = fmaf(qn[d], __bfloat162float(a.w_uk[((size_t)h * TR_DN + d) * TR_DL + c]), v);
        q[c] = v;
    }
    __syncthreads();
    float m = -INFINITY, l = 0.f, acc[TR_DL / 32];
#pragma unroll
    for (int j = 0; j < TR_DL / 32; j++) acc[j] = 0.f;
    for (int p = warp; p < s.len + s.n; p += TR_WARPS) {
        if (!((tree_tile_bits(word, s.len, s.n, p / 64) >> (p % 64)) & 1)) continue;
        long long row = paged_row(a.v, b, p);
        if (row < 0) {
            if (lane == 0) atomicCAS(a.err + 1, 0u, (unsigned)PAGED_PAGE);
            row = p % a.v.page_size;
        }
        const __nv_bfloat16 *c = a.latent + (size_t)row * TR_DL, *r = a.rope + (size_t)row * TR_DR;
        float x[TR_DL / 32], d = 0.f;
#pragma unroll
        for (int j = 0; j < TR_DL / 32; j++) {
            x[j] = __bfloat162float(c[lane + 32 * j]);
            d = fmaf(x[j], q[lane + 32 * j], d);
        }
#pragma unroll
        for (int j = 0; j < TR_DR / 32; j++)
            d = fmaf(__bfloat162float(r[lane + 32 * j]), q[TR_DL + lane + 32 * j], d);
#pragma unroll
        for (int w = 16; w; w >>= 1) d += __shfl_xor_sync(0xffffffffu, d, w);
        d *= a.scale;
        if (!isfinite(d) && p >= s.len) d = NAN;
        const float mn = fmaxf(m, d), f = m == mn ? 1.f : expf(m - mn), e = expf(d - mn);
        m = mn;
        l = l * f + e;
#pragma unroll
        for (int j = 0; j < TR_DL / 32; j++) acc[j] = acc[j] * f + e * x[j];
    }
#pragma unroll
    for (int j = 0; j < TR_DL / 32; j++) o[warp][lane + 32 * j] = acc[j];
    if (lane == 0) ml[warp][0] = m, ml[warp][1] = l;
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < TR_WARPS; w++) M = fmaxf(M, ml[w][0]);
    float f[TR_WARPS];
#pragma unroll
    for (int w = 0; w < TR_WARPS; w++) {
        f[w] = ml[w][1] == 0.f ? 0.f : expf(ml[w][0] - M);
        L += ml[w][1] * f[w];
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    for (int c = tid; c < TR_DL; c += 32 * TR_WARPS) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < TR_WARPS; w++)
            if (ml[w][1] != 0.f) v += f[w] * o[w][c];
        q[c] = v * inv;
    }
    __syncthreads();
    for (int j = warp; j < TR_DV; j += TR_WARPS) {
        float v = 0.f;
        for (int c = lane; c < TR_DL; c += 32)
            v = fmaf(q[c], __bfloat162float(a.w_uv[((size_t)h * TR_DV + j) * TR_DL + c]), v);
#pragma unroll
        for (int w = 16; w; w >>= 1) v += __shfl_xor_sync(0xffffffffu, v, w);
        if (lane == 0) io<OUT>::st(out + th * TR_DV + j, v);
    }
}

static int tree_shape(int B, int T, int H, int dn, int dr, int dl, int dv) {
    K3_ARG_CHECK(B >= 0 && T >= 0 && H >= 1 && H <= TR_H, "mla_tree_attend: bad B=%d T=%d H=%d", B,
                 T, H);
    if (dn != TR_DN || dr != TR_DR || dl != TR_DL || dv != TR_DV)
        return set_error(K3CUDA_ERR_UNSUPPORTED, "mla_tree_attend: dn=%d dr=%d dl=%d dv=%d not built",
                         dn, dr, dl, dv);
    return K3CUDA_OK;
}

}  // namespace k3

using namespace k3;

extern "C" int k3cuda_mla_tree_attend_workspace(int B, int T, int H, int dl, int dv,
                                                size_t *bytes) {
    K3_ARG_CHECK(bytes, "mla_tree_attend: null bytes");
    int rc = tree_shape(B, T, H, TR_DN, TR_DR, dl, dv);
    if (rc) return rc;
    *bytes = 0;
    return K3CUDA_OK;
}

extern "C" int k3cuda_mla_tree_attend(k3cuda_ctx *ctx, void *out, int out_dtype,
                                      const void *q_nope, const void *q_rope,
                                      const k3cuda_paged_cache *cache,
                                      const k3cuda_token_batch *batch,
                                      const unsigned long long *tree_mask, const void *w_uk,
                                      const void *w_uv, int H, int dn, int dr, int dl, int dv,
                                      float scale, void *workspace, size_t workspace_bytes) {
    const char *what = "mla_tree_attend";
    int rc = paged_args_ok(what, cache, batch);
    if (rc || (rc = tree_shape(batch->B, batch->T, H, dn, dr, dl, dv))) return rc;
    K3_ARG_CHECK(out_dtype == K3CUDA_F32 || out_dtype == K3CUDA_BF16, "%s: bad out_dtype %d", what,
                 out_dtype);
    if (batch->B == 0 || batch->T == 0) return enter(ctx);
    K3_ARG_CHECK(out && q_nope && q_rope && w_uk && w_uv, "%s: null pointer", what);
    const void *al[] = {out, q_nope, q_rope, w_uk, w_uv};
    for (const void *p : al)
        K3_ARG_CHECK(aligned(p, 16), "%s: pointers must be 16-byte aligned", what);
    K3_ARG_CHECK(aligned(tree_mask, 8), "%s: tree_mask must be 8-byte aligned", what);
    if ((rc = enter(ctx))) return rc;
    (void)workspace;
    (void)workspace_bytes;
    const TreeArgs a{paged_view(cache, batch),        (const __nv_bfloat16 *)cache->latent,
                     (const __nv_bfloat16 *)cache->rope, (const __nv_bfloat16 *)q_nope,
                     (const __nv_bfloat16 *)q_rope,   (const __nv_bfloat16 *)w_uk,
                     (const __nv_bfloat16 *)w_uv,     tree_mask,
                     H,                               scale,
                     ctx->err_word};
    const dim3 grid(batch->T, H);
    if (out_dtype == K3CUDA_BF16)
        mla_tree_attend_k<<<grid, 32 * TR_WARPS, 0, ctx->stream>>>(a, (__nv_bfloat16 *)out);
    else
        mla_tree_attend_k<<<grid, 32 * TR_WARPS, 0, ctx->stream>>>(a, (float *)out);
    return after_launch(ctx, what);
}
