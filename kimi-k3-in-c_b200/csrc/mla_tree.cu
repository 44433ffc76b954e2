// mla_tree.cu -- absorbed MLA attention of drafted tokens over a paged latent cache, on tcgen05.
//
// Token i of sequence b, head h (W_UK, W_UV: the head's blocks of kv_b):
//     qa    = W_UK^T q_nope                                      mla_absorb (mla_decode.cu)
//     s_r   = (qa . c_r + q_rope . r_r) scale                    mla_tree_attend_tc
//     o     = sum_r e^(s_r - m) c_r,  l = sum_r e^(s_r - m)      mla_tree_attend_tc
//     out   = W_UV o / l                                         mla_project (mla_decode.cu)
// over the cache rows r that i sees: the sequence's cached rows and the drafts whose bits are set
// in its word.
//
// The (token, head) pairs of a sequence's drafts are packed into row tiles of 128, the MMA's M, so
// that a few heads of one rank and many drafts fill it as well as 128 heads of one token do, and
// one read of the cache serves all of them.
//
// The accumulator of o (128 x 512 fp32) takes all of an SM's TMEM, so a row tile is worked on by a
// cluster of two CTAs with one job each. The score CTA holds the query in TMEM (288 columns, the A
// operand), streams the tile's 576-wide rows, forms S and the softmax, and sends the weights P to
// its peer as bf16 (asynchronous cluster stores that complete on an mbarrier), with the factor by
// which o is to be rescaled. The value CTA streams the same rows' 512 latent dims, from L2 by then,
// and accumulates o. P is double-buffered, so neither waits for the other in step.
// What decides this split (measured on a B200): cluster stores move 17 B a clock and SM, TMA reads
// from L2 over 70. Splitting the dims over the pair instead (each row read once, partial scores and
// P exchanged, 36 KB per 96 rows and CTA) is bound by the former: 5400 cycles per 96 rows.
// Tiles are 128 cache rows: an MMA takes about 60 cycles for any N up to 128 (60 at N = 64, 65.5 at
// 128, 128.6 at 256, A in TMEM), so smaller tiles run the scores below the full rate.
// Per SM:
//   score   TMEM: query 288 columns, S 128;  shared: 4 stages x 48 KB (three 64-dim blocks of 128
//           rows, K-major, 128-byte swizzle)
//   value   TMEM: o 512 columns;  shared: 4 stages x 32 KB (32 rows x 512 dims, MN-major), P 2 x 32 KB
// Warps: 0 loads (a lane per box), 1 issues the MMAs, 2-17 are four groups of one warp per lane
// quarter: in the score CTA a group takes 32 score columns of all rows, in the value CTA 128 dims
// of o (rescaling, read-out).
//
// Work: the (row tile, cache tile) pairs lie on a line, every row tile taking TT_FIXED more places
// for its fixed work; clusters take equal pieces (paged.cuh). A row tile that one cluster does
// whole is written as (o, l); one that is cut leaves partial (m, l, o) that mla_tree_join joins.
// The line is formed on the device from the batch's tables (mla_tree_plan), so that a captured
// call follows them.
//
// Hidden rows: a masked score gives weight 0 whatever it is, and a zero weight times a row of
// infinities must stay 0, so in tiles that reach past the cached rows the value CTA zeroes
// unwritten rows in shared memory, and non-finite elements of draft rows too; a draft row's score
// that is not finite counts as NaN for those that see it. Every wait is bounded (sm100.cuh).
#include "internal.cuh"
#include "paged.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace k3 {

using namespace sm100;

constexpr int TT_DN = 128, TT_DR = 64, TT_DL = 512, TT_DV = 128, TT_H = 128;
constexpr int TT_QW = TT_DL + TT_DR;       // absorbed query width
constexpr int TT_M = 128;                  // rows of a row tile
constexpr int TT_TILE = 128;               // cache rows of a tile
constexpr int TT_BOX = 32;                 // most rows of a load box
constexpr int TT_NST = 4;                  // stages of either CTA
constexpr int TT_KBLK = TT_TILE * 128;     // score: a 64-dim block of a tile; three to a stage
constexpr int TT_KSTAGE = 3 * TT_KBLK;
constexpr int TT_VROWS = 32;               // value: rows of a stage
constexpr int TT_VBLK = TT_VROWS * 128;    // a 64-dim block of a value stage; eight to a stage
constexpr int TT_VSTAGE = 8 * TT_VBLK;
constexpr int TT_CHUNKS = TT_TILE / TT_VROWS;
constexpr int TT_OFF_P = TT_NST * TT_VSTAGE;   // value: P, two buffers of two 64-column blocks
constexpr int TT_PBUF = 2 * TT_M * 128;
constexpr int TT_SMEM = TT_NST * TT_KSTAGE + 1024;
static_assert(TT_CHUNKS == TT_NST, "chunk c of every tile is in stage c");
static_assert(TT_OFF_P + 2 * TT_PBUF <= TT_SMEM - 1024, "both CTAs' layouts fit");
constexpr int TT_TM_Q = 0, TT_TM_S = 288, TT_TM_COLS = 512;
constexpr int TT_CW = TT_TILE / 4;         // score columns of a softmax warp
constexpr int TT_WORKERS = 16;             // warps 2 .. 17
constexpr int TT_THREADS = (2 + TT_WORKERS) * 32;
constexpr int TT_CLUSTERS = 74;            // 148 SMs of a B200
constexpr int TT_FIXED = 4;                // a row tile's fixed work, in tiles
constexpr int TT_MIN_TILES = 2;            // fewest tiles per cluster
constexpr int TT_PART = TT_DL + 4;         // floats of a partial row: o, m, l, pad
constexpr uint32_t TT_P_BYTES = TT_PBUF + TT_M * 4;  // P and the rescale factors of a tile

// the device-side plan, at the start of the workspace
struct TreePlan {
    long long total;   // places on the line
    int G;             // clusters that take part
};

struct TreeArgs {
    PagedView v;
    const TreePlan *plan;
    const long long *cum;      // [B + 1] first place of each sequence
    const unsigned long long *mask;
    const __nv_bfloat16 *qlat; // [T][H][576]
    float *part;               // [2 TT_CLUSTERS][128][TT_PART]
    __nv_bfloat16 *olat2;      // [T][H][hi 512 | lo 512]
    float *rowsum;             // [T][H]
    int H;
    float scale_log2e;
    unsigned *err;
};

struct TreeMaps {
    CUtensorMap lat, rope;
};

// A cluster's next piece of the line: tiles t0 .. t1 - 1 of row tile mt of sequence b.
struct TreeSeg {
    int b, mt, t0, t1, tiles;
    PagedSeq s;
    long long ustart;  // the row tile's first place
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == tiles; }
    // the partial's slot: the even one of a cluster for a row tile that began in an earlier cluster
    __device__ __forceinline__ int slot(int c) const { return 2 * c + (t0 == 0 ? 1 : 0); }
};

struct TreeWalk {
    const TreeArgs &a;
    long long c0, c1, at;  // this cluster's places; the next row tile's first place
    int b, mt, units;
    long long cost;
    PagedSeq s;
    __device__ __forceinline__ void seq() {
        s = paged_seq(a.v, b, K3CUDA_MAX_DRAFTS);
        units = (int)(((long long)s.n * a.H + TT_M - 1) / TT_M);
        cost = TT_FIXED + (s.len + s.n + TT_TILE - 1) / TT_TILE;
    }
    __device__ __forceinline__ TreeWalk(const TreeArgs &args, int c, long long total, int G)
        : a(args), c0(line_begin(total, G, c)), c1(line_begin(total, G, c + 1)) {
        b = last_at_most(a.cum, a.v.B, c0);
        seq();
        mt = (int)((c0 - a.cum[b]) / cost);
        at = a.cum[b] + mt * cost;
    }
    __device__ __forceinline__ bool next(TreeSeg &g) {
        while (at < c1) {
            if (mt >= units) {  // the next sequence with tokens
                if (++b >= a.v.B) return false;
                mt = 0;
                seq();
                continue;
            }
            const long long first = at + TT_FIXED;  // place of tile 0
            g.b = b;
            g.mt = mt;
            g.s = s;
            g.ustart = at;
            g.tiles = (int)(cost - TT_FIXED);
            g.t0 = (int)(c0 > first ? c0 - first : 0);
            g.t1 = (int)(c1 < first ? 0 : c1 - first < g.tiles ? c1 - first : g.tiles);
            at += cost;
            mt++;
            if (g.t0 < g.t1) return true;
        }
        return false;
    }
};

// Plan: the line's prefix over the sequences, which tokens count, and what is wrong with the tables.
__global__ void __launch_bounds__(1024) mla_tree_plan(PagedView v, int H, TreePlan *plan,
                                                      long long *cum, int *keep, int clusters,
                                                      unsigned *err) {
    __shared__ long long wsum[32], carry, tsum[32];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int t = tid; t < v.T; t += 1024) keep[t] = 0;
    if (tid == 0) carry = 0;
    __syncthreads();
    long long tiles_all = 0;
    for (int b0 = 0; b0 < v.B; b0 += 1024) {
        const int b = b0 + tid;
        long long cost = 0;
        if (b < v.B) {
            const PagedSeq s = paged_seq(v, b, K3CUDA_MAX_DRAFTS);
            if (s.code) atomicCAS(err + 1, 0u, (unsigned)s.code);
            for (int i = 0; i < s.n; i++) keep[s.first + i] = 1;
            const long long units = ((long long)s.n * H + TT_M - 1) / TT_M;
            const long long tiles = (s.len + s.n + TT_TILE - 1) / TT_TILE;
            cost = units * (tiles + TT_FIXED);
            tiles_all += units * tiles;
        }
        long long x = cost;  // inclusive prefix over the block
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) wsum[warp] = x;
        __syncthreads();
        long long before = carry;
        for (int w = 0; w < warp; w++) before += wsum[w];
        if (b < v.B) cum[b] = before + x - cost;
        __syncthreads();
        if (tid == 1023) carry = before + x;
        __syncthreads();
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) tiles_all += __shfl_xor_sync(0xffffffffu, tiles_all, o);
    if (lane == 0) tsum[warp] = tiles_all;
    __syncthreads();
    if (tid == 0) {
        long long tiles = 0;
        for (int w = 0; w < 32; w++) tiles += tsum[w];
        const long long want = (tiles + TT_MIN_TILES - 1) / TT_MIN_TILES;
        cum[v.B] = carry;
        plan->total = carry;
        plan->G = (int)(want < clusters ? want : clusters);
    }
}

// A bounded wait taken by one lane for its warp: 32 lanes that poll one barrier take the
// shared-memory pipe from everybody else.
template <bool kCluster = false>
__device__ __forceinline__ bool lane_wait(uint64_t *bar, uint32_t parity, unsigned *err,
                                          unsigned code) {
    bool ok = true;
    if ((threadIdx.x & 31) == 0) ok = mbar_wait_impl<kCluster>(bar, parity, err, code);
    __syncwarp();  // what lane 0 has seen, every lane sees
    return __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
}

struct TreeBars {
    uint64_t full[TT_NST], empty[TT_NST];  // stages
    uint64_t q_full, q_empty, s_full, s_empty;  // score
    uint64_t pair[4];           // score: per lane quarter, its four warps
    uint64_t p_in[2], p_full[2];  // value: P has come; o is ready for it
    uint64_t pv_done[2];        // both: o of the tile is done, P's buffer free
    uint64_t clean[TT_CHUNKS];  // value: the stages of a tile that reaches past the cached rows
    float val[2][4][TT_M];      // score: row maxima (or sums) of the four warps, by phase parity
    float fac[2][TT_M];         // value: rescale factors
    uint32_t tmem_base;
};

// n columns of o from addr: multiply by f
__device__ __forceinline__ void rescale_o(uint32_t addr, int n, float f) {
    for (int c = 0; c < n; c += 16) {
        float v[16];
        tmem_ld16(addr + c, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] *= f;
        tmem_st16(addr + c, v);
    }
    tmem_wait_st();
}

// A segment's o, latent dims dim .. dim + n - 1 (TMEM columns from addr) of row `row`: to the
// partial, or (a whole row tile) as the projection's bf16 hi/lo pair.
__device__ __forceinline__ void write_o(const TreeArgs &a, const TreeSeg &g, int cl, uint32_t addr,
                                        int row, int dim, int n) {
    const int lr = g.mt * TT_M + row;
    const bool ok = lr < g.s.n * a.H, whole = g.whole();
    const size_t th = (size_t)g.s.first * a.H + lr;
    float *dst = a.part + ((size_t)g.slot(cl) * TT_M + row) * TT_PART + dim;
    __nv_bfloat16 *hi = a.olat2 + th * 2 * TT_DL + dim;
    for (int c = 0; c < n; c += 16) {
        float v[16];
        tmem_ld16(addr + c, v);
        tmem_wait_ld();
        if (!ok) continue;
        if (!whole) {
            float4 *d4 = reinterpret_cast<float4 *>(dst + c);
#pragma unroll
            for (int i = 0; i < 4; i++)
                d4[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
            float lo[16];
#pragma unroll
            for (int i = 0; i < 16; i++)
                lo[i] = v[i] - __bfloat162float(__float2bfloat16_rn(v[i]));
            uint4 *h4 = reinterpret_cast<uint4 *>(hi + c), *l4 = h4 + TT_DL / 8;
            h4[0] = pack_bf8(v);
            h4[1] = pack_bf8(v + 8);
            l4[0] = pack_bf8(lo);
            l4[1] = pack_bf8(lo + 8);
        }
    }
}

// A row tile's queries into TMEM (lane = row, two bf16 per column): group grp of a quarter takes
// every fourth 64-dim block. Rows past the last token's are zero.
__device__ __forceinline__ void load_q(const TreeArgs &a, const TreeSeg &g, uint32_t lane_addr,
                                       int row, int grp) {
    const int lr = g.mt * TT_M + row;
    const bool ok = lr < g.s.n * a.H;
    const uint4 *q = reinterpret_cast<const uint4 *>(a.qlat + ((size_t)g.s.first * a.H + lr) * TT_QW);
    for (int h = 2 * grp; h < 18; h += h & 1 ? 7 : 1) {  // half blocks: 32 dims, 16 columns
        float v[16];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 w = ok ? q[4 * h + i] : make_uint4(0, 0, 0, 0);
            v[4 * i] = __uint_as_float(w.x);
            v[4 * i + 1] = __uint_as_float(w.y);
            v[4 * i + 2] = __uint_as_float(w.z);
            v[4 * i + 3] = __uint_as_float(w.w);
        }
        tmem_st16(lane_addr + TT_TM_Q + 16 * h, v);
    }
    tmem_wait_st();
}

// The rows of a tile's load boxes: box j holds rows j box .. of the tile.
__device__ __forceinline__ int box_row(const TreeArgs &a, const TreeSeg &g, long long pos,
                                       bool report) {
    long long r = paged_row(a.v, g.b, (int)pos);
    if (r < 0) {
        if (report) atomicCAS(a.err + 1, 0u, (unsigned)PAGED_PAGE);
        r = pos % a.v.page_size;
    }
    return (int)r;
}

// Zero what a draft row of bf16 pairs holds that is not finite.
__device__ __forceinline__ uint32_t finite_pair(uint32_t u) {
    if ((u & 0x7f80u) == 0x7f80u) u &= 0xffff0000u;
    if ((u & 0x7f800000u) == 0x7f800000u) u &= 0xffffu;
    return u;
}

// ---------------------------------------------------------------- score CTA
__device__ __forceinline__ void score_loads(const TreeMaps &maps, const TreeArgs &a, TreeWalk walk,
                                            uint8_t *sm, TreeBars &bars) {
    const int lane = threadIdx.x & 31;
    const int box = a.v.page_size < TT_BOX ? a.v.page_size : TT_BOX, boxes = TT_TILE / box;
    int i = 0;  // stages filled
    bool ok = true;
    TreeSeg sg;
    while (ok && walk.next(sg)) {
        for (int t = sg.t0; t < sg.t1 && ok; t++) {
            const long long p0 = (long long)t * TT_TILE;
            const int rows = sg.s.len + sg.s.n;
            const int live = (int)min((long long)boxes, (rows - p0 + box - 1) / box);
            // a lane's boxes are the same in each of the tile's three stages (boxes <= 16, three
            // blocks: up to two loads a lane)
            int row[2];
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int j = (lane + 32 * k) % boxes;
                row[k] = 0;
                if (lane + 32 * k < 3 * boxes && j < live)
                    row[k] = box_row(a, sg, p0 + j * box, true);
            }
            for (int c = 0; c < 3; c++, i++) {
                const int st = i % TT_NST, n = i / TT_NST;
                if (n > 0 && !(ok = lane_wait(&bars.empty[st], (n - 1) & 1, a.err, 0x502))) break;
                if (lane == 0) mbar_expect_tx(&bars.full[st], live * box * 3 * 128);
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int e = lane + 32 * k, j = e % boxes, kb = 3 * c + e / boxes;
                    if (e >= 3 * boxes || j >= live) continue;
                    uint8_t *dst = sm + st * TT_KSTAGE + (e / boxes) * TT_KBLK + j * box * 128;
                    if (kb < 8) tma_load_2d(dst, &maps.lat, &bars.full[st], kb * 64, row[k]);
                    else tma_load_2d(dst, &maps.rope, &bars.full[st], 0, row[k]);
                }
            }
        }
    }
    // loads still in flight are waited for (bounded) before the CTA may exit
    if (lane == 0)
        for (int st = 0; st < TT_NST && st < i; st++)
            mbar_wait_quiet(&bars.full[st], ((i - 1 - st) / TT_NST) & 1);
    __syncwarp();
}

__device__ __forceinline__ void score_mma(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                          TreeBars &bars, uint32_t tbase) {
    constexpr uint32_t id = idesc_f16(128, TT_TILE, false, false);
    int g = 0, i = 0, nq = 0;
    TreeSeg sg;
    while (walk.next(sg)) {
        if (!mbar_wait(&bars.q_full, nq++ & 1, a.err, 0x511)) return;
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            for (int c = 0; c < 3; c++, i++) {
                const int st = i % TT_NST;
                if (!mbar_wait(&bars.full[st], (i / TT_NST) & 1, a.err, 0x512)) return;
                if (c == 0 && g >= 1 && !mbar_wait(&bars.s_empty, (g - 1) & 1, a.err, 0x513)) return;
                tc_fence_after();
                const uint32_t kv = smem_u32(sm + st * TT_KSTAGE);
#pragma unroll
                for (int kb = 0; kb < 3; kb++)
#pragma unroll
                    for (int ks = 0; ks < 4; ks++)
                        mma_bf16_ts(tbase + TT_TM_S, tbase + TT_TM_Q + (3 * c + kb) * 32 + ks * 8,
                                    sdesc_kmajor(kv + kb * TT_KBLK + ks * 32), id,
                                    (c | kb | ks) ? 1u : 0u);
                mma_commit(&bars.empty[st]);
            }
            mma_commit(&bars.s_full);
            if (t + 1 == sg.t1) mma_commit(&bars.q_empty);
        }
    }
}

__device__ __forceinline__ void score_softmax(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                              TreeBars &bars, uint32_t tbase, int cl) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q4 = warp & 3, grp = (warp - 2) >> 2;  // lane quarter, group
    const int row = 32 * q4 + lane;                  // row of the row tile = TMEM lane
    const int c0 = TT_CW * grp;                      // first score column
    const uint32_t laddr = tbase + ((uint32_t)(32 * q4) << 16);
    const uint32_t ppeer = map_peer(smem_u32(sm + TT_OFF_P), 1);
    const uint32_t fpeer = map_peer(smem_u32(&bars.fac[0][row]), 1);
    const uint32_t bpeer = map_peer(smem_u32(&bars.p_in[0]), 1);
    float m_ref = -INFINITY, l = 0.f;  // l: this warp's columns
    int g = 0, nq = 0, np = 0;
    // the row's values of the quarter's four warps
    auto share = [&](float v, float (&o)[4]) -> bool {
        bars.val[np & 1][grp][row] = v;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.pair[q4]);
        if (!lane_wait(&bars.pair[q4], np & 1, a.err, 0x521)) return false;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = bars.val[np & 1][i][row];
        np++;
        return true;
    };
    TreeSeg sg;
    while (walk.next(sg)) {
        // this warp's part of the queries (the last row tile's S must be done)
        if (nq > 0 && !lane_wait(&bars.q_empty, (nq - 1) & 1, a.err, 0x522)) return;
        tc_fence_after();
        load_q(a, sg, laddr, row, grp);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.q_full);
        nq++;
        // the word of this row's token
        const int tok = min((sg.mt * TT_M + row) / a.H, sg.s.n - 1);
        const uint64_t word = a.mask ? a.mask[sg.s.first + tok] : (((uint64_t)2 << tok) - 1);
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            float s[TT_CW];
            if (!lane_wait(&bars.s_full, g & 1, a.err, 0x523)) return;
            tc_fence_after();
            tmem_ld32(laddr + TT_TM_S + c0, s);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.s_empty);
            const long long p0 = (long long)t * TT_TILE + c0;
            if (p0 + TT_CW > sg.s.len) {  // reaches past the cached rows
                const uint32_t see = (uint32_t)tree_bits(word, sg.s.len, sg.s.n, p0);
                const int d0 = (int)max(0ll, min((long long)TT_CW, sg.s.len - p0));
#pragma unroll
                for (int i = 0; i < TT_CW; i++) {
                    if (i >= d0 && !(fabsf(s[i]) < INFINITY)) s[i] = NAN;
                    // (a negative scale would turn the mask into +inf)
                    s[i] = (see >> i) & 1 ? s[i] * a.scale_log2e : -INFINITY;
                }
            } else {
#pragma unroll
                for (int i = 0; i < TT_CW; i++) s[i] *= a.scale_log2e;
            }
            float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < TT_CW; i++) m4[i & 3] = fmaxf(m4[i & 3], s[i]);
            float o[4];
            if (!share(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), o)) return;
            const float mx = fmaxf(fmaxf(o[0], o[1]), fmaxf(o[2], o[3]));
            float f = 1.f;
            if (t == sg.t0) {
                m_ref = mx;
                l = 0.f;
            } else if (mx > m_ref + MLA_RESCALE_LOG2) {
                f = exp2f(m_ref - mx);
                l *= f;
                m_ref = mx;
            }
            const float base = m_ref == -INFINITY ? 0.f : m_ref;  // nothing seen so far
            uint32_t w[TT_CW / 2];
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < TT_CW; i += 2) {
                const float a0 = ex2_approx(s[i] - base), a1 = ex2_approx(s[i + 1] - base);
                sum[(i >> 1) & 3] += a0 + a1;
                w[i / 2] = pack_bf2(a0, a1);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            // P to the peer: 16-byte chunk ch of a row, 64 columns to a block, swizzled
            const int pb = g & 1;
            if (g >= 2 && !lane_wait(&bars.pv_done[pb], ((g >> 1) - 1) & 1, a.err, 0x524)) return;
            const uint32_t rbar = bpeer + 8 * pb;
#pragma unroll
            for (int c = 0; c < TT_CW / 8; c++) {
                const int ch = c0 / 8 + c;
                st_async_v4(ppeer + pb * TT_PBUF + (ch >> 3) * (TT_M * 128) + swz(row, ch & 7),
                            __uint_as_float(w[4 * c]), __uint_as_float(w[4 * c + 1]),
                            __uint_as_float(w[4 * c + 2]), __uint_as_float(w[4 * c + 3]), rbar);
            }
            if (grp == 0) st_async_f32(fpeer + pb * TT_M * 4, f, rbar);
        }
        // the row's sum
        float o[4];
        if (!share(l, o)) return;
        const int lr = sg.mt * TT_M + row;
        if (grp == 0 && lr < sg.s.n * a.H) {
            const float lt = (o[0] + o[1]) + (o[2] + o[3]);
            if (sg.whole()) a.rowsum[(size_t)sg.s.first * a.H + lr] = lt;
            else {
                float *dst = a.part + ((size_t)sg.slot(cl) * TT_M + row) * TT_PART + TT_DL;
                dst[0] = m_ref;
                dst[1] = lt;
            }
        }
    }
    // the peer is done with every P (its last commits arrive on this CTA's barriers)
    for (int k = g >= 2 ? g - 2 : 0; k < g; k++)
        if (!lane_wait(&bars.pv_done[k & 1], (k >> 1) & 1, a.err, 0x525)) return;
}

// ---------------------------------------------------------------- value CTA
__device__ __forceinline__ void value_loads(const TreeMaps &maps, const TreeArgs &a, TreeWalk walk,
                                            uint8_t *sm, TreeBars &bars) {
    const int lane = threadIdx.x & 31;
    const int box = a.v.page_size < TT_BOX ? a.v.page_size : TT_BOX, boxes = TT_VROWS / box;
    int i = 0;
    bool ok = true;
    TreeSeg sg;
    while (ok && walk.next(sg)) {
        for (int t = sg.t0; t < sg.t1 && ok; t++) {
            const long long rows = sg.s.len + sg.s.n;
            for (int c = 0; c < TT_CHUNKS; c++, i++) {
                const int st = i % TT_NST, n = i / TT_NST;
                // lane: box lane % boxes of 64-dim block lane / boxes
                const int j = lane % boxes, kb = lane / boxes;
                const long long p0 = (long long)t * TT_TILE + c * TT_VROWS;
                const int live =
                    (int)max(0ll, min((long long)boxes, (rows - p0 + box - 1) / box));
                const bool some = j < live && kb < 8;
                const int row = some ? box_row(a, sg, p0 + j * box, false) : 0;
                if (n > 0 && !(ok = lane_wait(&bars.empty[st], (n - 1) & 1, a.err, 0x532))) break;
                if (lane == 0) mbar_expect_tx(&bars.full[st], live * box * 8 * 128);
                __syncwarp();
                if (some)
                    tma_load_2d(sm + st * TT_VSTAGE + kb * TT_VBLK + j * box * 128, &maps.lat,
                                &bars.full[st], kb * 64, row);
            }
        }
    }
    if (lane == 0)
        for (int st = 0; st < TT_NST && st < i; st++)
            mbar_wait_quiet(&bars.full[st], ((i - 1 - st) / TT_NST) & 1);
    __syncwarp();
}

__device__ __forceinline__ void value_mma(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                          TreeBars &bars, uint32_t tbase) {
    constexpr uint32_t id = idesc_f16(128, 256, false, true);
    int g = 0, i = 0, edges = 0;
    TreeSeg sg;
    while (walk.next(sg)) {
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            if (!mbar_wait(&bars.p_full[g & 1], (g >> 1) & 1, a.err, 0x541)) return;
            const bool edge = (long long)(t + 1) * TT_TILE > sg.s.len;
            const uint32_t P = smem_u32(sm + TT_OFF_P + (g & 1) * TT_PBUF);
            for (int c = 0; c < TT_CHUNKS; c++, i++) {
                const int st = i % TT_NST;
                if (!mbar_wait(&bars.full[st], (i / TT_NST) & 1, a.err, 0x542)) return;
                if (edge && !mbar_wait(&bars.clean[c], edges & 1, a.err, 0x543)) return;
                tc_fence_after();
                const uint32_t kv = smem_u32(sm + st * TT_VSTAGE);
#pragma unroll
                for (int ks = 0; ks < TT_VROWS / 16; ks++) {
                    const int k = c * (TT_VROWS / 16) + ks;  // 16 rows of the tile
#pragma unroll
                    for (int h = 0; h < 2; h++)
                        mma_bf16_ss(tbase + 256 * h,
                                    sdesc_kmajor(P + (k >> 2) * (TT_M * 128) + (k & 3) * 32),
                                    sdesc_mnmajor(kv + h * 4 * TT_VBLK + ks * 2048, TT_VBLK), id,
                                    (t == sg.t0 && k == 0) ? 0u : 1u);
                }
                mma_commit(&bars.empty[st]);
            }
            mma_commit_cluster(&bars.pv_done[g & 1], 3);
            edges += edge;
        }
    }
}

__device__ __forceinline__ void value_output(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                             TreeBars &bars, uint32_t tbase, int cl) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q4 = warp & 3, grp = (warp - 2) >> 2;
    const int row = 32 * q4 + lane;
    const uint32_t oaddr = tbase + ((uint32_t)(32 * q4) << 16) + 128 * grp;
    int g = 0, i = 0;
    TreeSeg sg, old;
    while (walk.next(sg)) {
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            const int pb = g & 1, before = (g - 1) & 1, ph = ((g - 1) >> 1) & 1;
            if (warp == 2 && lane == 0) mbar_expect_tx(&bars.p_in[pb], TT_P_BYTES);
            if (t == sg.t0 && g > 0) {  // the last row tile's o, before it is written over
                if (!lane_wait(&bars.pv_done[before], ph, a.err, 0x551)) return;
                tc_fence_after();
                write_o(a, old, cl, oaddr, row, 128 * grp, 128);
            }
            if (!lane_wait<true>(&bars.p_in[pb], (g >> 1) & 1, a.err, 0x552)) return;
            const float f = t == sg.t0 ? 1.f : bars.fac[pb][row];
            if (__any_sync(0xffffffffu, f != 1.f)) {
                if (!lane_wait(&bars.pv_done[before], ph, a.err, 0x553)) return;
                tc_fence_after();
                rescale_o(oaddr, 128, f);
            }
            fence_async_shared();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_full[pb]);
            if ((long long)(t + 1) * TT_TILE <= sg.s.len) {
                i += TT_CHUNKS;
                continue;
            }
            // rows past the cached ones: zero where nothing is written, and where a draft's element
            // is not finite
            for (int c = 0; c < TT_CHUNKS; c++, i++) {
                const int st = i % TT_NST;
                if (!lane_wait(&bars.full[st], (i / TT_NST) & 1, a.err, 0x554)) return;
                const long long d0 = sg.s.len - ((long long)t * TT_TILE + c * TT_VROWS);
                const long long d1 = d0 + sg.s.n;
                uint8_t *kv = sm + st * TT_VSTAGE;
                for (int e = threadIdx.x - 64; e < TT_VROWS * 64; e += TT_WORKERS * 32) {
                    const int r = e / 64, kb = (e / 8) % 8, ch = e % 8;
                    if (r < d0) continue;
                    uint4 *p = reinterpret_cast<uint4 *>(kv + kb * TT_VBLK + r * 128 + ch * 16);
                    uint4 w = make_uint4(0, 0, 0, 0);
                    if (r < d1) {
                        w = *p;
                        w = make_uint4(finite_pair(w.x), finite_pair(w.y), finite_pair(w.z),
                                       finite_pair(w.w));
                    }
                    *p = w;
                }
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars.clean[c]);
            }
        }
        old = sg;
    }
    if (g > 0 && lane_wait(&bars.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, a.err, 0x555)) {
        tc_fence_after();
        write_o(a, old, cl, oaddr, row, 128 * grp, 128);
    }
}

__global__ void __launch_bounds__(TT_THREADS, 1) __cluster_dims__(2, 1, 1)
mla_tree_attend_tc(const __grid_constant__ TreeMaps maps, const __grid_constant__ TreeArgs a) {
    extern __shared__ uint8_t smraw[];
    uint8_t *sm = (uint8_t *)(((uintptr_t)smraw + 1023) & ~(uintptr_t)1023);
    __shared__ TreeBars bars;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool score = cluster_rank() == 0;
    const int cl = blockIdx.x >> 1;
    pdl_trigger();
    pdl_wait();  // the plan, the queries and the cache come from earlier work
    const long long total = a.plan->total;
    const int G = a.plan->G;
    if (cl >= G) return;  // both CTAs of the pair

    if (threadIdx.x == 0) {
        for (int s = 0; s < TT_NST; s++) {
            mbar_init(&bars.full[s], 1);
            mbar_init(&bars.empty[s], 1);
        }
        mbar_init(&bars.q_full, TT_WORKERS);
        mbar_init(&bars.q_empty, 1);
        mbar_init(&bars.s_full, 1);
        mbar_init(&bars.s_empty, TT_WORKERS);
        for (int q = 0; q < 4; q++) mbar_init(&bars.pair[q], 4);
        for (int b = 0; b < 2; b++) {
            mbar_init(&bars.p_in[b], 1);
            mbar_init(&bars.p_full[b], TT_WORKERS);
            mbar_init(&bars.pv_done[b], 1);
        }
        for (int c = 0; c < TT_CHUNKS; c++) mbar_init(&bars.clean[c], TT_WORKERS);
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc(&bars.tmem_base, TT_TM_COLS);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers are ready before anything arrives on them
    tc_fence_after();
    const uint32_t tbase = bars.tmem_base;
    const TreeWalk walk(a, cl, total, G);

    if (warp == 0) {
        if (lane == 0) prefetch_tmap(&maps.lat);
        if (score) score_loads(maps, a, walk, sm, bars);
        else value_loads(maps, a, walk, sm, bars);
    } else if (warp == 1) {
        if (lane == 0) {
            if (score) score_mma(a, walk, sm, bars, tbase);
            else value_mma(a, walk, sm, bars, tbase);
        }
        __syncwarp();
    } else if (score) {
        score_softmax(a, walk, sm, bars, tbase, cl);
    } else {
        value_output(a, walk, sm, bars, tbase, cl);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // nothing of the peer's is on its way into this CTA's shared memory
    if (warp == 1) tmem_dealloc(tbase, TT_TM_COLS);
}

// Join a row tile that several clusters took (the flash-decoding identity), for the cluster in
// which it begins: one block per (cluster, row), thread t owns latent dims 4 t .. 4 t + 3.
__global__ void __launch_bounds__(128) mla_tree_join(const __grid_constant__ TreeArgs a) {
    pdl_trigger();
    pdl_wait();
    const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, G = a.plan->G;
    const long long total = a.plan->total;
    if (c + 1 >= G) return;
    // the row tile that holds the cluster's last place
    const long long end = line_begin(total, G, c + 1);
    const int b = last_at_most(a.cum, a.v.B, end - 1);
    const PagedSeq s = paged_seq(a.v, b, K3CUDA_MAX_DRAFTS);
    const long long cost = TT_FIXED + (s.len + s.n + TT_TILE - 1) / TT_TILE;
    const int mt = (int)((end - 1 - a.cum[b]) / cost);
    const long long first = a.cum[b] + mt * cost + TT_FIXED, last = first + cost - TT_FIXED - 1;
    // cut here, with its first tile in this cluster
    if (end <= first || last < end || first < line_begin(total, G, c)) return;
    const int lr = mt * TT_M + row;
    if (lr >= s.n * a.H) return;
    const int cn = line_cluster(total, G, last);
    const float *base = a.part + (size_t)row * TT_PART;
    const size_t stride = (size_t)2 * TT_M * TT_PART;  // between clusters
    auto part = [&](int k) { return base + k * stride + (k == c ? TT_M * TT_PART : 0); };
    float M = -INFINITY;
    for (int k = c; k <= cn; k++) M = fmaxf(M, part(k)[TT_DL]);
    float L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = c; k0 <= cn; k0 += 4) {
        float4 v[4];
        float w[4], pl[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            w[u] = pl[u] = 0.f;
            v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (k0 + u <= cn) {
                const float *p = part(k0 + u);
                const float m = p[TT_DL];
                pl[u] = p[TT_DL + 1];
                w[u] = m == -INFINITY && pl[u] == 0.f ? 0.f : exp2f(m - M);
                v[u] = reinterpret_cast<const float4 *>(p)[tid];
            }
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            L += w[u] * pl[u];
            o.x += w[u] * v[u].x; o.y += w[u] * v[u].y; o.z += w[u] * v[u].z; o.w += w[u] * v[u].w;
        }
    }
    const float ov[4] = {o.x, o.y, o.z, o.w};
    float lo[4];
#pragma unroll
    for (int i = 0; i < 4; i++) lo[i] = ov[i] - __bfloat162float(__float2bfloat16_rn(ov[i]));
    const size_t th = (size_t)s.first * a.H + lr;
    __nv_bfloat16 *dst = a.olat2 + th * 2 * TT_DL;
    reinterpret_cast<uint2 *>(dst)[tid] = make_uint2(pack_bf2(ov[0], ov[1]), pack_bf2(ov[2], ov[3]));
    reinterpret_cast<uint2 *>(dst + TT_DL)[tid] =
        make_uint2(pack_bf2(lo[0], lo[1]), pack_bf2(lo[2], lo[3]));
    if (tid == 0) a.rowsum[th] = L;
}

static int tree_shape(int B, int T, int H, int dn, int dr, int dl, int dv) {
    K3_ARG_CHECK(B >= 0 && T >= 0 && H >= 1 && H <= TT_H && B < (1 << 24),
                 "mla_tree_attend: bad B=%d T=%d H=%d", B, T, H);
    if (dn != TT_DN || dr != TT_DR || dl != TT_DL || dv != TT_DV)
        return set_error(K3CUDA_ERR_UNSUPPORTED,
                         "mla_tree_attend: dn=%d dr=%d dl=%d dv=%d not built", dn, dr, dl, dv);
    K3_ARG_CHECK(T < (1 << 23), "mla_tree_attend: T=%d", T);
    return K3CUDA_OK;
}

// The workspace: plan, cum [B + 1], keep [T], queries, partials, o as hi/lo pairs, row sums.
struct TreeWs {
    size_t cum, keep, qlat, part, olat2, rowsum, total;
};
static TreeWs tree_ws(int B, int T, int H) {
    size_t off = 0;
    auto take = [&](size_t n) {
        const size_t o = off;
        off += (n + 255) & ~(size_t)255;
        return o;
    };
    TreeWs w;
    take(sizeof(TreePlan));
    w.cum = take(((size_t)B + 1) * sizeof(long long));
    w.keep = take((size_t)T * sizeof(int));
    w.qlat = take((size_t)T * H * TT_QW * 2);
    w.part = take((size_t)2 * TT_CLUSTERS * TT_M * TT_PART * sizeof(float));
    w.olat2 = take((size_t)T * H * 2 * TT_DL * 2);
    w.rowsum = take((size_t)T * H * sizeof(float));
    w.total = off;
    return w;
}

}  // namespace k3

using namespace k3;

extern "C" int k3cuda_mla_tree_attend_workspace(int B, int T, int H, int dl, int dv,
                                                size_t *bytes) {
    K3_ARG_CHECK(bytes, "mla_tree_attend: null bytes");
    int rc = tree_shape(B, T, H, TT_DN, TT_DR, dl, dv);
    if (rc) return rc;
    *bytes = B == 0 || T == 0 ? 0 : tree_ws(B, T, H).total;
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
    const int B = batch->B, T = batch->T;
    if (B == 0 || T == 0) return enter(ctx);
    K3_ARG_CHECK(out && q_nope && q_rope && w_uk && w_uv, "%s: null pointer", what);
    const void *al[] = {out, q_nope, q_rope, w_uk, w_uv};
    for (const void *p : al)
        K3_ARG_CHECK(aligned(p, 16), "%s: pointers must be 16-byte aligned", what);
    K3_ARG_CHECK(aligned(tree_mask, 8), "%s: tree_mask must be 8-byte aligned", what);
    const TreeWs ws = tree_ws(B, T, H);
    if (!workspace || workspace_bytes < ws.total)
        return set_error(K3CUDA_ERR_WORKSPACE, "%s: workspace %zu < %zu", what, workspace_bytes,
                         ws.total);
    K3_ARG_CHECK(aligned(workspace, 256), "%s: workspace must be 256-byte aligned", what);
    if ((rc = enter(ctx))) return rc;

    char *w = (char *)workspace;
    TreePlan *plan = (TreePlan *)w;
    long long *cum = (long long *)(w + ws.cum);
    int *keep = (int *)(w + ws.keep);
    __nv_bfloat16 *qlat = (__nv_bfloat16 *)(w + ws.qlat);
    const TreeArgs a{paged_view(cache, batch), plan, cum, tree_mask, qlat,
                     (float *)(w + ws.part), (__nv_bfloat16 *)(w + ws.olat2),
                     (float *)(w + ws.rowsum), H, scale * 1.4426950408889634f, ctx->err_word};
    const uint64_t rows = (uint64_t)cache->n_pages * cache->page_size;
    const uint32_t box = cache->page_size < TT_BOX ? cache->page_size : TT_BOX;
    const CUtensorMapDataType BF = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    TreeMaps maps;
    rc = make_tmap_2d(&maps.lat, cache->latent, BF, 2, TT_DL, rows, TT_DL * 2, 64, box);
    if (!rc) rc = make_tmap_2d(&maps.rope, cache->rope, BF, 2, TT_DR, rows, TT_DR * 2, 64, box);
    if (rc || (rc = set_smem(mla_tree_attend_tc, TT_SMEM))) return rc;

    int clusters = ctx->sm_count / 2;
    if (clusters > TT_CLUSTERS) clusters = TT_CLUSTERS;
    if (clusters < 1) clusters = 1;
    rc = launch_pdl(ctx, ctx->stream, "mla_tree_plan", mla_tree_plan, dim3(1), dim3(1024), 0, a.v, H,
                    plan, cum, keep, clusters, ctx->err_word);
    if (!rc) rc = mla_absorb(ctx, qlat, H, q_nope, q_rope, w_uk, TT_DN, T, H);
    if (!rc)
        rc = launch_pdl(ctx, ctx->stream, "mla_tree_attend_tc", mla_tree_attend_tc,
                        dim3(2 * clusters), dim3(TT_THREADS), TT_SMEM, maps, a);
    if (!rc)
        rc = launch_pdl(ctx, ctx->stream, "mla_tree_join", mla_tree_join, dim3(clusters, TT_M),
                        dim3(128), 0, a);
    if (!rc)
        rc = mla_project(ctx, out, out_dtype, a.olat2, a.rowsum, keep, w_uv, TT_DV, T, H);
    return rc;
}
