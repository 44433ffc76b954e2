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
// cluster of two CTAs with one job each. The score CTA holds the query in TMEM (the A operand; its
// rope dims in shared memory), streams the tile's 576-wide rows, forms S and the softmax, and sends
// the weights P to its peer as bf16, with the factor by which o is to be rescaled. The value CTA
// streams the same rows' 512 latent dims, from L2 by then, and accumulates o. S and P are
// double-buffered, so neither CTA waits for the other in step.
// What decides this layout (measured on a B200, cycles of an SM):
//   * cluster stores move 17 B a clock and SM, TMA reads from L2 over 70. Splitting the dims over the
//     pair instead (each row read once, partial scores and P exchanged, 36 KB per 96 rows and CTA)
//     is bound by the former: 5400 cycles per 96 rows.
//   * an MMA (M 128, A in TMEM) takes 74 cycles at N = 128 and 37 at N = 64, and the queue before the
//     tensor core is a few MMAs deep: a wait of the issuing warp or a slow issue shows as idle tensor
//     time. So tiles are 128 rows (N = 128: 64-row tiles took 5600 cycles per 128 rows), each chunk's
//     barrier is looked at before the chunk before is fully issued, and P leaves by bulk copy (16-byte
//     cluster stores from the softmax warps held up the MMAs behind them: +480 cycles per 64 rows).
//   * a TMA instruction takes about 115 cycles to issue whatever it moves (4 KB boxes: 35 B a clock),
//     so a chunk comes in one, through a four-dimensional view of the cache that lays eight-row
//     groups [dim blocks][8 rows][128 B] one after another; pages of fewer rows take one each.
// Per SM:
//   score   TMEM: query 256 columns, S 2 x 128;  shared: 5 stages of 32 KB (128 rows x 128 dims,
//           K-major, a quarter of a tile), the tile's rope dims 16 KB, the query's 16 KB, P 32 KB on its
//           way out (four stages and no reading ahead in the page table: 64 x 1 193 us back to
//           back, now 184)
//   value   TMEM: o 512 columns;  shared: a tile in 4 stages of 32 KB (32 rows x 512 dims, MN-major),
//           P 2 x 32 KB
// Warps: 0 loads (a lane per page), 1 issues the MMAs, 2-9 are two groups of one warp per lane
// quarter: in the score CTA a group takes 64 score columns of all rows, in the value CTA 256 dims
// of o (rescaling, read-out). Warp 10 of the score CTA sends P, that of the value CTA brings rows into
// L2. The warps share four schedulers, and
// the score CTA's are busy half the time: sixteen softmax warps of 32 columns each slowed the loads
// and the MMA issue by more than they gained.
//
// Work: the (row tile, cache tile) pairs lie on a line, every row tile taking some more places for
// its fixed work; clusters take equal pieces (paged.cuh). A row tile that one cluster does
// whole is written as (o, l); one that is cut leaves partial (m, l, o) that mla_tree_join joins.
// The line is formed on the device from the batch's tables (mla_tree_plan), so that a captured
// call follows them.
//
// Measured (the five launches of a call, the caches cold; in brackets calls back to back): 64 x 1 token of
// 128 heads over 8192 rows 218 us (184), of which this kernel 153 (its floor is 97 us of HBM and 91 of
// MMAs); 48 x up to 13 tokens, 128 heads, 393 to 406 us (350 to 383) as the clock allows (294 in this
// kernel; 181 us of MMAs); one token after 509 rows 25 us (26). A tile takes about 4250 cycles where its
// MMAs in the score CTA need 2650. 3870 of the 4250 are the SM's own: so much it takes with 12 clusters at
// work instead of 74. What it waits for are the rows: 910 cycles for 10 TMA instructions (two pages of 64
// rows, 91 cycles each; 18 instructions, a block of 64 dims each: 4600 cycles a tile), and 147 KB of rows
// in the other 2960, 50 B a clock, beside the MMAs' reads of them and P in shared memory's 128. A row
// tile's start and end take some 14000 cycles.
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
constexpr int TT_KCH = 4, TT_VCH = 4;      // chunks of a tile: by dims, by rows
constexpr int TT_KST = 5, TT_VST = TT_VCH; // stages, a chunk each
constexpr int TT_KSTAGE = TT_TILE * TT_DL * 2 / TT_KCH;
constexpr int TT_VROWS = TT_TILE / TT_VCH;
constexpr int TT_VSTAGE = TT_VROWS * TT_DL * 2;
constexpr int TT_AHEAD = 3;                // tiles that rows are brought into L2 before their load
constexpr int TT_PACE = 1600;              // ns between the first of them
constexpr int TT_PBUF = 2 * TT_M * 128;    // two blocks of 64 columns
constexpr int TT_OFF_KR = TT_KST * TT_KSTAGE;     // score: rope dims of the tile
constexpr int TT_OFF_QR = TT_OFF_KR + TT_TILE * 128;  // and of the query
constexpr int TT_OFF_PS = TT_OFF_QR + TT_M * 128;     // P on its way out
constexpr int TT_OFF_FS = TT_OFF_PS + TT_PBUF;        // its rescale factors
constexpr int TT_GRP = 2;                  // groups of worker warps, one warp per lane quarter each
constexpr int TT_OFF_VAL = TT_OFF_FS + TT_M * 4;      // values shared by a row's warps
constexpr int TT_OFF_P = TT_VST * TT_VSTAGE;      // value: P, two buffers
constexpr int TT_OFF_F = TT_OFF_P + 2 * TT_PBUF;  // and their factors
constexpr int TT_OFF_W = TT_OFF_F + 1024;         // o on its way out, 4 KB a warp
constexpr int TT_SMEM_SCORE = TT_OFF_VAL + 2 * TT_GRP * TT_M * 4;
constexpr int TT_SMEM_VALUE = TT_OFF_W + 4 * TT_GRP * 4096;
constexpr int TT_OFF_BARS = TT_SMEM_SCORE > TT_SMEM_VALUE ? TT_SMEM_SCORE : TT_SMEM_VALUE;
static_assert(TT_OFF_W % 1024 == 0 && 2 * TT_M * 4 <= 1024, "the stages are swizzled");

constexpr int TT_TM_Q = 0, TT_TM_S = 256, TT_TM_COLS = 512;
constexpr int TT_CW = TT_TILE / TT_GRP;    // score columns of a softmax warp
constexpr int TT_OW = TT_DL / TT_GRP;      // dims of o of a warp in the value CTA
constexpr int TT_WORKERS = 4 * TT_GRP;     // warps 2 ..
constexpr int TT_THREADS = (3 + TT_WORKERS) * 32;
constexpr int TT_CLUSTERS = 74;            // 148 SMs of a B200
constexpr int TT_DRAIN = 1 << 17;          // clocks that a CTA stays after a wait that ran out
constexpr int TT_FIXED = 4;                // a row tile's fixed work, in tiles
// a partial, in floats: o [dims / 4][rows][4], m [rows], l [rows]
constexpr int TT_PART_M = TT_DL * TT_M, TT_PART_L = TT_PART_M + TT_M, TT_PART = TT_PART_L + TT_M;
// A row tile that is cut: the clusters with the first and the last part of it, its rows, and its first
// row among all (token, head) rows.
struct TreeCut {
    int first, last, rows;
    long long row0;
};

// Where a cluster's piece of the line begins: a row tile and its first place.
struct TreeStart {
    int b, mt;
    long long at;
};

// the device-side plan, at the start of the workspace
struct TreePlan {
    long long total;   // places on the line
    int B;             // sequences that count
    int G;             // clusters that take part
    int fixed;         // places of a row tile's fixed work
    int cuts;
    TreeCut cut[TT_CLUSTERS];
    TreeStart start[TT_CLUSTERS];
};

struct TreeArgs {
    PagedView v;
    const TreePlan *plan;
    const long long *cum;      // the sequences' first places
    const unsigned long long *mask;
    const __nv_bfloat16 *latent, *rope;  // the cache's rows
    float *part;               // [2 TT_CLUSTERS][TT_PART]
    __nv_bfloat16 *olat2;      // [T][H][hi 512 | lo 512]
    float *rowsum;             // [T][H]
    int H;
    float scale_log2e;
    unsigned *err;
};

struct TreeMaps {
    CUtensorMap lat_k, lat_v, rope, q, q_rope;
};

// A cluster's next piece of the line: tiles t0 .. t1 - 1 of row tile mt of sequence b.
struct TreeSeg {
    int b, mt, t0, t1, tiles;
    PagedSeq s;
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == tiles; }
    // the partial's slot: the even one of a cluster for a row tile that began in an earlier cluster
    __device__ __forceinline__ int slot(int c) const { return 2 * c + (t0 == 0 ? 1 : 0); }
};

// The sequence that holds a place of the line (a step at a time, millions of empty ones took longer than
// a wait may). Not expanded into the roles, which seldom need it.
__device__ __noinline__ int tree_find(const long long *cum, int B, long long x) {
    return last_at_most(cum, B, x);
}

struct TreeWalk {
    const TreeArgs &a;
    long long c0, c1, at;  // this cluster's places; the next row tile's first place
    int b, mt, units, fixed;
    long long cost;
    PagedSeq s;
    __device__ __forceinline__ void seq() {
        s = paged_seq(a.v, b, K3CUDA_MAX_DRAFTS);
        units = (int)(((long long)s.n * a.H + TT_M - 1) / TT_M);
        cost = fixed + (s.len + s.n + TT_TILE - 1) / TT_TILE;
    }
    __device__ __forceinline__ TreeWalk(const TreeArgs &args, int c, long long total, int G)
        : a(args), c0(line_begin(total, G, c)), c1(line_begin(total, G, c + 1)) {
        const TreeStart first = a.plan->start[c];
        fixed = a.plan->fixed;
        b = first.b;
        mt = first.mt;
        at = first.at;
        seq();
    }
    __device__ __forceinline__ bool next(TreeSeg &g) {
        while (at < c1) {
            if (mt >= units) {  // the next sequence with tokens, the one that holds place `at`
                if (++b >= a.v.B) return false;
                mt = 0;
                seq();
                if (units == 0) {
                    b = tree_find(a.cum, a.plan->B, at);
                    seq();
                }
                continue;
            }
            const long long first = at + fixed;  // place of tile 0
            g.b = b;
            g.mt = mt;
            g.s = s;
            g.tiles = (int)(cost - fixed);
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
// It runs beside mla_absorb, whose CTAs let it start once what came before is done, and waits for that
// kernel at its end, so that the attention waits for both.
__global__ void __launch_bounds__(1024) mla_tree_plan(PagedView v, int H, TreePlan *plan,
                                                      long long *cum, int *keep, int clusters,
                                                      unsigned *err) {
    __shared__ long long wsum[32], carry, all;
    __shared__ int ordered;
    pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int t = tid; t < v.T; t += 1024) keep[t] = 0;
    if (tid == 0) {
        carry = all = 0;
        ordered = v.B;
    }
    __syncthreads();
    long long tiles;
    for (;;) {
        tiles = 0;
        for (int b = tid; b < v.B; b += 1024) {
            const PagedSeq s = paged_seq(v, b, K3CUDA_MAX_DRAFTS);
            if (s.code) atomicCAS(err + 1, 0u, (unsigned)s.code);
            if (!paged_in_order(v, b)) atomicMin(&ordered, b);
            tiles += ((long long)s.n * H + TT_M - 1) / TT_M * ((s.len + s.n + TT_TILE - 1) / TT_TILE);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
        if (lane == 0) atomicAdd((unsigned long long *)&all, (unsigned long long)tiles);
        __syncthreads();
        tiles = all;
        if (ordered == v.B) break;
        v.B = ordered;  // once more without the sequences from the first that is out of order
        __syncthreads();
        if (tid == 0) all = 0;
        __syncthreads();
    }
    // A cluster has one tile at least. With no more than that for each, a row tile's fixed work is
    // left out of account, or the clusters that its places fall to would have no tile.
    const int G = (int)(tiles < clusters ? tiles : clusters);
    const int fixed = tiles > clusters ? TT_FIXED : 0;
    for (int b0 = 0; b0 < v.B; b0 += 1024) {
        const int b = b0 + tid;
        long long cost = 0;
        if (b < v.B) {
            const PagedSeq s = paged_seq(v, b, K3CUDA_MAX_DRAFTS);
            for (int i = 0; i < s.n; i++) keep[s.first + i] = 1;
            const long long units = ((long long)s.n * H + TT_M - 1) / TT_M;
            cost = units * (fixed + (s.len + s.n + TT_TILE - 1) / TT_TILE);
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
    if (tid == 0) {
        cum[v.B] = carry;
        plan->total = carry;
        plan->B = v.B;
        plan->G = G;
        plan->fixed = fixed;
    }
    __syncthreads();
    // the row tile that holds each cluster's first place
    const long long total = carry;
    if (tid < G) {
        TreeStart start;
        const long long c0 = line_begin(total, G, tid);
        start.b = last_at_most(cum, v.B, c0);
        const PagedSeq s = paged_seq(v, start.b, K3CUDA_MAX_DRAFTS);
        const long long cost = fixed + (s.len + s.n + TT_TILE - 1) / TT_TILE;
        start.mt = (int)((c0 - cum[start.b]) / cost);
        start.at = cum[start.b] + start.mt * cost;
        plan->start[tid] = start;
    }
    __shared__ TreeCut cut[TT_CLUSTERS];
    if (tid < TT_CLUSTERS) {
        cut[tid].last = -1;
        if (tid + 1 < G) {
            const long long end = line_begin(total, G, tid + 1);
            const int b = last_at_most(cum, v.B, end - 1);
            const PagedSeq s = paged_seq(v, b, K3CUDA_MAX_DRAFTS);
            const long long cost = fixed + (s.len + s.n + TT_TILE - 1) / TT_TILE;
            const int mt = (int)((end - 1 - cum[b]) / cost);
            const long long first = cum[b] + mt * cost + fixed, last = first + cost - fixed - 1;
            // some of its tiles are in this cluster, the first among them, and some are not
            if (first < end && end <= last && first >= line_begin(total, G, tid)) {
                cut[tid].first = tid;
                cut[tid].last = line_cluster(total, G, last);
                cut[tid].rows = min(TT_M, s.n * H - mt * TT_M);
                cut[tid].row0 = (long long)s.first * H + mt * TT_M;
            }
        }
    }
    __syncthreads();
    if (tid < TT_CLUSTERS) {
        int at = 0;
        for (int c = 0; c < tid; c++) at += cut[c].last >= 0;
        if (cut[tid].last >= 0) plan->cut[at++] = cut[tid];
        if (tid + 1 == TT_CLUSTERS) plan->cuts = at;
    }
    pdl_wait();
}

struct TreeBars {  // at TT_OFF_BARS
    uint64_t full[TT_KST], empty[TT_KST];  // stages
    uint64_t r_full, r_empty;              // score: the tile's rope dims
    uint64_t s_full[2], s_empty[2];        // score
    uint64_t pair[4];                      // score: per lane quarter, its two warps
    uint64_t p_out, p_ack;                 // score: P is written; the peer has it
    uint64_t p_in[2], p_full[2];           // value: P has come; o is ready for it
    uint64_t pv_done[2];                   // both: o of the tile is done, P's buffer free
    uint64_t clean[TT_VCH];                // value: stages that reach past the cached rows
    uint32_t tmem_base;
    int tile;                              // value: the tile being loaded
};
constexpr int TT_SMEM = TT_OFF_BARS + sizeof(TreeBars);
static_assert(TT_SMEM <= 232448, "all that a block can have, without slack for the alignment");
static_assert(TT_VST <= TT_KST, "the value CTA's stages have barriers");

// n columns of o from addr: multiply by f
__device__ __forceinline__ void rescale_o(uint32_t addr, int n, float f) {
#pragma unroll 1
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

// A segment's o, latent dims dim .. dim + n - 1 (TMEM columns from addr) of the warp's 32 rows from
// row0. A lane reads its row from TMEM. A partial is laid out for that: 16 bytes of 32 rows follow one
// another. A whole row tile goes out as the projection's bf16 hi/lo pair, through 4 KB of shared memory,
// so that 64 bytes of a row are stored at a time (stored from the lanes, 16 bytes of 32 rows each, this
// took 20000 cycles; through shared memory 13000; a partial takes 9000). Either is 256 KB of an SM, beside
// the loads of the next tiles.
// The loops stay rolled: what runs once per row tile is not in the instruction cache, and every 128
// bytes of it cost some 250 cycles.
__device__ __forceinline__ void write_o(const TreeArgs &a, const TreeSeg &g, int cl, uint32_t addr,
                                        uint8_t *stage, int row0, int dim, int n) {
    const int lane = threadIdx.x & 31, j = lane & 7;
    const int rows = min(32, g.s.n * a.H - (g.mt * TT_M + row0));  // that exist
    if (!g.whole()) {
        float4 *dst = reinterpret_cast<float4 *>(a.part + (size_t)g.slot(cl) * TT_PART) +
                      dim / 4 * TT_M + row0 + lane;
#pragma unroll 1
        for (int c = 0; c < n; c += 16, dst += 4 * TT_M) {
            float v[16];
            tmem_ld16(addr + c, v);
            tmem_wait_ld();
            if (lane < rows) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    dst[i * TT_M] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
        }
        return;
    }
    // this lane's 16-byte chunk of rows lane / 8, + 4, ..: of 32 hi and 32 lo halves
    char *dst = reinterpret_cast<char *>(
        a.olat2 + ((size_t)g.s.first * a.H + g.mt * TT_M + row0) * 2 * TT_DL + dim);
    dst += (j & 3) * 16 + (j >> 2) * TT_DL * 2 + (lane >> 3) * TT_DL * 4;
    float v[32];
    tmem_ld32(addr, v);
#pragma unroll 1
    for (int c = 0; c < n; c += 32, dst += 64) {
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint4 hi = pack_bf8(v + 8 * i);
            float h[8], lo[8];
            unpack_bf8(hi, h);
#pragma unroll
            for (int k = 0; k < 8; k++) lo[k] = v[8 * i + k] - h[k];
            st16s(stage + swz(lane, i), hi);
            st16s(stage + swz(lane, 4 + i), pack_bf8(lo));
        }
        __syncwarp();
        if (c + 32 < n) tmem_ld32(addr + c + 32, v);  // under the copy
        uint4 w[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            w[i] = *reinterpret_cast<const uint4 *>(stage + swz(4 * i + (lane >> 3), j));
        __syncwarp();
        char *d = dst;
#pragma unroll
        for (int i = 0; i < 8; i++, d += 4 * TT_DL * 4)
            if (4 * i + (lane >> 3) < rows) *reinterpret_cast<uint4 *>(d) = w[i];
    }
}

// Zero what a draft row of bf16 pairs holds that is not finite.
__device__ __forceinline__ uint32_t finite_pair(uint32_t u) {
    if ((u & 0x7f80u) == 0x7f80u) u &= 0xffff0000u;
    if ((u & 0x7f800000u) == 0x7f800000u) u &= 0xffffu;
    return u;
}

// A CTA's loads, chunk by chunk: for the score CTA 128 rows x 128 latent dims, the rope dims with
// the first; for the value CTA 32 rows x 512 dims. Chunk c of every tile is in stage c. In the score
// CTA a row tile's queries come through the same stages before its first tile.
template <bool kScore>
__device__ __forceinline__ bool tree_loads(const TreeMaps &maps, const TreeArgs &a, TreeWalk walk,
                                           uint8_t *sm, TreeBars &bars) {
    constexpr int CH = kScore ? TT_KCH : TT_VCH, ROWS = kScore ? TT_TILE : TT_VROWS;
    constexpr int ST = kScore ? TT_KST : TT_VST;
    constexpr int STAGE = kScore ? TT_KSTAGE : TT_VSTAGE, RB = STAGE / ROWS;  // bytes of a row
    const int lane = threadIdx.x & 31;
    const int box = min(a.v.page_size, ROWS), per = ROWS / box;  // rows of a box, boxes of a chunk
    int g = 0, loaded = 0;  // tiles; stages in use, and their phase
    int st = 0, fill = 0;   // the next stage and how often it was filled
    int ropes = 0;          // tiles whose rope dims are loaded
    // This lane's box of a tile: its page, read a tile before it is looked at (the read takes 700 cycles
    // and more behind the TMA's traffic, and what waits for it holds up the loads), and its first cache
    // row (of page 0 where the table names no page).
    auto box_page = [&](const TreeSeg &sg, int t) -> int {
        const int p = t * TT_TILE + lane * box;
        if (lane >= TT_TILE / box || p >= sg.s.len + sg.s.n) return 0;
        return a.v.table[(long long)sg.b * a.v.max_pages + (p >> a.v.shift)];
    };
    auto box_row = [&](int page, int t) -> int {
        if (page < 0 || page >= a.v.n_pages) {
            if (kScore) atomicCAS(a.err + 1, 0u, (unsigned)PAGED_PAGE);
            page = 0;
        }
        return (page << a.v.shift) + ((t * TT_TILE + lane * box) & (a.v.page_size - 1));
    };
    auto free = [&] { return fill == 0 || warp_spin(&bars.empty[st], (fill - 1) & 1, a.err, 0x501); };
    auto next = [&] {
        loaded = (loaded & ~(3 << (2 * st))) | ((fill & 1 ? 2 : 1) << (2 * st));
        if (++st == ST) st = 0, fill++;
    };
    // the last tile's products with its rope dims are done
    auto rope_free = [&] { return g == 0 || warp_spin(&bars.r_empty, (g - 1) & 1, a.err, 0x502); };
    TreeSeg sg;
    bool more = walk.next(sg), ok = true;
    int t = more ? sg.t0 : 0, page = more ? box_page(sg, t) : 0;
    for (; more && ok; g++) {
        const int live = (sg.s.len + sg.s.n - t * TT_TILE + box - 1) / box, at = box_row(page, t);
        if (!kScore && lane == 0) *(volatile int *)&bars.tile = g;
        if (kScore && t == sg.t0) {
            const int q0 = sg.s.first * a.H + sg.mt * TT_M;
#pragma unroll 1
            for (int c = 0; c < CH && (ok = free()); c++) {
                const bool rope = c == CH - 1;  // as late as may be: its place is in use longest
                if (rope && !(ok = rope_free())) break;
                if (lane == 0) {
                    mbar_expect_tx(&bars.full[st], STAGE + (rope ? TT_M * 128 : 0));
                    tma_load_3d(sm + st * STAGE, &maps.q, &bars.full[st], 0, q0, 2 * c);
                    if (rope) tma_load_2d(sm + TT_OFF_QR, &maps.q_rope, &bars.full[st], TT_DL, q0);
                }
                __syncwarp();
                next();
            }
            if (!ok) break;
        }
        const bool last = t + 1 >= sg.t1;
        if (!last) page = box_page(sg, ++t);
#pragma unroll 1
        for (int c = 0; c < CH && (ok = free()); c++) {
            // the lanes whose boxes this chunk takes: all of them, or those of its rows
            const int first = kScore ? 0 : c * per, j = lane - first;
            const int n = max(0, min(per, live - first));
            if (lane == 0) mbar_expect_tx(&bars.full[st], n * box * RB);
            __syncwarp();
            if (j >= 0 && j < n)
                tma_load_4d(sm + st * STAGE + j * box * RB, kScore ? &maps.lat_k : &maps.lat_v,
                            &bars.full[st], 0, 0, kScore ? c * (RB / 128) : 0, at / 8);
            next();
            if (kScore && c == 0) {
                if (!(ok = rope_free())) break;
                if (lane == 0) mbar_expect_tx(&bars.r_full, n * box * 128);
                __syncwarp();
                if (j < n)
                    tma_load_2d(sm + TT_OFF_KR + j * box * 128, &maps.rope, &bars.r_full, 0, at);
                ropes++;
            }
        }
        if (last) {
            more = walk.next(sg);
            t = more ? sg.t0 : 0;
            page = more ? box_page(sg, t) : 0;
        }
    }
    // loads still in flight are waited for (bounded) before the CTA may exit
    if (ropes && lane == 0) mbar_wait_quiet(&bars.r_full, (ropes - 1) & 1);
    if (lane == 0)
        for (int c = 0; c < ST; c++)
            if ((loaded >> (2 * c)) & 3) mbar_wait_quiet(&bars.full[c], (loaded >> (2 * c)) & 2 ? 1 : 0);
    __syncwarp();
    return ok;
}

// ---------------------------------------------------------------- score CTA
__device__ __forceinline__ bool score_mma(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                          TreeBars &bars, uint32_t tbase) {
    constexpr uint32_t id = idesc_f16(128, TT_TILE, false, false);
    int g = 0, st = 0;                              // tiles; the next stage
    uint32_t ph = 0;                                // and its phase
    bool data = false, rope = false, room = true;   // next chunk, rope dims, score buffer: as seen before
    auto next = [&] {
        if (++st == TT_KST) st = 0, ph ^= 1;
    };
    TreeSeg sg;
    while (walk.next(sg)) {
        // The queries into TMEM, 16 dims at a time, once the last row tile's scores are formed. (Taken
        // there by the softmax warps, a row tile's first scores came 5000 cycles later.)
        if (g > 0 && !warp_spin(&bars.s_full[(g - 1) & 1], ((g - 1) >> 1) & 1, a.err, 0x511))
            return false;
#pragma unroll 1
        for (int c = 0; c < TT_KCH; c++) {
            if (!data && !warp_spin(&bars.full[st], ph, a.err, 0x514)) return false;
            tc_fence_after();
            uint64_t q = sdesc_kmajor(smem_u32(sm + st * TT_KSTAGE));
            uint32_t d = tbase + TT_TM_Q + 64 * c;
#pragma unroll 1
            for (int half = 0; half < 2; half++, q += (TT_M * 128) >> 4, d += 32) {
#pragma unroll
                for (int ks = 0; ks < 4; ks++) warp_copy(d + ks * 8, q + ks * (32 >> 4));
            }
            warp_commit(&bars.empty[st]);
            next();
            data = false;
        }
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            const int sb = g & 1;
            const uint32_t d = tbase + TT_TM_S + sb * TT_TILE;
            uint32_t q = tbase + TT_TM_Q;
            if (!room && !warp_spin(&bars.s_empty[sb], ((g >> 1) - 1) & 1, a.err, 0x512))
                return false;
            if (!rope && !warp_spin(&bars.r_full, g & 1, a.err, 0x515)) return false;
            tc_fence_after();
            {
                const uint64_t qr = sdesc_kmajor(smem_u32(sm + TT_OFF_QR));
                const uint64_t kr = sdesc_kmajor(smem_u32(sm + TT_OFF_KR));
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
                    warp_mma_ss(d, qr + ks * (32 >> 4), kr + ks * (32 >> 4), id, ks ? 1u : 0u);
                warp_commit(&bars.r_empty);
            }
#pragma unroll 1
            for (int c = 0; c < TT_KCH; c++) {
                if (!data && !warp_spin(&bars.full[st], ph, a.err, 0x513)) return false;
                tc_fence_after();
                uint64_t b = sdesc(smem_u32(sm + st * TT_KSTAGE), 16, 2048);
                const int used = st;
#pragma unroll
                for (int ks = 0; ks < 4; ks++) warp_mma_ts(d, q + ks * 8, b + ks * (32 >> 4), id, 1u);
                next();
                data = __all_sync(0xffffffffu, mbar_test(&bars.full[st], ph));
                if (c + 1 == TT_KCH) {
                    rope = __all_sync(0xffffffffu, mbar_test(&bars.r_full, (g + 1) & 1));
                    room = g < 1 || __all_sync(0xffffffffu, mbar_test(&bars.s_empty[sb ^ 1],
                                                                          (((g + 1) >> 1) - 1) & 1));
                }
                q += 32;
                b += 1024 >> 4;
#pragma unroll
                for (int ks = 0; ks < 4; ks++) warp_mma_ts(d, q + ks * 8, b + ks * (32 >> 4), id, 1u);
                q += 32;
                if (c + 1 == TT_KCH) warp_commit(&bars.s_full[sb]);
                warp_commit(&bars.empty[used]);
            }
        }
    }
    return true;
}

__device__ __forceinline__ bool score_softmax(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                              TreeBars &bars, uint32_t tbase, int cl) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q4 = warp & 3, grp = (warp - 2) >> 2;  // lane quarter, group
    const int row = 32 * q4 + lane;                  // row of the row tile = TMEM lane
    const int c0 = TT_CW * grp;                      // first score column
    const uint32_t laddr = tbase + ((uint32_t)(32 * q4) << 16);
    uint8_t *P = sm + TT_OFF_PS + grp * (TT_M * 128);  // this warp's 64-column block
    float *val = reinterpret_cast<float *>(sm + TT_OFF_VAL) + row;  // [2][TT_GRP][TT_M]
    // Scores are scaled to log2 units with the maximum's subtraction, by a positive factor, so that a
    // masked -inf stays one; the sign of a negative scale, or a scale of zero, is taken before.
    const float sign = a.scale_log2e > 0.f ? 1.f : a.scale_log2e < 0.f ? -1.f : 0.f;
    const float scale = a.scale_log2e == 0.f ? 1.f : fabsf(a.scale_log2e);
    float m_ref = -INFINITY, l = 0.f;  // l: this warp's columns
    int g = 0, np = 0;
    // the other warp's value of the row
    auto share = [&](float v, float &o) -> bool {
        float *at = val + (np & 1) * TT_GRP * TT_M;
        at[grp * TT_M] = v;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.pair[q4]);
        if (!warp_spin(&bars.pair[q4], np & 1, a.err, 0x521)) return false;
        o = at[(grp ^ 1) * TT_M];
        np++;
        return true;
    };
    TreeSeg sg;
    while (walk.next(sg)) {
        // the word of this row's token
        const int tok = min((sg.mt * TT_M + row) / a.H, sg.s.n - 1);
        const uint64_t word = a.mask ? a.mask[sg.s.first + tok] : (((uint64_t)2 << tok) - 1);
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            const int sb = g & 1;
            float s[TT_CW];
            if (!warp_spin(&bars.s_full[sb], (g >> 1) & 1, a.err, 0x523)) return false;
            tc_fence_after();
            const int p0 = t * TT_TILE + c0;
            if (p0 + TT_CW > sg.s.len || sign != 1.f) {  // past the cached rows: masked in TMEM
                const uint64_t see = tree_bits(word, sg.s.len, sg.s.n, p0);
                const int d0 = sg.s.len - p0;
#pragma unroll 1
                for (int c = 0; c < TT_CW; c += 16) {
                    float x[16];
                    tmem_ld16(laddr + TT_TM_S + sb * TT_TILE + c0 + c, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        x[i] *= sign;
                        if (c + i >= d0 && !(fabsf(x[i]) < INFINITY)) x[i] = NAN;
                        if (!((see >> (c + i)) & 1)) x[i] = -INFINITY;
                    }
                    tmem_st16(laddr + TT_TM_S + sb * TT_TILE + c0 + c, x);
                }
                tmem_wait_st();
            }
            tmem_ld32(laddr + TT_TM_S + sb * TT_TILE + c0, s);
            tmem_ld32(laddr + TT_TM_S + sb * TT_TILE + c0 + 32, s + 32);
            tmem_wait_ld();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.s_empty[sb]);
            float m4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int i = 4; i < TT_CW; i += 8)
#pragma unroll
                for (int j = 0; j < 4; j++) m4[j] = max3(m4[j], s[i + j], i + 4 < TT_CW ? s[i + 4 + j] : s[i + j]);
            float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * scale, o;
            if (!share(mx, o)) return false;
            mx = fmaxf(mx, o);
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
            const float2 k2 = make_float2(scale, scale), b2 = make_float2(-base, -base);
            float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int i = 0; i < TT_CW; i += 2) {
                float2 e = fma2(make_float2(s[i], s[i + 1]), k2, b2);
                e.x = ex2_approx(e.x);
                e.y = ex2_approx(e.y);
                sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], e);
                w[i / 2] = pack_bf2(e.x, e.y);
            }
            sum[0] = add2(sum[0], sum[1]);
            l += sum[0].x + sum[0].y;
            // P as the MMA will read it: 16-byte chunk ch of a row of 64 columns, swizzled
            if (g >= 1 && !warp_spin<true>(&bars.p_ack, (g - 1) & 1, a.err, 0x524)) return false;
#pragma unroll
            for (int c = 0; c < TT_CW / 8; c++)
                st16s(P + swz(row, c),
                      make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]));
            if (grp == 0) reinterpret_cast<float *>(sm + TT_OFF_FS)[row] = f;
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_out);
        }
        // the row's sum
        float o;
        if (!share(l, o)) return false;
        const int lr = sg.mt * TT_M + row;
        if (grp == 0 && lr < sg.s.n * a.H) {
            const float lt = l + o;
            if (sg.whole()) a.rowsum[(size_t)sg.s.first * a.H + lr] = lt;
            else {
                float *dst = a.part + (size_t)sg.slot(cl) * TT_PART + row;
                dst[TT_PART_M] = m_ref;
                dst[TT_PART_L] = lt;
            }
        }
    }
    return true;
}

// P to the peer as soon as it is written and the buffer there is free.
__device__ __forceinline__ bool score_send(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                           TreeBars &bars) {
    const uint32_t ps = smem_u32(sm + TT_OFF_PS), fs = smem_u32(sm + TT_OFF_FS);
    const uint32_t pd = map_peer(smem_u32(sm + TT_OFF_P), 1), fd = map_peer(smem_u32(sm + TT_OFF_F), 1);
    const uint32_t bar = map_peer(smem_u32(&bars.p_in[0]), 1);
    const bool lead = (threadIdx.x & 31) == 0;
    int g = 0;
    TreeSeg sg;
    while (walk.next(sg)) {
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            const int pb = g & 1;
            if (!warp_spin(&bars.p_out, g & 1, a.err, 0x531)) return false;
            if (g >= 2 && !warp_spin(&bars.pv_done[pb], ((g >> 1) - 1) & 1, a.err, 0x532))
                return false;
            if (lead) {
                bulk_send(pd + pb * TT_PBUF, ps, TT_PBUF, bar + 8 * pb);
                bulk_send(fd + pb * TT_M * 4, fs, TT_M * 4, bar + 8 * pb);
            }
            __syncwarp();
        }
    }
    // the peer's last arrivals on this CTA's barriers
    if (g > 0 && !warp_spin<true>(&bars.p_ack, (g - 1) & 1, a.err, 0x533)) return false;
    for (int k = g >= 2 ? g - 2 : 0; k < g; k++)
        if (!warp_spin(&bars.pv_done[k & 1], (k >> 1) & 1, a.err, 0x534)) return false;
    return true;
}

// ---------------------------------------------------------------- value CTA
__device__ __forceinline__ bool value_mma(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                          TreeBars &bars, uint32_t tbase) {
    constexpr uint32_t id = idesc_f16(128, 256, false, true);
    int g = 0, edges = 0;
    bool data = false, ready = false;  // the next chunk and P, as seen in advance
    TreeSeg sg;
    while (walk.next(sg)) {
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            const int pb = g & 1;
            const bool edge = (long long)(t + 1) * TT_TILE > sg.s.len;
            const int live = min(TT_TILE, sg.s.len + sg.s.n - t * TT_TILE);  // rows of the tile
            if (!ready && !warp_spin(&bars.p_full[pb], (g >> 1) & 1, a.err, 0x541)) return false;
#pragma unroll 1
            for (int c = 0; c < TT_VCH; c++) {
                if (!data && !warp_spin(&bars.full[c], g & 1, a.err, 0x542)) return false;
                if (edge && c * TT_VROWS < live && !warp_spin(&bars.clean[c], edges & 1, a.err, 0x543))
                    return false;
                tc_fence_after();
                // 16 rows at a time: P's columns, the rows' 512 dims in two halves
                const uint64_t kv = sdesc(smem_u32(sm + c * TT_VSTAGE), 1024, 8192);
                const uint64_t pd = sdesc_kmajor(
                    smem_u32(sm + TT_OFF_P + pb * TT_PBUF + (c >> 1) * TT_M * 128 + (c & 1) * 64));
                const uint32_t acc = (t == sg.t0 && c == 0) ? 0u : 1u;
                const bool some = c * TT_VROWS < live;  // else its weights are all zero
                if (some) {
                    warp_mma_ss(tbase, pd, kv, id, acc);
                    warp_mma_ss(tbase + 256, pd, kv + (4096 >> 4), id, acc);
                    warp_mma_ss(tbase, pd + (32 >> 4), kv + (16384 >> 4), id, 1u);
                }
                if (c + 1 < TT_VCH) {
                    data = __all_sync(0xffffffffu, mbar_test(&bars.full[c + 1], g & 1));
                } else {
                    data = __all_sync(0xffffffffu, mbar_test(&bars.full[0], (g + 1) & 1));
                    ready = __all_sync(0xffffffffu,
                                       mbar_test(&bars.p_full[pb ^ 1], ((g + 1) >> 1) & 1));
                }
                if (some) warp_mma_ss(tbase + 256, pd + (32 >> 4), kv + (20480 >> 4), id, 1u);
                if (c + 1 == TT_VCH) warp_commit_cluster(&bars.pv_done[pb], 3);
                warp_commit(&bars.empty[c]);
            }
            edges += edge;
        }
    }
    return true;
}

// Bring the rows of the tiles to come into L2 (both CTAs' loads find them there): the score CTA's
// stages do not cover the latency of HBM under load, about 3000 cycles. Plain prefetches: TMA's take
// as much of its time as the loads. The score CTA's loads run two to three tiles before this CTA's.
// At the start the clusters' first tiles share HBM's rate, so the others wait: TT_PACE is what it takes
// to bring one tile to every cluster (without the wait the first scores came 15000 cycles later).
__device__ __forceinline__ void value_prefetch(const TreeArgs &a, TreeWalk walk, TreeBars &bars) {
    const int lane = threadIdx.x & 31, box = min(a.v.page_size, TT_TILE);
    int g = 0;
    TreeSeg sg;
    while (walk.next(sg)) {
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            const long long t0 = clock64();
            while (g > *(volatile int *)&bars.tile + TT_AHEAD) {
                __nanosleep(400);
                if (*(volatile unsigned *)a.err || clock64() - t0 > wait_limit(a.err)) return;
            }
            if (g > 0 && g <= TT_AHEAD) __nanosleep(TT_PACE);
            const int end = min((t + 1) * TT_TILE, sg.s.len + sg.s.n);
            for (int p = t * TT_TILE; p < end; p += box) {
                const long long row = paged_row(a.v, sg.b, p);
                if (row < 0) continue;
                const int rows = min(box, end - p);
                const char *lat = reinterpret_cast<const char *>(a.latent + row * TT_DL);
                const char *rope = reinterpret_cast<const char *>(a.rope + row * TT_DR);
                for (int e = lane; e < rows * 8; e += 32)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(lat + e * 128));
                for (int e = lane; e < rows; e += 32)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(rope + e * 128));
            }
        }
    }
}

__device__ __forceinline__ bool value_output(const TreeArgs &a, TreeWalk walk, uint8_t *sm,
                                             TreeBars &bars, uint32_t tbase, int cl) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int q4 = warp & 3, grp = (warp - 2) >> 2;
    const int row = 32 * q4 + lane;
    const uint32_t oaddr = tbase + ((uint32_t)(32 * q4) << 16) + TT_OW * grp;
    const float *fac = reinterpret_cast<const float *>(sm + TT_OFF_F) + row;
    uint8_t *stage = sm + TT_OFF_W + (warp - 2) * 4096;
    int g = 0;
    TreeSeg sg, old;
    while (walk.next(sg)) {
        for (int t = sg.t0; t < sg.t1; t++, g++) {
            const int pb = g & 1, before = (g - 1) & 1, ph = ((g - 1) >> 1) & 1;
            if (warp == 2 && lane == 0) mbar_expect_tx(&bars.p_in[pb], TT_PBUF + TT_M * 4);
            if (t == sg.t0 && g > 0) {  // the last row tile's o, before it is written over
                if (!warp_spin(&bars.pv_done[before], ph, a.err, 0x551)) return false;
                tc_fence_after();
                write_o(a, old, cl, oaddr, stage, 32 * q4, TT_OW * grp, TT_OW);
            }
            if (!warp_spin<true>(&bars.p_in[pb], (g >> 1) & 1, a.err, 0x552)) return false;
            if (warp == 2 && lane == 0) mbar_arrive_cluster_relaxed(&bars.p_ack, 0);
            const float f = t == sg.t0 ? 1.f : fac[pb * TT_M];
            if (__any_sync(0xffffffffu, f != 1.f)) {
                if (!warp_spin(&bars.pv_done[before], ph, a.err, 0x553)) return false;
                tc_fence_after();
                rescale_o(oaddr, TT_OW, f);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars.p_full[pb]);
            if ((long long)(t + 1) * TT_TILE <= sg.s.len) continue;
            // Rows past the cached ones: zero where nothing is written, and where a draft's element
            // is not finite (a chunk without rows is left out of the products). The last tile's
            // products are waited for first. P may come before that tile's rows have, and the stages'
            // barriers, of which a wait sees one bit, would show its phase as this tile's; and the MMA
            // warp may still be about to look at `clean` for that tile, which the arrivals below
            // would take a phase further.
            if (g > 0 && !warp_spin(&bars.pv_done[before], ph, a.err, 0x556)) return false;
            const int live = sg.s.len + sg.s.n - t * TT_TILE;
#pragma unroll 1
            for (int c = 0; c < TT_VCH; c++) {
                if (c * TT_VROWS < live) {
                    if (!warp_spin(&bars.full[c], g & 1, a.err, 0x554)) return false;
                    const int d0 = max(0, sg.s.len - (t * TT_TILE + c * TT_VROWS));
                    const int d1 = live - c * TT_VROWS;
                    // a warp per row; a lane's 16 bytes of two 64-dim blocks
#pragma unroll 1
                    for (int e = 2 * d0 + warp - 2; e < 2 * TT_VROWS; e += TT_WORKERS) {
                        const int r = e / 2;
                        uint4 *p = reinterpret_cast<uint4 *>(
                            sm + c * TT_VSTAGE + (r / 8) * 8192 + (4 * (e & 1) + lane / 8) * 1024 +
                            (r % 8) * 128 + (lane % 8) * 16);
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
                }
                if (lane == 0) mbar_arrive(&bars.clean[c]);
            }
        }
        old = sg;
    }
    if (g == 0) return true;
    if (!warp_spin(&bars.pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, a.err, 0x555)) return false;
    tc_fence_after();
    write_o(a, old, cl, oaddr, stage, 32 * q4, TT_OW * grp, TT_OW);
    return true;
}

__device__ __forceinline__ void tree_roles(const TreeMaps &maps, const TreeArgs &a,
                                           const TreeWalk &walk, uint8_t *sm, TreeBars &bars,
                                           uint32_t tbase, int cl, bool score) {
    const int warp = threadIdx.x >> 5;
    bool ok = true;
    if (warp == 0) {
        ok = score ? tree_loads<true>(maps, a, walk, sm, bars)
                   : tree_loads<false>(maps, a, walk, sm, bars);
    } else if (warp == 1) {
        ok = score ? score_mma(a, walk, sm, bars, tbase) : value_mma(a, walk, sm, bars, tbase);
    } else if (warp == 2 + TT_WORKERS) {
        if (score) ok = score_send(a, walk, sm, bars);
        else value_prefetch(a, walk, bars);
    } else if (score) {
        ok = score_softmax(a, walk, sm, bars, tbase, cl);
    } else {
        ok = value_output(a, walk, sm, bars, tbase, cl);
    }
    // After a wait that ran out, the CTAs stay until what is still on its way has arrived: P to the
    // peer, whose barrier alone would show it, and products in TMEM, which take some microseconds.
    if (!ok)
        for (const long long t0 = clock64(); clock64() - t0 < TT_DRAIN;) __nanosleep(1000);
}

__global__ void __launch_bounds__(TT_THREADS, 1) __cluster_dims__(2, 1, 1)
mla_tree_attend_tc(const __grid_constant__ TreeMaps maps, const __grid_constant__ TreeArgs a) {
    extern __shared__ __align__(1024) uint8_t sm[];
    TreeBars &bars = *reinterpret_cast<TreeBars *>(sm + TT_OFF_BARS);
    const int warp = threadIdx.x >> 5;
    const bool score = cluster_rank() == 0;
    const int cl = blockIdx.x >> 1;
    if (smem_u32(sm) & 1023) {  // nothing else is in shared memory, so this does not happen
        if (threadIdx.x == 0) atomicCAS(a.err, 0u, 0x500u);
        return;
    }
    pdl_trigger();
    if (threadIdx.x == 0) {
        mbar_init(&bars.r_full, 1);
        mbar_init(&bars.r_empty, 1);
        for (int c = 0; c < TT_KST; c++) {
            mbar_init(&bars.full[c], 1);
            mbar_init(&bars.empty[c], 1);
        }
        for (int c = 0; c < TT_VCH; c++) mbar_init(&bars.clean[c], TT_WORKERS);
        for (int q = 0; q < 4; q++) mbar_init(&bars.pair[q], TT_GRP);
        mbar_init(&bars.p_out, TT_WORKERS);
        mbar_init(&bars.p_ack, 1);
        for (int b = 0; b < 2; b++) {
            mbar_init(&bars.s_full[b], 1);
            mbar_init(&bars.s_empty[b], TT_WORKERS);
            mbar_init(&bars.p_in[b], 1);
            mbar_init(&bars.p_full[b], TT_WORKERS);
            mbar_init(&bars.pv_done[b], 1);
        }
        bars.tile = -1;
        fence_barrier_init();
        prefetch_tmap(score ? &maps.lat_k : &maps.lat_v);
    }
    __syncthreads();
    cluster_sync();  // the peer's barriers are ready before anything arrives on them
    pdl_wait();      // the plan, the queries and the cache come from earlier work
    if (warp == 1) tmem_alloc(&bars.tmem_base, TT_TM_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = bars.tmem_base;
    const int G = a.plan->G;
    if (cl < G) tree_roles(maps, a, TreeWalk(a, cl, a.plan->total, G), sm, bars, tbase, cl, score);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // nothing of the peer's is on its way into this CTA's shared memory
    if (warp == 1) tmem_dealloc(tbase, TT_TM_COLS);
}

// Join the row tiles that several clusters took (the flash-decoding identity). A warp takes 8 dims of
// 32 rows, a row to a lane, as the partials lie, TJ_UP parts at a time with a running maximum. Bound by
// L2's latency: a warp has few items after one another and few loads that wait for others (a row per
// block of 128 threads took 16 us for 73 cut tiles).
constexpr int TJ_WARPS = 4, TJ_UP = 4;
constexpr int TJ_ITEMS = TT_M / 32 * (TT_DL / 8);  // of a cut row tile
__global__ void __launch_bounds__(TJ_WARPS * 32, 8) mla_tree_join(const __grid_constant__ TreeArgs a) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, items = a.plan->cuts * TJ_ITEMS;
    for (int i = blockIdx.x * TJ_WARPS + (threadIdx.x >> 5); i < items; i += gridDim.x * TJ_WARPS) {
        const TreeCut cut = a.plan->cut[i / TJ_ITEMS];
        const int row = i % (TT_M / 32) * 32 + lane, dim = i % TJ_ITEMS / (TT_M / 32) * 8;
        if (row >= cut.rows) continue;
        float M = -INFINITY, L = 0.f, o[8] = {};
        for (int k0 = cut.first; k0 <= cut.last; k0 += TJ_UP) {
            float m[TJ_UP], l[TJ_UP];
            float4 v[TJ_UP][2];
#pragma unroll
            for (int u = 0; u < TJ_UP; u++) {
                const int k = k0 + u;
                m[u] = -INFINITY;
                l[u] = 0.f;
                v[u][0] = v[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (k > cut.last) continue;
                // the first cluster's part is its odd slot, the others' the even ones
                const float *p = a.part + (size_t)(2 * k + (k == cut.first)) * TT_PART;
                m[u] = p[TT_PART_M + row];
                l[u] = p[TT_PART_L + row];
                v[u][0] = reinterpret_cast<const float4 *>(p)[dim / 4 * TT_M + row];
                v[u][1] = reinterpret_cast<const float4 *>(p)[(dim / 4 + 1) * TT_M + row];
            }
            float M1 = M;
#pragma unroll
            for (int u = 0; u < TJ_UP; u++) M1 = fmaxf(M1, m[u]);
            const float f = M == M1 ? 1.f : exp2f(M - M1);
            M = M1;
            L *= f;
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] *= f;
#pragma unroll
            for (int u = 0; u < TJ_UP; u++) {
                const float w = m[u] == -INFINITY && l[u] == 0.f ? 0.f : exp2f(m[u] - M);
                L += w * l[u];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    o[4 * j] = fmaf(w, v[u][j].x, o[4 * j]);
                    o[4 * j + 1] = fmaf(w, v[u][j].y, o[4 * j + 1]);
                    o[4 * j + 2] = fmaf(w, v[u][j].z, o[4 * j + 2]);
                    o[4 * j + 3] = fmaf(w, v[u][j].w, o[4 * j + 3]);
                }
            }
        }
        const size_t th = (size_t)cut.row0 + row;
        uint4 *dst = reinterpret_cast<uint4 *>(a.olat2 + th * 2 * TT_DL + dim);
        const uint4 hi = pack_bf8(o);
        float h[8], lo[8];
        unpack_bf8(hi, h);
#pragma unroll
        for (int e = 0; e < 8; e++) lo[e] = o[e] - h[e];
        dst[0] = hi;
        dst[TT_DL / 8] = pack_bf8(lo);
        if (dim == 0) a.rowsum[th] = L;
    }
}

static int tree_shape(int B, int T, int H, int dn, int dr, int dl, int dv) {
    K3_ARG_CHECK(B >= 0 && T >= 0 && H >= 1 && H <= TT_H && B < (1 << 24),
                 "mla_tree_attend: bad B=%d T=%d H=%d", B, T, H);
    if (dn != TT_DN || dr != TT_DR || dl != TT_DL || dv != TT_DV)
        return set_error(K3CUDA_ERR_UNSUPPORTED,
                         "mla_tree_attend: dn=%d dr=%d dl=%d dv=%d not built", dn, dr, dl, dv);
    // the per-head products take 128 tokens to a row of their grid
    K3_ARG_CHECK(T <= 65535 * 128, "mla_tree_attend: T=%d", T);
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
    w.part = take((size_t)2 * TT_CLUSTERS * TT_PART * sizeof(float));
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
    const float scale_log2e = scale * 1.4426950408889634f;
    K3_ARG_CHECK(isfinite(scale_log2e), "%s: bad scale %g", what, scale);
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
    const TreeArgs a{paged_view(cache, batch), plan, cum, tree_mask,
                     (const __nv_bfloat16 *)cache->latent, (const __nv_bfloat16 *)cache->rope,
                     (float *)(w + ws.part), (__nv_bfloat16 *)(w + ws.olat2),
                     (float *)(w + ws.rowsum), H, scale_log2e, ctx->err_word};
    const uint64_t rows = (uint64_t)cache->n_pages * cache->page_size;
    const uint32_t kbox = cache->page_size < TT_TILE ? cache->page_size : TT_TILE;
    const uint32_t vbox = cache->page_size < TT_VROWS ? cache->page_size : TT_VROWS;
    TreeMaps maps;
    rc = make_tmap_rows8(&maps.lat_k, cache->latent, TT_DL, rows, TT_DL / 64 / TT_KCH, kbox);
    if (!rc) rc = make_tmap_rows8(&maps.lat_v, cache->latent, TT_DL, rows, TT_DL / 64, vbox);
    if (!rc)
        rc = make_tmap_2d(&maps.rope, cache->rope, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, TT_DR, rows,
                          TT_DR * 2, 64, kbox);
    const uint64_t qrows = (uint64_t)T * H;
    if (!rc)
        rc = make_tmap_3d(&maps.q, qlat, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 64, qrows, TT_DL / 64,
                          TT_QW * 2, 128, 64, TT_M, 2);
    if (!rc)
        rc = make_tmap_2d(&maps.q_rope, qlat, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, TT_QW, qrows,
                          TT_QW * 2, 64, TT_M);
    if (rc || (rc = set_smem(mla_tree_attend_tc, TT_SMEM))) return rc;

    int clusters = ctx->sm_count / 2;
    if (clusters > TT_CLUSTERS) clusters = TT_CLUSTERS;
    if (clusters < 1) clusters = 1;
    rc = mla_absorb(ctx, qlat, H, q_nope, q_rope, w_uk, TT_DN, T, H);
    if (!rc)
        rc = launch_pdl(ctx, ctx->stream, "mla_tree_plan", mla_tree_plan, dim3(1), dim3(1024), 0, a.v,
                        H, plan, cum, keep, clusters, ctx->err_word);
    if (!rc)
        rc = launch_pdl(ctx, ctx->stream, "mla_tree_attend_tc", mla_tree_attend_tc,
                        dim3(2 * clusters), dim3(TT_THREADS), TT_SMEM, maps, a);
    if (!rc)
        rc = launch_pdl(ctx, ctx->stream, "mla_tree_join", mla_tree_join, dim3(8 * ctx->sm_count),
                        dim3(TJ_WARPS * 32), 0, a);
    if (!rc)
        rc = mla_project(ctx, out, out_dtype, a.olat2, a.rowsum, keep, w_uv, TT_DV, T, H);
    return rc;
}
