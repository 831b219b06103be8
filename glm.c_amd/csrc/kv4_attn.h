// kv4_attn.h -- MLA attention of a step's tokens over the paged cache in 4 bits (gmoe_kv4_attend).
//
// Work split. A request's fresh tokens times heads are its query rows; a tile is 8 MT of them (MT 1, 2
// or 3) and a unit a tile against KA_P positions. All units of a launch lie on one axis, tile after
// tile, each tile led by KA_LEAD for what it costs to begin one; the axis is cut into one equal
// share a block, so that every block has the same work whatever the lengths. A tile inside one
// share is written where it belongs; one that the cuts part leaves a partial result a block, which
// k_kv4_merge joins. A block has at most two partial results, of its first tile and its last. The
// lengths are device data, so every block works out the axis by itself; a tile's place on it is a
// formula (ka_place), near its units' number, and the units in a share follow from the place alone
// (ka_cut), so that neighbours agree.
//
// Products. Both run on v_mfma_f32_16x16x32_f16. The cache's values are exact in fp16 (e2m1 times a
// power of two that the format holds to fp16's range), so only the queries and the exponentials
// are split into two fp16 parts, x = hi + lo to 22 bits: two products where split operands on both sides
// take three. The two parts of eight rows make the 16 operand rows of a tile, in the order
// (hi hi lo lo) of rows 2g, 2g + 1: then a row's two sums lie in the same lane.
//
// A block (8 waves, one block a CU) takes KA_P = 64 positions at a time:
//   scores   wave (h, g) has half h of the columns (nine blocks of 32) and positions 16 g .. + 15. A lane
//            loads 16 bytes, a block of 32 codes, which are four steps' operands when the steps run over
//            the blocks' eighths (the sum over columns may run in any order); v_cvt_scalef32_pk_f16_fp4
//            turns a byte of codes and their scale into two halves. The queries stay in registers
//            (108). The halves go to shared memory as they are, a row a position.
//   softmax  wave w has rows 3 w .. + 2, a lane a position; the exponentials go to shared memory as
//            operands.
//   values   wave w has columns 64 w .. + 63: the rows of halves through the transposing read.
// The softmax of a tile and the scores of the next share a phase, in opposite order on the two waves of
// a SIMD, so that the one's vector instructions run beside the other's matrix instructions; two barriers
// a tile. Codes are requested a tile ahead, their pages two.
//
// Measured, 20 heads, ranks 512 + 64 (kernel + join): one token at 4096 positions 14.2 + 5.1 us, 64 requests
// of 8 to 8192 positions 31.9 + 6.3 (36.7 MB of rows, 1.2 TB/s), 1023 tokens after 2977 389 + 12 (155
// GFLOP, twice that with the split: 0.8 PFLOP/s of matrix instructions). What bounds it: a unit of three
// operand tiles takes some 5400 clocks of a CU, of which its matrix instructions are 1630 of a SIMD's, its
// vector instructions 2050 and shared memory 1800; two waves a SIMD (the registers hold no more) and two barriers a unit
// overlap a third of that. Few rows: the beginning (lengths, table, codes: three waits on memory) and the join.
//
// Softmax reference: exponentials are taken against a row's reference, which follows the running
// maximum only when a score passes it by 2^KA_SLACK, so that sums are rescaled a few times a
// chunk. They are scaled by 2^KA_UP for the split, whose error is then 2^-33 of the largest.
#pragma once

#include <algorithm>

#include "kv4.h"
#include "split16.h"

#define KA_P 64
#define KA_BLOCK 512
#define KA_WAVES (KA_BLOCK / 64)
#define KA_ROWS 24    // rows of the largest tile
#define KA_HALF 9     // column blocks of a wave's half
#define KA_GRID 256   // blocks: one a CU
#define KA_LEAD 4     // of a tile's beginning, in units (64 ragged requests: 39 us with 2, 32 with 4, 34 with 7)
#define KA_SLACK 6.0f
#define KA_UP 8
#define KA_VROW 512  // halves of a row of values in shared memory
#define KA_SROW 24   // floats of a position's scores
#define KA_PROW 64   // halves of an operand row of exponentials
#define KA_QROW 584  // halves of an operand row of queries (while they are staged)
static_assert(2 * KA_HALF >= KV4_BLOCKS_MAX, "two halves hold a row");
static_assert(2 * KA_ROWS * KA_QROW <= 2 * KA_P * KA_VROW, "the queries are staged where the values come later");

// What a block leaves for k_kv4_merge: the cut tile that ends in its share (k > 1 partial results).
struct KaCut {
    int k;           // 0: none
    int first, next; // slots of its partial results: first, next, next + 2, next + 4, ...
    int t0, row0, nr;
};
static_assert(sizeof(KaCut) == 6 * sizeof(int), "read as six words");

struct Kv4Attn {
    Kv4Cache c;
    int R, max_pages, H;
    float scale;
    double slope;    // units that a tile has more than the one before it, halved: rows / (2 KA_P H)
    const int32_t *table, *offsets, *context;
    const float *q_abs, *q_pe;
    int64_t ld_q_abs, ld_q_pe, ld_out;
    float *out;
    float *part;     // [2 KA_GRID][KA_ROWS][kv]
    float *part_ml;  // [2 KA_GRID][KA_ROWS][2]: a part's reference (of base 2, to a constant) and its sum of exponentials
    KaCut *cuts;     // [KA_GRID]
};

// ---- the split of a launch -------------------------------------------------------------------

// (fresh * H < 2^27)
__device__ static inline unsigned ka_tiles(const Kv4Attn &a, int fresh, int rows) { return (unsigned)(fresh * a.H + rows - 1) / rows; }

// The place on the axis of tile i of a request whose first token has `first` positions before it: a
// trapezoid's area, rounded, so that it needs no sum over the tiles. Rises by over KA_LEAD a tile.
__device__ static inline uint64_t ka_place(const Kv4Attn &a, uint64_t i, int first) {
    return i * (KA_LEAD + 1) + i * (unsigned)max(0, first) / KA_P + (uint64_t)((double)(i * i) * a.slope);
}
// The units before place x of a tile of n units at place p, whose next tile is at e.
__device__ static inline int ka_cut(uint64_t x, uint64_t p, uint64_t e, int n) {
    return x >= e ? n : x <= p + KA_LEAD ? 0 : (int)min((uint64_t)n, x - p - KA_LEAD);
}

// A tile, and its place.
struct KaItem {
    int r, tile, t0, fresh, context;  // request, tile of it; the request's first token, its tokens, its positions
    uint64_t p, e;
};

// The axis of a launch. With at most 64 requests every wave has them all, a lane each, and finds
// tiles by itself; with more a thread of the block has every KA_BLOCK-th run of them, and the one that
// has a tile hands it over in shared memory.
struct KaPlan {
    int r0, r1;                   // the thread's requests
    int t0, fresh, context;       // of the first
    double at, size;              // their place on the axis (whole numbers below 2^53)
    uint64_t total, share;
};
struct KaShared {
    double red[KA_WAVES];
    KaItem item;
};

__device__ static inline double ka_size(const Kv4Attn &a, int fresh, int context, int rows) {
    return (double)ka_place(a, ka_tiles(a, fresh, rows), context - fresh);
}

__device__ static inline KaPlan ka_plan(const Kv4Attn &a, int rows, KaShared &sh) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const bool few = a.R <= 64;
    const int per = few ? 1 : (a.R + KA_BLOCK - 1) / KA_BLOCK, mine = few ? lane : tid;
    KaPlan p;
    p.r0 = min(a.R, mine * per);
    p.r1 = min(a.R, p.r0 + per);
    p.t0 = p.fresh = p.context = 0;
    p.size = 0.0;
    for (int r = p.r0; r < p.r1; r++) {
        const int t0 = a.offsets[r], fresh = max(0, a.offsets[r + 1] - t0), context = a.context[r];
        if (r == p.r0) {
            p.t0 = t0;
            p.fresh = fresh;
            p.context = context;
        }
        p.size += ka_size(a, fresh, context, rows);
    }
    const double s = wave_incl_scan_dpp(p.size);
    double before = 0.0, total = readlane_d(s, 63);
    if (!few) {
        if (lane == 63) sh.red[w] = s;
        __syncthreads();
        total = 0.0;
#pragma unroll
        for (int i = 0; i < KA_WAVES; i++) {
            if (i < w) before += sh.red[i];
            total += sh.red[i];
        }
    }
    p.at = before + s - p.size;
    p.total = (uint64_t)readlane_d(total, 0);
    p.share = max((uint64_t)1, (p.total + KA_GRID - 1) / KA_GRID);  // (2 at least: a token at 4096 15.6 us, with 1 14.2)
    return p;
}

// The tile of a request, from place `at` on, that has place x.
__device__ static inline KaItem ka_tile(const Kv4Attn &a, int rows, uint64_t x, int r, int t0, int fresh, int context, uint64_t at) {
    uint64_t lo = 0, hi = ka_tiles(a, fresh, rows);
    while (hi - lo > 1) {  // the last tile whose place is at most x, by halving
        const uint64_t mid = (lo + hi) >> 1;
        if (at + ka_place(a, mid, context - fresh) <= x) lo = mid;
        else hi = mid;
    }
    return KaItem{r, (int)lo, t0, fresh, max(0, context), at + ka_place(a, lo, context - fresh), at + ka_place(a, lo + 1, context - fresh)};
}

// The tile at place x, to every thread of the block.
__device__ static inline KaItem ka_find(const Kv4Attn &a, const KaPlan &p, int rows, uint64_t x, KaShared &sh) {
    const double d = (double)x;
    const bool has = d >= p.at && d < p.at + p.size;
    if (a.R <= 64) {
        const int l = __ffsll(__ballot(has)) - 1;
        return ka_tile(a, rows, x, l, __builtin_amdgcn_readlane(p.t0, l), __builtin_amdgcn_readlane(p.fresh, l),
                       __builtin_amdgcn_readlane(p.context, l), (uint64_t)readlane_d(p.at, l));
    }
    __syncthreads();
    if (has) {
        double at = p.at;
        for (int r = p.r0; r < p.r1; r++) {
            const int t0 = a.offsets[r], fresh = max(0, a.offsets[r + 1] - t0), context = a.context[r];
            const double size = ka_size(a, fresh, context, rows);
            if (d < at + size) {
                sh.item = ka_tile(a, rows, x, r, t0, fresh, context, (uint64_t)at);
                break;
            }
            at += size;
        }
    }
    __syncthreads();
    return sh.item;
}

// A tile in scalar registers.
__device__ static inline KaItem ka_uniform(KaItem m) {
    auto u32 = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    auto u64 = [&](uint64_t v) { return (uint64_t)(unsigned)u32((int)v) | (uint64_t)(unsigned)u32((int)(v >> 32)) << 32; };
    return KaItem{u32(m.r), u32(m.tile), u32(m.t0), u32(m.fresh), u32(m.context), u64(m.p), u64(m.e)};
}

// ---- the kernel ------------------------------------------------------------------------------

typedef _Float16 ka_h2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32_any __attribute__((aligned(1)));

// Eight codes and their scale to eight halves.
__device__ static inline a16_h8 ka_halves(unsigned codes, float scale) {
    const ka_h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 1);
    const ka_h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, 3);
    return (a16_h8){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The codes and scales of a lane's position and half, as loaded.
struct KaRaw {
    u32x4 q0, q1;  // blocks j and 4 + j of the half (j = lane / 16)
    unsigned q2;   // the lane's eighth of block 8
    unsigned w[3]; // twelve scale bytes, the half's among them
    unsigned on;   // all ones, or 0 where there is no such position
};

// The thread's index as the compiler cannot know it, so that addresses made from it are not kept in
// registers (or out of them) across the loop over items.
__device__ static inline int ka_tid() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

template <int MT>
__global__ __launch_bounds__(KA_BLOCK, 2) void k_kv4_attend(Kv4Attn a) {
    constexpr int ROWS = 8 * MT, OPS = 16 * MT, RPW = MT;  // rows, operand rows, rows of a wave's softmax
    static_assert(RPW * KA_WAVES == ROWS, "every row has a wave");
    // Rows of 16-byte pieces, 16 pieces 256 bytes; piece i of a row lies at i ^ (a number of the row), so that
    // neither the eight rows that are written side by side nor the eight that the transposing read takes
    // a pair of pieces from meet in a bank
    __shared__ __align__(16) _Float16 val[2][KA_P * KA_VROW];
    __shared__ __align__(16) float sc[2][2][KA_P * KA_SROW];
    __shared__ __align__(16) _Float16 pr[OPS * KA_PROW];
    __shared__ __align__(8) float cr[ROWS], rl[ROWS], rm[ROWS];
    __shared__ __align__(8) unsigned char moved[KA_WAVES];
    __shared__ KaShared sh;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kh = w >> 2, pg = w & 3;
    const int kv = a.c.kv, rope = a.c.rope, nb = a.c.blocks, shift = a.c.shift;
    const KaPlan plan = ka_plan(a, ROWS, sh);
    const float scale = __fmul_rn(a.scale, 1.44269504f);  // scores of base 2
    const uint64_t x0 = blockIdx.x * plan.share, x1 = min(plan.total, x0 + plan.share);
    if (threadIdx.x == 0) a.cuts[blockIdx.x].k = 0;

    for (uint64_t at = x0; at < x1;) {
        const KaItem m = ka_uniform(ka_find(a, plan, ROWS, at, sh));
        at = m.e;
        const int rows = m.fresh * a.H, row0 = m.tile * ROWS, nr = min(ROWS, rows - row0);
        const int first = m.context - m.fresh;  // the position of the request's first token
        const int end = (int)min((long long)max(0, first + min(m.fresh, (row0 + nr - 1) / a.H + 1)), (long long)a.max_pages << shift);
        const int units = (end + KA_P - 1) / KA_P;
        const int u0 = ka_cut(x0, m.p, m.e, units), u1 = ka_cut(x1, m.p, m.e, units);
        // the places of its first unit and its last; the block that has the one and the other has it whole
        const uint64_t head = units > 0 ? m.p + KA_LEAD : m.p, tail = units > 0 ? min(m.p + KA_LEAD + units, m.e) - 1 : m.p;
        const bool ends = x0 <= tail && tail < x1, whole = ends && x0 <= head;
        if (units > 0 ? u0 == u1 : !whole) continue;
        __syncthreads();  // (what the tile before left in shared memory is read)
        const int s0 = KA_P * u0, s1 = min(end, KA_P * u1), nt = u1 - u0;
        const int slot = 2 * blockIdx.x + (m.p > x0 ? 1 : 0);  // of a partial result: the block's first tile, or its last
        const int32_t *table = a.table + (size_t)m.r * a.max_pages;
        const int tid = ka_tid(), lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
        // The lane's blocks of its half, and which of the half's bytes are their scales. A block past the
        // row's last reads codes of another at scale 0.
        const int b0 = KA_HALF * kh + lg, b1 = b0 + 4, b2 = KA_HALF * kh + 8;
        // (twelve bytes from `from` on, which the row has: it ends 16 bytes past its codes, 32 where it has over 16 blocks)
        const int from = kh == 0 ? 0 : nb > 16 ? KA_HALF : 4, w0 = KA_HALF * kh - from + lg;
        const unsigned none = 0x0c0c0c0cu, sel0 = b0 < nb ? 0x0c0c0c00u + w0 : none, sel1 = b1 < nb ? 0x0c0c0c00u + w0 : none,
                       sel2 = b2 < nb ? 0x0c0c0c00u + w0 - lg : none;
        const int at0 = b0 < nb ? 16 * b0 : 0, at1 = b1 < nb ? 16 * b1 : 0, at2 = b2 < nb ? 16 * b2 + 4 * lg : 0;
        const int ats = 16 * nb + from;
        const bool v0 = 32 * b0 < kv, v1 = 32 * b1 < kv, v2 = 32 * b2 < kv;  // blocks of the entry, not of the rope part

        // the lane's position of tile j: its page, as the table has it (nothing looks at it before fetch(),
        // so that nothing waits for it), and from the page its row
        auto page_of = [&](int j) { return *gbl(table + (min(s0 + KA_P * j + 16 * pg + l16, s1 - 1) >> shift)); };
        auto fetch = [&](KaRaw &x, int j, int page) {
            const int s = s0 + KA_P * j + 16 * pg + l16;
            x.on = s < s1 && page >= 0 && page < a.c.n_pages ? ~0u : 0u;
            const unsigned slot = x.on & (((unsigned)page << shift) + (s & ((1 << shift) - 1)));
            const uint8_t *row = a.c.rows + (size_t)slot * (unsigned)a.c.row_bytes;
            x.q0 = *gbl((const u32x4 *)(row + at0));
            x.q1 = *gbl((const u32x4 *)(row + at1));
            x.q2 = *gbl((const unsigned *)(row + at2));
            // (word by word: a vector of three may be loaded as four, past the end of the pool's last row)
#pragma unroll
            for (int k = 0; k < 3; k++) x.w[k] = ((const GM_GLOBAL u32_any *)(row + ats))[k];
        };
        // the first pages, then the queries, then the first codes, so that they are under way together
        int page0 = -1, page = -1;
        if (nt > 0) page0 = page_of(0);
        if (nt > 1) page = page_of(1);
        _Float16 *stage = val[0];
        const int plane = ka_tid() & 63;
        float lsum[RPW], top[RPW];  // a row's sum, and its reference + KA_SLACK (of base 2)
        int eq[RPW], last[RPW];
        bool on[RPW];
        // wave w stages rows RPW w .. as operand rows of halves, scaled by 2^-e
        float v[RPW][KV4_BLOCKS_MAX / 2];
#pragma unroll
        for (int i = 0; i < RPW; i++) {
            const int g = row0 + min(RPW * w + i, nr - 1), t = g / a.H, h = g - t * a.H;
            const float *qa = a.q_abs + (m.t0 + t) * a.ld_q_abs + (int64_t)h * kv, *qp = a.q_pe + (m.t0 + t) * a.ld_q_pe + (int64_t)h * rope;
#pragma unroll
            for (int k = 0; k < KV4_BLOCKS_MAX / 2; k++) {
                const int col = 64 * k + plane;
                v[i][k] = 0.0f;
                if (col < kv) v[i][k] = *gbl(qa + col);
                else if (col - kv < rope) v[i][k] = *gbl(qp + col - kv);
            }
            last[i] = min(first + t, s1 - 1);
            lsum[i] = 0.0f;
            top[i] = -INFINITY;
        }
        KaRaw raw;
        if (nt > 0) fetch(raw, 0, page0);
#pragma unroll
        for (int i = 0; i < RPW; i++) {
            const int r = RPW * w + i;
            float mx = 0.0f;
#pragma unroll
            for (int k = 0; k < KV4_BLOCKS_MAX / 2; k++) mx = fmaxf(mx, fabsf(v[i][k]));
            mx = wave_max_dpp_f(mx);
            eq[i] = mx < INFINITY ? spl_exp(mx) : 0;
            _Float16 *hi = stage + (16 * (r >> 3) + 4 * ((r & 7) >> 1) + (r & 1)) * KA_QROW, *lo = hi + 2 * KA_QROW;
#pragma unroll
            for (int k = 0; k < KV4_BLOCKS_MAX / 2; k++) {
                _Float16 x, y;
                spl_split(ldexpf(v[i][k], -eq[i]), x, y);
                hi[64 * k + plane] = x;
                lo[64 * k + plane] = y;
            }
        }
        block_barrier();
        a16_h8 q[KA_HALF][MT];  // steps 0..3: eighths of blocks j; 4..7: of blocks 4 + j; 8: block 8
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const _Float16 *src = stage + (16 * mt + l16) * KA_QROW;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                q[k][mt] = *(const a16_h8 *)(src + 32 * b0 + 8 * k);
                q[4 + k][mt] = *(const a16_h8 *)(src + 32 * b1 + 8 * k);
            }
            q[8][mt] = *(const a16_h8 *)(src + 32 * b2 + 8 * lg);
        }
        aq_f4 acc[4][MT];
#pragma unroll
        for (int c = 0; c < 4; c++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++) acc[c][mt] = (aq_f4){0.0f, 0.0f, 0.0f, 0.0f};
        block_barrier();  // the staged queries are read; values may come

        // where the lane writes values (pieces 4 b0 .. + 3, then b1's 16 on, and its eighth of block 2) and scores
        const int mix = (2 * (l16 & 7)) ^ (l16 >> 2 & 1);
        int wat[4];
#pragma unroll
        for (int k = 0; k < 4; k++) wat[k] = 8 * ((4 * b0 + k) ^ mix);
        const int wat2 = 8 * ((4 * b2 + lg) ^ mix);
        const int sat = (16 * pg + l16) * KA_SROW + ((2 * lg) ^ (l16 & 8) >> 1 ^ (pg & 1) << 1);
        // tile j's scores (this half's part) from `raw`, its values to shared memory
        auto scores = [&](int j) {
            unsigned e0 = __builtin_amdgcn_perm(raw.w[1], raw.w[0], sel0) & raw.on, e1 = __builtin_amdgcn_perm(raw.w[2], raw.w[1], sel1) & raw.on,
                     e2 = __builtin_amdgcn_perm(0u, raw.w[2], sel2) & raw.on;
            unsigned long long spoilt = __ballot(max(max(e0, e1), e2) == KV4_BYTE_NAN);
            if (spoilt) {  // such a block's values count as zeros, and its position's scores as NaN
                if (e0 == KV4_BYTE_NAN) e0 = 0;
                if (e1 == KV4_BYTE_NAN) e1 = 0;
                if (e2 == KV4_BYTE_NAN) e2 = 0;
                spoilt |= spoilt >> 32;
                spoilt |= spoilt >> 16;
            }
            const float f0 = __uint_as_float(e0 << 23), f1 = __uint_as_float(e1 << 23), f2 = __uint_as_float(e2 << 23);
            _Float16 *dst = val[j & 1] + (16 * pg + l16) * KA_VROW;
            aq_f4 d[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) d[mt] = (aq_f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < 4; g++) {  // two eighths at a time
                a16_h8 x[2];
#pragma unroll
                for (int k = 0; k < 2; k++) x[k] = ka_halves(g < 2 ? raw.q0[2 * g + k] : raw.q1[2 * (g - 2) + k], g < 2 ? f0 : f1);
                if (g < 2 ? v0 : v1)
#pragma unroll
                    for (int k = 0; k < 2; k++) *(a16_h8 *)(dst + wat[2 * (g & 1) + k] + 128 * (g >> 1)) = x[k];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) d[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[2 * g + k][mt], x[k], d[mt], 0, 0, 0);
            }
            const a16_h8 x = ka_halves(raw.q2, f2);
            if (v2) *(a16_h8 *)(dst + wat2) = x;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) d[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[8][mt], x, d[mt], 0, 0, 0);
            float2 t[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) t[mt] = make_float2(d[mt][0] + d[mt][2], d[mt][1] + d[mt][3]);
            if (spoilt || !__all(raw.on)) {
                const float odd = !raw.on ? -INFINITY : __uint_as_float(0x7fc00000u);
                if (!raw.on || ((unsigned)spoilt >> l16 & 1))
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) t[mt] = make_float2(odd, odd);
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++) *(float2 *)&sc[j & 1][kh][sat + 8 * mt] = t[mt];
        };
        // tile j's exponentials from its scores
        // where the lane finds its position's scores and puts its pair of positions' first parts, or the second,
        // but for the row
        const int rat = lane * KA_SROW, rmix = (lane & 8) >> 1 ^ (lane & 16) >> 3;
        const int pat = (32 * (lane >> 5) + 8 * ((lane & 15) >> 2) + 4 * ((lane & 31) >> 4) + (lane & 2)) ^ 16 * (lane & 1);
        const int podd = 2 * KA_PROW * (lane & 1);
        const unsigned pick = lane & 1 ? 0x03020706u : 0x05040100u;  // of (the partner's, the lane's) pair of parts
        auto softmax = [&](int j) {
            const int s = s0 + KA_P * j + lane;
            float t[RPW];
            bool up[RPW], any = false;
            float xa[RPW], xb[RPW];
#pragma unroll
            for (int i = 0; i < RPW; i++) {
                const int at = rat + ((RPW * w + i) ^ rmix);
                xa[i] = sc[j & 1][0][at];
                xb[i] = sc[j & 1][1][at];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < RPW; i++) {
                const float x = xa[i] + xb[i];
                t[i] = ldexpf(x, eq[i]);
                on[i] = s <= last[i] && x != -INFINITY;
                up[i] = on[i] && t[i] * scale > top[i];
                any |= up[i];
            }
            const bool move = __any(any);
            float mine = 1.0f;  // lane i: row i's factor
            if (move) {
#pragma unroll
                for (int i = 0; i < RPW; i++) {
                    const float mx = wave_max_dpp_f(on[i] ? t[i] * scale : -INFINITY);
                    float f = 1.0f;
                    if (mx > top[i]) {
                        f = __builtin_amdgcn_exp2f((top[i] - KA_SLACK) - mx);  // 0 before the first position
                        top[i] = mx + KA_SLACK;
                    }
                    lsum[i] *= f;
                    mine = lane == i ? f : mine;
                }
            }
            if (lane < RPW) cr[RPW * w + lane] = mine;
            if (lane == 0) moved[w] = move;
#pragma unroll
            for (int i = 0; i < RPW; i++) {
                const float ref = top[i] - (KA_SLACK + KA_UP);
                const float e = on[i] ? __builtin_amdgcn_exp2f(fmaf(t[i], scale, -ref)) : 0.0f;
                lsum[i] += e;
                ka_h2 both;
                both.x = (_Float16)e;
                both.y = (_Float16)fmaf((float)both.x, -1.0f, e);
                const unsigned me = __builtin_bit_cast(unsigned, both);
                const unsigned other = (unsigned)__builtin_amdgcn_update_dpp(0, (int)me, DPP_QUAD_1032, 0xF, 0xF, false);
                const int r = RPW * w + i, o = 16 * (r >> 3) + 4 * ((r & 7) >> 1) + (r & 1);  // (the second part's row is o + 2)
                *(unsigned *)&pr[o * KA_PROW + podd + (pat ^ 8 * ((o & 7) ^ (o >> 3 & 1)))] = __builtin_amdgcn_perm(other, me, pick);
            }
        };
        // where the lane reads exponentials, and four rows' values of each 16 columns
        const int pin = l16 * KA_PROW + 8 * (lg ^ (l16 & 7) ^ (l16 >> 3));
        int vin[4];
        {
            const int row = 4 * lg + (l16 >> 2), m2 = (2 * (row & 7)) ^ (row >> 2 & 1);
#pragma unroll
            for (int c = 0; c < 4; c++) vin[c] = row * KA_VROW + 8 * ((8 * w + 2 * c + (l16 >> 1 & 1)) ^ m2) + 4 * (l16 & 1);
        }
        // tile j's values weighted
        auto values = [&](int j) {
            const u32x2 mv = *(const u32x2 *)moved;
            const _Float16 *src = val[j & 1];
            a16_h8 p[MT], v[4];
            auto load = [&](int ks) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++) p[mt] = *(const a16_h8 *)(pr + 16 * mt * KA_PROW + (ks ? pin ^ 32 : pin));
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const a16_h4 x = a16_tr(src + vin[c] + 32 * ks * KA_VROW), y = a16_tr(src + vin[c] + (32 * ks + 16) * KA_VROW);
                    v[c] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
                }
            };
            load(0);
            if (__builtin_amdgcn_readfirstlane(mv[0] | mv[1])) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    const float2 f = *(const float2 *)&cr[8 * mt + 2 * lg];
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[c][mt] *= (aq_f4){f.x, f.y, f.x, f.y};
                }
            }
#pragma unroll
            for (int ks = 0; ks < KA_P / 32; ks++) {
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) acc[c][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[mt], v[c], acc[c][mt], 0, 0, 0);
                if (ks + 1 < KA_P / 32) load(ks + 1);
            }
        };
        const bool mine = 64 * w < kv;  // the wave has columns
        auto ahead = [&](int j) {  // tile j's scores, and the request of the next one's codes
            scores(j);
            if (j + 1 < nt) {
                fetch(raw, j + 1, page);
                if (j + 2 < nt) page = page_of(j + 2);
            }
        };
        if (nt > 0) {
            ahead(0);
            block_barrier();
            for (int j = 0; j < nt; j++) {
                if (kh == 0 && j + 1 < nt) ahead(j + 1);
                softmax(j);
                if (kh != 0 && j + 1 < nt) ahead(j + 1);
                block_barrier();
                if (mine) values(j);
                block_barrier();
            }
        }
        // the rows' sums to every wave, and the results
        const int etid = ka_tid(), elane = etid & 63;
#pragma unroll
        for (int i = 0; i < RPW; i++) {
            float l = row_sum_dpp_f(lsum[i]);
            l = (readlane_f(l, 0) + readlane_f(l, 16)) + (readlane_f(l, 32) + readlane_f(l, 48));
            if (elane == 0) {
                rl[RPW * w + i] = l;
                rm[RPW * w + i] = top[i];
            }
        }
        __syncthreads();
        if (ends && !whole && etid == 0) {
            const int bf = (int)(head / plan.share);  // the block of the first part
            a.cuts[blockIdx.x] = KaCut{(int)blockIdx.x - bf + 1, 2 * bf + (m.p > bf * plan.share ? 1 : 0), 2 * bf + 2, m.t0, row0, nr};
        }
        if (!whole && etid < nr) {
            float *ml = a.part_ml + ((size_t)slot * KA_ROWS + etid) * 2;
            ml[0] = rm[etid];
            ml[1] = rl[etid];
        }
        if (mine) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int r = 8 * mt + 2 * (elane >> 4) + i;
                    if (r >= nr) continue;
                    float *dst;
                    float f = 1.0f;
                    if (!whole) {
                        dst = a.part + ((size_t)slot * KA_ROWS + r) * kv;
                    } else {
                        const int g = row0 + r, t = g / a.H;
                        dst = a.out + (m.t0 + t) * a.ld_out + (int64_t)(g - t * a.H) * kv;
                        f = rl[r] == 0.0f ? 0.0f : 1.0f / rl[r];
                    }
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int col = 64 * w + 16 * c + (elane & 15);
                        if (col < kv) dst[col] = (acc[c][mt][i] + acc[c][mt][i + 2]) * f;
                    }
                }
        }
    }
}

// The cut tiles' partial results joined: out = sum_c w_c part_c / sum_c w_c l_c with w_c = 2^(ref_c - max
// ref). A block has two rows of the blockIdx.y-th cut tile and one of QUARTERS parts of their columns; a
// row's threads have four columns each and every 2 QUARTERS-th part. Few tiles (one long sequence) are
// joined by four times the blocks.
#define KM_ROWS 2
#define KM_FEW 8  // tiles (joining a token's 64 parts: 5.1 us with quarters, 6.4 without; 64 tiles: 10.6 and 6.3)
#define KM_THREADS (KA_BLOCK / KM_ROWS)
template <int QUARTERS>
__global__ __launch_bounds__(KA_BLOCK) void k_kv4_merge(Kv4Attn a) {
    constexpr int COLS = 128 / QUARTERS, GROUPS = KM_THREADS / COLS;  // threads of a row's part, groups of them
    static_assert(4 * 128 >= 512 && KM_THREADS % COLS == 0, "the parts cover a row");
    __shared__ int cut[6];
    __shared__ int found[KA_GRID / 64];
    __shared__ float wgt[KM_ROWS][KA_GRID];
    __shared__ float red[KM_ROWS][4], red2[KM_ROWS][4];
    __shared__ __align__(16) float4 sum[KM_ROWS][GROUPS - 1][COLS];
    const int kv = a.c.kv, tid = threadIdx.x, pair = blockIdx.x / QUARTERS;
    // the blockIdx.y-th of the shares that a cut tile ends in
    const bool has = tid < KA_GRID;
    // (word by word: as a struct of each thread's the compiler keeps it in shared memory, and reads the launch's
    // packet for its place there: 14 us)
    const int *share = (const int *)(a.cuts + (has ? tid : 0));
    int f[6];
#pragma unroll
    for (int i = 0; i < 6; i++) f[i] = share[i];
    const unsigned long long ends = __ballot(has && f[0] > 0);
    if (has && (tid & 63) == 0) found[tid >> 6] = __popcll(ends);
    __syncthreads();
    int rank = __popcll(ends & ((1ull << (tid & 63)) - 1)), all = 0;
#pragma unroll
    for (int i = 0; i < KA_GRID / 64; i++) {
        if (i < tid >> 6) rank += found[i];
        all += found[i];
    }
    if ((int)blockIdx.y >= all) return;
    if (has && f[0] > 0 && rank == (int)blockIdx.y)
#pragma unroll
        for (int i = 0; i < 6; i++) cut[i] = f[i];
    __syncthreads();
    const KaCut m = {cut[0], cut[1], cut[2], cut[3], cut[4], cut[5]};
    if (pair * KM_ROWS >= m.nr) return;
    const int sub = __builtin_amdgcn_readfirstlane(tid / KM_THREADS), t = tid % KM_THREADS, rr = pair * KM_ROWS + sub;
    const bool there = rr < m.nr;
    auto at = [&](int c) { return (size_t)(c == 0 ? m.first : m.next + 2 * (c - 1)) * KA_ROWS + rr; };
    static_assert(KA_GRID <= KM_THREADS, "a thread a part");
    float pm = -INFINITY, pl = 0.0f;
    if (there && t < m.k) {
        pm = a.part_ml[at(t) * 2];
        pl = a.part_ml[at(t) * 2 + 1];
    }
    const float wm = wave_max_dpp_f(pm);
    if ((t & 63) == 0) red[sub][t >> 6] = wm;
    __syncthreads();
    const float mx = fmaxf(fmaxf(red[sub][0], red[sub][1]), fmaxf(red[sub][2], red[sub][3]));
    const float e = pl == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(pm - mx);
    if (t < m.k) wgt[sub][t] = e;
    float l = row_sum_dpp_f(pl == 0.0f ? 0.0f : e * pl);
    l = (readlane_f(l, 0) + readlane_f(l, 16)) + (readlane_f(l, 32) + readlane_f(l, 48));
    if ((t & 63) == 0) red2[sub][t >> 6] = l;
    __syncthreads();
    l = (red2[sub][0] + red2[sub][1]) + (red2[sub][2] + red2[sub][3]);
    const int grp = t / COLS, col = 4 * (t % COLS + COLS * (blockIdx.x % QUARTERS));
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (there && col < kv) {
#pragma unroll 8
        for (int c = grp; c < m.k; c += GROUPS) {
            const float4 v = *(const float4 *)(a.part + at(c) * kv + col);
            const float x = wgt[sub][c];
            s.x = fmaf(x, v.x, s.x);
            s.y = fmaf(x, v.y, s.y);
            s.z = fmaf(x, v.z, s.z);
            s.w = fmaf(x, v.w, s.w);
        }
    }
    if (grp > 0) sum[sub][grp - 1][t % COLS] = s;
    __syncthreads();
    if (there && col < kv && grp == 0) {
#pragma unroll
        for (int i = 0; i + 1 < GROUPS; i++) {
            const float4 v = sum[sub][i][t % COLS];
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
        const int g = m.row0 + rr, tok = g / a.H;
        float *dst = a.out + (m.t0 + tok) * a.ld_out + (int64_t)(g - tok * a.H) * kv + col;
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        dst[0] = s.x * f;
        dst[1] = s.y * f;
        dst[2] = s.z * f;
        dst[3] = s.w * f;
    }
}
static_assert(KM_THREADS == 256, "four waves a row");

// The most tiles a launch can cut, of those that a step of up to `tokens` tokens of R requests has.
static inline int ka_cut_tiles(long long tokens, int R, int H, int mt) {
    return (int)std::min<long long>(KA_GRID, tokens * H / (8 * mt) + R);
}

// Operand tiles a row tile for rows of a request's step, by the cost of the tiles it takes: each
// converts the cache's codes once (about one operand tile's products) and multiplies MT operand tiles.
static inline int ka_operand_tiles(long long rows) {
    int best = 1;
    long long least = 1ll << 62;
    for (int mt = 1; mt <= KA_ROWS / 8; mt++) {
        const long long cost = (rows + 8 * mt - 1) / (8 * mt) * (1 + mt);
        if (cost < least) {
            least = cost;
            best = mt;
        }
    }
    return best;
}
