// kv4_attn.h -- MLA attention of a step's tokens over the paged cache in 4 bits (gmoe_kv4_attend).
//
// Work split. A request's fresh tokens times heads are its query rows; a tile is 8 MT of them
// (MT 1, 2 or 3), and an item is a tile against a chunk of the request's positions. All chunks of a launch are
// one length, a multiple of KA_P positions, the least that makes at most KA_ITEMS items beside
// the one a tile needs (ka_plan): few long requests are cut fine, many are not cut at all. The
// lengths are device data, so every block works out the split by itself from the requests'
// lengths, and the grid is a fixed number of blocks that walk the items. A tile of one chunk is
// written where it belongs; the others leave partial results that k_kv4_merge joins.
//
// Products. Both run on v_mfma_f32_16x16x32_f16. The cache's values are exact in fp16 (e2m1 times a
// power of two that the format holds to fp16's range), so only the queries and the exponentials
// are split into two fp16 parts, x = hi + lo to 22 bits: two products where split operands on both sides
// take three. The two parts of eight rows make the 16 operand rows of a tile, in the order
// (hi hi lo lo) of rows 2g, 2g + 1: then a row's two sums lie in the same lane.
//
// A block (8 waves, one a CU) takes KA_P = 64 positions at a time:
//   scores   wave (h, g) has half h of the columns (nine blocks of 32) and positions 16 g .. + 15. A lane
//            loads 16 bytes, a block of 32 codes, which are four steps' operands when the steps run over
//            the blocks' eighths (the sum over columns may run in any order); v_cvt_scalef32_pk_f16_fp4
//            turns a byte of codes and their scale into two halves. The queries stay in registers
//            (108). The halves go to shared memory as they are, a row a position.
//   softmax  wave w has rows 3 w .. + 2, a lane a position; the exponentials go to shared memory as
//            operands.
//   values   wave w has columns 64 w .. + 63: the rows of halves through the transposing read.
// The values of a tile and the scores of the next share a phase, so two barriers a tile; codes
// are requested a tile ahead, pages two.
//
// Softmax reference: exponentials are taken against a row's reference, which follows the running
// maximum only when a score passes it by 2^KA_SLACK, so that sums are rescaled a few times a
// chunk. They are scaled by 2^KA_UP for the split, whose error is then 2^-33 of the largest.
#pragma once

#include "kv4.h"
#include "split16.h"

#define KA_P 64
#define KA_BLOCK 512
#define KA_WAVES (KA_BLOCK / 64)
#define KA_ROWS 24    // rows of the largest tile
#define KA_HALF 9     // column blocks of a wave's half
#define KA_GRID 256
#define KA_ITEMS 512
#define KA_MAX_PARTS (2 * KA_ITEMS)  // a cut tile has over U/c + 1 <= 2 U/c chunks, U/c of all at most KA_ITEMS
#define KA_SLACK 6.0f
#define KA_UP 8
#define KA_VROW 528  // halves of a row of values in shared memory: rows 8 banks apart (of 64)
#define KA_SROW 26   // floats of a position's scores
#define KA_PROW 72   // halves of an operand row of exponentials
#define KA_QROW 584  // halves of an operand row of queries (while they are staged)
static_assert(2 * KA_HALF >= KV4_BLOCKS_MAX, "two halves hold a row");
static_assert(2 * KA_ROWS * KA_QROW <= 2 * KA_P * KA_VROW, "the queries are staged where the values come later");

struct Kv4Attn {
    Kv4Cache c;
    int R, max_pages, H;
    float scale;
    const int32_t *table, *offsets, *context;
    const float *q_abs, *q_pe;
    int64_t ld_q_abs, ld_q_pe, ld_out;
    float *out;
    float *part;     // [KA_MAX_PARTS][KA_ROWS][kv]
    float *part_ml;  // [KA_MAX_PARTS][KA_ROWS][2]: a chunk's reference (of base 2, to a constant) and its sum of exponentials
};

// ---- the split of a launch -------------------------------------------------------------------

__device__ static inline unsigned ka_tiles(const Kv4Attn &a, int r, int rows) {
    const int fresh = a.offsets[r + 1] - a.offsets[r];
    return fresh > 0 ? (unsigned)(fresh * a.H + rows - 1) / rows : 0u;  // (fresh * H < 2^27)
}
__device__ static inline unsigned ka_units(const Kv4Attn &a, int r) {
    const long long n = min((long long)a.context[r], (long long)a.max_pages << a.c.shift);  // what the table names
    return n > 0 ? ((unsigned)n + KA_P - 1) / KA_P : 0u;
}

// A thread's share of the requests, and what lies before it. Cut tiles are those of more than one chunk.
struct KaPlan {
    int r0, r1;
    unsigned items0, items, cuts0, cuts, parts0;
    unsigned chunk, total, total_cuts;  // units of a chunk; all items; all cut tiles
};
struct KaShared {
    unsigned red[KA_WAVES];
    unsigned long long red2[KA_WAVES];
};

__device__ static inline unsigned ka_chunks(unsigned units, unsigned chunk) { return max(1u, (units + chunk - 1) / chunk); }

__device__ static inline KaPlan ka_plan(const Kv4Attn &a, int rows, KaShared &sh) {
    const int tid = threadIdx.x, nw = blockDim.x >> 6, per = (a.R + blockDim.x - 1) / blockDim.x;
    KaPlan p;
    p.r0 = min(a.R, tid * per);
    p.r1 = min(a.R, p.r0 + per);
    unsigned long long work = 0;
    for (int r = p.r0; r < p.r1; r++) work += (unsigned long long)ka_tiles(a, r, rows) * ka_units(a, r);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) work += __shfl_xor(work, d);
    if ((tid & 63) == 0) sh.red2[tid >> 6] = work;
    __syncthreads();
    work = 0;
    for (int i = 0; i < nw; i++) work += sh.red2[i];
    p.chunk = (unsigned)max(1ull, min((work + KA_ITEMS - 1) / KA_ITEMS, 1ull << 30));
    p.items = p.cuts = 0;
    unsigned parts = 0;
    for (int r = p.r0; r < p.r1; r++) {
        const unsigned t = ka_tiles(a, r, rows), k = ka_chunks(ka_units(a, r), p.chunk);
        p.items += t * k;
        if (k > 1) {
            p.cuts += t;
            parts += t * k;
        }
    }
    unsigned n;
    p.items0 = block_scan_u(p.items, sh.red, &p.total);
    p.cuts0 = block_scan_u(p.cuts, sh.red, &p.total_cuts);
    p.parts0 = block_scan_u(parts, sh.red, &n);
    return p;
}

// One item of the split.
struct KaItem {
    int r, tile, k, chunk;     // request, tile of it, its chunks, this one
    int t0, fresh, context;    // the request's first token, its tokens, its positions
    unsigned part;             // partial-result slot of the item (k > 1)
};

// The item of number `i` (of the cut tiles, first chunk, when CUT) by the thread that has it.
template <bool CUT>
__device__ static inline void ka_find(const Kv4Attn &a, const KaPlan &p, int rows, unsigned i, KaItem *out) {
    const unsigned base = CUT ? p.cuts0 : p.items0, mine = CUT ? p.cuts : p.items;
    if (i - base >= mine) return;
    unsigned left = i - base, part = p.parts0;
    for (int r = p.r0; r < p.r1; r++) {
        const unsigned t = ka_tiles(a, r, rows), k = ka_chunks(ka_units(a, r), p.chunk), n = CUT ? (k > 1 ? t : 0) : t * k;
        if (left < n) {
            KaItem m;
            m.r = r;
            m.k = (int)k;
            m.tile = (int)(CUT ? left : left / k);
            m.chunk = (int)(CUT ? 0 : left % k);
            m.t0 = a.offsets[r];
            m.fresh = a.offsets[r + 1] - m.t0;
            m.context = max(0, a.context[r]);
            m.part = part + m.tile * k + m.chunk;
            *out = m;
            return;
        }
        left -= n;
        if (k > 1) part += t * k;
    }
}

// ---- the kernel ------------------------------------------------------------------------------

typedef _Float16 ka_h2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

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
    u32x2 w0;      // the half's scale bytes, from byte 0 (first half) or 1 on: eight,
    unsigned w1;   // and the next four
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
    __shared__ __align__(16) _Float16 val[2][KA_P * KA_VROW];
    __shared__ __align__(16) float sc[2][KA_P][KA_SROW];
    __shared__ __align__(16) _Float16 pr[OPS][KA_PROW];
    __shared__ __align__(8) float cr[ROWS], rl[ROWS], rm[ROWS];
    __shared__ __align__(8) unsigned char moved[KA_WAVES];
    __shared__ KaShared sh;
    __shared__ KaItem item;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kh = w >> 2, pg = w & 3;
    const int kv = a.c.kv, rope = a.c.rope, nb = a.c.blocks, shift = a.c.shift;
    const KaPlan plan = ka_plan(a, ROWS, sh);
    const float scale = __fmul_rn(a.scale, 1.44269504f);  // scores of base 2

    for (unsigned it = blockIdx.x; it < plan.total; it += gridDim.x) {
        __syncthreads();
        ka_find<false>(a, plan, ROWS, it, &item);
        __syncthreads();
        const KaItem m = item;
        const int rows = m.fresh * a.H, row0 = m.tile * ROWS, nr = min(ROWS, rows - row0);
        const int first = m.context - m.fresh;  // the position of the request's first token
        const int end = (int)min((long long)max(0, first + min(m.fresh, (row0 + nr - 1) / a.H + 1)), (long long)a.max_pages << shift);
        const long long c0 = (long long)m.chunk * plan.chunk * KA_P;
        const int s0 = (int)min(c0, (long long)end), s1 = (int)min(c0 + (long long)plan.chunk * KA_P, (long long)end);
        const int nt = (s1 - s0 + KA_P - 1) / KA_P;
        const int32_t *table = a.table + (size_t)m.r * a.max_pages;

        const int tid = ka_tid(), lane = tid & 63, l16 = lane & 15, lg = lane >> 4;
        // The lane's blocks of its half, and which of the half's bytes are their scales. A block past the
        // row's last reads codes of another at scale 0.
        const int b0 = KA_HALF * kh + lg, b1 = b0 + 4, b2 = KA_HALF * kh + 8;
        const unsigned none = 0x0c0c0c0cu, sel0 = b0 < nb ? 0x0c0c0c00u + kh + lg : none, sel1 = b1 < nb ? 0x0c0c0c00u + kh + lg : none,
                       sel2 = b2 < nb ? 0x0c0c0c00u + kh : none;
        const int at0 = b0 < nb ? 16 * b0 : 0, at1 = b1 < nb ? 16 * b1 : 0, at2 = b2 < nb ? 16 * b2 + 4 * lg : 0;
        // (a row ends 16 bytes past its codes, 32 where it has over 16 blocks)
        const int ats = 16 * nb + (KA_HALF * kh < nb ? 8 * kh : 0), atw = 16 * nb + (kh == 0 ? 8 : nb > 16 ? 16 : 0);
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
            x.w0 = *gbl((const u32x2 *)(row + ats));
            x.w1 = *gbl((const unsigned *)(row + atw));
        };
        int page = -1;
        KaRaw raw;
        if (nt > 0) {
            fetch(raw, 0, page_of(0));
            if (nt > 1) page = page_of(1);
        }

        // the queries: wave w stages rows RPW w .. as operand rows of halves, scaled by 2^-e
        _Float16 *stage = val[0];
        const int plane = ka_tid() & 63;
        float lsum[RPW], top[RPW];  // a row's sum, and its reference + KA_SLACK (of base 2)
        int eq[RPW], last[RPW];
        bool on[RPW];
#pragma unroll
        for (int i = 0; i < RPW; i++) {
            const int r = RPW * w + i, g = row0 + min(r, nr - 1), t = g / a.H, h = g - t * a.H;
            const float *qa = a.q_abs + (m.t0 + t) * a.ld_q_abs + (int64_t)h * kv, *qp = a.q_pe + (m.t0 + t) * a.ld_q_pe + (int64_t)h * rope;
            float v[KV4_BLOCKS_MAX / 2];
            float mx = 0.0f;
#pragma unroll
            for (int k = 0; k < KV4_BLOCKS_MAX / 2; k++) {
                const int col = 64 * k + plane;
                v[k] = col < kv ? qa[col] : col - kv < rope ? qp[col - kv] : 0.0f;
                mx = fmaxf(mx, fabsf(v[k]));
            }
            mx = wave_max_dpp_f(mx);
            const int e = mx < INFINITY ? spl_exp(mx) : 0;
            _Float16 *hi = stage + (16 * (r >> 3) + 4 * ((r & 7) >> 1) + (r & 1)) * KA_QROW, *lo = hi + 2 * KA_QROW;
#pragma unroll
            for (int k = 0; k < KV4_BLOCKS_MAX / 2; k++) {
                _Float16 x, y;
                spl_split(ldexpf(v[k], -e), x, y);
                hi[64 * k + plane] = x;
                lo[64 * k + plane] = y;
            }
            eq[i] = e;
            last[i] = min(first + t, s1 - 1);
            lsum[i] = 0.0f;
            top[i] = -INFINITY;
        }
        __syncthreads();
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
        __syncthreads();  // the staged queries are read; values may come

        // tile j's scores (this half's part) from `raw`, its values to shared memory
        auto scores = [&](int j) {
            unsigned e0 = __builtin_amdgcn_perm(raw.w0[1], raw.w0[0], sel0) & raw.on, e1 = __builtin_amdgcn_perm(raw.w1, raw.w0[1], sel1) & raw.on,
                     e2 = __builtin_amdgcn_perm(0u, raw.w1, sel2) & raw.on;
            unsigned long long spoilt = __ballot(max(max(e0, e1), e2) == KV4_BYTE_NAN);
            if (spoilt) {  // such a block's values count as zeros, and its position's scores as NaN
                if (e0 == KV4_BYTE_NAN) e0 = 0;
                if (e1 == KV4_BYTE_NAN) e1 = 0;
                if (e2 == KV4_BYTE_NAN) e2 = 0;
                spoilt |= spoilt >> 32;
                spoilt |= spoilt >> 16;
            }
            const float f0 = __uint_as_float(e0 << 23), f1 = __uint_as_float(e1 << 23), f2 = __uint_as_float(e2 << 23);
            const int p = 16 * pg + l16;
            // rows r and r + 8 have the halves of 16 columns the other way round, in other banks
            _Float16 *dst = val[j & 1] + p * KA_VROW;
            const int flip = p & 8;
            aq_f4 d[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) d[mt] = (aq_f4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int g = 0; g < 2; g++) {
                a16_h8 x[4];
#pragma unroll
                for (int k = 0; k < 4; k++) x[k] = ka_halves(g ? raw.q1[k] : raw.q0[k], g ? f1 : f0);
                if (g ? v1 : v0) {
                    _Float16 *at = dst + 32 * (g ? b1 : b0);
#pragma unroll
                    for (int k = 0; k < 4; k++) *(a16_h8 *)(at + ((8 * k) ^ flip)) = x[k];
                }
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) d[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[4 * g + k][mt], x[k], d[mt], 0, 0, 0);
            }
            const a16_h8 x = ka_halves(raw.q2, f2);
            if (v2) *(a16_h8 *)(dst + 32 * b2 + ((8 * lg) ^ flip)) = x;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) d[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q[8][mt], x, d[mt], 0, 0, 0);
            float2 t[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) t[mt] = make_float2(d[mt][0] + d[mt][2], d[mt][1] + d[mt][3]);
            if (spoilt || !__all(raw.on)) {
                const float odd = !raw.on ? -INFINITY : __uint_as_float(0x7fc00000u);
                if (!raw.on || (spoilt >> l16 & 1))
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) t[mt] = make_float2(odd, odd);
            }
#pragma unroll
            for (int mt = 0; mt < MT; mt++) *(float2 *)&sc[kh][p][8 * mt + 2 * lg] = t[mt];
        };
        // tile j's exponentials from its scores
        const int slot_at = 32 * (lane >> 5) + 8 * ((lane & 15) >> 2) + 4 * ((lane & 31) >> 4) + (lane & 3);  // a position's operand slot
        _Float16 *const pdst = &pr[0][slot_at];
        auto softmax = [&](int j) {
            const int s = s0 + KA_P * j + lane;
            float t[RPW];
            bool up[RPW], any = false;
#pragma unroll
            for (int i = 0; i < RPW; i++) {
                const float x = sc[0][lane][RPW * w + i] + sc[1][lane][RPW * w + i];
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
                const int r = RPW * w + i;
                const float ref = top[i] - (KA_SLACK + KA_UP);
                const float e = on[i] ? __builtin_amdgcn_exp2f(fmaf(t[i], scale, -ref)) : 0.0f;
                lsum[i] += e;
                _Float16 *dst = pdst + (16 * (r >> 3) + 4 * ((r & 7) >> 1) + (r & 1)) * KA_PROW;
                const _Float16 hi = (_Float16)e;
                dst[0] = hi;
                dst[2 * KA_PROW] = (_Float16)fmaf((float)hi, -1.0f, e);
            }
        };
        // tile j's values weighted
        auto values = [&](int j) {
            const u32x2 mv = *(const u32x2 *)moved;
            if (__builtin_amdgcn_readfirstlane(mv[0] | mv[1])) {
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    const float2 f = *(const float2 *)&cr[8 * mt + 2 * lg];
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[c][mt] *= (aq_f4){f.x, f.y, f.x, f.y};
                }
            }
            const _Float16 *src = val[j & 1] + (4 * lg + (l16 >> 2)) * KA_VROW + ((64 * w + 4 * (l16 & 3)) ^ (lg & 2 ? 8 : 0));
#pragma unroll
            for (int ks = 0; ks < KA_P / 32; ks++) {
                a16_h8 p[MT];
#pragma unroll
                for (int mt = 0; mt < MT; mt++) p[mt] = *(const a16_h8 *)&pr[16 * mt + l16][32 * ks + 8 * lg];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const a16_h4 x = a16_tr(src + 32 * ks * KA_VROW + 16 * c), y = a16_tr(src + (32 * ks + 16) * KA_VROW + 16 * c);
                    const a16_h8 v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) acc[c][mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[mt], v, acc[c][mt], 0, 0, 0);
                }
            }
        };
        const bool mine = 64 * w < kv;  // the wave has columns
        if (nt > 0) {
            for (int j = 0; j <= nt; j++) {
                if (j < nt) {
                    scores(j);
                    if (j + 1 < nt) {
                        fetch(raw, j + 1, page);
                        if (j + 2 < nt) page = page_of(j + 2);
                    }
                }
                if (j > 0 && mine) values(j - 1);
                block_barrier();
                if (j < nt) {
                    softmax(j);
                    block_barrier();
                }
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
        if (m.k > 1 && etid < nr) {
            float *ml = a.part_ml + ((size_t)m.part * KA_ROWS + etid) * 2;
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
                    if (m.k > 1) {
                        dst = a.part + ((size_t)m.part * KA_ROWS + r) * kv;
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

// The cut tiles' partial results joined, a block a query row: out = sum_c w_c part_c / sum_c w_c l_c
// with w_c = 2^(ref_c - max ref). Threads have four columns each; the groups that cover a row share
// its chunks.
__global__ __launch_bounds__(KA_BLOCK) void k_kv4_merge(Kv4Attn a, int rows) {
    __shared__ KaShared sh;
    __shared__ KaItem item;
    __shared__ float wgt[KA_ITEMS];
    __shared__ float red[KA_WAVES];
    __shared__ __align__(16) float4 sum[KA_BLOCK];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, kv = a.c.kv;
    const KaPlan plan = ka_plan(a, rows, sh);
    const int cols = kv / 4, groups = KA_BLOCK / cols, grp = tid / cols, col = tid - grp * cols;
    for (unsigned unit = blockIdx.x; unit < plan.total_cuts * rows; unit += gridDim.x) {
        const unsigned ti = unit / rows;
        const int rr = (int)(unit - ti * rows);
        __syncthreads();
        ka_find<true>(a, plan, rows, ti, &item);
        __syncthreads();
        const KaItem m = item;
        const int g = m.tile * rows + rr;
        if (g >= m.fresh * a.H) continue;
        const float *ml = a.part_ml + ((size_t)m.part * KA_ROWS + rr) * 2;
        float pm = -INFINITY, pl = 0.0f;
        if (tid < m.k) {
            pm = ml[(size_t)tid * KA_ROWS * 2];
            pl = ml[(size_t)tid * KA_ROWS * 2 + 1];
        }
        const float wm = wave_max_dpp_f(pm);
        if (lane == 0) red[w] = wm;
        __syncthreads();
        float mx = red[0];
#pragma unroll
        for (int i = 1; i < KA_WAVES; i++) mx = fmaxf(mx, red[i]);
        __syncthreads();
        const float e = pl == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(pm - mx);
        if (tid < m.k) wgt[tid] = e;
        float l = row_sum_dpp_f(e * pl);
        l = (readlane_f(l, 0) + readlane_f(l, 16)) + (readlane_f(l, 32) + readlane_f(l, 48));
        if (lane == 0) red[w] = l;
        __syncthreads();
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < KA_WAVES; i++) l += red[i];
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (grp < groups) {
            const float *pc = a.part + ((size_t)m.part * KA_ROWS + rr) * kv + 4 * col;
#pragma unroll 4
            for (int c = grp; c < m.k; c += groups) {
                const float4 v = *(const float4 *)(pc + (size_t)c * KA_ROWS * kv);
                const float x = wgt[c];
                s.x = fmaf(x, v.x, s.x);
                s.y = fmaf(x, v.y, s.y);
                s.z = fmaf(x, v.z, s.z);
                s.w = fmaf(x, v.w, s.w);
            }
        }
        sum[tid] = s;
        __syncthreads();
        if (tid < cols) {
            for (int k = 1; k < groups; k++) {
                const float4 v = sum[tid + k * cols];
                s.x += v.x;
                s.y += v.y;
                s.z += v.z;
                s.w += v.w;
            }
            const int t = g / a.H;
            float *dst = a.out + (m.t0 + t) * a.ld_out + (int64_t)(g - t * a.H) * kv + 4 * tid;
            const float f = l == 0.0f ? 0.0f : 1.0f / l;
            dst[0] = s.x * f;
            dst[1] = s.y * f;
            dst[2] = s.z * f;
            dst[3] = s.w * f;
        }
    }
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
