// kv4_attn.h -- MLA attention of a step's tokens over the paged cache in 4 bits (gmoe_kv4_attend).
//
// Work split. A request's fresh tokens times heads are its query rows; a tile is KA_ROWS of them,
// and an item is a tile against a chunk of the request's positions. All chunks of a launch are
// one length, a multiple of KA_UNIT positions, the least that makes at most KA_ITEMS items beside
// the one a tile needs (kv4_plan): few long requests are cut fine, many are not cut at all. The
// lengths are device data, so every block works out the split by itself, from the requests'
// lengths, and the grid is a fixed number of blocks that walk the items. A tile of one chunk is
// written where it belongs; the others leave partial results that k_kv4_merge joins.
#pragma once

#include "kv4.h"

#define KA_ROWS 24
#define KA_UNIT 64
#define KA_ITEMS 512
#define KA_MAX_PARTS (2 * KA_ITEMS)  // a cut tile has over U/c + 1 <= 2 U/c chunks, U/c of all at most KA_ITEMS
#define KA_BLOCK 256

struct Kv4Attn {
    Kv4Cache c;
    int R, max_pages, H;
    float scale;
    const int32_t *table, *offsets, *context;
    const float *q_abs, *q_pe;
    int64_t ld_q_abs, ld_q_pe, ld_out;
    float *out;
    float *part;     // [KA_MAX_PARTS][KA_ROWS][kv]
    float *part_ml;  // [KA_MAX_PARTS][KA_ROWS][2]: a chunk's largest score and its sum of exponentials
};

// The split of a launch, in shared memory.
struct Kv4Plan {
    unsigned items[PM_MAX_R];  // items up to and with the request
    unsigned parts[PM_MAX_R];  // partial results before the request
    unsigned red[KA_BLOCK / 64];
    unsigned long long red2[KA_BLOCK / 64];
    unsigned total, chunk;  // items; units of a chunk
};

__device__ static inline unsigned ka_tiles(const Kv4Attn &a, int r) {
    const int fresh = a.offsets[r + 1] - a.offsets[r];
    return fresh > 0 ? (unsigned)(((long long)fresh * a.H + KA_ROWS - 1) / KA_ROWS) : 0u;
}
__device__ static inline unsigned ka_units(const Kv4Attn &a, int r) {
    const long long n = min((long long)a.context[r], (long long)a.max_pages << a.c.shift);  // what the table names
    return n > 0 ? ((unsigned)n + KA_UNIT - 1) / KA_UNIT : 0u;
}

__device__ static inline void kv4_plan(const Kv4Attn &a, Kv4Plan &p) {
    const int tid = threadIdx.x, R = a.R, per = (R + KA_BLOCK - 1) / KA_BLOCK, r0 = tid * per, r1 = min(R, r0 + per);
    unsigned long long work = 0;
    for (int r = r0; r < r1; r++) work += (unsigned long long)ka_tiles(a, r) * ka_units(a, r);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) work += __shfl_xor(work, d);
    if ((tid & 63) == 0) p.red2[tid >> 6] = work;
    __syncthreads();
    work = 0;
    for (int i = 0; i < KA_BLOCK / 64; i++) work += p.red2[i];
    const unsigned chunk = (unsigned)max(1ull, min((work + KA_ITEMS - 1) / KA_ITEMS, 1ull << 30));
    unsigned items = 0, parts = 0;
    for (int r = r0; r < r1; r++) {
        const unsigned t = ka_tiles(a, r), k = max(1u, (ka_units(a, r) + chunk - 1) / chunk);
        items += t * k;
        if (k > 1) parts += t * k;
    }
    unsigned n, np;
    unsigned i0 = block_scan_u(items, p.red, &n), p0 = block_scan_u(parts, p.red, &np);
    for (int r = r0; r < r1; r++) {
        const unsigned t = ka_tiles(a, r), k = max(1u, (ka_units(a, r) + chunk - 1) / chunk);
        i0 += t * k;
        p.items[r] = i0;
        p.parts[r] = p0;
        if (k > 1) p0 += t * k;
    }
    if (tid == 0) {
        p.total = n;
        p.chunk = chunk;
    }
    __syncthreads();
}

// One item of the split.
struct Kv4Item {
    int r, tile, k, chunk;     // request, tile of it, its chunks, this one
    int t0, fresh, context;    // the request's first token, its tokens, its positions
    int s0, s1;                // positions of the chunk that any row of the tile attends
    unsigned part;             // partial-result slot (k > 1)
};
__device__ static inline Kv4Item kv4_item(const Kv4Attn &a, const Kv4Plan &p, unsigned i) {
    Kv4Item m;
    m.r = upper_bound_u(p.items, a.R, i);
    const unsigned local = i - (m.r > 0 ? p.items[m.r - 1] : 0u);
    m.k = (int)max(1u, (ka_units(a, m.r) + p.chunk - 1) / p.chunk);
    m.tile = (int)(local / m.k);
    m.chunk = (int)(local % m.k);
    m.part = p.parts[m.r] + local;
    m.t0 = a.offsets[m.r];
    m.fresh = a.offsets[m.r + 1] - m.t0;
    m.context = max(0, a.context[m.r]);
    const int last = min(m.fresh - 1, (int)(((long long)(m.tile + 1) * KA_ROWS - 1) / a.H));  // the tile's last token
    const long long c0 = (long long)m.chunk * p.chunk * KA_UNIT, c1 = c0 + (long long)p.chunk * KA_UNIT;
    const int end = (int)min((long long)max(0, m.context - m.fresh + last + 1), (long long)a.max_pages << a.c.shift);
    m.s0 = (int)min(c0, (long long)end);
    m.s1 = (int)min(c1, (long long)end);
    return m;
}

// A plain form for any shape: a tile's queries and 32 positions' values in shared memory in fp32.
#define KS_P 32
#define KS_LD (KV4_BLOCKS_MAX * 32 + 4)
__global__ __launch_bounds__(KA_BLOCK) void k_kv4_attend(Kv4Attn a) {
    __shared__ Kv4Plan plan;
    __shared__ float q[KA_ROWS][KS_LD];
    __shared__ float kt[KS_P / 2][KS_LD];
    __shared__ float sc[KA_ROWS][KS_P / 2];
    __shared__ float ml[KA_ROWS][2], cr[KA_ROWS];
    __shared__ int on[KS_P / 2];
    constexpr int P = KS_P / 2;
    const int tid = threadIdx.x, kv = a.c.kv, rope = a.c.rope, cols = 32 * a.c.blocks, lanes = 4 * a.c.blocks;
    kv4_plan(a, plan);
    for (unsigned it = blockIdx.x; it < plan.total; it += gridDim.x) {
        const Kv4Item m = kv4_item(a, plan, it);
        const long long rows = (long long)m.fresh * a.H, row0 = (long long)m.tile * KA_ROWS;
        const int nr = (int)min((long long)KA_ROWS, rows - row0);
        __syncthreads();
        for (int i = tid; i < KA_ROWS * cols; i += KA_BLOCK) {
            const int rr = i / cols, col = i % cols;
            float v = 0.0f;
            if (rr < nr) {
                const long long g = row0 + rr, t = m.t0 + g / a.H;
                const int h = (int)(g % a.H);
                if (col < kv) v = a.q_abs[t * a.ld_q_abs + (long long)h * kv + col];
                else if (col - kv < rope) v = a.q_pe[t * a.ld_q_pe + (long long)h * rope + col - kv];
            }
            q[rr][col] = v;
        }
        float acc[KA_ROWS][2];
#pragma unroll
        for (int rr = 0; rr < KA_ROWS; rr++) acc[rr][0] = acc[rr][1] = 0.0f;
        if (tid < KA_ROWS) {
            ml[tid][0] = -INFINITY;
            ml[tid][1] = 0.0f;
        }
        for (int s0 = m.s0; s0 < m.s1; s0 += P) {
            __syncthreads();
            for (int i = tid; i < P * lanes; i += KA_BLOCK) {
                const int j = i / lanes, w = i % lanes, s = s0 + j;
                float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
                bool ok = s < m.s1;
                if (ok) {
                    const int page = a.table[(size_t)m.r * a.max_pages + (s >> a.c.shift)];
                    ok = page >= 0 && page < a.c.n_pages;
                    if (ok) {
                        const size_t slot = ((size_t)page << a.c.shift) + (s & ((1 << a.c.shift) - 1));
                        const uint8_t *row = a.c.rows + slot * a.c.row_bytes;
                        kv4_values(((const unsigned *)row)[w], row[16 * a.c.blocks + (w >> 2)], v);
                    }
                }
                if (w == 0) on[j] = ok;
#pragma unroll
                for (int k = 0; k < 8; k++) kt[j][8 * w + k] = v[k];
            }
            __syncthreads();
            for (int i = tid; i < KA_ROWS * P; i += KA_BLOCK) {
                const int rr = i / P, j = i % P;
                float d = 0.0f;
                for (int col = 0; col < cols; col++) d = fmaf(q[rr][col], kt[j][col], d);
                const long long last = m.context - m.fresh + (row0 + rr) / a.H;
                sc[rr][j] = rr < nr && on[j] && s0 + j <= last ? d * a.scale : -INFINITY;
            }
            __syncthreads();
            if (tid < KA_ROWS) {
                float mx = ml[tid][0], l = ml[tid][1];
                for (int j = 0; j < P; j++) mx = fmaxf(mx, sc[tid][j]);
                const float ref = mx == -INFINITY ? 0.0f : mx, back = ml[tid][0] == -INFINITY ? 0.0f : expf(ml[tid][0] - ref);
                l *= back;
                for (int j = 0; j < P; j++) {
                    const float x = sc[tid][j], e = x == -INFINITY ? 0.0f : expf(x - ref);
                    sc[tid][j] = e;
                    l += e;
                }
                ml[tid][0] = mx;
                ml[tid][1] = l;
                cr[tid] = back;
            }
            __syncthreads();
            for (int rr = 0; rr < KA_ROWS; rr++) {
                acc[rr][0] *= cr[rr];
                acc[rr][1] *= cr[rr];
            }
            for (int j = 0; j < P; j++) {
                const float v0 = kt[j][tid], v1 = kt[j][tid + KA_BLOCK];
                for (int rr = 0; rr < KA_ROWS; rr++) {
                    const float e = sc[rr][j];
                    if (e != 0.0f) {  // a masked position's value may be NaN
                        acc[rr][0] = fmaf(e, v0, acc[rr][0]);
                        acc[rr][1] = fmaf(e, v1, acc[rr][1]);
                    }
                }
            }
        }
        __syncthreads();
        for (int rr = 0; rr < nr; rr++) {
            const float l = ml[rr][1];
            float *dst;
            float f = 1.0f;
            if (m.k > 1) {
                dst = a.part + ((size_t)m.part * KA_ROWS + rr) * kv;
                if (tid < 2) a.part_ml[((size_t)m.part * KA_ROWS + rr) * 2 + tid] = ml[rr][tid];
            } else {
                const long long g = row0 + rr, t = m.t0 + g / a.H;
                dst = a.out + t * a.ld_out + (g % a.H) * kv;
                f = l == 0.0f ? 0.0f : 1.0f / l;
            }
            if (tid < kv) dst[tid] = f == 0.0f ? 0.0f : acc[rr][0] * f;
            if (tid + KA_BLOCK < kv) dst[tid + KA_BLOCK] = f == 0.0f ? 0.0f : acc[rr][1] * f;
        }
    }
}

// The cut tiles' partial results joined, a block a query row: out = sum_c w_c part_c / sum_c w_c l_c
// with w_c = exp(m_c - m).
__global__ __launch_bounds__(KA_BLOCK) void k_kv4_merge(Kv4Attn a) {
    __shared__ Kv4Plan plan;
    __shared__ float wgt[KA_MAX_PARTS];
    __shared__ float red[KA_BLOCK / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, kv = a.c.kv;
    kv4_plan(a, plan);
    unsigned i = 0;
    for (unsigned unit = blockIdx.x;; unit += gridDim.x) {
        // the unit-th row slot of the cut tiles
        const unsigned ti = unit / KA_ROWS, rr = unit % KA_ROWS;
        // walk the items to the ti-th cut tile
        unsigned seen = 0;
        bool found = false;
        for (int r = 0; r < a.R; r++) {
            const unsigned n = plan.items[r] - (r > 0 ? plan.items[r - 1] : 0u);
            const unsigned k = max(1u, (ka_units(a, r) + plan.chunk - 1) / plan.chunk);
            if (k < 2 || n == 0) continue;
            if (ti < seen + n / k) {
                i = (r > 0 ? plan.items[r - 1] : 0u) + (ti - seen) * k;
                found = true;
                break;
            }
            seen += n / k;
        }
        if (!found) return;
        const Kv4Item m = kv4_item(a, plan, i);
        const long long g = (long long)m.tile * KA_ROWS + rr;
        if (g >= (long long)m.fresh * a.H) continue;
        const float *pml = a.part_ml + ((size_t)m.part * KA_ROWS + rr) * 2;
        float mx = -INFINITY;
        for (int c = tid; c < m.k; c += KA_BLOCK) mx = fmaxf(mx, pml[(size_t)c * KA_ROWS * 2]);
        mx = wave_max_dpp_f(mx);
        __syncthreads();
        if (lane == 0) red[w] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        __syncthreads();
        float l = 0.0f;
        for (int c = tid; c < m.k; c += KA_BLOCK) {
            const float pm = pml[(size_t)c * KA_ROWS * 2], pl = pml[(size_t)c * KA_ROWS * 2 + 1];
            const float e = pl == 0.0f ? 0.0f : expf(pm - mx);
            wgt[c] = e;
            l = fmaf(pl, e, l);
        }
        for (int d = 32; d > 0; d >>= 1) l += __shfl_xor(l, d);
        if (lane == 0) red[w] = l;
        __syncthreads();
        l = (red[0] + red[1]) + (red[2] + red[3]);
        float *dst = a.out + (m.t0 + g / a.H) * a.ld_out + (g % a.H) * kv;
        for (int col = tid; col < kv; col += KA_BLOCK) {
            const float *pc = a.part + ((size_t)m.part * KA_ROWS + rr) * kv + col;
            float s = 0.0f;
            for (int c = 0; c < m.k; c++)
                if (wgt[c] != 0.0f) s = fmaf(wgt[c], pc[(size_t)c * KA_ROWS * kv], s);
            dst[col] = l == 0.0f ? 0.0f : s / l;
        }
    }
}
