// logprobs.h -- log probabilities of given tokens, entropy and top alternatives of rows of logits
// (gmoe_logprobs), in one pass over the logits.
//
// Mathematics. With m a row's largest logit and S the sum of exp(x - m) over every other token,
// ln p = (x - m) - log1p(S) and the entropy is log1p(S) + D / (1 + S), D = sum exp(x - m) (m - x): sums
// of terms of one sign, which keep their relative precision where one token has nearly all of p
// (S far below 1). (m, S, D) of two parts join by moving the part of the lower m to the higher:
// S' = f S, D' = f (D + dm S), f = e^-dm, and the lower m itself joins as one more term. A thread
// keeps a triple of its own, so the pass has no exchange; a tile's values meet in a knockout
// (max and min of pairs), whose winner is the tile's maximum and whose losers are the terms.
//
// Top alternatives. Keys order the logits by value, then the lower index, and no two are
// equal. A block keeps the list of keys that may be among its `top` largest: those above a
// threshold, which starts from the first tile's per-thread maxima (a value that `top` of them reach,
// a quarter in each wave) and is set to the list's top-th key each time the list is cut to
// `top`. After the first tiles nearly no value passes, so that a tile costs one comparison a
// thread. Later tiles hold higher indexes, so a value equal to the threshold does not pass.
//
// Split. A block takes a run of tiles of a row; with more than one run a row (few rows) the
// runs' triples and keys go through the workspace and k_lp_join joins them, a block a row.
#pragma once

#include <float.h>

#include "common.h"
#include "gmoe_serve.h"
#include "pages.h"

#define LP_BLOCK 256
#define LP_E 8           // logits a thread holds: with 16, half the blocks fit a CU (801 rows: 117 us against 98)
#define LP_TILE (LP_BLOCK * LP_E)
#define LP_SEGS 256     // most runs of a row: a thread each in k_lp_join
#define LP_LIST 192     // list entries besides a tile's (LP_CUT and more: eight blocks' shared memory fits a CU)
#define LP_CUT 160      // the list is cut to `top` when it is longer
static_assert(LP_LIST >= LP_CUT && LP_CUT >= GMOE_TOP_MAX, "a tile's values fit behind a list that is not cut");

// A run's result: the triple, its keys' number, whether a value is NaN.
struct LpRun {
    float m, s, d;
    int n;  // -1: a NaN
};

struct LpArgs {
    gmoe_logprobs_args a;
    int segs, per;  // runs a row, tiles a run
    LpRun *runs;                // [n][segs]
    unsigned long long *keys;   // [n][segs][top], the largest first
};

// A value and its index as one integer that orders rows of logits: by value, then the lower index
// first. Not for NaN. 0 is below every key.
__device__ static inline unsigned long long lp_key(float x, int i) {
    const unsigned b = __float_as_uint(x + 0.0f);  // (-0 equals +0)
    const unsigned o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)o << 32 | (unsigned)~i;
}
__device__ static inline float lp_value(unsigned long long key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ static inline int lp_index(unsigned long long key) { return (int)~(unsigned)key; }

// e^y for y <= 0 (0 for -inf): the product's rounding is 2^-24 |y| of a result of e^y.
__device__ static inline float lp_exp(float y) { return __builtin_amdgcn_exp2f(y * 1.44269504f); }

struct LpSum {
    float m, s, d;
    // The running sums moved to a reference of at least m.
    __device__ inline void move(float ref) {
        const float f = lp_exp(m - ref), dm = fminf(ref - m, 1000.0f);  // (f is 0 by then)
        d = f * fmaf(dm, s, d);
        s *= f;
    }
    __device__ inline void term(float x, float ref) {
        const float y = x - ref, e = lp_exp(y);
        s += e;
        d = fmaf(-e, fmaxf(y, -1000.0f), d);  // (0 * inf is no term)
    }
};

// Sum over the 64 lanes of a wave, to every lane.
__device__ static inline float wave_sum_dpp_f(float v) {
    v = row_sum_dpp_f(v);
    return (readlane_f(v, 0) + readlane_f(v, 16)) + (readlane_f(v, 32) + readlane_f(v, 48));
}

// The block's triples joined into one, in every thread; red: 3 * LP_BLOCK / 64 floats.
__device__ static inline LpSum lp_join(LpSum v, float *red) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    constexpr int W = LP_BLOCK / 64;
    float M = wave_max_dpp_f(v.m);
    __syncthreads();
    if (lane == 0) red[w] = M;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < W; k++) M = fmaxf(M, red[k]);
    int first = 0;  // the first wave that holds the maximum: its first such lane's own term is left out
    while (first < W - 1 && red[first] != M) first++;
    const unsigned long long has = __ballot(v.m == M);
    const bool mine = w == first && has && lane == __ffsll((unsigned long long)has) - 1;
    const float ref = fmaxf(M, -FLT_MAX), m0 = v.m;
    v.move(ref);
    if (!mine) v.term(m0, ref);
    v.s = wave_sum_dpp_f(v.s);
    v.d = wave_sum_dpp_f(v.d);
    if (lane == 0) {
        red[W + w] = v.s;
        red[2 * W + w] = v.d;
    }
    __syncthreads();
    v.m = M;
    v.s = (red[W] + red[W + 1]) + (red[W + 2] + red[W + 3]);
    v.d = (red[2 * W] + red[2 * W + 1]) + (red[2 * W + 2] + red[2 * W + 3]);
    return v;
}
static_assert(LP_BLOCK == 256, "lp_join adds four waves");

// The list of keys of a block, in shared memory, with what cutting it needs.
template <int CAP>
struct LpList {
    unsigned long long key[CAP];
    unsigned long long best[GMOE_TOP_MAX];
    unsigned hist[256];
    unsigned scan[LP_BLOCK / 64];
    unsigned n, digit, left, fill;
};

// Cuts the list's first n keys to its `top` largest (n where there are fewer), the largest first,
// and returns how many those are; every thread calls it with the same n, after a barrier.
template <int CAP>
__device__ static int lp_cut(LpList<CAP> &l, int n, int top) {
    const int tid = threadIdx.x;
    const unsigned long long *src = l.key;
    if (n > 2 * LP_BLOCK) {
        // the top-th largest key, digit by digit from the highest: `left` of the keys that
        // share the digits so far are wanted
        unsigned long long prefix = 0;
        int shift = 56;
        unsigned left = top;
        for (;; shift -= 8) {
            l.hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += LP_BLOCK) {
                const unsigned long long k = l.key[i];
                if (shift == 56 || k >> (shift + 8) == prefix) atomicAdd(&l.hist[(k >> shift) & 255], 1u);
            }
            __syncthreads();
            const unsigned c = l.hist[255 - tid];
            unsigned all;
            const unsigned above = block_scan_u(c, l.scan, &all);
            if (above < left && left <= above + c) {
                l.digit = 255 - tid;
                l.left = left - above;
                l.fill = c;
            }
            __syncthreads();
            prefix = prefix << 8 | l.digit;
            left = l.left;
            const bool whole = left == l.fill;  // the whole bin is wanted
            __syncthreads();
            if (whole || shift == 0) break;
        }
        const unsigned long long least = prefix << shift;
        if (tid == 0) l.fill = 0;
        __syncthreads();
        for (int i = tid; i < n; i += LP_BLOCK)
            if (l.key[i] >= least) l.best[atomicAdd(&l.fill, 1u)] = l.key[i];
        __syncthreads();
        src = l.best;
        n = top;
    }
    // ranked by counting the larger ones
    const unsigned long long k0 = tid < n ? src[tid] : 0, k1 = tid + LP_BLOCK < n ? src[tid + LP_BLOCK] : 0;
    int r0 = 0, r1 = 0;
    if (n <= LP_BLOCK) {
        if ((tid & ~63) < n)  // (the other waves hold none)
#pragma unroll 8
            for (int j = 0; j < n; j++) r0 += src[j] > k0;
    } else {
#pragma unroll 8
        for (int j = 0; j < n; j++) {
            const unsigned long long k = src[j];
            r0 += k > k0;
            r1 += k > k1;
        }
    }
    __syncthreads();
    if (tid < n && r0 < top) l.key[r0] = k0;
    if (tid + LP_BLOCK < n && r1 < top) l.key[r1] = k1;
    __syncthreads();
    return min(n, top);
}

// The logit of the row's given token g, NaN outside the vocabulary.
__device__ static inline float lp_given(const gmoe_logprobs_args &a, int row, int g) {
    const int id = a.given[(size_t)row * a.n_given + g];
    return id < 0 || id >= a.vocab ? __uint_as_float(0x7fc00000u) : a.logits[(size_t)row * a.ld + id];
}

// The row's results from its joined triple and its alternatives (k of them, the largest first);
// given: the thread's lp_given of the first LP_BLOCK tokens, requested long before.
__device__ static inline void lp_finish(const gmoe_logprobs_args &a, int row, const LpSum &t, bool nan, const unsigned long long *key,
                                        int k, float given) {
    const int tid = threadIdx.x;
    const float NaN = __uint_as_float(0x7fc00000u), ls = log1pf(t.s);
    const bool bad = nan || !(t.m < INFINITY), none = t.m == -INFINITY;
    auto lp = [&](float v) { return bad || v != v ? NaN : none ? -INFINITY : (v - t.m) - ls; };
    if (tid == 0 && a.entropy) a.entropy[row] = bad ? NaN : none ? 0.0f : ls + t.d / (1.0f + t.s);
    for (int g = tid; g < a.n_given; g += LP_BLOCK)
        a.logprob[(size_t)row * a.n_given + g] = lp(g == tid ? given : lp_given(a, row, g));
    if (tid < a.top) {
        const bool no = tid >= k;
        a.top_id[(size_t)row * a.top + tid] = no || bad || none ? -1 : lp_index(key[tid]);
        a.top_logprob[(size_t)row * a.top + tid] = bad ? NaN : no ? -INFINITY : lp(lp_value(key[tid]));
    }
}

// A run of a row, runs side by side: `per` tiles of LP_TILE logits. Tiles start at the 16-byte
// line of the row's first logit, so that every load but a row's first and last is whole.
__global__ __launch_bounds__(LP_BLOCK, 8) void k_lp_run(LpArgs g) {
    constexpr int E = LP_E, TILE = LP_TILE;
    __shared__ LpList<TILE + LP_LIST> l;
    __shared__ float red[3 * LP_BLOCK / 64];
    __shared__ float tops[LP_BLOCK / 64];
    const gmoe_logprobs_args &a = g.a;
    const int tid = threadIdx.x, row = blockIdx.x / g.segs, seg = blockIdx.x - row * g.segs, V = a.vocab, top = a.top;
    const float *x = a.logits + (size_t)row * a.ld;
    const int lead = (int)((uintptr_t)x >> 2 & 3);  // logits of the first line before the row's
    const int end = V + lead, i0 = seg * g.per * TILE, i1 = min(end, i0 + g.per * TILE);
    const float *line = x - lead;
    LpSum t = {-INFINITY, 0.0f, 0.0f};
    const float given = g.segs == 1 && tid < a.n_given ? lp_given(a, row, tid) : 0.0f;
    bool nan = false;
    float over = -INFINITY;  // a value passes above it
    if (tid == 0) l.n = 0;
    __syncthreads();
    int n = 0, cut = 0;  // the list's length, and what it was cut to
    for (int base = i0; base < i1; base += TILE) {
        float v[E];
        const bool edge = base < lead || base + TILE > end;
#pragma unroll
        for (int k = 0; k < E / 4; k++) {
            const int i = base + 4 * (k * LP_BLOCK + tid);
            if (!edge || (i >= lead && i + 4 <= end)) {
                // read once, so non-temporal: 801 rows of 151551 97 us, 102 with plain loads; 64 of 154880 18.4, 18.0
                typedef float f4 __attribute__((ext_vector_type(4)));
                *(f4 *)&v[4 * k] = __builtin_nontemporal_load((const f4 *)(line + i));
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) v[4 * k + j] = i + j >= lead && i + j < end ? line[i + j] : -INFINITY;
            }
        }
        float p[E];
#pragma unroll
        for (int k = 0; k < E; k++) {
            p[k] = v[k];
            nan |= v[k] != v[k];
        }
#pragma unroll
        for (int w = E / 2; w >= 1; w >>= 1)
#pragma unroll
            for (int k = 0; k < w; k++) {
                const float hi = fmaxf(p[k], p[k + w]), lo = fminf(p[k], p[k + w]);
                p[k] = hi;
                p[k + w] = lo;
            }
        const float tm = p[0], lo = fminf(t.m, tm), mn = fmaxf(t.m, tm), ref = fmaxf(mn, -FLT_MAX);
        t.move(ref);
        t.m = mn;
        t.term(lo, ref);
#pragma unroll
        for (int k = 1; k < E; k++) t.term(p[k], ref);
        if (top == 0) continue;
        const bool first = base == i0;
        if (first) {
            // a value that a quarter of `top` of each wave's maxima reach, so that `top` values do
            const int quarter = (top + LP_BLOCK / 64 - 1) / (LP_BLOCK / 64);
            float best = wave_max_dpp_f(tm), rest = tm;
            for (int j = 1; j < quarter; j++) {  // the largest below the ones before, of which there was one at least each
                rest = rest < best ? rest : -INFINITY;
                best = wave_max_dpp_f(rest);
            }
            if ((tid & 63) == 0) tops[tid >> 6] = best;
            __syncthreads();
            over = fminf(fminf(tops[0], tops[1]), fminf(tops[2], tops[3]));
        }
        if (first ? tm >= over : tm > over) {
#pragma unroll
            for (int k = 0; k < E; k++) {
                const int i = base + 4 * ((k >> 2) * LP_BLOCK + tid) + (k & 3);
                if ((first ? v[k] >= over : v[k] > over) && i >= lead && i < end) l.key[atomicAdd(&l.n, 1u)] = lp_key(v[k], i - lead);
            }
        }
        block_barrier();
        n = (int)l.n;
        block_barrier();
        if (first || n > LP_CUT) {
            n = cut = lp_cut(l, n, top);
            if (n == top) over = lp_value(l.key[top - 1]);
            if (tid == 0) l.n = n;
            __syncthreads();
        }
    }
    nan = __syncthreads_or(nan);
    t = lp_join(t, red);
    if (n > cut) n = lp_cut(l, n, top);
    if (g.segs == 1) {
        lp_finish(a, row, t, nan, l.key, n, given);
        return;
    }
    const size_t at = (size_t)row * g.segs + seg;
    if (tid == 0) g.runs[at] = LpRun{t.m, t.s, t.d, nan ? -1 : n};
    if (tid < n) g.keys[at * top + tid] = l.key[tid];
}

// A row's runs joined. Keys: those no smaller than the top-th largest of the runs' first keys, which
// come from `top` runs at most.
__global__ __launch_bounds__(LP_BLOCK) void k_lp_join(LpArgs g) {
    constexpr int CAP = GMOE_TOP_MAX * GMOE_TOP_MAX;
    __shared__ LpList<CAP> l;
    __shared__ float red[3 * LP_BLOCK / 64];
    __shared__ unsigned long long firsts[LP_SEGS];
    __shared__ int counts[LP_SEGS], from[GMOE_TOP_MAX];
    __shared__ unsigned long long bound;
    const int tid = threadIdx.x, row = blockIdx.x, top = g.a.top, segs = g.segs;
    const size_t at = (size_t)row * segs;
    LpSum t = {-INFINITY, 0.0f, 0.0f};
    int n = 0;
    unsigned long long mine = 0;
    const float given = tid < g.a.n_given ? lp_given(g.a, row, tid) : 0.0f;
    if (tid < segs) {
        const LpRun r = g.runs[at + tid];
        if (top > 0) mine = g.keys[(at + tid) * top];
        t = {r.m, r.s, r.d};
        n = r.n;
        mine = n > 0 ? mine : 0;
    }
    const bool nan = __syncthreads_or(n < 0);
    t = lp_join(t, red);
    if (top > 0) {
        firsts[tid] = mine;
        counts[tid] = max(n, 0);
        if (tid == 0) {
            l.n = 0;
            bound = 0;
        }
        __syncthreads();
        int above = 0;  // runs with a larger first key
#pragma unroll 8
        for (int j = 0; j < segs; j++) above += firsts[j] > mine;
        if (mine && above < top) from[above] = tid;
        if (mine && above == top - 1) bound = mine;
        const int live = min(top, __syncthreads_count(mine != 0));
        const unsigned long long least = bound;
#pragma unroll 2
        for (int i = tid; i < live * top; i += LP_BLOCK) {
            const int s = from[i / top], j = i % top;
            const unsigned long long k = j < counts[s] ? g.keys[(at + s) * top + j] : 0;
            if (k && k >= least) l.key[atomicAdd(&l.n, 1u)] = k;
        }
        __syncthreads();
        n = lp_cut(l, (int)l.n, top);
    }
    lp_finish(g.a, row, t, nan, l.key, n, given);
}

// How a call is split: as many runs a row as the GPU holds at once (eight blocks a CU), so that
// every block starts at once and none is left for a second turn. 801 rows of 151551 (1602 blocks):
// 98 us, and 113 with 2403 blocks, 139 with 801; 64 rows of 154880: 17 us with 26 runs a row, 20 with 13.
#define LP_FILL 2048
struct LpSplit {
    int segs, per;  // runs a row, tiles a run
};
static inline LpSplit lp_split(int n, int vocab) {
    const int tiles = (vocab + 3 + LP_TILE - 1) / LP_TILE, want = std::max(1, std::min({tiles, LP_FILL / n, LP_SEGS}));
    LpSplit s;
    s.per = (tiles + want - 1) / want;
    s.segs = (tiles + s.per - 1) / s.per;
    return s;
}
