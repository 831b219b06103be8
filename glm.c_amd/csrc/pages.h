// pages.h -- page tables and slot maps of a step over several requests (gmoe_page_maps): prefix
// sums over the requests' tokens and page needs, then one thread a token.
//
// Every block repeats the two prefix sums over all requests (at most PM_MAX_R, 16 KB of lengths
// from L2) and keeps them in shared memory, so that one launch does: the tokens are then
// independent, and a token finds its request by a binary search over the sums. The pages a step
// takes are written by the tokens that begin them: page j of a request starts at position
// j * page_size, which is one of its new tokens exactly where j is a new page.
#pragma once

#include "common.h"
#include "gmoe_serve.h"

#define PM_BLOCK 256
#define PM_TOKENS 1024  // tokens a block
#define PM_MAX_R GMOE_MAX_REQUESTS
#define PM_PER (PM_MAX_R / PM_BLOCK)
#define PM_MAX_LEN (1 << 30)

// Exclusive prefix sum over the block's threads, and the total, through shared memory (one
// word a wave). Wraps modulo 2^32.
__device__ static inline unsigned block_scan_u(unsigned v, unsigned *red, unsigned *total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    unsigned s = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_up(s, d);
        if (lane >= d) s += o;
    }
    __syncthreads();  // (red may still be read from a call before)
    if (lane == 63) red[w] = s;
    __syncthreads();
    unsigned before = 0, all = 0;
    for (int i = 0; i < nw; i++) {
        if (i < w) before += red[i];
        all += red[i];
    }
    *total = all;
    return before + s - v;
}

// The first i of 0..n-1 with v[i] > x (v rising); n where there is none.
__device__ static inline int upper_bound_u(const unsigned *v, int n, unsigned x) {
    int lo = 0;
    while (n > 0) {
        const int half = n >> 1;
        if (v[lo + half] <= x) {
            lo += half + 1;
            n -= half + 1;
        } else {
            n = half;
        }
    }
    return lo;
}

__global__ __launch_bounds__(PM_BLOCK) void k_page_maps(gmoe_batch b, int shift) {
    __shared__ unsigned ends[PM_MAX_R];   // tokens up to and with the request, of any fit
    __shared__ unsigned before[PM_MAX_R]; // pages taken before the request; PM_SHORT: it is short
    __shared__ unsigned red[PM_BLOCK / 64];
    constexpr unsigned PM_SHORT = 0xffffffffu;
    const int tid = threadIdx.x, R = b.n_requests;
    const unsigned T = b.max_tokens;
    const int per = (R + PM_BLOCK - 1) / PM_BLOCK, r0 = tid * per, r1 = min(R, r0 + per);
    // a request's tokens count up to T + 1 here, so that R of them stay below 2^32
    unsigned sum = 0;
    for (int r = r0; r < r1; r++) sum += min((unsigned)max(b.fresh[r], 0), T + 1);
    unsigned tokens;
    unsigned at = block_scan_u(sum, red, &tokens);
    unsigned pages = 0;
    for (int r = r0; r < r1; r++) {
        const int seen = b.seen[r], fresh = b.fresh[r];
        at += min((unsigned)max(fresh, 0), T + 1);
        ends[r] = at;
        unsigned need = PM_SHORT;
        if (seen >= 0 && fresh >= 0 && seen <= PM_MAX_LEN && fresh <= PM_MAX_LEN && at <= T) {
            const unsigned mask = (1u << shift) - 1;
            const unsigned have = ((unsigned)seen + mask) >> shift, want = ((unsigned)seen + (unsigned)fresh + mask) >> shift;
            if (want <= (unsigned)b.max_pages) need = want - have;
        }
        before[r] = need;
        if (need != PM_SHORT) pages += need;
    }
    unsigned all;
    unsigned first = block_scan_u(pages, red, &all);
    const unsigned n_free = (unsigned)max(*b.n_free, 0);
    unsigned taken = 0, shorts = 0;
    for (int r = r0; r < r1; r++) {
        const unsigned need = before[r];
        if (need == PM_SHORT) {
            shorts++;
            continue;
        }
        if (need > 0 && first + need > n_free) {
            before[r] = PM_SHORT;
            shorts++;
        } else {
            before[r] = first;
            taken += need;
        }
        first += need;
    }
    unsigned all_taken, all_short;
    block_scan_u(taken, red, &all_taken);
    block_scan_u(shorts, red, &all_short);  // (its barriers also end the writes of ends and before)
    tokens = min(tokens, T);
    if (blockIdx.x == 0 && tid == 0) {
        b.offsets[0] = 0;
        b.totals[0] = (int)tokens;
        b.totals[1] = (int)all_taken;
        b.totals[2] = (int)all_short;
    }
    for (int r = blockIdx.x * PM_BLOCK + tid; r < R; r += gridDim.x * PM_BLOCK) {
        b.offsets[r + 1] = (int)min(ends[r], T);
        b.context[r] = before[r] == PM_SHORT ? 0 : b.seen[r] + b.fresh[r];
    }
#pragma unroll
    for (int k = 0; k < PM_TOKENS / PM_BLOCK; k++) {
        const unsigned t = blockIdx.x * PM_TOKENS + k * PM_BLOCK + tid;
        if (t >= T) break;
        int r = -1, pos = -1, slot = -1;
        if (t < tokens) {
            r = upper_bound_u(ends, R, t);
            const unsigned begin = before[r];
            if (begin != PM_SHORT) {
                const int seen = b.seen[r];
                pos = seen + (int)(t - (r > 0 ? ends[r - 1] : 0u));
                const unsigned have = ((unsigned)seen + (1u << shift) - 1) >> shift, j = (unsigned)pos >> shift;
                int *row = b.table + (size_t)r * b.max_pages;
                int page;
                if (j >= have) {
                    page = b.free_pages[n_free - 1 - (begin + (j - have))];
                    if (pos == (int)(j << shift)) row[j] = page;
                } else {
                    page = row[j];
                }
                const long long s = ((long long)page << shift) + (pos & ((1 << shift) - 1));
                slot = page < 0 || s > 0x7fffffffLL ? -1 : (int)s;
            }
        }
        b.request[t] = r;
        b.position[t] = pos;
        b.slot[t] = slot;
    }
}
