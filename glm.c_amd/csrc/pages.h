// pages.h -- page tables and slot maps of a step over several requests (gmoe_page_maps): prefix
// sums over the requests' tokens and page needs, then one thread a token.
//
// Every block repeats the two prefix sums over all requests (at most PM_MAX_R, 16 KB of lengths
// from L2) and keeps them in shared memory, so that one launch does: the tokens are then
// independent, and a token finds its request by a binary search over the sums. The pages a step
// takes are written by the tokens that begin them: page j of a request starts at position
// j * page_size, which is one of its new tokens exactly where j is a new page.
//
// Latency bound at every size (a call moves 0.1 MB for 1000 requests): a wait on the lengths, two sums, a
// search, a wait on the page. 1000 requests with 7411 tokens: 6.7 us a call, as one request's (a launch
// from the host alone is about that), with a token a thread and the first lengths in registers; 9.7
// with four tokens a thread and lengths reread.
#pragma once

#include "common.h"
#include "gmoe_serve.h"

#define PM_BLOCK 256
#define PM_MAX_R GMOE_MAX_REQUESTS
#define PM_MAX_LEN (1 << 30)

// Inclusive prefix sum over a wave's lanes, modulo 2^32, by moves within rows of 16 lanes.
__device__ static inline unsigned wave_incl_scan_u(unsigned v) {
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_SHR(1), 0xF, 0xF, false);
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_SHR(2), 0xF, 0xF, false);
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_SHR(4), 0xF, 0xF, false);
    v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, DPP_ROW_SHR(8), 0xF, 0xF, false);
    const unsigned r0 = (unsigned)__builtin_amdgcn_readlane((int)v, 15), r1 = (unsigned)__builtin_amdgcn_readlane((int)v, 31),
                   r2 = (unsigned)__builtin_amdgcn_readlane((int)v, 47);
    const int row = (threadIdx.x & 63) >> 4;
    return v + (row >= 1 ? r0 : 0u) + (row >= 2 ? r1 : 0u) + (row >= 3 ? r2 : 0u);
}

// Exclusive prefix sum over the block's threads, and the total, through shared memory (one
// word a wave). Wraps modulo 2^32.
__device__ static inline unsigned block_scan_u(unsigned v, unsigned *red, unsigned *total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const unsigned s = wave_incl_scan_u(v);
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

// One thread's requests: r0 .. r1 - 1, the first one's lengths in registers (they are all there are with up
// to PM_BLOCK requests, so that one wait on memory does).
__global__ __launch_bounds__(PM_BLOCK) void k_page_maps(gmoe_batch b, int shift) {
    __shared__ unsigned ends[PM_MAX_R];   // tokens up to and with the request, of any fit
    __shared__ unsigned before[PM_MAX_R]; // pages taken before the request; PM_SHORT: it is short
    __shared__ unsigned red[PM_BLOCK / 64], red2[PM_BLOCK / 64];
    constexpr unsigned PM_SHORT = 0xffffffffu;
    const int tid = threadIdx.x, R = b.n_requests;
    const unsigned T = b.max_tokens, mask = (1u << shift) - 1;
    const int per = (R + PM_BLOCK - 1) / PM_BLOCK, r0 = min(R, tid * per), r1 = min(R, r0 + per);
    const int n_free_ = *b.n_free, seen0 = r0 < r1 ? b.seen[r0] : 0, fresh0 = r0 < r1 ? b.fresh[r0] : 0;
    auto seen_of = [&](int r) { return r == r0 ? seen0 : b.seen[r]; };
    auto fresh_of = [&](int r) { return r == r0 ? fresh0 : b.fresh[r]; };
    // a request's tokens count up to T + 1 here, so that R of them stay below 2^32
    auto tokens_of = [&](int r) { return min((unsigned)max(fresh_of(r), 0), T + 1); };
    unsigned sum = 0;
    for (int r = r0; r < r1; r++) sum += tokens_of(r);
    unsigned tokens;
    unsigned at = block_scan_u(sum, red, &tokens);
    unsigned pages = 0;
    for (int r = r0; r < r1; r++) {
        const int seen = seen_of(r), fresh = fresh_of(r);
        at += tokens_of(r);
        ends[r] = at;
        unsigned need = PM_SHORT;
        if (seen >= 0 && fresh >= 0 && seen <= PM_MAX_LEN && fresh <= PM_MAX_LEN && at <= T) {
            const unsigned have = ((unsigned)seen + mask) >> shift, want = ((unsigned)seen + (unsigned)fresh + mask) >> shift;
            if (want <= (unsigned)b.max_pages) need = want - have;
        }
        before[r] = need;
        if (need != PM_SHORT) pages += need;
    }
    unsigned all;
    unsigned first = block_scan_u(pages, red2, &all);
    const unsigned n_free = (unsigned)max(n_free_, 0);
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
    __syncthreads();
    tokens = min(tokens, T);
    const unsigned t = blockIdx.x * PM_BLOCK + tid;
    if (t < T) {
        int r = -1, pos = -1, slot = -1;
        if (t < tokens) {
            r = upper_bound_u(ends, R, t);
            const unsigned begin = before[r];
            if (begin != PM_SHORT) {
                const int seen = b.seen[r];
                pos = seen + (int)(t - (r > 0 ? ends[r - 1] : 0u));
                const unsigned have = ((unsigned)seen + mask) >> shift, j = (unsigned)pos >> shift;
                int *row = b.table + (size_t)r * b.max_pages;
                int page;
                if (j >= have) {
                    page = b.free_pages[n_free - 1 - (begin + (j - have))];
                    if (pos == (int)(j << shift)) row[j] = page;
                } else {
                    page = row[j];
                }
                const long long s = ((long long)page << shift) + (pos & (int)mask);
                slot = page < 0 || s > 0x7fffffffLL ? -1 : (int)s;
            }
        }
        b.request[t] = r;
        b.position[t] = pos;
        b.slot[t] = slot;
    }
    for (int r = blockIdx.x * PM_BLOCK + tid; r < R; r += gridDim.x * PM_BLOCK) {
        b.offsets[r + 1] = (int)min(ends[r], T);
        b.context[r] = before[r] == PM_SHORT ? 0 : b.seen[r] + b.fresh[r];
    }
    if (blockIdx.x > 0) return;
    unsigned all_taken, all_short;
    block_scan_u(taken, red, &all_taken);
    block_scan_u(shorts, red2, &all_short);
    if (tid == 0) {
        b.offsets[0] = 0;
        b.totals[0] = (int)tokens;
        b.totals[1] = (int)all_taken;
        b.totals[2] = (int)all_short;
    }
}
