// logprobs.h -- log probabilities of given tokens, entropy and top alternatives of rows of logits
// (gmoe_logprobs).
//
// With m a row's largest logit and S the sum of exp(x - m) over every other token, ln p = (x - m) -
// log1p(S) and the entropy is log1p(S) + sum p (m - x): sums of terms of one sign, which keep their
// relative precision where one token has nearly all of p (S far below 1).
#pragma once

#include "common.h"
#include "gmoe_serve.h"

#define LP_BLOCK 256

// A value and its index as one integer that orders rows of logits: by value, then the lower index
// first; a NaN above every number. 0 is below every key.
__device__ static inline unsigned long long lp_key(float x, int i) {
    const unsigned b = __float_as_uint(x);
    unsigned o = b & 0x80000000u ? ~b : b | 0x80000000u;
    if (x != x) o = 0xffffffffu;
    if (b == 0x80000000u) o = 0x80000000u;  // -0 equals +0
    return (unsigned long long)o << 32 | (unsigned)~i;
}
__device__ static inline float lp_value(unsigned long long key) {
    const unsigned o = (unsigned)(key >> 32);
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ static inline int lp_index(unsigned long long key) { return (int)~(unsigned)key; }

__device__ static inline unsigned long long wave_max_u64(unsigned long long v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const unsigned long long o = __shfl_xor(v, d);
        v = o > v ? o : v;
    }
    return v;
}

// A plain form: a block a row, one pass for each alternative.
__global__ __launch_bounds__(LP_BLOCK) void k_logprobs(gmoe_logprobs_args a) {
    __shared__ unsigned long long rk[LP_BLOCK / 64];
    __shared__ float rs[2][LP_BLOCK / 64];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, V = a.vocab;
    const float *x = a.logits + blockIdx.x * a.ld;
    auto below = [&](unsigned long long lim) {  // the row's largest key under lim
        unsigned long long best = 0;
        for (int i = tid; i < V; i += LP_BLOCK) {
            const unsigned long long k = lp_key(x[i], i);
            if (k < lim && k > best) best = k;
        }
        best = wave_max_u64(best);
        __syncthreads();
        if (lane == 0) rk[w] = best;
        __syncthreads();
        for (int k = 0; k < LP_BLOCK / 64; k++) best = rk[k] > best ? rk[k] : best;
        return best;
    };
    const unsigned long long top = below(~0ull);
    const float m = lp_value(top);
    const int im = lp_index(top);
    const bool none = m == -INFINITY, bad = !(m < INFINITY);
    float s = 0.0f, d = 0.0f;
    for (int i = tid; i < V; i += LP_BLOCK) {
        const float y = x[i] - m, e = expf(y);
        if (i != im) s += e;
        if (e > 0.0f) d = fmaf(e, -y, d);
    }
    for (int k = 32; k > 0; k >>= 1) {
        s += __shfl_xor(s, k);
        d += __shfl_xor(d, k);
    }
    if (lane == 0) {
        rs[0][w] = s;
        rs[1][w] = d;
    }
    __syncthreads();
    s = (rs[0][0] + rs[0][1]) + (rs[0][2] + rs[0][3]);
    d = (rs[1][0] + rs[1][1]) + (rs[1][2] + rs[1][3]);
    const float nan = __uint_as_float(0x7fc00000u), ls = log1pf(s);
    auto lp = [&](float v) { return bad ? nan : none ? -INFINITY : (v - m) - ls; };
    if (tid == 0 && a.entropy) a.entropy[blockIdx.x] = bad ? nan : none ? 0.0f : ls + d / (1.0f + s);
    for (int g = tid; g < a.n_given; g += LP_BLOCK) {
        const int id = a.given[(size_t)blockIdx.x * a.n_given + g];
        a.logprob[(size_t)blockIdx.x * a.n_given + g] = id < 0 || id >= V ? nan : lp(x[id]);
    }
    unsigned long long lim = ~0ull;
    for (int k = 0; k < a.top; k++) {
        lim = below(lim);
        if (tid == 0) {
            const bool no = lim == 0;
            a.top_id[(size_t)blockIdx.x * a.top + k] = no || bad || none ? -1 : lp_index(lim);
            a.top_logprob[(size_t)blockIdx.x * a.top + k] = bad ? nan : no ? -INFINITY : lp(lp_value(lim));
        }
    }
}
