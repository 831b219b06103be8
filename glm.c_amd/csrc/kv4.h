// kv4.h -- the latent cache in 4 bits: rows of e2m1 codes in blocks of 32 columns with a
// power-of-two scale each (gmoe_serve.h), written, read back and attended.
#pragma once

#include "common.h"
#include "gmoe_serve.h"
#include "pages.h"

#define KV4_BYTE_LO 104  // scale 2^-23: the least step a block may have, half of it fp16's least
#define KV4_BYTE_HI 140  // scale 2^13: 6 steps are 49152, below fp16's largest
#define KV4_BYTE_NAN 255
#define KV4_BLOCK 256
#define KV4_BLOCKS_MAX 18  // column blocks of the widest row

// One layer's cache as the kernels take it.
struct Kv4Cache {
    uint8_t *rows;
    int kv, rope;
    int blocks;     // column blocks of a row: kv / 32 + ceil(rope / 32)
    int row_bytes;
    int n_slots, n_pages, shift;
};

__host__ __device__ static inline int kv4_blocks(int kv, int rope) { return kv / 32 + (rope + 31) / 32; }

// ---- writing and reading back ------------------------------------------------------------
//
// Four lanes a block of 32 columns, eight columns a lane, a row's lanes side by side: a lane's
// eight values are two 16-byte loads where the rows are aligned to that (VEC), its eight codes
// one 4-byte store. Bound by the memory traffic, most of it the fp32 values: 8191 rows of 512 + 64 take 7.0 us
// to write (21.5 MB, 3.1 TB/s) and 6.3 to read back (3.4 TB/s), 64 rows 3.4 and 3.1 (a launch).

// The code of |v| = mag steps (mag >= 0): halves up to 2, ones up to 4, then twos, each rounded
// to the even one at a tie (rint), at most 6.
__device__ static inline unsigned kv4_code(float mag) {
    const float lo = rintf(2.0f * mag), mid = 2.0f + rintf(mag), hi = fminf(4.0f + rintf(0.5f * mag), 7.0f);
    return (unsigned)(mag < 1.75f ? lo : mag < 3.5f ? mid : hi);
}

// The largest of the four lanes of a quad.
__device__ static inline unsigned quad_max_u(unsigned v) {
    v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, DPP_QUAD_1032, 0xF, 0xF, false));
    return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, DPP_QUAD_2301, 0xF, 0xF, false));
}

template <bool VEC>
__global__ __launch_bounds__(KV4_BLOCK) void k_kv4_append(Kv4Cache c, int n, const float *__restrict__ comp, int64_t ld_comp,
                                                          const float *__restrict__ pe, int64_t ld_pe,
                                                          const int32_t *__restrict__ slot) {
    const int lanes = 4 * c.blocks;  // of a row
    const unsigned g = blockIdx.x * KV4_BLOCK + threadIdx.x;  // (n * lanes < 2^26)
    const int t = (int)(g / (unsigned)lanes), i = (int)(g % (unsigned)lanes);
    if (t >= n) return;  // (whole quads: a row's lanes are a multiple of four)
    const int s = slot[t];
    if (s < 0 || s >= c.n_slots) return;
    const int col = 8 * i;
    const bool tail = col >= c.kv;
    const float *src = tail ? pe + t * ld_pe + (col - c.kv) : comp + t * ld_comp + col;
    const int have = tail ? min(8, max(0, c.rope - (col - c.kv))) : 8;
    float v[8];
    if (VEC && have == 8) {
        *(float4 *)&v[0] = *(const float4 *)src;
        *(float4 *)&v[4] = *(const float4 *)(src + 4);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = k < have ? src[k] : 0.0f;
    }
    unsigned amax = 0;  // by the bits: finite < infinity < NaN
#pragma unroll
    for (int k = 0; k < 8; k++) amax = max(amax, __float_as_uint(v[k]) & 0x7fffffffu);
    amax = quad_max_u(amax);
    const bool bad = amax >= 0x7f800000u;
    // 2^e <= amax < 2^(e+1) has scale 2^(e-2), or 2^(e-1) when amax is over 7 of those steps
    const int byte = bad ? KV4_BYTE_NAN : min(max((int)((amax + 0x1fffffu) >> 23) - 2, KV4_BYTE_LO), KV4_BYTE_HI);
    const float inv = __uint_as_float((unsigned)(254 - byte) << 23);  // (not used where bad)
    unsigned word = 0;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const unsigned code = kv4_code(fabsf(v[k]) * inv) | (__float_as_uint(v[k]) >> 31) << 3;
        word |= bad ? 0u : code << (4 * k);
    }
    uint8_t *row = c.rows + (size_t)s * c.row_bytes;
    ((unsigned *)row)[i] = word;
    if ((i & 3) == 0) row[16 * c.blocks + (i >> 2)] = (uint8_t)byte;
    const int pad = c.row_bytes - 17 * c.blocks;  // the row's last bytes are zeros
    for (int k = i; k < pad; k += lanes) row[17 * c.blocks + k] = 0;
}

// The eight values of a word of codes at scale 2^(byte - 127).
__device__ static inline void kv4_values(unsigned word, int byte, float (&v)[8]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const float scale = __uint_as_float((unsigned)byte << 23);
    const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 1);
    const f2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, 3);
    const bool bad = byte == KV4_BYTE_NAN;
    const float nan = __uint_as_float(0x7fc00000u);
    v[0] = bad ? nan : a.x;
    v[1] = bad ? nan : a.y;
    v[2] = bad ? nan : b.x;
    v[3] = bad ? nan : b.y;
    v[4] = bad ? nan : d.x;
    v[5] = bad ? nan : d.y;
    v[6] = bad ? nan : e.x;
    v[7] = bad ? nan : e.y;
}

template <bool VEC>
__global__ __launch_bounds__(KV4_BLOCK) void k_kv4_read(Kv4Cache c, int n, const int32_t *__restrict__ slot, float *__restrict__ comp,
                                                        int64_t ld_comp, float *__restrict__ pe, int64_t ld_pe) {
    const int lanes = 4 * c.blocks;
    const unsigned g = blockIdx.x * KV4_BLOCK + threadIdx.x;  // (n * lanes < 2^26)
    const int t = (int)(g / (unsigned)lanes), i = (int)(g % (unsigned)lanes);
    if (t >= n) return;
    const int col = 8 * i;
    const bool tail = col >= c.kv;
    float *base = tail ? pe : comp;
    if (!base) return;
    float *dst = tail ? pe + t * ld_pe + (col - c.kv) : comp + t * ld_comp + col;
    const int have = tail ? min(8, max(0, c.rope - (col - c.kv))) : 8;
    const int s = slot[t];
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (s >= 0 && s < c.n_slots) {
        const uint8_t *row = c.rows + (size_t)s * c.row_bytes;
        kv4_values(((const unsigned *)row)[i], row[16 * c.blocks + (i >> 2)], v);
    }
    if (VEC && have == 8) {
        // non-temporal: the values are a stream nobody reads back here, and the rows stay in the caches
        // (8191 rows of 512 + 64: 6.3 us, 8.9 with plain stores; the next append 7.0, 7.7 after those)
        typedef float f4 __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(*(const f4 *)&v[0], (f4 *)dst);
        __builtin_nontemporal_store(*(const f4 *)&v[4], (f4 *)(dst + 4));
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < have) dst[k] = v[k];
    }
}
