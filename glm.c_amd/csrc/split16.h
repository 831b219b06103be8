// split16.h -- fp32 values as two fp16 parts for the fp16 matrix cores, and those cores' operands:
// shared by the attentions on them (attn16.h, kv4_attn.h).
#pragma once

#include "common.h"

typedef float aq_f4 __attribute__((ext_vector_type(4)));
typedef _Float16 a16_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 a16_h4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) a16_h4 a16_lds_h4;

// The 16-lane group's 4 rows x 16 columns of halves, transposed: lane i of the group names
// the 8 bytes at row i / 4, columns 4 (i % 4) .. + 3, and gets column i of the four rows.
__device__ static inline a16_h4 a16_tr(const _Float16 *p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    return __builtin_bit_cast(a16_h4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)p));
}

#define SPL_EMPTY (-1000)

// The exponent e with |x| 2^-e < 2^15 for every |x| <= mx (SPL_EMPTY when mx is 0).
__device__ static inline int spl_exp(float mx) {
    if (!(mx > 0.0f)) return SPL_EMPTY;
    int k;
    (void)frexpf(mx, &k);  // mx < 2^k
    return k - 15;
}

// x = hi + lo: hi the nearest fp16, lo the nearest fp16 to the (exact) remainder.
__device__ static inline void spl_split(float x, _Float16 &hi, _Float16 &lo) {
    hi = (_Float16)x;
    lo = (_Float16)(x - (float)hi);
}
