// serve.hip -- the C entries of include/gmoe_serve.h: the arguments' checks and the launches.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gmoe_serve.h"
#include "common.h"
#include "pages.h"
#include "kv4.h"
#include "kv4_attn.h"
#include "logprobs.h"

// gmoe.hip
void gm_set_err(const char *fmt, ...);

namespace {

// `device` as the current device for a scope.
struct OnDevice {
    int before = -1;
    hipError_t err;
    explicit OnDevice(int device) {
        err = hipGetDevice(&before);
        if (err == hipSuccess && before != device) err = hipSetDevice(device);
        else before = -1;  // nothing to put back
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

int invalid(const char *fmt, long long a = 0, long long b = 0, long long c = 0, long long d = 0) {
    gm_set_err(fmt, a, b, c, d);
    return GMOE_ERR_INVALID;
}

int failed(const char *what, hipError_t e) {
    gm_set_err("%s failed: %s", what, hipGetErrorString(e));
    return GMOE_ERR_HIP;
}

int page_shift(int page_size) {
    if (page_size < 1 || page_size > 65536 || (page_size & (page_size - 1))) return -1;
    return __builtin_ctz((unsigned)page_size);
}

bool ranks_ok(int kv, int rope) { return kv >= 32 && kv <= 512 && kv % 32 == 0 && rope >= 2 && rope <= 64 && rope % 2 == 0; }

int check_batch(const char *who, const gmoe_batch *b) {
    if (b->n_requests < 1 || b->n_requests > GMOE_MAX_REQUESTS || b->max_tokens < 1 || b->max_tokens > GMOE_MAX_STEP_TOKENS ||
        b->max_pages < 1 || b->max_pages > GMOE_MAX_TABLE || page_shift(b->page_size) < 0) {
        gm_set_err("%s: %d requests, %d tokens, %d pages a request of %d positions: outside 1..%d, 1..%d, 1..%d or not a "
                   "power of two up to 65536",
                   who, b->n_requests, b->max_tokens, b->max_pages, b->page_size, GMOE_MAX_REQUESTS, GMOE_MAX_STEP_TOKENS,
                   GMOE_MAX_TABLE);
        return GMOE_ERR_INVALID;
    }
    return GMOE_OK;
}

int cache_of(const char *who, const gmoe_kv4 *c, Kv4Cache *k) {
    const int shift = page_shift(c->page_size);
    if (!c->rows || ((uintptr_t)c->rows & 15) || !ranks_ok(c->kv_lora_rank, c->rope_dim) || shift < 0 || c->n_pages < 1 ||
        ((long long)c->n_pages << shift) >= (1ll << 31)) {
        gm_set_err("%s: cache of ranks %d + %d, %d pages of %d positions at %p: ranks a multiple of 32 in 32..512 and even in "
                   "2..64, a power of two of positions up to 65536, fewer than 2^31 in all, 16-byte aligned",
                   who, c->kv_lora_rank, c->rope_dim, c->n_pages, c->page_size, c->rows);
        return GMOE_ERR_INVALID;
    }
    k->rows = (uint8_t *)c->rows;
    k->kv = c->kv_lora_rank;
    k->rope = c->rope_dim;
    k->blocks = kv4_blocks(k->kv, k->rope);
    k->row_bytes = (int)gmoe_kv4_row_bytes(k->kv, k->rope);
    k->n_pages = c->n_pages;
    k->n_slots = c->n_pages << shift;
    k->shift = shift;
    return GMOE_OK;
}

// Whether rows of floats `ld` apart from p (and q) are all 16-byte aligned.
bool rows16(const void *p, int64_t ld, const void *q, int64_t lq) {
    return !(((uintptr_t)p | (uintptr_t)q) & 15) && ld % 4 == 0 && lq % 4 == 0;
}
bool floats(const void *p) { return !((uintptr_t)p & 3); }

}  // namespace

extern "C" int gmoe_page_maps(int device, const gmoe_batch *b, void *stream) {
    if (!b || !b->seen || !b->fresh || !b->free_pages || !b->n_free || !b->table || !b->offsets || !b->context || !b->request ||
        !b->position || !b->slot || !b->totals)
        return invalid("gmoe_page_maps: null argument");
    if (int rc = check_batch("gmoe_page_maps", b)) return rc;
    OnDevice on(device);
    if (on.err != hipSuccess) return failed("gmoe_page_maps: the device", on.err);
    const unsigned grid = (unsigned)((b->max_tokens + PM_BLOCK - 1) / PM_BLOCK);
    hipLaunchKernelGGL(k_page_maps, dim3(grid), dim3(PM_BLOCK), 0, (hipStream_t)stream, *b, page_shift(b->page_size));
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GMOE_OK : failed("gmoe_page_maps", e);
}

extern "C" size_t gmoe_kv4_row_bytes(int kv_lora_rank, int rope_dim) {
    if (!ranks_ok(kv_lora_rank, rope_dim)) return 0;
    return ((size_t)17 * kv4_blocks(kv_lora_rank, rope_dim) + 15) / 16 * 16;
}

extern "C" int gmoe_kv4_append(int device, const gmoe_kv4 *c, int n, const float *comp, int64_t ld_comp, const float *pe,
                               int64_t ld_pe, const int32_t *slot, void *stream) {
    if (!c || (n != 0 && (!comp || !pe || !slot))) return invalid("gmoe_kv4_append: null argument");
    Kv4Cache k;
    if (int rc = cache_of("gmoe_kv4_append", c, &k)) return rc;
    if (n < 0 || n > GMOE_MAX_STEP_TOKENS || ld_comp < 0 || ld_pe < 0 || !floats(comp) || !floats(pe) || !floats(slot))
        return invalid("gmoe_kv4_append: %lld tokens (0..%lld) of rows %lld and %lld floats apart (not negative, 4-byte aligned)", n,
                       GMOE_MAX_STEP_TOKENS, ld_comp, ld_pe);
    if (n == 0) return GMOE_OK;
    OnDevice on(device);
    if (on.err != hipSuccess) return failed("gmoe_kv4_append: the device", on.err);
    const dim3 grid((unsigned)(((long long)n * 4 * k.blocks + KV4_BLOCK - 1) / KV4_BLOCK)), block(KV4_BLOCK);
    hipStream_t st = (hipStream_t)stream;
    if (rows16(comp, ld_comp, pe, ld_pe)) hipLaunchKernelGGL(k_kv4_append<true>, grid, block, 0, st, k, n, comp, ld_comp, pe, ld_pe, slot);
    else hipLaunchKernelGGL(k_kv4_append<false>, grid, block, 0, st, k, n, comp, ld_comp, pe, ld_pe, slot);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GMOE_OK : failed("gmoe_kv4_append", e);
}

extern "C" int gmoe_kv4_read(int device, const gmoe_kv4 *c, int n, const int32_t *slot, float *comp, int64_t ld_comp, float *pe,
                             int64_t ld_pe, void *stream) {
    if (!c || (n != 0 && (!slot || (!comp && !pe)))) return invalid("gmoe_kv4_read: null argument");
    Kv4Cache k;
    if (int rc = cache_of("gmoe_kv4_read", c, &k)) return rc;
    if (n < 0 || n > GMOE_MAX_STEP_TOKENS || (comp && ld_comp < k.kv && n > 1) || (pe && ld_pe < k.rope && n > 1) || !floats(comp) ||
        !floats(pe) || !floats(slot))
        return invalid("gmoe_kv4_read: %lld slots (0..%lld) into rows %lld and %lld floats apart (not below the ranks, 4-byte aligned)",
                       n, GMOE_MAX_STEP_TOKENS, ld_comp, ld_pe);
    if (n == 0) return GMOE_OK;
    OnDevice on(device);
    if (on.err != hipSuccess) return failed("gmoe_kv4_read: the device", on.err);
    const dim3 grid((unsigned)(((long long)n * 4 * k.blocks + KV4_BLOCK - 1) / KV4_BLOCK)), block(KV4_BLOCK);
    hipStream_t st = (hipStream_t)stream;
    if (rows16(comp, ld_comp, pe, ld_pe)) hipLaunchKernelGGL(k_kv4_read<true>, grid, block, 0, st, k, n, slot, comp, ld_comp, pe, ld_pe);
    else hipLaunchKernelGGL(k_kv4_read<false>, grid, block, 0, st, k, n, slot, comp, ld_comp, pe, ld_pe);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GMOE_OK : failed("gmoe_kv4_read", e);
}

extern "C" size_t gmoe_kv4_attend_workspace(int n_heads, int kv_lora_rank) {
    if (n_heads < 1 || n_heads > 256 || !ranks_ok(kv_lora_rank, 2)) return 0;
    return (size_t)2 * KA_GRID * KA_ROWS * (kv_lora_rank + 2) * sizeof(float) + KA_GRID * sizeof(KaCut);
}

extern "C" int gmoe_kv4_attend(int device, const gmoe_kv4 *c, const gmoe_batch *b, const gmoe_kv4_heads *h, void *stream) {
    if (!c || !b || !h || !b->table || !b->offsets || !b->context || !h->q_abs || !h->q_pe || !h->out)
        return invalid("gmoe_kv4_attend: null argument");
    if (int rc = check_batch("gmoe_kv4_attend", b)) return rc;
    Kv4Attn a;
    if (int rc = cache_of("gmoe_kv4_attend", c, &a.c)) return rc;
    if (b->page_size != c->page_size)
        return invalid("gmoe_kv4_attend: the cache has pages of %lld positions, the batch of %lld", c->page_size, b->page_size);
    if (h->n_heads < 1 || h->n_heads > 256) return invalid("gmoe_kv4_attend: %lld heads outside 1..256", h->n_heads);
    const int64_t HV = (int64_t)h->n_heads * a.c.kv;
    if (h->ld_q_abs < 0 || h->ld_q_pe < 0 || h->ld_out < HV || !floats(h->q_abs) || !floats(h->q_pe) || !floats(h->out))
        return invalid("gmoe_kv4_attend: rows %lld, %lld and %lld floats apart (not negative, results at least %lld, 4-byte aligned)",
                       h->ld_q_abs, h->ld_q_pe, h->ld_out, HV);
    const size_t need = gmoe_kv4_attend_workspace(h->n_heads, a.c.kv);
    if (!h->work || ((uintptr_t)h->work & 15) || h->work_bytes < need)
        return invalid("gmoe_kv4_attend: a workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", (long long)need,
                       (long long)h->work_bytes);
    a.R = b->n_requests;
    a.max_pages = b->max_pages;
    a.H = h->n_heads;
    a.scale = h->scale;
    a.table = b->table;
    a.offsets = b->offsets;
    a.context = b->context;
    a.q_abs = h->q_abs;
    a.q_pe = h->q_pe;
    a.ld_q_abs = h->ld_q_abs;
    a.ld_q_pe = h->ld_q_pe;
    a.out = h->out;
    a.ld_out = h->ld_out;
    a.part = (float *)h->work;
    a.part_ml = a.part + (size_t)2 * KA_GRID * KA_ROWS * a.c.kv;
    a.cuts = (KaCut *)(a.part_ml + (size_t)2 * KA_GRID * KA_ROWS * 2);
    OnDevice on(device);
    if (on.err != hipSuccess) return failed("gmoe_kv4_attend: the device", on.err);
    hipStream_t st = (hipStream_t)stream;
    // the host knows no request's tokens: it takes them all alike
    const int mt = ka_operand_tiles((long long)a.H * ((b->max_tokens + a.R - 1) / a.R));
    a.slope = 8.0 * mt / (2.0 * KA_P * a.H);
    if (mt == 1) hipLaunchKernelGGL(k_kv4_attend<1>, dim3(KA_GRID), dim3(KA_BLOCK), 0, st, a);
    else if (mt == 2) hipLaunchKernelGGL(k_kv4_attend<2>, dim3(KA_GRID), dim3(KA_BLOCK), 0, st, a);
    else hipLaunchKernelGGL(k_kv4_attend<3>, dim3(KA_GRID), dim3(KA_BLOCK), 0, st, a);
    const unsigned tiles = (unsigned)ka_cut_tiles(b->max_tokens, a.R, a.H, mt), pairs = 8 * mt / KM_ROWS;
    if (tiles <= KM_FEW) hipLaunchKernelGGL(k_kv4_merge<4>, dim3(4 * pairs, tiles), dim3(KA_BLOCK), 0, st, a);
    else hipLaunchKernelGGL(k_kv4_merge<1>, dim3(pairs, tiles), dim3(KA_BLOCK), 0, st, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GMOE_OK : failed("gmoe_kv4_attend", e);
}

extern "C" size_t gmoe_logprobs_workspace(int n, int vocab, int top) {
    if (n < 1 || n > (1 << 24) || vocab < 1 || vocab > (1 << 24) || top < 0 || top > GMOE_TOP_MAX) return 0;
    const LpSplit s = lp_split(n, vocab);
    return s.segs > 1 ? (size_t)n * s.segs * (sizeof(LpRun) + top * sizeof(unsigned long long)) : 0;
}

extern "C" int gmoe_logprobs(int device, const gmoe_logprobs_args *a, void *stream) {
    if (!a) return invalid("gmoe_logprobs: null argument");
    if (a->n < 0 || a->n > (1 << 24) || a->vocab < 1 || a->vocab > (1 << 24) || a->n_given < 0 || a->top < 0 || a->top > GMOE_TOP_MAX ||
        (a->ld < a->vocab && a->n > 1))
        return invalid("gmoe_logprobs: %lld rows of %lld logits, %lld given, %lld alternatives: outside 0..2^24, 1..2^24, 0.., "
                       "0..64, or rows closer than that",
                       a->n, a->vocab, a->n_given, a->top);
    if (a->n == 0) return GMOE_OK;
    if (!a->logits || (a->n_given > 0 && (!a->given || !a->logprob)) || (a->top > 0 && (!a->top_id || !a->top_logprob)))
        return invalid("gmoe_logprobs: null argument");
    if (!floats(a->logits)) return invalid("gmoe_logprobs: logits are not 4-byte aligned");
    const size_t need = gmoe_logprobs_workspace(a->n, a->vocab, a->top);
    if (need > 0 && (!a->work || ((uintptr_t)a->work & 15) || a->work_bytes < need))
        return invalid("gmoe_logprobs: a workspace of %lld bytes, 16-byte aligned, is needed (got %lld)", (long long)need,
                       (long long)a->work_bytes);
    OnDevice on(device);
    if (on.err != hipSuccess) return failed("gmoe_logprobs: the device", on.err);
    const LpSplit s = lp_split(a->n, a->vocab);
    LpArgs g;
    g.a = *a;
    g.segs = s.segs;
    g.per = s.per;
    g.runs = (LpRun *)a->work;
    g.keys = (unsigned long long *)(g.runs + (size_t)a->n * s.segs);
    hipStream_t st = (hipStream_t)stream;
    const dim3 grid((unsigned)a->n * (unsigned)s.segs);
    hipLaunchKernelGGL(k_lp_run, grid, dim3(LP_BLOCK), 0, st, g);
    if (s.segs > 1) hipLaunchKernelGGL(k_lp_join, dim3((unsigned)a->n), dim3(LP_BLOCK), 0, st, g);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GMOE_OK : failed("gmoe_logprobs", e);
}
