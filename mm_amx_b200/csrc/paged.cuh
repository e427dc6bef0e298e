// The paged cache as the kernels see it (device side of paged.h) and the checks of its descriptor.
#pragma once
#include "common.cuh"
#include "paged.h"

namespace b200fc {

struct PagedView {
    unsigned char* k; unsigned char* v;
    long long page_stride, head_stride, token_stride;       // bytes
    float* k_scale; float* v_scale; long long scale_stride; // scale_stride: floats
    const int* table; long long table_stride;               // entries
    const int* seq_lens; const int* row_start;
    int B, T, max_rows, Hkv, pages, page_shift;
    long long capacity;                                     // tokens that a row of the table has room for
    int* status;
};

// Checks of what both calls take; `what` names the call in messages.
inline int paged_view(const b200fc_paged_cache_t* c, const char* what, int T, int max_rows, const int32_t* row_start, PagedView* out) {
    if (!c) { set_error("%s: null cache", what); return B200FC_ERR_INVALID; }
    if (c->D != 64 && c->D != 128) { set_error("%s: head size must be 64 or 128", what); return B200FC_ERR_UNSUPPORTED; }
    int shift = 4;
    while (shift < 7 && (1 << shift) != c->page_tokens) shift++;
    if ((1 << shift) != c->page_tokens) { set_error("%s: page_tokens must be 16, 32, 64 or 128", what); return B200FC_ERR_UNSUPPORTED; }
    if (c->dtype != B200FC_BF16 && c->dtype != B200FC_S8) { set_error("%s: the cache is bf16 or s8", what); return B200FC_ERR_INVALID; }
    if (c->B < 0 || T < 0 || max_rows < 0 || c->pages < 0 || c->max_pages < 0 || c->Hkv <= 0 || c->Hkv > 65535) {
        set_error("%s: a negative size, or kv heads outside 1..65535", what);
        return B200FC_ERR_INVALID;
    }
    if (c->B > (1 << 20) || T > (1 << 24)) { set_error("%s: at most 2^20 sequences and 2^24 rows per call", what); return B200FC_ERR_INVALID; }
    if (!row_start && T != c->B) { set_error("%s: without row_start there is one row per sequence, T = B", what); return B200FC_ERR_INVALID; }
    if (!c->k || !c->v || !c->page_table || !c->seq_lens) { set_error("%s: null pointer in the cache", what); return B200FC_ERR_INVALID; }
    const long long row = (long long)c->D * (c->dtype == B200FC_BF16 ? 2 : 1);
    if (((uintptr_t)c->k & 15) || ((uintptr_t)c->v & 15) || ((c->page_stride | c->head_stride | c->token_stride) & 15) || c->token_stride < row ||
        c->page_stride < 0 || c->head_stride < 0) {
        set_error("%s: the cache needs 16-byte aligned pointers and strides, none negative, token stride >= a token", what);
        return B200FC_ERR_INVALID;
    }
    if (((uintptr_t)c->page_table & 3) || (c->table_stride & 3) || c->table_stride < (int64_t)c->max_pages * 4 || ((uintptr_t)c->seq_lens & 3) ||
        ((uintptr_t)row_start & 3)) {
        set_error("%s: page_table, seq_lens and row_start need 4-byte alignment, and the table a stride of at least a row", what);
        return B200FC_ERR_INVALID;
    }
    if (c->dtype == B200FC_S8 && (!c->k_scale || !c->v_scale || (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) || (c->scale_page_stride & 3) ||
                                  c->scale_page_stride < (int64_t)c->Hkv * 4)) {
        set_error("%s: an 8-bit cache needs aligned k_scale and v_scale with a factor for each page and head", what);
        return B200FC_ERR_INVALID;
    }
    PagedView v;
    v.k = (unsigned char*)c->k; v.v = (unsigned char*)c->v;
    v.page_stride = c->page_stride; v.head_stride = c->head_stride; v.token_stride = c->token_stride;
    v.k_scale = c->k_scale; v.v_scale = c->v_scale; v.scale_stride = c->scale_page_stride / 4;
    v.table = c->page_table; v.table_stride = c->table_stride / 4;
    v.seq_lens = c->seq_lens; v.row_start = row_start;
    v.B = c->B; v.T = T; v.max_rows = max_rows; v.Hkv = c->Hkv; v.pages = c->pages; v.page_shift = shift;
    v.capacity = (long long)c->max_pages << shift;
    v.status = nullptr;
    *out = v;
    return B200FC_OK;
}
// the word that reports land in; asked for once everything else is checked
inline int paged_status(const char* what, PagedView* v) {
    v->status = kernel_status_word();
    if (!v->status) { set_error("%s: no kernel status word on this device", what); return B200FC_ERR_CUDA; }
    return B200FC_OK;
}
inline bool unaligned16(const void* p, int64_t s0, int64_t s1) { return ((uintptr_t)p | (uintptr_t)s0 | (uintptr_t)s1) & 15; }

#ifdef __CUDACC__
__device__ __forceinline__ void report_paged(const PagedView& c) { atomicCAS(c.status, 0, kStatusPaged); }

// rows of sequence b; false: its numbers lie outside their buffers
__device__ __forceinline__ bool load_seq(const PagedView& c, int b, SeqRows* s) {
    const int r0 = c.row_start ? __ldg(c.row_start + b) : b, r1 = c.row_start ? __ldg(c.row_start + b + 1) : b + 1;
    return seq_rows(r0, r1, __ldg(c.seq_lens + b), c.T, c.max_rows, c.capacity, s);
}
// The last sequence whose first row is <= r, or -1; whether it owns r is seen from its rows.  By a whole warp: a round of 32 probes instead of five
// dependent loads.
__device__ __forceinline__ int find_sequence(const PagedView& c, int r) {
    if (!c.row_start) return r;
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = c.B;
    bool found = false;
    while (hi > lo) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, at < hi && __ldg(c.row_start + (at < hi ? at : lo)) <= r);
        if (!m) return found ? lo : -1;
        found = true;
        lo += (31 - __clz(m)) * step;
        if (step == 1) return lo;
        hi = min(hi, lo + step);
    }
    return -1;
}
// page of entry i of sequence b's table, -1 outside the pool
__device__ __forceinline__ int table_page(const PagedView& c, int b, int i) {
    const int p = __ldg(c.table + (long long)b * c.table_stride + i);
    return (unsigned)p < (unsigned)c.pages ? p : -1;
}
#endif

}  // namespace b200fc
