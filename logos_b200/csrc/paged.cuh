// paged.cuh -- what the kernels over the paged INT8 cache share: the device view of a cache and of a batch, and the
// checked way from a token row to its sequence and page row.  Every table entry is checked against the bounds
// before it is used as an index, whatever the tables hold.
#pragma once

#include "common.cuh"

namespace logos {

struct PagedArgs {
    int8_t *k, *v;
    float *ks, *vs;
    const int32_t *cu_q, *kv_len, *table;
    int* status;
    int pages, page_shift, H;               // page_size = 1 << page_shift
    int B, max_pages, rows, max_q, max_kv;
};

inline PagedArgs paged_args(const logos_ctx* ctx, const logos_paged_cache* c, const logos_paged_batch* b) {
    PagedArgs a;
    a.k = c->k; a.v = c->v; a.ks = c->k_scale; a.vs = c->v_scale;
    a.cu_q = b->cu_q; a.kv_len = b->kv_len; a.table = b->page_table;
    a.status = ctx->tc_status;
    a.pages = c->pages;
    a.page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
    a.H = c->H;
    a.B = b->B; a.max_pages = b->max_pages; a.rows = b->rows; a.max_q = b->max_q; a.max_kv = b->max_kv;
    return a;
}

struct PagedSeq { int q0, n, kv; bool ok; };      // first row, new tokens, tokens held

__host__ __device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b) {
    PagedSeq s;
    const int q1 = a.cu_q[b + 1];
    s.q0 = a.cu_q[b];
    s.kv = a.kv_len[b];
    s.ok = s.q0 >= 0 && q1 >= s.q0 && q1 <= a.rows && s.kv >= 0 && s.kv <= a.max_kv;
    s.n = s.ok ? q1 - s.q0 : 0;
    s.ok = s.ok && s.n <= a.max_q && s.n <= s.kv;
    return s;
}

// the page of position `pos` (0 <= pos < max_kv, so the table entry exists), -1 when it is outside the cache
__host__ __device__ __forceinline__ int paged_page(const PagedArgs& a, int b, int pos) {
    const int page = a.table[(size_t)b * a.max_pages + (pos >> a.page_shift)];
    return (unsigned)page < (unsigned)a.pages ? page : -1;
}

// first row of head h in a page: row r of it has its DH bytes at (that + r) * DH and its scale at that + r
__host__ __device__ __forceinline__ size_t paged_row(const PagedArgs& a, int page, int h) {
    return ((size_t)page * a.H + h) << a.page_shift;
}

}  // namespace logos
