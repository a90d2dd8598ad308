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

// First row of head h in a page: row r of it has its DH bytes at (that + r) * DH and its scale at that + r.  Rows fit 32
// bits (paged_check; a row takes 136 bytes at least), their byte offsets do not: widen before the multiplication.
__host__ __device__ __forceinline__ uint32_t paged_row(const PagedArgs& a, int page, int h) {
    return ((uint32_t)page * (uint32_t)a.H + (uint32_t)h) << a.page_shift;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}
// two biased bytes (b + 128) under the exponent of 1024, minus 1152
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t biased, uint32_t sel) {
    const uint32_t w = prmt(biased, 0x64646464u, sel), bias = 0x64806480u;
    __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<uint32_t*>(&h);
}
// two raw bytes u under 0x43: BF16 128 + (u & 127), minus 128 or, for a negative one, 256
__device__ __forceinline__ uint32_t bytes_to_bf162(uint32_t bytes, uint32_t sel) {
    const uint32_t w = prmt(bytes, 0x43434343u, sel), p = w & 0xff7fff7fu, c = w & 0xff80ff80u;
    __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&p), *reinterpret_cast<const __nv_bfloat162*>(&c));
    return *reinterpret_cast<uint32_t*>(&r);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A query row in FP16 by a power of two: `top` = max|q| of the row.  The factor puts it at 2^13 ... 2^14, so a BF16
// row keeps every bit of values down to 2^-27 of its largest; rows of zeros, infinities or NaN keep factor 1.
__device__ __forceinline__ void row_power(float top, float& mul, float& inv) {
    const int be = (int)(__float_as_uint(top) >> 23);
    const int up = (be == 0 || be >= 255) ? 127 : min(max(267 - be, 1), 253);   // biased exponent of the factor
    mul = __uint_as_float((uint32_t)up << 23);
    inv = __uint_as_float((uint32_t)(254 - up) << 23);
}

// paged_chunk.cu: the sequences with more than min_rows query rows per key/value head
size_t paged_chunk_workspace_bytes(const logos_ctx* ctx, int DH);
int paged_chunk(logos_ctx* ctx, const PagedArgs& p, int DH, const void* Q, void* O, const logos_row_strides& q,
                const logos_row_strides& o, int G, bool f16, const logos_attn_params* prm, int min_rows);

constexpr float kMoveMax = 15.0f;         // log2 units by which a row may outgrow its reference maximum (weights up to 2^15: FP16 ends at 2^16)
constexpr float kLeastScale = 1e-30f;     // a value scale below this (a row nobody wrote) counts as this: its log2 stays finite

}  // namespace logos
