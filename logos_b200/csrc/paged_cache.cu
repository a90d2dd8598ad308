// paged_cache.cu -- new tokens' K and V quantised into their pages (logos_paged_append) and the cache's values read
// back (logos_paged_read).  The quantiser is nikhilam_compress (cuda/ModelGPU.cu:293-386 of LOGOS) applied to one row
// of one head: scale = (max|x| + 1e-8) / 127.5, q = round-half-even(x / scale) held to +-127, IEEE division.
//
// Both move every byte once; reading is bound by HBM on prompts, appending by its rounding, both on single tokens by the chain
// "cu_q -> kv_len -> page table -> row" on single tokens.  DH / 8 lanes hold a row, 8 channels each (the maximum is
// a shuffle over them); a thread keeps one token, finds its page row once and walks over heads of K, then of V.
// Measured, 16 heads x 64, BF16: append of 33,000 tokens 60 us = 3.4 TB/s, where its instructions bound it; reading
// 32 sequences of 900 to 4096 tokens 90 us, 0.9 of a plain copy; single tokens of 64 sequences 3 us each.
#include "paged.cuh"

namespace logos {
namespace {

constexpr int kCacheThreads = 256;

struct CacheArgs {
    PagedArgs p;
    void *k, *v;                                   // token tensors
    long long k_row, k_head, v_row, v_head;
    int per, chunks;                               // heads per CTA; CTA rows of the grid per tensor
};

// Row of the sequence tables that owns token t: the number of sequences that end at or before it.  A warp's
// lanes read the ends together and every group of lanes counts for its own token; -1 when no sequence owns it.
template <int L>
__device__ __forceinline__ int owner_of(const PagedArgs& a, int t) {
    constexpr int G = 32 / L;                      // tokens of a warp
    const int lane = threadIdx.x & 31;
    int mine = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
        const bool in = b0 + lane < a.B;
        const int end = in ? a.cu_q[b0 + lane + 1] : 0;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int tg = __shfl_sync(0xffffffffu, t, g * L);
            const int n = __popc(__ballot_sync(0xffffffffu, in && end <= tg));
            if (lane / L == g) mine += n;
        }
    }
    return mine < a.B ? mine : -1;
}

// page row (in units of DH bytes, head 0) of token t, -1 when it has none
template <int L>
__device__ __forceinline__ long long slot_of(const PagedArgs& a, int t) {
    const int b = owner_of<L>(a, t);
    if (t >= a.rows || b < 0) return -1;
    const PagedSeq s = paged_seq(a, b);
    if (!s.ok || t < s.q0 || t >= s.q0 + s.n) {
        if (!s.ok) report_batch(a.status, b, false);
        return -1;
    }
    const int pos = s.kv - s.n + (t - s.q0);
    const int page = paged_page(a, b, pos);
    if (page < 0) { report_batch(a.status, b, true); return -1; }
    return (long long)(((size_t)page * a.H) << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
}

template <int L> __device__ __forceinline__ float row_max(float v) {   // over the L lanes of a row
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// grid (token blocks, chunks of `per` heads of K, then of V)
template <typename T, int D>
__global__ void __launch_bounds__(kCacheThreads)
paged_append_kernel(const CacheArgs a) {
    constexpr int L = D / 8, kTokens = kCacheThreads / L, U = 4, W = sizeof(T) / 2;
    const int chunk = threadIdx.x % L;
    const int token = blockIdx.x * kTokens + threadIdx.x / L;
    const bool is_v = (int)blockIdx.y >= a.chunks;
    const int h0 = ((int)blockIdx.y - (is_v ? a.chunks : 0)) * a.per, h1 = min(h0 + a.per, a.p.H);
    const long long at = token < a.p.rows ? token : 0;
    const long long xh = is_v ? a.v_head : a.k_head;
    const T* x = static_cast<const T*>(is_v ? a.v : a.k) + at * (is_v ? a.v_row : a.k_row) + 8 * chunk;
    uint4 raw[U][W];                               // in flight while the page row is looked up
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (h0 + u < h1) {
#pragma unroll
            for (int i = 0; i < W; ++i) raw[u][i] = reinterpret_cast<const uint4*>(x + (h0 + u) * xh)[i];
        }
    const long long slot = slot_of<L>(a.p, token);
    int8_t* c8 = (is_v ? a.p.v : a.p.k);
    float* cs = (is_v ? a.p.vs : a.p.ks);
    for (int h = h0; h < h1; h += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h + u >= h1) break;
            float v[8];
            const T* t = reinterpret_cast<const T*>(raw[u]);
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) { v[e] = to_f32<T>(t[e]); top = fmaxf(top, fabsf(v[e])); }
            if (h + u + U < h1) {
#pragma unroll
                for (int i = 0; i < W; ++i) raw[u][i] = reinterpret_cast<const uint4*>(x + (h + u + U) * xh)[i];
            }
            const float scale = __fdiv_rn(row_max<L>(top) + 1e-8f, 127.5f);
            // x / scale, rounded twice (to fp32, to a whole number), is x * (1 / scale) rounded once unless that product lies
            // within 1e-4 of a half: it is off by 127 * 2^-21 at most.  Only then the division is done.  (The row's largest value
            // is held to 127 either way, so it is taken out first.)  The kernel is bound by its instructions: 70 us with eight
            // divisions a lane for the append of 33,000 tokens x 16 heads, 60 this way, 42 if no channel ever met a half.
            const float inv = __fdividef(1.0f, scale);
            const float2 inv2 = make_float2(inv, inv), magic = make_float2(12582912.0f, 12582912.0f), less = make_float2(-12582912.0f, -12582912.0f);
            uint32_t w[2], bits[8];
            float far = 0.0f;
            float2 odd = make_float2(0.0f, 0.0f);              // NaN when one of the values is, or is an infinity
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                float2 t = __fmul2_rn(make_float2(v[e], v[e + 1]), inv2);
                odd = __ffma2_rn(make_float2(v[e], v[e + 1]), make_float2(0.0f, 0.0f), odd);
                t = make_float2(fminf(fmaxf(t.x, -127.0f), 127.0f), fminf(fmaxf(t.y, -127.0f), 127.0f));
                const float2 r = __fadd2_rn(t, magic);        // 1.5 * 2^23 and more: the last bits are the whole number
                const float2 n = __fadd2_rn(r, less);
                bits[e] = __float_as_uint(r.x);
                bits[e + 1] = __float_as_uint(r.y);
                far = fmaxf(fmaxf(far, fabsf(t.x - n.x)), fabsf(t.y - n.y));
            }
            if (!(far <= 0.4999f) || !(odd.x + odd.y == 0.0f)) {
                // (16-bit rows meet exact halves often: only the channels that do are divided)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float t = fminf(fmaxf(v[e] * inv, -127.0f), 127.0f);
                    if (!(fabsf(t - (__uint_as_float(bits[e]) - 12582912.0f)) <= 0.4999f) || !(odd.x + odd.y == 0.0f))
                        bits[e] = (uint32_t)max(-127, min(127, __float2int_rn(__fdiv_rn(v[e], scale))));
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                w[i] = prmt(prmt(bits[4 * i], bits[4 * i + 1], 0x0040), prmt(bits[4 * i + 2], bits[4 * i + 3], 0x0040), 0x5410);
            if (slot >= 0) {
                const size_t row = (size_t)slot + ((size_t)(h + u) << a.p.page_shift);
                *reinterpret_cast<uint2*>(c8 + row * D + 8 * chunk) = make_uint2(w[0], w[1]);
                if (chunk == 0) cs[row] = scale;
            }
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kCacheThreads)
paged_read_kernel(const CacheArgs a) {
    constexpr int L = D / 8, kTokens = kCacheThreads / L, U = 4, W = sizeof(T) / 2;
    const int chunk = threadIdx.x % L;
    const int token = blockIdx.x * kTokens + threadIdx.x / L;
    const bool is_v = (int)blockIdx.y >= a.chunks;
    const int h0 = ((int)blockIdx.y - (is_v ? a.chunks : 0)) * a.per, h1 = min(h0 + a.per, a.p.H);
    const long long slot = slot_of<L>(a.p, token);
    if (slot < 0) return;
    const long long yh = is_v ? a.v_head : a.k_head;
    T* y = static_cast<T*>(is_v ? a.v : a.k) + (long long)token * (is_v ? a.v_row : a.k_row) + 8 * chunk;
    const int8_t* c8 = (is_v ? a.p.v : a.p.k);
    const float* cs = (is_v ? a.p.vs : a.p.ks);
    for (int h = h0; h < h1; h += U) {
        uint2 w[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h + u >= h1) break;
            const size_t row = (size_t)slot + ((size_t)(h + u) << a.p.page_shift);
            w[u] = *reinterpret_cast<const uint2*>(c8 + row * D + 8 * chunk);
            s[u] = cs[row];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h + u >= h1) break;
            uint4 out[W];
            T* t = reinterpret_cast<T*>(out);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                t[e] = from_f32<T>((float)(int8_t)((e < 4 ? w[u].x : w[u].y) >> (8 * (e & 3))) * s[u]);
#pragma unroll
            for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(y + (h + u) * yh)[i] = out[i];
        }
    }
}

template <typename T, int D>
int launch_cache(logos_ctx* ctx, CacheArgs& a, bool read) {
    constexpr int kTokens = kCacheThreads / (D / 8);
    const int n_tb = (a.p.rows + kTokens - 1) / kTokens;
    // heads per CTA: as many as leave 8 CTAs per SM, at most 16 (the page row is found once per token and chunk)
    const long long per = (long long)n_tb * 2 * a.p.H / (8LL * ctx->sm_count);
    a.per = per < 1 ? 1 : per > 16 ? 16 : (int)per;
    a.chunks = (a.p.H + a.per - 1) / a.per;
    const dim3 grid(n_tb, 2 * a.chunks);
    if (read) paged_read_kernel<T, D><<<grid, kCacheThreads, 0, ctx->stream>>>(a);
    else paged_append_kernel<T, D><<<grid, kCacheThreads, 0, ctx->stream>>>(a);
    LOGOS_LAUNCH_CHECK(ctx, read ? "paged_read_kernel" : "paged_append_kernel");
    return LOGOS_OK;
}

template <typename T>
int dispatch_cache(logos_ctx* ctx, CacheArgs& a, int DH, bool read) {
    return DH == 64 ? launch_cache<T, 64>(ctx, a, read) : launch_cache<T, 128>(ctx, a, read);
}

int run_cache(logos_ctx* ctx, const char* what, int dtype, void* K, void* V, const logos_row_strides* ks,
              const logos_row_strides* vs, const logos_paged_cache* cache, const logos_paged_batch* batch, bool read) {
    if (int rc = paged_check(ctx, what, cache, batch)) return rc;
    if (!dtype_ok(dtype)) return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: unknown dtype", what);
    if (batch->rows == 0 || batch->B == 0 || batch->max_q == 0) return LOGOS_OK;
    if (!K || !V) return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: null pointer", what);
    if (!aligned16(K) || !aligned16(V)) return fail(ctx, LOGOS_ERR_ALIGNMENT, "%s: tensors must be 16-byte aligned", what);
    const size_t esz = dtype_size(dtype);
    const logos_row_strides packed{(int64_t)cache->H * cache->DH, cache->DH};
    const logos_row_strides k = ks ? *ks : packed, v = vs ? *vs : packed;
    if (!rows_aligned(k, esz) || !rows_aligned(v, esz))
        return fail(ctx, LOGOS_ERR_ALIGNMENT, "%s: negative strides, or rows that are not 16-byte aligned", what);
    if (read && (!rows_apart(k, batch->rows, cache->H, cache->DH) || !rows_apart(v, batch->rows, cache->H, cache->DH)))
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: the rows of an output overlap", what);
    CacheArgs a;
    a.p = paged_args(ctx, cache, batch);
    a.k = K; a.v = V;
    a.k_row = k.row; a.k_head = k.head; a.v_row = v.row; a.v_head = v.head;
    if (dtype == LOGOS_F32) return dispatch_cache<float>(ctx, a, cache->DH, read);
    if (dtype == LOGOS_F16) return dispatch_cache<__half>(ctx, a, cache->DH, read);
    return dispatch_cache<__nv_bfloat16>(ctx, a, cache->DH, read);
}

}  // namespace

int paged_check(logos_ctx* ctx, const char* what, const logos_paged_cache* c, const logos_paged_batch* b) {
    if (!c || !b) return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: null cache or batch", what);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || c->pages <= 0 || c->H <= 0 || c->H > 1024)
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: bad cache (pointers, pages, 1 to 1024 heads)", what);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return fail(ctx, LOGOS_ERR_UNSUPPORTED, "%s: page_size %d (16, 32, 64 or 128)", what, c->page_size);
    if (c->DH != 64 && c->DH != 128) return fail(ctx, LOGOS_ERR_UNSUPPORTED, "%s: DH = %d (64 or 128)", what, c->DH);
    if ((int64_t)c->pages * c->H * c->page_size > 0x7fffffffLL)
        return fail(ctx, LOGOS_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows in a cache (pages x H x page_size)", what);
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale))
        return fail(ctx, LOGOS_ERR_ALIGNMENT, "%s: the cache must be 16-byte aligned", what);
    if (b->B < 0 || b->rows < 0 || b->max_q < 0 || b->max_kv < 0 || b->max_pages < 0 || b->B > 65535 ||
        (int64_t)b->max_kv > (int64_t)b->max_pages * c->page_size || b->max_q > b->max_kv)
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: bad batch (B %d up to 65535, rows %d, max_q %d <= max_kv %d <= %d pages x %d)",
                    what, b->B, b->rows, b->max_q, b->max_kv, b->max_pages, c->page_size);
    if (b->rows > kMostRows || b->max_kv > kMostRows)        // the kernels round row numbers and positions up in 32 bits
        return fail(ctx, LOGOS_ERR_UNSUPPORTED, "%s: rows %d, max_kv %d (2^30 at most)", what, b->rows, b->max_kv);
    if (b->B > 0 && (!b->cu_q || !b->kv_len || (b->max_kv > 0 && !b->page_table)))
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: null table", what);
    return LOGOS_OK;
}

int paged_append(logos_ctx* ctx, int dtype, const void* K, const void* V, const logos_row_strides* k_in,
                 const logos_row_strides* v_in, const logos_paged_cache* cache, const logos_paged_batch* batch) {
    return run_cache(ctx, "paged_append", dtype, const_cast<void*>(K), const_cast<void*>(V), k_in, v_in, cache, batch, false);
}

int paged_read(logos_ctx* ctx, int dtype, const logos_paged_cache* cache, const logos_paged_batch* batch, void* K, void* V,
               const logos_row_strides* k_out, const logos_row_strides* v_out) {
    return run_cache(ctx, "paged_read", dtype, K, V, k_out, v_out, cache, batch, true);
}

}  // namespace logos
