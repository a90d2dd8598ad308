// qk_rope.cu -- RMS norm of every head of the queries and keys and their rotation by position, in one pass, and the
// backward pass of it (logos_qk_norm_rope, logos_qk_norm_rope_bwd; formulas in include/logos_attn.h).
//
// Both are bound by HBM: forward 2 e, backward 3 e bytes per value (e bytes a value), a dozen operations per value.
// So nothing but the rows moves: DH / 8 lanes hold a row, 8 channels each; a lane's angles depend on the token alone,
// so a thread keeps ONE token and walks over heads, its cosines and sines (16 registers) computed once.
// The angle p f is wanted modulo one turn and p goes up to 2^31: the frequency comes as a 64-bit fixed-point number of
// turns, the product p F wraps modulo 2^64 by itself and its upper word is the fraction of a turn to 2^-32.  (A float
// product is off by 2^-24 p f radians: useless from p f ~ 10^5 on.)
//
// Measured: forward, 65,536 tokens x 32 heads x 64 BF16, 98 us = 5.5 TB/s (0.84 of a plain copy); backward, 16,384 tokens x
// 40 heads x 128 BF16 with both weights' gradients, 101 us = 5.0 TB/s, the sum of the partial gradients mostly under it;
// 32 tokens 3 us, which is the launch.
#include <cmath>

#include "common.cuh"

namespace logos {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeParts = 1184;        // most partial sums of a weight gradient (8 CTAs on each of 148 SMs)
constexpr int kRopeReduceWarps = 32;

struct RopeArgs {
    unsigned long long turns[LOGOS_ROPE_MAX_PAIRS];   // frequency of pair k in turns per position, times 2^64
    const void *q, *k, *gq, *gk;                      // rows; backward: gradients of the outputs
    void *yq, *yk;                                    // outputs; backward: gradients of the rows
    const float *wq, *wk;
    const int32_t* pos;
    float* part;                                      // backward: [parts][DH] partial weight gradients, Q's first
    long long q_row, q_head, k_row, k_head, yq_row, yq_head, yk_row, yk_head, gq_row, gq_head, gk_row, gk_head;
    float eps;
    int dims, rows, Hq, Hk, per, q_chunks;            // heads per CTA; CTA rows of the grid that belong to Q
};

// eight channels of a row
template <typename T> struct Raw8 { uint4 w[sizeof(T) / 2]; };
template <typename T> __device__ __forceinline__ Raw8<T> load8(const T* p) {
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const uint4*>(p)[i];
    return r;
}
template <typename T> __device__ __forceinline__ void widen8(const Raw8<T>& r, float (&x)[8]) {
    const T* t = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f32<T>(t[e]);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&y)[8]) {
    Raw8<T> r;
    T* t = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = from_f32<T>(y[e]);
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

template <int L> __device__ __forceinline__ float row_sum(float v) {   // over the L lanes of a row
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// What a lane needs to rotate its 8 channels: y_e = n_e cos_e + (partner's n) sin_e, the sign in sin_e.  Pairs of
// halves: the partner channel sits in lane `partner`; neighbours: in the lane itself.  Channels that are not
// rotated have cos 1, sin 0.
struct Turn { float c[8], s[8]; int partner; };
template <bool NEIGHBOURS>
__device__ __forceinline__ Turn lane_turn(const RopeArgs& a, int chunk, int pos) {
    Turn t;
    t.partner = chunk;
    const bool rotated = 8 * chunk < a.dims;
    const int half = a.dims >> 1;
    const bool upper = !NEIGHBOURS && rotated && 8 * chunk >= half;
    if (!NEIGHBOURS && rotated) t.partner = upper ? chunk - (half >> 3) : chunk + (half >> 3);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (NEIGHBOURS && (e & 1)) { t.c[e] = t.c[e - 1]; t.s[e] = -t.s[e - 1]; continue; }
        t.c[e] = 1.0f;
        t.s[e] = 0.0f;
        if (rotated) {
            const int k = NEIGHBOURS ? 4 * chunk + (e >> 1) : 8 * chunk + e - (upper ? half : 0);
            const unsigned long long frac = (unsigned long long)(long long)pos * a.turns[k];
            float sn, cs;
            sincospif((float)(int)(frac >> 32) * 0x1p-31f, &sn, &cs);   // (-1/2, 1/2] turns as multiples of pi
            t.c[e] = cs;
            t.s[e] = upper ? sn : -sn;
        }
    }
    return t;
}
// sign = +1: rotate, -1: rotate back
template <bool NEIGHBOURS, int L>
__device__ __forceinline__ void rotate8(const Turn& t, float sign, const float (&n)[8], float (&y)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float other = NEIGHBOURS ? n[e ^ 1] : __shfl_sync(0xffffffffu, n[e], t.partner, L);
        y[e] = fmaf(other, sign * t.s[e], n[e] * t.c[e]);
    }
}

// grid (token blocks, chunks of `per` heads: Q's first, then K's)
template <typename T, int D, bool NEIGHBOURS>
__global__ void __launch_bounds__(kRopeThreads)
qk_norm_rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int L = D / 8, kTokens = kRopeThreads / L, U = 4;
    const int chunk = threadIdx.x % L;
    const int token = blockIdx.x * kTokens + threadIdx.x / L;
    const bool live = token < a.rows;                     // every lane stays for the shuffles
    const bool is_k = (int)blockIdx.y >= a.q_chunks;
    const int h0 = ((int)blockIdx.y - (is_k ? a.q_chunks : 0)) * a.per;
    const int h1 = min(h0 + a.per, is_k ? a.Hk : a.Hq);
    const long long xh = is_k ? a.k_head : a.q_head, yh = is_k ? a.yk_head : a.yq_head;
    const long long at = live ? token : 0;
    const T* x = static_cast<const T*>(is_k ? a.k : a.q) + at * (is_k ? a.k_row : a.q_row) + 8 * chunk;
    T* y = static_cast<T*>(is_k ? a.yk : a.yq) + at * (is_k ? a.yk_row : a.yq_row) + 8 * chunk;
    const float* w = is_k ? a.wk : a.wq;
    const bool norm = w != nullptr;
    Raw8<T> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (h0 + u < h1) raw[u] = load8<T>(x + (h0 + u) * xh);
    float wt[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) wt[e] = norm ? w[8 * chunk + e] : 1.0f;
    const Turn t = lane_turn<NEIGHBOURS>(a, chunk, a.pos[at]);
    for (int h = h0; h < h1; h += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h + u >= h1) break;
            float v[8], n[8], out[8];
            widen8<T>(raw[u], v);
            if (h + u + U < h1) raw[u] = load8<T>(x + (h + u + U) * xh);
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(v[e], v[e], ss);
            const float r = norm ? rsqrtf(row_sum<L>(ss) * (1.0f / D) + a.eps) : 1.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) n[e] = v[e] * r * wt[e];
            rotate8<NEIGHBOURS, L>(t, 1.0f, n, out);
            if (live) store8<T>(y + (h + u) * yh, out);
        }
    }
}

// Backward.  g = rotation back of dy; dw += g x r; h = g w; dx = r (h - x r^2 mean(h x)).
// A CTA walks over token blocks and leaves one partial weight gradient: the sums' order is that of the launch,
// which the sizes alone decide.
template <typename T, int D, bool NEIGHBOURS>
__global__ void __launch_bounds__(kRopeThreads)
qk_norm_rope_bwd_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int L = D / 8, kTokens = kRopeThreads / L, U = 2;
    __shared__ float s_part[kRopeThreads / 32][D];
    grid_release_dependents();
    const int chunk = threadIdx.x % L;
    const bool is_k = (int)blockIdx.y >= a.q_chunks;
    const int h0 = ((int)blockIdx.y - (is_k ? a.q_chunks : 0)) * a.per;
    const int h1 = min(h0 + a.per, is_k ? a.Hk : a.Hq);
    const long long xh = is_k ? a.k_head : a.q_head, yh = is_k ? a.yk_head : a.yq_head, gh = is_k ? a.gk_head : a.gq_head;
    const float* w = is_k ? a.wk : a.wq;
    const bool norm = w != nullptr;
    float wt[8], dw[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) { wt[e] = norm ? w[8 * chunk + e] : 1.0f; dw[e] = 0.0f; }
    for (int tb = blockIdx.x; tb * kTokens < a.rows; tb += gridDim.x) {
        const int token = tb * kTokens + threadIdx.x / L;
        const bool live = token < a.rows;
        const long long at = live ? token : 0;
        const T* x = static_cast<const T*>(is_k ? a.k : a.q) + at * (is_k ? a.k_row : a.q_row) + 8 * chunk;
        const T* g_in = static_cast<const T*>(is_k ? a.gk : a.gq) + at * (is_k ? a.gk_row : a.gq_row) + 8 * chunk;
        T* y = static_cast<T*>(is_k ? a.yk : a.yq) + at * (is_k ? a.yk_row : a.yq_row) + 8 * chunk;
        Raw8<T> rx[U], rg[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (h0 + u < h1) { rx[u] = load8<T>(x + (h0 + u) * xh); rg[u] = load8<T>(g_in + (h0 + u) * gh); }
        const Turn t = lane_turn<NEIGHBOURS>(a, chunk, a.pos[at]);
        for (int h = h0; h < h1; h += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (h + u >= h1) break;
                float v[8], dy[8], g[8], out[8];
                widen8<T>(rx[u], v);
                widen8<T>(rg[u], dy);
                if (h + u + U < h1) { rx[u] = load8<T>(x + (h + u + U) * xh); rg[u] = load8<T>(g_in + (h + u + U) * gh); }
                rotate8<NEIGHBOURS, L>(t, -1.0f, dy, g);
                if (norm) {
                    float ss = 0.0f, dot = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) { ss = fmaf(v[e], v[e], ss); dot = fmaf(g[e] * wt[e], v[e], dot); }
                    const float r = rsqrtf(row_sum<L>(ss) * (1.0f / D) + a.eps);
                    const float back = row_sum<L>(dot) * (1.0f / D) * r * r;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (live) dw[e] = fmaf(g[e], v[e] * r, dw[e]);
                        out[e] = r * (g[e] * wt[e] - v[e] * back);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) out[e] = g[e];
                }
                if (live) store8<T>(y + (h + u) * yh, out);
            }
        }
    }
    if (!norm) return;
    // the CTA's sum per channel: over the rows of a warp, then over the warps
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int o = L; o < 32; o <<= 1) dw[e] += __shfl_xor_sync(0xffffffffu, dw[e], o);
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane < L) {
#pragma unroll
        for (int e = 0; e < 8; ++e) s_part[warp][8 * lane + e] = dw[e];
    }
    __syncthreads();
    if (threadIdx.x < D) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kRopeThreads / 32; ++i) sum += s_part[i][threadIdx.x];
        a.part[((size_t)blockIdx.y * gridDim.x + blockIdx.x) * D + threadIdx.x] = sum;
    }
}

// sums the partial weight gradients: grid (DH / 32, Q and K), a lane per channel, a warp per every 32nd partial row
__global__ void __launch_bounds__(32 * kRopeReduceWarps)
rope_weight_grad_kernel(const float* part, int D, int q_parts, int k_parts, float* dwq, float* dwk) {
    __shared__ float s_sum[kRopeReduceWarps][33];
    const bool is_k = blockIdx.y == 1;
    float* out = is_k ? dwk : dwq;
    const int n = is_k ? k_parts : q_parts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    const float* p = part + (is_k ? (size_t)q_parts * D : 0) + c;
    grid_wait_for_earlier();
    if (!out) return;
    float sum = 0.0f;
#pragma unroll 8
    for (int i = warp; i < n; i += kRopeReduceWarps) sum += p[(size_t)i * D];
    s_sum[warp][lane] = sum;
    __syncthreads();
    if (warp == 0) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < kRopeReduceWarps; ++i) total += s_sum[i][lane];
        out[c] = total;
    }
}


template <typename T, int D, bool NEIGHBOURS>
int launch(logos_ctx* ctx, RopeArgs& a, bool bwd, float* dwq, float* dwk) {
    constexpr int kTokens = kRopeThreads / (D / 8);
    const int n_tb = (a.rows + kTokens - 1) / kTokens, H = a.Hq + a.Hk;
    // Heads per CTA: as many as leave the device filled (8 CTAs per SM), at most 16; the angles are computed once per
    // token and chunk of heads, so few heads per CTA cost arithmetic and many cost parallelism.
    const long long want = 8LL * ctx->sm_count;
    long long per = (long long)n_tb * H / want;
    if (per < (H + 511) / 512) per = (H + 511) / 512;       // so that the chunks never outnumber the partial sums
    if (bwd && per < 2) per = 2;       // the two that a thread has in flight, and half the sums: 1,237 tokens x 32 heads 9.2 -> 6.5 us
    a.per = per > 16 ? 16 : (int)per;
    a.q_chunks = (a.Hq + a.per - 1) / a.per;
    const int chunks = a.q_chunks + (a.Hk + a.per - 1) / a.per;
    if (!bwd) {
        qk_norm_rope_kernel<T, D, NEIGHBOURS><<<dim3(n_tb, chunks), kRopeThreads, 0, ctx->stream>>>(a);
        LOGOS_LAUNCH_CHECK(ctx, "qk_norm_rope_kernel");
        return LOGOS_OK;
    }
    // one partial sum per CTA, at most kRopeParts of them: CTAs then walk over token blocks
    const int most = kRopeParts / chunks;
    const int gx = n_tb < most ? n_tb : most;
    qk_norm_rope_bwd_kernel<T, D, NEIGHBOURS><<<dim3(gx, chunks), kRopeThreads, 0, ctx->stream>>>(a);
    LOGOS_LAUNCH_CHECK(ctx, "qk_norm_rope_bwd_kernel");
    if (dwq || dwk) {
        LOGOS_CUDA_TRY(ctx, launch_overlapped(rope_weight_grad_kernel, dim3(D / 32, 2), dim3(32 * kRopeReduceWarps), 0, ctx->stream,
                                              static_cast<const float*>(a.part), D, gx * a.q_chunks, gx * (chunks - a.q_chunks), dwq, dwk));
    }
    return LOGOS_OK;
}

template <typename T>
int dispatch(logos_ctx* ctx, RopeArgs& a, int DH, bool neighbours, bool bwd, float* dwq, float* dwk) {
    if (DH == 64) return neighbours ? launch<T, 64, true>(ctx, a, bwd, dwq, dwk) : launch<T, 64, false>(ctx, a, bwd, dwq, dwk);
    return neighbours ? launch<T, 128, true>(ctx, a, bwd, dwq, dwk) : launch<T, 128, false>(ctx, a, bwd, dwq, dwk);
}

}  // namespace

size_t qk_norm_rope_bwd_workspace_bytes(int DH) { return kWorkspaceCounterBytes + (size_t)kRopeParts * DH * sizeof(float); }

// forward: dQ_out, dK_out, dq_weight, dk_weight NULL and `bwd` false; backward: Y are the gradients of the rows
int qk_norm_rope(logos_ctx* ctx, int dtype, bool bwd, const void* Q, const void* K, const void* GQ, const void* GK,
                 const float* wq, const float* wk, const int32_t* positions, const logos_rope* rope, float eps, void* YQ,
                 void* YK, float* dwq, float* dwk, int rows, int Hq, int Hk, int DH, const logos_row_strides* q_in,
                 const logos_row_strides* k_in, const logos_row_strides* gq_in, const logos_row_strides* gk_in,
                 const logos_row_strides* q_out, const logos_row_strides* k_out) {
    const char* what = bwd ? "qk_norm_rope_bwd" : "qk_norm_rope";
    if (!dtype_ok(dtype)) return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: unknown dtype", what);
    if (!rope || rows < 0 || Hq < 0 || Hk < 0 || Hq + Hk == 0)
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: bad pointer or extent", what);
    if (DH != 64 && DH != 128) return fail(ctx, LOGOS_ERR_UNSUPPORTED, "%s: DH = %d (64 or 128)", what, DH);
    if (rope->dims < 0 || rope->dims > DH || rope->dims % 16)
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: rope dims %d (a multiple of 16 up to DH)", what, rope->dims);
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: eps must be finite and not negative", what);
    if (Hq > 1024 || Hk > 1024) return fail(ctx, LOGOS_ERR_UNSUPPORTED, "%s: more than 1024 heads", what);
    if (rows > kMostRows) return fail(ctx, LOGOS_ERR_UNSUPPORTED, "%s: %d rows (2^30 at most)", what, rows);
    RopeArgs a = {};
    for (int k = 0; k < rope->dims / 2; ++k) {
        const double f = rope->inv_freq[k];
        if (!std::isfinite(f)) return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: inv_freq[%d] is not finite", what, k);
        // (a frequency's 53 bits leave 2^31 positions 2^-22 of a turn: below fp32's own error of the angle)
        const double turns = f * 0.15915494309189535;               // 1 / (2 pi)
        const double frac = turns - std::floor(turns);
        a.turns[k] = frac < 1.0 ? (unsigned long long)(frac * 0x1p64) : 0ull;
    }
    if (bwd && ((wq == nullptr) != (dwq == nullptr) || (wk == nullptr) != (dwk == nullptr)))
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: a weight and its gradient are given together", what);
    if (rows == 0) {                                    // nothing to do but the empty sums
        if (dwq) LOGOS_CUDA_TRY(ctx, cudaMemsetAsync(dwq, 0, DH * sizeof(float), ctx->stream));
        if (dwk) LOGOS_CUDA_TRY(ctx, cudaMemsetAsync(dwk, 0, DH * sizeof(float), ctx->stream));
        return LOGOS_OK;
    }
    if (!positions || (Hq && (!Q || !YQ || (bwd && !GQ))) || (Hk && (!K || !YK || (bwd && !GK))))
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: null pointer", what);
    const size_t esz = dtype_size(dtype);
    const logos_row_strides pq{(int64_t)Hq * DH, DH}, pk{(int64_t)Hk * DH, DH};
    const logos_row_strides qi = q_in ? *q_in : pq, ki = k_in ? *k_in : pk, qo = q_out ? *q_out : pq, ko = k_out ? *k_out : pk;
    const logos_row_strides gqi = gq_in ? *gq_in : pq, gki = gk_in ? *gk_in : pk;
    for (const void* p : {Q, K, GQ, GK, (const void*)YQ, (const void*)YK, (const void*)wq, (const void*)wk})
        if (!aligned16(p)) return fail(ctx, LOGOS_ERR_ALIGNMENT, "%s: tensors and weights must be 16-byte aligned", what);
    if (!rows_aligned(qi, esz) || !rows_aligned(ki, esz) || !rows_aligned(qo, esz) || !rows_aligned(ko, esz) ||
        !rows_aligned(gqi, esz) || !rows_aligned(gki, esz))
        return fail(ctx, LOGOS_ERR_ALIGNMENT, "%s: negative strides, or rows that are not 16-byte aligned", what);
    if (!rows_apart(qo, rows, Hq, DH) || !rows_apart(ko, rows, Hk, DH))
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "%s: the rows of an output overlap", what);
    a.q = Q; a.k = K; a.gq = GQ; a.gk = GK; a.yq = YQ; a.yk = YK; a.wq = wq; a.wk = wk; a.pos = positions;
    a.q_row = qi.row; a.q_head = qi.head; a.k_row = ki.row; a.k_head = ki.head;
    a.yq_row = qo.row; a.yq_head = qo.head; a.yk_row = ko.row; a.yk_head = ko.head;
    a.gq_row = gqi.row; a.gq_head = gqi.head; a.gk_row = gki.row; a.gk_head = gki.head;
    a.eps = eps; a.dims = rope->dims; a.rows = rows; a.Hq = Hq; a.Hk = Hk;
    if (bwd) {
        if (!ctx->workspace || ctx->workspace_bytes < qk_norm_rope_bwd_workspace_bytes(DH))
            return fail(ctx, LOGOS_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, the context has %zu", what,
                        qk_norm_rope_bwd_workspace_bytes(DH), ctx->workspace ? ctx->workspace_bytes : 0);
        a.part = reinterpret_cast<float*>(static_cast<char*>(ctx->workspace) + kWorkspaceCounterBytes);
    }
    if (dtype == LOGOS_F32) return dispatch<float>(ctx, a, DH, rope->interleaved != 0, bwd, dwq, dwk);
    if (dtype == LOGOS_F16) return dispatch<__half>(ctx, a, DH, rope->interleaved != 0, bwd, dwq, dwk);
    return dispatch<__nv_bfloat16>(ctx, a, DH, rope->interleaved != 0, bwd, dwq, dwk);
}

}  // namespace logos
