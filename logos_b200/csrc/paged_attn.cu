// paged_attn.cu -- attention of new tokens over the paged INT8 cache (logos_paged_attention): the kernel for few query
// rows per key/value head (single tokens, speculative steps, short chunks), and the dispatch.
//
// Mathematics.  With K_j = ks_j k8_j and V_j = vs_j v8_j (int8 rows, one fp32 scale each) and a query row q,
//   x_j = (q . k8_j) scale log2(e) ks_j + log2(vs_j),   m = max x_j,   p_j = 2^(x_j - m),
//   O = sum_j p_j v8_j,   l = sum_j p_j / vs_j,   o = O / l:
// the scale of V rides in the exponent, so a weight p_j <= 1 meets plain integers, and both products run on FP16
// operands that hold the cache's bytes exactly.  q is brought into FP16 by a power of two per row (a BF16 value fits
// FP16's mantissa; the row's largest value becomes 2^13 ... 2^14, so only values 2^-27 below it lose bits).  p is
// rounded to FP16 once (2^-11 relative); everything else is fp32.
//
// What bounds it: HBM, 2 DH + 8 bytes per cached token and head.  Both contractions sit on mma.sync m16n8k16, whose
// fragments come straight from global memory: S = q K^T has the rows as M and the keys as N, O^T = V^T p has the
// channels as M and the rows as N, and the accumulator of the first is the B operand of the second as it is, so p
// never moves between threads.  The order of the channels inside a product is free, so a thread's share of a K row is
// 16 consecutive bytes and its share of a V row DH / 8.  Blocks of 32 keys and their scales come by
// cp.async into a ring of each warp's own, kStages blocks in flight and no registers spent on them.  (By cp.async.bulk, one
// lane for all, it took 80 instructions more a block, for the operands of its eight copies: 237 us where this took 197, 64 sequences x
// 16 heads x 8192 tokens.)  (tcgen05 needs 128 rows to be busy and its operands in shared memory; here a head has 1 to 16.)
// int8 -> FP16 costs five instructions for four values: bytes biased to unsigned, spliced under the exponent of 1024
// and the bias subtracted.
//
// A CTA takes one sequence, head, tile of 8 or 16 rows and one chunk of the keys; its four warps take the chunk's
// blocks in turn, each with its own running maximum, and join in shared memory.  Chunks join through the workspace:
// the last CTA to arrive sums the partial results in the order of the chunks.
//
// Measured: one token each of 64 sequences x 16 heads x 8192 tokens, DH 64, 194 us = 5.9 TB/s (0.90 of a plain copy);
// 4 sequences of 1,300 to 9,000 tokens, 32 heads over 8, DH 128, 21 us, 5 of them the join, at 3 CTAs per SM unevenly filled.
#include "paged.cuh"

namespace logos {
namespace {

constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = 32 * kSplitWarps;
constexpr int kStages = 2;                       // blocks in a warp's ring
constexpr int kSpan = 2048;                      // keys whose pages a warp's lanes hold, one 16-key block each
// Query rows per head up to which a sequence is this kernel's.  It reads the keys once per 16 rows (from L2 after the first),
// the other once per 256 with a longer start.  8 heads over 4000 tokens, this kernel / the other, us: one sequence, 64 rows
// 21 / 43 (DH 64), 34 / 48 (DH 128); 16 sequences 81 / 101 and 133 / 122; 128 rows 29 / 43, 47 / 50; 140 / 103, 230 / 126.
constexpr int kFewRows = 64;
constexpr int kSplitCounters = (int)(kWorkspaceCounterBytes / sizeof(int));

struct SplitArgs {
    PagedArgs p;
    const void* q;
    void* o;
    long long q_row, q_head, o_row, o_head;
    float c;                                     // scale * log2(e)
    int G, is_f16, causal, window, stride;
    int max_rows;                                // sequences with more query rows per head belong to paged_chunk_kernel
    int chunk, splits, tiles;                    // keys per chunk; most chunks and row tiles of a (sequence, head)
    float* part;                                 // [(sequence, head, tile)][splits][rows][DH + 2]
    int* counters;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int D>
__device__ __forceinline__ void store_out(const SplitArgs& a, int token, int head, int d, float x, float y) {
    const long long at = (long long)token * a.o_row + (long long)head * a.o_head + d;
    if (a.is_f16) *reinterpret_cast<__half2*>(static_cast<__half*>(a.o) + at) = __floats2half2_rn(x, y);
    else *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.o) + at) = __floats2bfloat162_rn(x, y);
}

// shared memory of a CTA: the warps' rings; the join of the warps uses their space
template <int D, int NQ> struct SplitShape {
    static constexpr int kRows = 8 * NQ, kKB = 32;            // keys of a block
    static constexpr int kOffV = kKB * D, kOffKs = 2 * kKB * D, kOffVs = kOffKs + 4 * kKB, kStage = kOffVs + 4 * kKB;
    static constexpr int kScaled = 8 * kKB;                   // log2 vs and 1 / vs of the warp's current block
    static constexpr int kRings = kSplitWarps * (kStages * kStage + kScaled);
    static constexpr int kPitch = D + 4;
    static constexpr int kJoin = kSplitWarps * kRows * (kPitch + 2) * 4;
    static constexpr int kSmem = kRings > kJoin ? kRings : kJoin;
};

// NQ: groups of 8 query rows in the tile
template <int D, int NQ>
__global__ void __launch_bounds__(kSplitThreads)
paged_split_kernel(const __grid_constant__ SplitArgs a) {
    using C = SplitShape<D, NQ>;
    constexpr int ROWS = C::kRows, KB = C::kKB, SUB = KB / 16;   // SUB: 16-key pieces of a block
    constexpr int KG = KB / 8, KS = D / 16, MT = D / 16, VW = D / 32;   // key groups; k steps of S; channel tiles; words of a V share
    constexpr int PITCH = C::kPitch;
    extern __shared__ __align__(128) unsigned char smem[];
    float (*s_o)[ROWS][PITCH] = reinterpret_cast<float (*)[ROWS][PITCH]>(smem);
    float (*s_m)[ROWS] = reinterpret_cast<float (*)[ROWS]>(smem + kSplitWarps * ROWS * PITCH * 4);
    float (*s_l)[ROWS] = s_m + kSplitWarps;
    __shared__ int s_last;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int b = blockIdx.y;
    int x = blockIdx.x;
    const int split = x % a.splits;
    x /= a.splits;
    const int h = x % a.p.H, tile = x / a.p.H;
    const PagedSeq s = paged_seq(a.p, b);
    if (!s.ok) {
        if (tid == 0 && blockIdx.x == 0) report_batch(a.p.status, b, false);
        return;
    }
    const int r0 = tile * ROWS, n_rows = min(ROWS, s.n * a.G - r0);
    if (n_rows <= 0 || (long long)s.n * a.G > a.max_rows) return;
    const int first = s.kv - s.n + r0 / a.G, last = s.kv - s.n + (r0 + n_rows - 1) / a.G;   // positions of the tile's rows
    const bool shun = shunyam_active(a.window, s.kv);
    const bool pure = shun && a.stride <= 0;     // a window without landmarks bounds the keys on both sides
    const int k_end = (a.causal || pure) ? last + 1 : s.kv;
    const int k_begin = pure ? (max(0, first - a.window) & ~(KB - 1)) : 0;
    const int n_splits = (k_end - k_begin + a.chunk - 1) / a.chunk;
    if (split >= n_splits) return;
    const int c0 = k_begin + split * a.chunk, c1 = min(c0 + a.chunk, k_end);

    unsigned char* ring = smem + warp * (kStages * C::kStage + C::kScaled);
    float* scaled = reinterpret_cast<float*>(ring + kStages * C::kStage);
    const uint32_t ring_addr = (uint32_t)__cvta_generic_to_shared(ring);
    // The chunk is walked in spans of 2048 keys.  Block i of a warp in a span is keys s0 + (4 i + warp) KB ...; lane
    // SUB i + j holds the page of its j-th 16 keys (a page never ends inside 16 keys).
    int s0 = c0, s1 = c0, n_iter = 0, my_page = -1;
    bool whole = true;                            // every page of the warp's blocks is there
    auto open_span = [&](int at0) {
        s0 = at0;
        s1 = min(s0 + kSpan, c1);
        n_iter = (s1 - s0 - warp * KB + kSplitWarps * KB - 1) / (kSplitWarps * KB);
        const int at = s0 + ((lane / SUB) * kSplitWarps + warp) * KB + (lane % SUB) * 16;
        my_page = -1;
        if (at < s1) {
            my_page = paged_page(a.p, b, at);
            if (my_page < 0) report_batch(a.p.status, b, true);
        }
        whole = __all_sync(0xffffffffu, at >= s1 || my_page >= 0);
    };
    open_span(c0);
    int st_in = 0, st_out = 0;                    // stages of the next block requested and taken
    // Requests block `it` of the span.  A page that is not there is read as page 0 and masked later.  (The lanes have read
    // the stage's last block: the __syncwarp before.)
    auto request = [&](int it) {
        if (it < n_iter) {
            const uint32_t dst = ring_addr + st_in * C::kStage + 16 * lane;
            const int key = s0 + (it * kSplitWarps + warp) * KB;
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                const int page = max(__shfl_sync(0xffffffffu, my_page, (it * SUB + j) & 31), 0);
                const uint32_t row = paged_row(a.p, page, h) + ((key + 16 * j) & ((1 << a.p.page_shift) - 1));
                const int8_t *k = a.p.k + (size_t)row * D + 16 * lane, *v = a.p.v + (size_t)row * D + 16 * lane;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    cp_async16(dst + 16 * j * D + 512 * i, k + 512 * i);
                    cp_async16(dst + C::kOffV + 16 * j * D + 512 * i, v + 512 * i);
                }
                if (lane < 8)                     // 64 bytes of each kind of scale
                    cp_async16(dst + (lane < 4 ? C::kOffKs : C::kOffVs - 64) + 64 * j, (lane < 4 ? a.p.ks : a.p.vs - 16) + row + 4 * lane);
            }
            st_in = st_in + 1 == kStages ? 0 : st_in + 1;
        }
        cp_async_commit();
    };
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) request(i);

    // the rows' A fragments: k step 4 i + e of the products holds channels 64 i + 16 t + 4 e ... + 3 of this thread
    uint32_t qa[KS][4];
    float alpha[NQ];                             // scale log2(e), with the row's power of two taken out again
    int pos[NQ];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        if (n >= NQ) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qa[ks][1] = qa[ks][3] = 0;
            break;
        }
        const int r = 8 * n + g;
        const bool in = r < n_rows;
        const int token = (r0 + (in ? r : 0)) / a.G, head = h * a.G + (r0 + (in ? r : 0)) % a.G;
        pos[n] = s.kv - s.n + token;
        float f[D / 4];
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + (long long)(s.q0 + token) * a.q_row + (long long)head * a.q_head + 16 * t;
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const uint4 w = in ? *reinterpret_cast<const uint4*>(src + 64 * (i >> 1) + 8 * (i & 1)) : make_uint4(0, 0, 0, 0);
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float2 v;
                if (a.is_f16) v = __half22float2(*reinterpret_cast<const __half2*>(&ww[e]));
                else v = make_float2(__uint_as_float(ww[e] << 16), __uint_as_float(ww[e] & 0xffff0000u));
                f[8 * i + 2 * e] = v.x;
                f[8 * i + 2 * e + 1] = v.y;
                top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float mul, unmul;
        row_power(top, mul, unmul);
        alpha[n] = a.c * unmul;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const __half2 lo = __floats2half2_rn(f[4 * ks] * mul, f[4 * ks + 1] * mul), hi = __floats2half2_rn(f[4 * ks + 2] * mul, f[4 * ks + 3] * mul);
            qa[ks][n] = *reinterpret_cast<const uint32_t*>(&lo);
            qa[ks][2 + n] = *reinterpret_cast<const uint32_t*>(&hi);
        }
    }

    float o[NQ][MT][4];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
    }

    for (;;) {
    for (int it = 0; it < n_iter; ++it) {
        const int k0 = s0 + (it * kSplitWarps + warp) * KB;
        const unsigned char* blk = ring + st_out * C::kStage;
        st_out = st_out + 1 == kStages ? 0 : st_out + 1;
        cp_async_wait<kStages - 1>();
        __syncwarp();                            // every lane's part of the block is there
        // each value scale's logarithm and reciprocal once, not by all eight threads that need them
        {
            const float v = fmaxf(reinterpret_cast<const float*>(blk + C::kOffVs)[lane], kLeastScale);
            scaled[lane] = __log2f(v);
            scaled[KB + lane] = __fdividef(1.0f, v);
        }
        __syncwarp();
        float sc[KG][4];
#pragma unroll
        for (int u = 0; u < KG; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[u][e] = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const uint4 kr = *reinterpret_cast<const uint4*>(blk + (8 * u + g) * D + 64 * i + 16 * t);
                const uint32_t w[4] = {kr.x ^ 0x80808080u, kr.y ^ 0x80808080u, kr.z ^ 0x80808080u, kr.w ^ 0x80808080u};
#pragma unroll
                for (int e = 0; e < 4; ++e) mma_f16(sc[u], qa[4 * i + e], bytes_to_half2(w[e], 0x4140), bytes_to_half2(w[e], 0x4342));
            }
            const float2 ksr = *reinterpret_cast<const float2*>(blk + C::kOffKs + 32 * u + 8 * t), lv = *reinterpret_cast<const float2*>(scaled + 8 * u + 2 * t);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                sc[u][2 * n] = fmaf(sc[u][2 * n], alpha[n] * ksr.x, lv.x);
                sc[u][2 * n + 1] = fmaf(sc[u][2 * n + 1], alpha[n] * ksr.y, lv.y);
            }
        }
        if (!whole || shun || k0 + KB > c1 || (a.causal && k0 + KB - 1 > first)) {
#pragma unroll
            for (int u = 0; u < KG; ++u) {
                const bool there = __shfl_sync(0xffffffffu, my_page, (it * SUB + (u >> 1)) & 31) >= 0;
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = k0 + 8 * u + 2 * t + e;
                        if (!there || key >= c1 || !key_allowed(pos[n], key, a.causal != 0, shun, a.window, a.stride)) sc[u][2 * n + e] = -INFINITY;
                    }
            }
        }
        float f[NQ];
        bool moved = false;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float top = fmaxf(sc[0][2 * n], sc[0][2 * n + 1]);
#pragma unroll
            for (int u = 1; u < KG; ++u) top = fmaxf(top, fmaxf(sc[u][2 * n], sc[u][2 * n + 1]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the reference maximum moves only when a weight would pass 2^15 (FP16 ends at 2^16), or at the first key
            const bool move = top > m[n] + kMoveMax || (m[n] == -INFINITY && top > -INFINITY);
            f[n] = (move && m[n] > -INFINITY) ? exp2_fast(m[n] - top) : 1.0f;
            moved |= move && m[n] > -INFINITY;
            if (move) m[n] = top;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                l[n] *= f[n];
                const float f0 = __shfl_sync(0xffffffffu, f[n], 8 * t), f1 = __shfl_sync(0xffffffffu, f[n], 8 * t + 4);   // rows 2t, 2t + 1
#pragma unroll
                for (int i = 0; i < MT; ++i) { o[n][i][0] *= f0; o[n][i][1] *= f1; o[n][i][2] *= f0; o[n][i][3] *= f1; }
            }
        }
        uint32_t pb[NQ][KG];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float ref = m[n] == -INFINITY ? 0.0f : m[n];
#pragma unroll
            for (int u = 0; u < KG; ++u) {
                const float2 inv = *reinterpret_cast<const float2*>(scaled + KB + 8 * u + 2 * t);
                const float p0 = exp2_fast(sc[u][2 * n] - ref), p1 = exp2_fast(sc[u][2 * n + 1] - ref);
                l[n] = fmaf(p0, inv.x, l[n]);
                l[n] = fmaf(p1, inv.y, l[n]);
                const __half2 w = __floats2half2_rn(p0, p1);
                pb[n][u] = *reinterpret_cast<const uint32_t*>(&w);
            }
        }
        // O^T += V^T p: the thread's channels are g DH / 8 + 2 tile, + 1
#pragma unroll
        for (int u2 = 0; u2 < KG / 2; ++u2) {
            uint32_t vr[4][VW];                  // keys 2t, 2t + 1, 2t + 8, 2t + 9 of the 16
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned char* at = blk + C::kOffV + (16 * u2 + 2 * t + 8 * (i >> 1) + (i & 1)) * D + g * (D / 8);
                if (D == 64) {
                    const uint2 x = *reinterpret_cast<const uint2*>(at);
                    vr[i][0] = x.x ^ 0x80808080u; vr[i][1] = x.y ^ 0x80808080u;
                } else {
                    const uint4 x = *reinterpret_cast<const uint4*>(at);
                    vr[i][0] = x.x ^ 0x80808080u; vr[i][1] = x.y ^ 0x80808080u;
                    vr[i][VW - 2] = x.z ^ 0x80808080u; vr[i][VW - 1] = x.w ^ 0x80808080u;
                }
            }
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                const uint32_t x0 = vr[0][w], x1 = vr[1][w], y0 = vr[2][w], y1 = vr[3][w];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t mx = prmt(x0, x1, half ? 0x7362 : 0x5140), my = prmt(y0, y1, half ? 0x7362 : 0x5140);
                    const uint32_t va[4] = {bytes_to_half2(mx, 0x4140), bytes_to_half2(mx, 0x4342),
                                            bytes_to_half2(my, 0x4140), bytes_to_half2(my, 0x4342)};
#pragma unroll
                    for (int n = 0; n < NQ; ++n) mma_f16(o[n][2 * w + half], va, pb[n][2 * u2], pb[n][2 * u2 + 1]);
                }
            }
        }
        __syncwarp();                            // the block has been read by every lane
        request(it + kStages);
    }
    if (s1 >= c1) break;
    open_span(s1);
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) request(i);
    }
    cp_async_wait<0>();
    __syncthreads();                             // no block is on its way any more: the rings' space is free

    // join the warps: statistics of row 8 n + g, then the outputs scaled to the CTA's maximum
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 1);
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], 2);
        if (m[n] == -INFINITY && !(l[n] == 0.0f)) m[n] = 0.0f;   // scores that are all NaN: not an empty row
        if (t == 0) { s_m[warp][8 * n + g] = m[n]; s_l[warp][8 * n + g] = l[n]; }
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = 8 * n + 2 * t + e;
            float top = s_m[0][r];
#pragma unroll
            for (int w = 1; w < kSplitWarps; ++w) top = fmaxf(top, s_m[w][r]);
            const float mine = s_m[warp][r];
            const float f = mine == -INFINITY ? 0.0f : exp2_fast(mine - top);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                s_o[warp][r][g * (D / 8) + 2 * i] = o[n][i][e] * f;
                s_o[warp][r][g * (D / 8) + 2 * i + 1] = o[n][i][2 + e] * f;
            }
        }
    __syncthreads();
    const size_t unit = ((size_t)b * a.p.H + h) * a.tiles + tile;
    float* part = a.part + unit * a.splits * ROWS * (D + 2);
    for (int i = tid; i < n_rows * (D / 2); i += kSplitThreads) {
        const int r = i / (D / 2), d = 2 * (i % (D / 2));
        float top = s_m[0][r], sum = 0.0f, x0 = 0.0f, x1 = 0.0f;
#pragma unroll
        for (int w = 1; w < kSplitWarps; ++w) top = fmaxf(top, s_m[w][r]);
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) {
            if (s_m[w][r] == -INFINITY) continue;
            sum = fmaf(s_l[w][r], exp2_fast(s_m[w][r] - top), sum);
            x0 += s_o[w][r][d];
            x1 += s_o[w][r][d + 1];
        }
        if (n_splits == 1) {
            const float n = top == -INFINITY ? 0.0f : 1.0f / sum;
            store_out<D>(a, s.q0 + (r0 + r) / a.G, h * a.G + (r0 + r) % a.G, d, x0 * n, x1 * n);
        } else {
            float* rec = part + ((size_t)split * ROWS + r) * (D + 2);
            *reinterpret_cast<float2*>(rec + 2 + d) = make_float2(x0, x1);
            if (d == 0) *reinterpret_cast<float2*>(rec) = make_float2(top, sum);
        }
    }
    if (n_splits == 1) return;
    __threadfence();
    __syncthreads();
    if (tid == 0) s_last = atomicAdd(a.counters + unit, 1) == n_splits - 1;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    if (tid == 0) a.counters[unit] = 0;          // as the next launch expects it
    // A warp per row; the statistics of 32 chunks at a time, a lane each, then the chunks' outputs, several loads in flight.
    for (int r = warp; r < n_rows; r += kSplitWarps) {
        const float* rec = part + (size_t)r * (D + 2);
        constexpr size_t kNext = (size_t)ROWS * (D + 2);
        float top = -INFINITY;
        for (int sp = lane; sp < n_splits; sp += 32) top = fmaxf(top, __ldcg(rec + sp * kNext));
        top = warp_max(top);
        float sum = 0.0f;
        float2 x[D / 64];
#pragma unroll
        for (int i = 0; i < D / 64; ++i) x[i] = make_float2(0.0f, 0.0f);
        for (int base = 0; base < n_splits; base += 32) {
            float f = 0.0f;
            if (base + lane < n_splits) {
                const float2 st = __ldcg(reinterpret_cast<const float2*>(rec + (base + lane) * kNext));
                f = st.x == -INFINITY ? 0.0f : exp2_fast(st.x - top);
                sum = fmaf(st.y, f, sum);
            }
            const int n = min(32, n_splits - base);
#pragma unroll 16
            for (int j = 0; j < n; ++j) {
                const float2* v = reinterpret_cast<const float2*>(rec + (base + j) * kNext + 2) + lane;
                const float fj = __shfl_sync(0xffffffffu, f, j);
#pragma unroll
                for (int i = 0; i < D / 64; ++i) {
                    const float2 y = __ldcg(v + 32 * i);
                    x[i].x = fmaf(y.x, fj, x[i].x);
                    x[i].y = fmaf(y.y, fj, x[i].y);
                }
            }
        }
        sum = warp_sum(sum);
        const float n = top == -INFINITY ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int i = 0; i < D / 64; ++i)
            store_out<D>(a, s.q0 + (r0 + r) / a.G, h * a.G + (r0 + r) % a.G, 64 * i + 2 * lane, x[i].x * n, x[i].y * n);
    }
}

// how a batch is cut: row tiles of 8 or 16, chunks of keys
struct SplitPlan { int rows, tiles, chunk, splits; size_t bytes; bool chunks; };
SplitPlan plan_split(const logos_ctx* ctx, const logos_paged_cache* c, const logos_paged_batch* b, int G) {
    SplitPlan p;
    int64_t most = (int64_t)b->max_q * G;                    // query rows of a (sequence, head)
    p.chunks = most > kFewRows;                              // some may be paged_chunk_kernel's
    if (p.chunks) most = kFewRows;
    p.rows = most <= 8 ? 8 : 16;
    p.tiles = (int)((most + p.rows - 1) / p.rows);
    const int64_t units = (int64_t)b->B * c->H * p.tiles;
    // enough chunks for four CTAs on every SM, none shorter than 128 keys (a block per warp at DH 64)
    const int64_t want = (4LL * ctx->sm_count + units - 1) / (units > 0 ? units : 1);
    int64_t chunk = (b->max_kv + want - 1) / want;
    chunk = chunk > kSpan && units <= kSplitCounters ? kSpan : chunk;
    if (units > kSplitCounters) chunk = b->max_kv;           // no counters to join chunks with, and CTAs enough
    chunk = (chunk + 127) / 128 * 128;
    p.chunk = chunk < 128 ? 128 : (int)chunk;
    p.splits = (b->max_kv + p.chunk - 1) / p.chunk;
    p.bytes = kWorkspaceCounterBytes + (size_t)units * p.splits * p.rows * (c->DH + 2) * sizeof(float);
    if (p.chunks) {                                          // the two kernels run one after the other
        const size_t other = paged_chunk_workspace_bytes(ctx, c->DH);
        if (other > p.bytes) p.bytes = other;
    }
    return p;
}

template <int D, int NQ>
int launch_split(logos_ctx* ctx, const SplitArgs& a) {
    const dim3 grid((unsigned)((int64_t)a.splits * a.p.H * a.tiles), a.p.B);
    auto* fn = paged_split_kernel<D, NQ>;
    if (int rc = ensure_smem_limit(ctx, fn, SplitShape<D, NQ>::kSmem)) return rc;
    fn<<<grid, kSplitThreads, SplitShape<D, NQ>::kSmem, ctx->stream>>>(a);
    LOGOS_LAUNCH_CHECK(ctx, "paged_split_kernel");
    return LOGOS_OK;
}
template <int D>
int launch_split(logos_ctx* ctx, const SplitArgs& a, int rows) {
    return rows == 8 ? launch_split<D, 1>(ctx, a) : launch_split<D, 2>(ctx, a);
}

}  // namespace

size_t paged_attention_workspace_bytes(logos_ctx* ctx, const logos_paged_cache* c, const logos_paged_batch* b, int Hq) {
    if (b->B == 0 || b->rows == 0 || b->max_q == 0) return kWorkspaceCounterBytes;
    return plan_split(ctx, c, b, Hq / c->H).bytes;
}

int paged_attention(logos_ctx* ctx, int dtype, const void* Q, const logos_paged_cache* cache, const logos_paged_batch* batch,
                    int Hq, const logos_attn_params* prm, void* O, const logos_row_strides* q_in, const logos_row_strides* o_out) {
    if (int rc = paged_check(ctx, "paged_attention", cache, batch)) return rc;
    if (dtype != LOGOS_BF16 && dtype != LOGOS_F16)
        return fail(ctx, dtype_ok(dtype) ? LOGOS_ERR_UNSUPPORTED : LOGOS_ERR_INVALID_ARG, "paged_attention: Q and O are BF16 or FP16");
    if (Hq <= 0 || Hq > 1024 || Hq % cache->H)
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "paged_attention: %d query heads over %d key/value heads (a multiple, at most 1024)", Hq, cache->H);
    if (!(prm->scale > 0.0f) || !(prm->scale < INFINITY))
        return fail(ctx, LOGOS_ERR_UNSUPPORTED, "paged_attention: scale must be positive and finite");
    if (prm->ns_alpha > 0.0f && (prm->ns_eta != 0.0f || (prm->diffuse_mode != LOGOS_DIFFUSE_NONE && prm->ns_nu != 0.0f)))
        return fail(ctx, LOGOS_ERR_UNSUPPORTED, "paged_attention: the Navier-Stokes terms are not offered over pages");
    if (batch->B == 0 || batch->rows == 0 || batch->max_q == 0) return LOGOS_OK;
    if (!Q || !O) return fail(ctx, LOGOS_ERR_INVALID_ARG, "paged_attention: null pointer");
    if (!aligned16(Q) || !aligned16(O)) return fail(ctx, LOGOS_ERR_ALIGNMENT, "paged_attention: tensors must be 16-byte aligned");
    const logos_row_strides packed{(int64_t)Hq * cache->DH, cache->DH};
    const logos_row_strides q = q_in ? *q_in : packed, o = o_out ? *o_out : packed;
    if (!rows_aligned(q, 2) || !rows_aligned(o, 2))
        return fail(ctx, LOGOS_ERR_ALIGNMENT, "paged_attention: negative strides, or rows that are not 16-byte aligned");
    if (!rows_apart(o, batch->rows, Hq, cache->DH))
        return fail(ctx, LOGOS_ERR_INVALID_ARG, "paged_attention: the rows of the output overlap");
    const int G = Hq / cache->H;
    const SplitPlan plan = plan_split(ctx, cache, batch, G);
    if ((int64_t)plan.splits * cache->H * plan.tiles > 0x7fffffffLL)
        return fail(ctx, LOGOS_ERR_UNSUPPORTED, "paged_attention: the batch needs more than 2^31 CTAs");
    if (!ctx->workspace || ctx->workspace_bytes < plan.bytes)
        return fail(ctx, LOGOS_ERR_WORKSPACE, "paged_attention: needs %zu bytes of workspace, the context has %zu", plan.bytes,
                    ctx->workspace ? ctx->workspace_bytes : 0);
    SplitArgs a;
    a.p = paged_args(ctx, cache, batch);
    a.q = Q; a.o = O;
    a.q_row = q.row; a.q_head = q.head; a.o_row = o.row; a.o_head = o.head;
    a.c = prm->scale * 1.4426950408889634f;
    a.G = G; a.is_f16 = dtype == LOGOS_F16;
    a.causal = prm->causal != 0; a.window = prm->window; a.stride = prm->stride;
    a.max_rows = kFewRows;
    a.chunk = plan.chunk; a.splits = plan.splits; a.tiles = plan.tiles;
    a.counters = static_cast<int*>(ctx->workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(ctx->workspace) + kWorkspaceCounterBytes);
    if (int rc = cache->DH == 64 ? launch_split<64>(ctx, a, plan.rows) : launch_split<128>(ctx, a, plan.rows)) return rc;
    if (!plan.chunks) return LOGOS_OK;
    return paged_chunk(ctx, a.p, cache->DH, Q, O, q, o, G, a.is_f16 != 0, prm, kFewRows);
}

}  // namespace logos
