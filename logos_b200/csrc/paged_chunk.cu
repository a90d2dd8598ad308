// paged_chunk.cu -- attention of chunks of new tokens over the paged INT8 cache on the 5th-generation tensor cores: the
// sequences of a logos_paged_attention call that have many query rows per key/value head.
//
// The mathematics is that of paged_attn.cu: x_j = (q . k8_j) (scale log2(e) ks_j) + log2(vs_j), weights 2^(x_j - m) in
// FP16 against plain integers, l = sum p_j / vs_j.  A key is three fp32 numbers then, (a, b, 1/vs), which travel
// beside its bytes through shared memory.
//
// What bounds it: per 256 rows x 128 keys the exponentials (16 a clock and SM: 2048 clocks) and the products
// (M128 N128 K16 in 67 clocks, N64 in 57 to 63: 1500 clocks at DH 64, 2150 at DH 128); the cache itself is read once
// per 256 rows and comes from L2 after the first.  So the threads' chain per tile decides, and everything that is not
// softmax is taken off the softmax threads.
//
// A CTA (512 threads, one per SM) holds two 128-row tiles of one (sequence, head) -- row r is token r / G, query head
// r % G of the group, so grouped heads share every K and V tile -- and walks over key tiles of 128.  Roles:
//   warps 0-3 / 4-7   softmax of tile 0 / 1, one thread per row (TMEM lane), the row's 128 scores in registers
//   warps 8,9 / 10,11 K / V: pages -> registers one tile ahead -> FP16 -> 128B-swizzled tiles in shared memory
//   warps 12,13       MMA issuers, one per tile: S = Q K^T from shared memory, O += P V with P read from TMEM
//   warp 14           the schedule
// TMEM (512 columns), DH 64: S 2 x 128, O 2 x 64, P 2 x 64, so the next scores are computed under this tile's
// exponentials.  DH 128: S 2 x 128, O 2 x 128; P lies on the first half of its own S, the next scores follow this
// tile's PV in the pipe and the other tile's exponentials cover both.
//
// Schedule.  The key tiles of all (sequence, head, 256 rows) items form one line, cut into equal shares, one per CTA:
// ragged batches, few rows over a long context and many rows alike fill the device.  An item cut between CTAs leaves
// partial results (at most two per CTA) in the workspace, and paged_join_kernel sums them in the order of the keys.
// Every wait is bounded: when one runs out the CTA raises its abort flag, all roles leave and the status word says so.
#include "paged.cuh"
#include "tcgen05_ptx.cuh"

namespace logos {
namespace {

using namespace tc;

constexpr int kChunkThreads = 512;
constexpr int kChunkRows = 256;              // query rows of an item
constexpr int kBN = 128;                     // keys of a tile
constexpr int kConvWarp = 8, kMmaWarp = 12, kPlanWarp = 14;
constexpr int kRegsSoftmax = 184, kRegsConvert = 104, kRegsRest = 40;
static_assert(256 * kRegsSoftmax + 128 * kRegsConvert + 128 * kRegsRest <= 65536 && 65536 / kChunkThreads == 128, "registers");
constexpr int kScaleStages = 4, kSegStages = 4;
constexpr int kSegReaders = kPlanWarp;       // warps 0 ... 13 read every segment
constexpr int kJoinRows = 32;                // rows a CTA of the join takes

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

template <int D> struct Shape {
    static constexpr int kTile = kBN * D * 2;                 // one FP16 tile of 128 rows
    static constexpr int kStages = D == 64 ? 3 : 2;
    static constexpr bool kOwnP = D == 64;                    // P has TMEM columns of its own
    static constexpr int kOffQ = 0, kOffK = kOffQ + 2 * kTile, kOffV = kOffK + kStages * kTile;
    static constexpr int kOffScale = kOffV + kStages * kTile; // kScaleStages x {a, b, 1/vs: 128 floats each, 4 words of landmarks}
    static constexpr int kScaleBytes = 3 * kBN * 4 + 16;
    static constexpr int kOffSeg = kOffScale + kScaleStages * kScaleBytes;
    static constexpr int kOffBar = kOffSeg + kSegStages * 64;
    static constexpr int kNumBars = 4 * kStages + 2 * kScaleStages + 2 * kSegStages + 5 * 2 + 1;
    static constexpr int kOffScan = kOffBar + kNumBars * 8;
    static constexpr int kSmem = kOffScan + 128 + 1024;       // + alignment slack
    static constexpr int kColO = 256, kColP = 384;
};
static_assert(Shape<128>::kSmem <= 232448 && Shape<64>::kSmem <= 232448, "shared memory");

struct Segment {          // a run of key tiles of one item
    int b, h, row0;       // sequence, head, first query row
    int n_rows;           // query rows of the whole (sequence, head)
    int q0, n, kv;        // the sequence: first token row, new tokens, tokens held
    int begin, end;       // keys of the item
    int i0, n_iter;       // first tile of the run, its tiles; n_iter 0: no more segments
    int slot;             // where a partial result goes; -1: the run is the whole item
};
static_assert(sizeof(Segment) <= 64, "segment slot");

struct JoinMeta { int parts, slot, b, h, row0, n_rows, q0, pad; };   // an item that starts in this CTA and does not end there

struct ChunkArgs {
    PagedArgs p;
    const void* q;
    void* o;
    long long q_row, q_head, o_row, o_head;
    float c;                                  // scale * log2(e)
    int G, is_f16, causal, window, stride;
    int min_rows;                             // sequences of at most this many query rows belong to the other kernel
    JoinMeta* meta;                           // [CTAs]
    float2* stat;                             // [CTAs][2][256]: m, l
    float* part;                              // [CTAs][2][256][DH]
};

struct Item { int begin, end, tiles; };
// keys that some of the query rows [row0, row0 + rows) see
__device__ __forceinline__ Item item_keys(const ChunkArgs& a, const PagedSeq& s, int row0, int rows) {
    const int first = s.kv - s.n + row0 / a.G, last = s.kv - s.n + (row0 + rows - 1) / a.G;
    const bool pure = shunyam_active(a.window, s.kv) && a.stride <= 0;
    Item it;
    it.end = (a.causal || pure) ? last + 1 : s.kv;
    it.begin = pure ? (max(0, first - a.window) & ~(kBN - 1)) : 0;
    it.tiles = (it.end - it.begin + kBN - 1) / kBN;
    return it;
}
// key tiles of one head of a sequence; 0 when the sequence is not this kernel's
__device__ __forceinline__ long long seq_tiles(const ChunkArgs& a, int b) {
    const PagedSeq s = paged_seq(a.p, b);
    if (!s.ok || (long long)s.n * a.G <= a.min_rows) return 0;
    long long sum = 0;
    for (int r = 0; r < s.n * a.G; r += kChunkRows) sum += item_keys(a, s, r, min(kChunkRows, s.n * a.G - r)).tiles;
    return sum;
}

template <int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
paged_chunk_kernel(const __grid_constant__ ChunkArgs a) {
    using C = Shape<D>;
    constexpr int ST = C::kStages;
    enum Bar { KFULL = 0, KEMPTY = KFULL + ST, VFULL = KEMPTY + ST, VEMPTY = VFULL + ST, SCFULL = VEMPTY + ST,
               SCEMPTY = SCFULL + kScaleStages, SEGFULL = SCEMPTY + kScaleStages, SEGEMPTY = SEGFULL + kSegStages,
               SFULL = SEGEMPTY + kSegStages, SEMPTY = SFULL + 2, PFULL = SEMPTY + 2, PVDONE = PFULL + 2, QREADY = PVDONE + 2,
               DRAIN = QREADY + 2, NBARS };
    static_assert(NBARS == C::kNumBars, "barrier count");
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t sbase = smem_u32(smem), bar0 = sbase + C::kOffBar;
    auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
    long long* scan = reinterpret_cast<long long*>(smem + C::kOffScan);       // the prologue's warp totals
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    __shared__ long long s_before;
    __shared__ int s_start_b;
    volatile int* abort_flag = &abort_word;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < ST; ++i) { mbar_init(bar(KFULL + i), 64); mbar_init(bar(KEMPTY + i), 2); mbar_init(bar(VFULL + i), 64); mbar_init(bar(VEMPTY + i), 2); }
        for (int i = 0; i < kScaleStages; ++i) { mbar_init(bar(SCFULL + i), 64); mbar_init(bar(SCEMPTY + i), 256); }
        for (int i = 0; i < kSegStages; ++i) { mbar_init(bar(SEGFULL + i), 1); mbar_init(bar(SEGEMPTY + i), kSegReaders); }
        for (int g = 0; g < 2; ++g) {
            mbar_init(bar(SFULL + g), 1); mbar_init(bar(SEMPTY + g), 128); mbar_init(bar(PFULL + g), 128);
            mbar_init(bar(PVDONE + g), 1); mbar_init(bar(QREADY + g), 128);
        }
        mbar_init(bar(DRAIN), 2);
        abort_word = 0;
        a.meta[blockIdx.x].parts = 0;                       // nothing to join, unless the schedule says otherwise
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // the line of key tiles: its length, then the sequence in which this CTA's share begins
    long long total = 0, share = 0, my0 = 0, my1 = 0;
    for (int pass = 0; pass < 2; ++pass) {
        long long run = 0;
        for (int b0 = 0; b0 < a.p.B; b0 += kChunkThreads) {
            const int b = b0 + tid;
            const long long mine = b < a.p.B ? seq_tiles(a, b) * a.p.H : 0;
            long long inc = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long up = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += up;
            }
            if (lane == 31) scan[warp] = inc;
            __syncthreads();
            long long before = run, block = 0;
            for (int w = 0; w < kChunkThreads / 32; ++w) { if (w < warp) before += scan[w]; block += scan[w]; }
            const long long end = before + inc, start = end - mine;
            if (pass == 1 && mine > 0 && my0 >= start && my0 < end) { s_start_b = b; s_before = start; }
            run += block;
            __syncthreads();
        }
        if (pass == 0) {
            total = run;
            share = (total + gridDim.x - 1) / gridDim.x;
            if (share < 2) share = 2;                       // a shorter run costs more in joining than it saves
            my0 = (long long)blockIdx.x * share;
            my1 = my0 + share < total ? my0 + share : total;
            if (my0 >= total) break;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const bool work = my0 < total;

    if (warp >= kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsRest));
        if (work && warp == kPlanWarp) {
            // ================= the schedule: this CTA's share as segments =================
            if (lane == 0) {
                int b = s_start_b, n_seg = 0;
                long long at = my0, base = s_before;         // base: where sequence b begins on the line
                JoinMeta meta = {0, 0, 0, 0, 0, 0, 0, 0};
                bool ok = true;
                for (; ok && at < my1; ++b) {
                    if (b >= a.p.B) break;
                    const long long per_head = seq_tiles(a, b);
                    if (per_head == 0) continue;
                    const PagedSeq s = paged_seq(a.p, b);
                    const int n_rows = s.n * a.G;
                    int h = (int)((at - base) / per_head);
                    long long off = (at - base) % per_head;  // into head h's tiles
                    for (; ok && h < a.p.H && at < my1; ++h) {
                        for (int row0 = 0; ok && row0 < n_rows && at < my1; row0 += kChunkRows) {
                            const Item it = item_keys(a, s, row0, min(kChunkRows, n_rows - row0));
                            if (off >= it.tiles) { off -= it.tiles; continue; }
                            Segment g;
                            g.b = b; g.h = h; g.row0 = row0; g.n_rows = n_rows;
                            g.q0 = s.q0; g.n = s.n; g.kv = s.kv; g.begin = it.begin; g.end = it.end;
                            g.i0 = (int)off;
                            const long long left = my1 - at, rest = it.tiles - off;
                            g.n_iter = (int)(rest < left ? rest : left);
                            const bool whole = g.i0 == 0 && g.n_iter == it.tiles;
                            g.slot = whole ? -1 : (int)blockIdx.x * 2 + (n_seg > 0 ? 1 : 0);
                            if (g.i0 == 0 && !whole) {       // it goes on in the next CTAs: this one names it for the join
                                const long long item0 = at;
                                meta.parts = (int)((item0 + it.tiles - 1) / share - item0 / share) + 1;
                                meta.slot = g.slot; meta.b = b; meta.h = h; meta.row0 = row0; meta.n_rows = n_rows; meta.q0 = s.q0;
                            }
                            const int st = n_seg % kSegStages;
                            if (n_seg >= kSegStages && !mbar_wait(bar(SEGEMPTY + st), ((n_seg / kSegStages) - 1) & 1, abort_flag)) { ok = false; break; }
                            *reinterpret_cast<Segment*>(smem + C::kOffSeg + st * 64) = g;
                            mbar_arrive(bar(SEGFULL + st));
                            ++n_seg;
                            at += g.n_iter;
                            off = 0;
                        }
                    }
                    base += per_head * a.p.H;
                }
                if (ok) {
                    const int st = n_seg % kSegStages;
                    if (n_seg < kSegStages || mbar_wait(bar(SEGEMPTY + st), ((n_seg / kSegStages) - 1) & 1, abort_flag)) {
                        reinterpret_cast<Segment*>(smem + C::kOffSeg + st * 64)->n_iter = 0;
                        mbar_arrive(bar(SEGFULL + st));
                    }
                }
                a.meta[blockIdx.x] = meta;
            }
        } else if (work && warp < kPlanWarp) {
            // ================= MMA issuers =================
            const int g = warp - kMmaWarp;
            uint32_t elected;
            asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(elected));
            const bool leader = elected != 0;
            auto wait_w = [&](uint32_t bb, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bb, parity, abort_flag)) != 0; };
            constexpr uint32_t idesc_qk = instr_desc(0, 0, 0, kBN), idesc_pv = instr_desc(0, 0, 1 /* V is MN-major */, D);
            const uint32_t desc_hi = (uint32_t)(smem_desc(0) >> 32);
            // K-major: the leading offset is not used; MN-major: 64 channels are one swizzle atom, the next 64 lie 16 KiB on
            auto lo_of = [](uint32_t addr, uint32_t lead) { return ((addr >> 4) & 0x3FFFu) | ((lead >> 4) << 16); };
            auto desc = [&](uint32_t lo) { return ((uint64_t)desc_hi << 32) | lo; };
            const uint32_t q_lo = lo_of(sbase + C::kOffQ + g * C::kTile, 16), k_lo0 = lo_of(sbase + C::kOffK, 16), v_lo0 = lo_of(sbase + C::kOffV, 16384);
            const uint32_t d_s = tmem + (uint32_t)g * 128u, d_o = tmem + C::kColO + (uint32_t)(g * D);
            const uint32_t a_p = C::kOwnP ? tmem + C::kColP + (uint32_t)g * 64u : d_s;
            int nk = 0, nv = 0, s_qk = 0, s_pv = 0, n_seg = 0;
            bool ok = true;
            for (; ok; ++n_seg) {
                const int sst = n_seg % kSegStages;
                if (!wait_w(bar(SEGFULL + sst), (n_seg / kSegStages) & 1)) break;
                const Segment sg = *reinterpret_cast<const Segment*>(smem + C::kOffSeg + sst * 64);
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(SEGEMPTY + sst));
                if (sg.n_iter == 0) break;
                PagedSeq s; s.q0 = sg.q0; s.n = sg.n; s.kv = sg.kv; s.ok = true;
                const int r0 = sg.row0 + 128 * g;
                int lo = 0, hi = 0;                          // tiles of the item that this row tile takes part in
                if (r0 < sg.n_rows) {
                    const Item mine = item_keys(a, s, r0, min(128, sg.n_rows - r0));
                    lo = (mine.begin - sg.begin) / kBN;
                    hi = (mine.end - sg.begin + kBN - 1) / kBN;
                }
                if (!wait_w(bar(QREADY + g), n_seg & 1)) break;
                auto issue_qk = [&](int i) {
                    const int st = nk % ST;
                    if (!wait_w(bar(KFULL + st), (nk / ST) & 1)) return false;
                    if (i >= lo && i < hi) {
                        if (C::kOwnP && s_qk > 0 && !wait_w(bar(SEMPTY + g), (s_qk - 1) & 1)) return false;
                        tc_fence_after();
                        const uint32_t kl = k_lo0 + (uint32_t)st * (C::kTile >> 4);
                        if (leader) {
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk) {
                                const uint32_t step = (uint32_t)((kk / 4) * (16384 >> 4) + 2 * (kk % 4));
                                tc_mma_f16(d_s, desc(q_lo + step), desc(kl + step), idesc_qk, kk > 0 ? 1u : 0u);
                            }
                            tc_commit(bar(SFULL + g));
                        }
                        ++s_qk;
                    }
                    if (leader) tc_commit(bar(KEMPTY + st));
                    ++nk;
                    __syncwarp();
                    return true;
                };
                auto issue_pv = [&](int i, bool first) {
                    const int st = nv % ST;
                    const bool on = i >= lo && i < hi;
                    if (on && !wait_w(bar(PFULL + g), s_pv & 1)) return false;
                    if (!wait_w(bar(VFULL + st), (nv / ST) & 1)) return false;
                    if (on) {
                        tc_fence_after();
                        const uint32_t vl = v_lo0 + (uint32_t)st * (C::kTile >> 4);
                        if (leader) {
#pragma unroll
                            for (int kk = 0; kk < kBN / 16; ++kk)
                                tc_mma_f16_ta(d_o, a_p + 8u * (uint32_t)kk, desc(vl + kk * (2048 >> 4)), idesc_pv, (!first || kk > 0) ? 1u : 0u);
                            tc_commit(bar(PVDONE + g));
                        }
                        ++s_pv;
                    }
                    if (leader) tc_commit(bar(VEMPTY + st));
                    ++nv;
                    __syncwarp();
                    return true;
                };
                const int i_end = sg.i0 + sg.n_iter, i_first = max(lo, sg.i0);
                ok = issue_qk(sg.i0);
                for (int i = sg.i0; ok && i < i_end; ++i) {
                    if (C::kOwnP) {                          // the next scores only need this tile's to have left TMEM
                        if (i + 1 < i_end) ok = issue_qk(i + 1);
                        if (ok) ok = issue_pv(i, i == i_first);
                    } else {                                 // the next scores land on this tile's weights: behind its PV
                        ok = issue_pv(i, i == i_first);
                        if (ok && i + 1 < i_end) ok = issue_qk(i + 1);
                    }
                }
            }
            // nothing of this warp is in flight when the CTA gives its tensor memory back, aborted or not
            if (leader) tc_commit(bar(DRAIN));
            __syncwarp();
            for (uint32_t it = 0; it < kSpinLimit && !mbar_try(bar(DRAIN), 0); ++it) {}
        }
    } else if (warp >= kConvWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
        if (work) {
            // ================= K (warps 8, 9) and V (10, 11) to FP16 =================
            constexpr int LR = D / 16, RI = 32 / LR, NI = 64 / RI;   // lanes of a row, rows of a load, loads of a tile's half
            const bool is_v = warp >= kConvWarp + 2;
            const int w64 = 64 * (warp & 1);                         // this warp's rows of the tile
            const int FULL = is_v ? VFULL : KFULL, EMPTY = is_v ? VEMPTY : KEMPTY;
            unsigned char* tiles = smem + (is_v ? C::kOffV : C::kOffK);
            const int8_t* src = is_v ? a.p.v : a.p.k;
            const int c16 = lane % LR;                               // 16 channels of a row
            int n_t = 0;
            bool ok = true;
            for (int n_seg = 0; ok; ++n_seg) {
                const int sst = n_seg % kSegStages;
                if (!__all_sync(0xffffffffu, mbar_wait(bar(SEGFULL + sst), (n_seg / kSegStages) & 1, abort_flag))) break;
                const Segment sg = *reinterpret_cast<const Segment*>(smem + C::kOffSeg + sst * 64);
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(SEGEMPTY + sst));
                if (sg.n_iter == 0) break;
                // Pages, eight tiles at a time and the next eight ahead: lane 4 i + j holds the page of keys 16 j ... of this
                // warp's half of tile i.
                auto pages_from = [&](int i) {
                    const int key = sg.begin + (sg.i0 + i + (lane >> 2)) * kBN + w64 + 16 * (lane & 3);
                    if (i + (lane >> 2) >= sg.n_iter || key >= sg.end) return -1;
                    const int page = paged_page(a.p, sg.b, key);
                    if (page < 0) report_batch(a.p.status, sg.b, true);
                    return page;
                };
                int pg = pages_from(0), pg_next = pages_from(8);
                uint4 buf[NI];
                float2 ks = make_float2(0.0f, 0.0f), vs = make_float2(0.0f, 0.0f);
                bool there = false;                                  // the two keys whose scales this thread holds
                auto load_tile = [&](int i) {                        // tile i of the segment; nothing beyond its last
                    if (i >= sg.n_iter) return;
                    if ((i & 7) == 0 && i > 0) { pg = pg_next; pg_next = pages_from(i + 8); }
                    const int key0 = sg.begin + (sg.i0 + i) * kBN + w64;
#pragma unroll
                    for (int u = 0; u < NI; ++u) {
                        const int r = RI * u + lane / LR;
                        const int page = __shfl_sync(0xffffffffu, pg, 4 * (i & 7) + (RI * u >> 4));
                        const size_t row = paged_row(a.p, page < 0 ? 0 : page, sg.h) + ((key0 + r) & ((1 << a.p.page_shift) - 1));
                        buf[u] = page >= 0 ? __ldg(reinterpret_cast<const uint4*>(src + row * D) + c16) : make_uint4(0, 0, 0, 0);
                    }
                    if (!is_v) {
                        const int page = __shfl_sync(0xffffffffu, pg, 4 * (i & 7) + (lane >> 3));
                        const int key = key0 + 2 * lane;
                        there = page >= 0;
                        const size_t row = paged_row(a.p, there ? page : 0, sg.h) + (key & ((1 << a.p.page_shift) - 1));
                        if (there) {
                            ks = __ldg(reinterpret_cast<const float2*>(a.p.ks + row));
                            vs = __ldg(reinterpret_cast<const float2*>(a.p.vs + row));
                        }
                    }
                };
                load_tile(0);
                for (int i = 0; ok && i < sg.n_iter; ++i, ++n_t) {
                    if (!is_v) {
                        const int sc = n_t % kScaleStages;
                        if (n_t >= kScaleStages && !__all_sync(0xffffffffu, mbar_wait(bar(SCEMPTY + sc), ((n_t / kScaleStages) - 1) & 1, abort_flag))) { ok = false; break; }
                        float* sa = reinterpret_cast<float*>(smem + C::kOffScale + sc * C::kScaleBytes);
                        const int key0 = sg.begin + (sg.i0 + i) * kBN + w64, j = w64 + 2 * lane;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const bool in = there && key0 + 2 * lane + e < sg.end;      // a key that is not there weighs 2^-inf
                            const float v = fmaxf(e ? vs.y : vs.x, kLeastScale);
                            sa[j + e] = in ? a.c * (e ? ks.y : ks.x) : 0.0f;
                            sa[kBN + j + e] = in ? __log2f(v) : -INFINITY;
                            sa[2 * kBN + j + e] = in ? __fdividef(1.0f, v) : 0.0f;
                        }
                        if (a.stride > 0) {                                               // landmark bits of the tile's keys
                            const uint32_t m0 = __ballot_sync(0xffffffffu, (key0 + lane) % a.stride == 0);
                            const uint32_t m1 = __ballot_sync(0xffffffffu, (key0 + 32 + lane) % a.stride == 0);
                            if (lane == 0) {
                                uint32_t* marks = reinterpret_cast<uint32_t*>(sa + 3 * kBN) + 2 * (warp & 1);
                                marks[0] = m0;
                                marks[1] = m1;
                            }
                            __syncwarp();
                        }
                        mbar_arrive(bar(SCFULL + sc));
                    }
                    const int st = n_t % ST;
                    if (n_t >= ST && !__all_sync(0xffffffffu, mbar_wait(bar(EMPTY + st), ((n_t / ST) - 1) & 1, abort_flag))) { ok = false; break; }
                    unsigned char* tile = tiles + st * C::kTile + (c16 >> 2) * 16384;
#pragma unroll
                    for (int u = 0; u < NI; ++u) {
                        const int r = w64 + RI * u + lane / LR;
                        const uint32_t w[4] = {buf[u].x ^ 0x80808080u, buf[u].y ^ 0x80808080u, buf[u].z ^ 0x80808080u, buf[u].w ^ 0x80808080u};
                        unsigned char* row = tile + r * 128;
                        const int ch = 2 * (c16 & 3);
                        *reinterpret_cast<uint4*>(row + ((ch ^ (r & 7)) << 4)) =
                            make_uint4(bytes_to_half2(w[0], 0x4140), bytes_to_half2(w[0], 0x4342), bytes_to_half2(w[1], 0x4140), bytes_to_half2(w[1], 0x4342));
                        *reinterpret_cast<uint4*>(row + (((ch + 1) ^ (r & 7)) << 4)) =
                            make_uint4(bytes_to_half2(w[2], 0x4140), bytes_to_half2(w[2], 0x4342), bytes_to_half2(w[3], 0x4140), bytes_to_half2(w[3], 0x4342));
                    }
                    load_tile(i + 1);
                    fence_async_smem();
                    mbar_arrive(bar(FULL + st));
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        if (work) {
            // ================= softmax: one thread per query row =================
            const int g = warp >> 2, r = (warp & 3) * 32 + lane;
            const uint32_t lane_addr = ((uint32_t)((warp & 3) * 32)) << 16;
            const uint32_t tmem_S = tmem + (uint32_t)g * 128u + lane_addr, tmem_O = tmem + C::kColO + (uint32_t)(g * D) + lane_addr;
            const uint32_t tmem_P = C::kOwnP ? tmem + C::kColP + (uint32_t)g * 64u + lane_addr : tmem_S;
            // the TMEM accesses below are the whole warp's: so are the verdicts of its waits
            auto wait_w = [&](uint32_t bb, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bb, parity, abort_flag)) != 0; };
            int n_t = 0, s_run = 0;                   // key tiles seen, score tiles of this row tile taken
            bool ok = true;
            for (int n_seg = 0; ok; ++n_seg) {
                const int sst = n_seg % kSegStages;
                if (!wait_w(bar(SEGFULL + sst), (n_seg / kSegStages) & 1)) break;
                const Segment sg = *reinterpret_cast<const Segment*>(smem + C::kOffSeg + sst * 64);
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(SEGEMPTY + sst));
                if (sg.n_iter == 0) break;
                PagedSeq s; s.q0 = sg.q0; s.n = sg.n; s.kv = sg.kv; s.ok = true;
                const int r0 = sg.row0 + 128 * g, row = r0 + r;
                const bool live = row < sg.n_rows;
                const int token = (live ? row : sg.row0) / a.G, head = sg.h * a.G + (live ? row : sg.row0) % a.G;
                const int pos = sg.kv - sg.n + token;
                int lo = 0, hi = 0, first = 0, last = 0;
                if (r0 < sg.n_rows) {
                    const int rows = min(128, sg.n_rows - r0);
                    const Item mine = item_keys(a, s, r0, rows);
                    lo = (mine.begin - sg.begin) / kBN;
                    hi = (mine.end - sg.begin + kBN - 1) / kBN;
                    first = sg.kv - sg.n + r0 / a.G;
                    last = sg.kv - sg.n + (r0 + rows - 1) / a.G;
                }
                const bool shun = shunyam_active(a.window, sg.kv);
                // the row into shared memory as FP16 times a power of two (its products so far are all done)
                float alpha;
                {
                    uint4 w[D / 8];
                    const uint16_t* src = static_cast<const uint16_t*>(a.q) + (long long)(sg.q0 + token) * a.q_row + (long long)head * a.q_head;
                    float top = 0.0f;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) w[i] = live ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0, 0, 0, 0);
                    auto wide = [&](uint32_t x) {
                        return a.is_f16 ? __half22float2(*reinterpret_cast<const __half2*>(&x)) : make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
                    };
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) { const float2 f = wide(ww[e]); top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y))); }
                    }
                    float mul;
                    row_power(top, mul, alpha);
                    unsigned char* dst = smem + C::kOffQ + g * C::kTile + r * 128;
#pragma unroll
                    for (int i = 0; i < D / 8; ++i) {
                        const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                        uint32_t h[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) { const float2 f = wide(ww[e]); h[e] = f32x2_to_16(f.x * mul, f.y * mul, true); }
                        *reinterpret_cast<uint4*>(dst + (i >> 3) * 16384 + (((i & 7) ^ (r & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                }
                fence_async_smem();
                mbar_arrive(bar(QREADY + g));

                float m_run = -INFINITY, l_run = 0.0f;
                int taken = 0;
                for (int i = sg.i0; ok && i < sg.i0 + sg.n_iter; ++i, ++n_t) {
                    const int sc = n_t % kScaleStages;
                    if (!wait_w(bar(SCFULL + sc), (n_t / kScaleStages) & 1)) { ok = false; break; }
                    if (i < lo || i >= hi) { mbar_arrive(bar(SCEMPTY + sc)); continue; }
                    const float* sa = reinterpret_cast<const float*>(smem + C::kOffScale + sc * C::kScaleBytes);
                    if (!wait_w(bar(SFULL + g), s_run & 1)) { ok = false; break; }
                    tc_fence_after();
                    float x[kBN];
                    tc_ld32(tmem_S, x);
                    tc_ld32(tmem_S + 32, x + 32);
                    tc_ld32(tmem_S + 64, x + 64);
                    tc_ld32(tmem_S + 96, x + 96);
                    tc_wait_ld();
                    if (C::kOwnP) {                   // the next scores may overwrite these columns
                        tc_fence_before();
                        mbar_arrive(bar(SEMPTY + g));
                    }
                    const float2 al2 = make_float2(alpha, alpha);
                    const float4* a4 = reinterpret_cast<const float4*>(sa);
                    const float4* b4 = reinterpret_cast<const float4*>(sa + kBN);
#pragma unroll
                    for (int j = 0; j < kBN / 4; ++j) {
                        const float4 ka = a4[j], kb = b4[j];
                        const float2 f0 = __fmul2_rn(make_float2(ka.x, ka.y), al2), f1 = __fmul2_rn(make_float2(ka.z, ka.w), al2);
                        const float2 y0 = __ffma2_rn(make_float2(x[4 * j], x[4 * j + 1]), f0, make_float2(kb.x, kb.y));
                        const float2 y1 = __ffma2_rn(make_float2(x[4 * j + 2], x[4 * j + 3]), f1, make_float2(kb.z, kb.w));
                        x[4 * j] = y0.x; x[4 * j + 1] = y0.y; x[4 * j + 2] = y1.x; x[4 * j + 3] = y1.y;
                    }
                    const int k0 = sg.begin + i * kBN;
                    if ((a.causal && k0 + kBN - 1 > first) || (shun && k0 < last - a.window) || (shun && k0 + kBN - 1 > first)) {
                        const uint32_t* marks = reinterpret_cast<const uint32_t*>(sa + 3 * kBN);
                        const int top = pos - k0, low = shun ? pos - a.window - k0 : -1;       // window columns [low, top]
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int hi_q = top - 32 * q, lo_q = low - 32 * q;
                            const uint32_t upto = hi_q < 0 ? 0u : hi_q >= 31 ? 0xffffffffu : (2u << hi_q) - 1u;
                            const uint32_t from = lo_q <= 0 ? 0xffffffffu : lo_q > 31 ? 0u : 0xffffffffu << lo_q;
                            uint32_t vis = (a.causal || shun) ? upto : 0xffffffffu;
                            if (shun) {
                                vis &= from;
                                if (a.stride > 0) vis |= marks[q] & (a.causal ? upto : 0xffffffffu);
                            }
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!(vis & (1u << j))) x[32 * q + j] = -INFINITY;
                        }
                    }
                    float mx;
                    {
                        float mc[8];
#pragma unroll
                        for (int q = 0; q < 8; ++q) mc[q] = fmaxf(x[2 * q], x[2 * q + 1]);
#pragma unroll
                        for (int j = 16; j < kBN; j += 16)
#pragma unroll
                            for (int q = 0; q < 8; ++q) mc[q] = fmaxf(fmaxf(mc[q], x[j + 2 * q]), x[j + 2 * q + 1]);
                        mx = fmaxf(fmaxf(fmaxf(mc[0], mc[1]), fmaxf(mc[2], mc[3])), fmaxf(fmaxf(mc[4], mc[5]), fmaxf(mc[6], mc[7])));
                    }
                    // the reference moves only when a weight would pass 2^8; the correction of O is warp-wide (TMEM access)
                    const bool want = mx > m_run + kMoveMax || (m_run == -INFINITY && mx > -INFINITY);
                    const bool any = __any_sync(0xffffffffu, want && taken > 0 && m_run > -INFINITY);
                    float m_new = want ? mx : m_run;
                    if (any && m_new < mx) m_new = mx;
                    bool pv_done = taken == 0 || !C::kOwnP;       // without columns of its own, P's S came behind the last PV
                    if (any) {
                        if (!pv_done && !wait_w(bar(PVDONE + g), (s_run - 1) & 1)) { ok = false; break; }
                        pv_done = true;
                        tc_fence_after();
                        const float f = m_run == -INFINITY ? 0.0f : ex2(m_run - m_new);
#pragma unroll
                        for (int hc = 0; hc < D / 16; ++hc) {
                            float o[16];
                            tc_ld16(tmem_O + 16 * hc, o);
                            tc_wait_ld();
                            uint32_t ow[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) ow[j] = __float_as_uint(m_run == -INFINITY ? 0.0f : o[j] * f);
                            tc_st8(tmem_O + 16 * hc, ow);
                            tc_st8(tmem_O + 16 * hc + 8, ow + 8);
                        }
                        tc_wait_st();
                        tc_fence_before();
                        l_run *= f;
                    }
                    m_run = m_new;
                    const float neg_m = m_run == -INFINITY ? 0.0f : -m_run;
                    const float2 nm2 = make_float2(neg_m, neg_m);
                    const float4* c4 = reinterpret_cast<const float4*>(sa + 2 * kBN);
                    float2 la = make_float2(0.0f, 0.0f), lb = make_float2(0.0f, 0.0f);
                    if (!pv_done) {                   // the last PV still reads P's columns until it is done
                        if (!wait_w(bar(PVDONE + g), (s_run - 1) & 1)) { ok = false; break; }
                        tc_fence_after();
                    }
#pragma unroll
                    for (int cb = 0; cb < kBN / 16; ++cb) {
                        uint32_t pk[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = 16 * cb + 4 * e;
                            const float2 t0 = __fadd2_rn(make_float2(x[j], x[j + 1]), nm2), t1 = __fadd2_rn(make_float2(x[j + 2], x[j + 3]), nm2);
                            const float2 p0 = make_float2(ex2(t0.x), ex2(t0.y)), p1 = make_float2(ex2(t1.x), ex2(t1.y));
                            const float4 ci = c4[j / 4];
                            la = __ffma2_rn(p0, make_float2(ci.x, ci.y), la);
                            lb = __ffma2_rn(p1, make_float2(ci.z, ci.w), lb);
                            pk[2 * e] = f32x2_to_16(p0.x, p0.y, true);
                            pk[2 * e + 1] = f32x2_to_16(p1.x, p1.y, true);
                        }
                        tc_st8(tmem_P + 8 * cb, pk);
                    }
                    mbar_arrive(bar(SCEMPTY + sc));
                    l_run += (la.x + la.y) + (lb.x + lb.y);
                    tc_wait_st();
                    tc_fence_before();
                    mbar_arrive(bar(PFULL + g));
                    ++s_run;
                    ++taken;
                }
                if (!ok) break;
                // ---- the segment's result: an output row, or a partial one ----
                if (taken > 0) {
                    if (!wait_w(bar(PVDONE + g), (s_run - 1) & 1)) break;
                    tc_fence_after();
                }
                if (m_run == -INFINITY && !(l_run == 0.0f)) m_run = 0.0f;      // scores that are all NaN: not an empty row
                const bool empty = taken == 0 || m_run == -INFINITY;
                const size_t rec = (size_t)(sg.slot < 0 ? 0 : sg.slot) * kChunkRows + 128 * g + r;
                if (sg.slot >= 0 && live) a.stat[rec] = make_float2(empty ? -INFINITY : m_run, l_run);
                const float inv = empty ? 0.0f : 1.0f / l_run;
#pragma unroll
                for (int hc = 0; hc < D / 16; ++hc) {
                    float o[16];
                    __syncwarp();
                    if (taken > 0) {                  // warp-uniform: the row tile took part
                        tc_ld16(tmem_O + 16 * hc, o);
                        tc_wait_ld();
                    }
                    if (!live) continue;
#pragma unroll
                    for (int j = 0; j < 16; ++j) o[j] = empty ? 0.0f : o[j];
                    if (sg.slot >= 0) {
                        float4* dst = reinterpret_cast<float4*>(a.part + rec * D + 16 * hc);
#pragma unroll
                        for (int j = 0; j < 4; ++j) dst[j] = make_float4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                    } else {
                        uint32_t w[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = f32x2_to_16(o[2 * j] * inv, o[2 * j + 1] * inv, a.is_f16 != 0);
                        uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + (long long)(sg.q0 + token) * a.o_row + (long long)head * a.o_head + 16 * hc);
                        dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
                        dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
                tc_fence_before();
            }
        }
    }

    // ---- teardown: every role comes here, aborted or not ----
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && tid == 0) {
        const int f = *abort_flag;
        atomicExch(a.p.status, (f & ~0xffff) | ((f - (int)(bar0 & 0xffffu)) & 0xffff));
    }
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// Joins the items that were cut: CTA (c, y) takes rows [32 y, 32 y + 32) of the item that begins in CTA c of the chunk
// kernel.  A warp per row; the parts follow one another in the order of the keys.
template <int D>
__global__ void __launch_bounds__(256)
paged_join_kernel(const __grid_constant__ ChunkArgs a) {
    constexpr int V = D / 32;
    grid_wait_for_earlier();
    const JoinMeta meta = a.meta[blockIdx.x];
    if (meta.parts <= 1 || meta.parts > (int)(gridDim.x - blockIdx.x)) return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int r = kJoinRows * blockIdx.y + warp; r < kJoinRows * ((int)blockIdx.y + 1); r += 8) {
        const int row = meta.row0 + r;
        if (row >= meta.n_rows) return;
        auto rec = [&](int k) { return (size_t)(k == 0 ? meta.slot : 2 * ((int)blockIdx.x + k)) * kChunkRows + r; };
        float top = -INFINITY;
        for (int k = lane; k < meta.parts; k += 32) top = fmaxf(top, a.stat[rec(k)].x);
        top = warp_max(top);
        float sum = 0.0f, o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.0f;
#pragma unroll 4
        for (int k = 0; k < meta.parts; ++k) {
            const float2 st = a.stat[rec(k)];
            const float* p = a.part + rec(k) * D + V * lane;
            float v[V];
            if (V == 2) { const float2 t = *reinterpret_cast<const float2*>(p); v[0] = t.x; v[1] = t.y; }
            else { const float4 t = *reinterpret_cast<const float4*>(p); v[0] = t.x; v[1] = t.y; v[V - 2] = t.z; v[V - 1] = t.w; }
            const float f = st.x == -INFINITY ? 0.0f : ex2(st.x - top);
            sum = fmaf(st.y, f, sum);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = fmaf(v[i], f, o[i]);
        }
        const float inv = top == -INFINITY ? 0.0f : 1.0f / sum;
        uint16_t* dst = static_cast<uint16_t*>(a.o) + (long long)(meta.q0 + row / a.G) * a.o_row +
                        (long long)(meta.h * a.G + row % a.G) * a.o_head + V * lane;
#pragma unroll
        for (int i = 0; i < V; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = f32x2_to_16(o[i] * inv, o[i + 1] * inv, a.is_f16 != 0);
    }
}

template <int D>
int launch_chunk(logos_ctx* ctx, const ChunkArgs& a) {
    auto* fn = paged_chunk_kernel<D>;
    if (int rc = ensure_smem_limit(ctx, fn, Shape<D>::kSmem)) return rc;
    fn<<<ctx->sm_count, kChunkThreads, Shape<D>::kSmem, ctx->stream>>>(a);
    LOGOS_LAUNCH_CHECK(ctx, "paged_chunk_kernel");
    LOGOS_CUDA_TRY(ctx, launch_overlapped(paged_join_kernel<D>, dim3(ctx->sm_count, kChunkRows / kJoinRows), dim3(256), 0, ctx->stream, a));
    return LOGOS_OK;
}

struct ChunkLayout { size_t meta, stat, part, total; };
ChunkLayout chunk_layout(const logos_ctx* ctx, int DH) {
    ChunkLayout l;
    const size_t n = (size_t)ctx->sm_count;
    l.meta = kWorkspaceCounterBytes;
    l.stat = (l.meta + n * sizeof(JoinMeta) + 255) & ~(size_t)255;
    l.part = (l.stat + n * 2 * kChunkRows * sizeof(float2) + 255) & ~(size_t)255;
    l.total = l.part + n * 2 * kChunkRows * (size_t)DH * sizeof(float);
    return l;
}

}  // namespace

size_t paged_chunk_workspace_bytes(const logos_ctx* ctx, int DH) { return chunk_layout(ctx, DH).total; }

int paged_chunk(logos_ctx* ctx, const PagedArgs& p, int DH, const void* Q, void* O, const logos_row_strides& q,
                const logos_row_strides& o, int G, bool f16, const logos_attn_params* prm, int min_rows) {
    const ChunkLayout l = chunk_layout(ctx, DH);
    char* ws = static_cast<char*>(ctx->workspace);
    ChunkArgs a;
    a.p = p;
    a.q = Q; a.o = O;
    a.q_row = q.row; a.q_head = q.head; a.o_row = o.row; a.o_head = o.head;
    a.c = prm->scale * 1.4426950408889634f;
    a.G = G; a.is_f16 = f16;
    a.causal = prm->causal != 0; a.window = prm->window; a.stride = prm->stride;
    a.min_rows = min_rows;
    a.meta = reinterpret_cast<JoinMeta*>(ws + l.meta);
    a.stat = reinterpret_cast<float2*>(ws + l.stat);
    a.part = reinterpret_cast<float*>(ws + l.part);
    return DH == 64 ? launch_chunk<64>(ctx, a) : launch_chunk<128>(ctx, a);
}

}  // namespace logos
