// paged_chunk.cu -- attention of chunks of new tokens over the paged INT8 cache on the 5th-generation tensor cores: the
// sequences of a logos_paged_attention call that have many query rows per key/value head.
//
// The mathematics is that of paged_attn.cu: x_j = (q . k8_j) (scale log2(e) ks_j) + log2(vs_j), weights 2^(x_j - m) in
// FP16 against plain integers, l = sum p_j / vs_j.  A key is three fp32 numbers then, (a, b, 1/vs), which travel
// beside its bytes through shared memory.
//
// What bounds it: per 256 rows x 128 keys the exponentials (16 a clock and SM: 2048 clocks) and the products
// (M128 N128 K16 in 67 clocks, N64 in 57 to 63: 1500 clocks at DH 64, 2150 at DH 128); the cache itself is read once
// per 256 rows and comes from L2 after the first.  Measured it is the threads: some 13,400 instructions of a warp per
// 256 x 128 scores at DH 128, issued in 0.45 of a scheduler's clocks; the rest are waits for tensor memory that 16 softmax
// warps, all that the registers allow, do not cover.  2048 tokens over 16,384, 32 heads over 8, DH 128: 756 us =
// 680 TFLOP/s (0.42 of a plain product), 14 us more for the join.  Hence:
//  - 16 softmax warps of 16 rows, each thread 32 keys of two rows through 16x256-bit TMEM loads: the three numbers of a key
//    then cost a quarter of the shared-memory reads that one thread per row makes (a broadcast takes its 128 bytes a
//    clock like any other read): 1162 -> 1075 us;
//  - no maximum before the exponentials: a row's reference is the last tile's, and only a weight above 2^kMoveMax makes
//    the warp take the tile again with a new one: 1075 -> 963;
//  - the softmax loop without a spill (200 KB of shared memory leave local memory little L1): 920 -> 830;
//  - pages looked up per tile, rows fetched a tile ahead, everything on warps of its own: 830 -> 763.
//
// A CTA (896 threads, one per SM) holds two 128-row tiles of one (sequence, head) -- row r is token r / G, query head
// r % G of the group, so grouped heads share every K and V tile -- and walks over key tiles of 128.  Roles:
//   warps 0-7 / 8-15  softmax of tile 0 / 1, 16 rows a warp
//   warps 16-19 / 20-23 K / V: pages -> shared memory, asynchronously -> 16 bits -> 128B-swizzled tiles in shared memory
//   warps 24,25       MMA issuers, one per tile: S = Q K^T from shared memory, O += P V with P read from TMEM
//   warp 26           the schedule
// TMEM (512 columns), DH 64: S 2 x 128, O 2 x 64, P 2 x 64, so the next scores are computed under this tile's
// exponentials.  DH 128: S 2 x 128, O 2 x 128; P lies on the second half of its own S, the next scores follow this
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

constexpr int kChunkThreads = 896;
constexpr int kChunkRows = 256;              // query rows of an item
constexpr int kBN = 128;                     // keys of a tile
constexpr int kConvWarp = 16, kMmaWarp = 24, kPlanWarp = 26;
constexpr int kRegsSoftmax = 88, kRegsConvert = 48, kRegsRest = 56;      // the launch gives every thread 72
static_assert(512 * kRegsSoftmax + 256 * kRegsConvert + 128 * kRegsRest <= kChunkThreads * 72 && kChunkThreads * 72 <= 65536, "registers");
constexpr int kScaleStages = 4, kSegStages = 4;
constexpr int kSegReaders = kPlanWarp;       // warps 0 ... 25 read every segment
constexpr int kItemCost = 4;                  // what an item costs beside its tiles (queries in, pipeline filled, rows out), in tiles
constexpr float kLeastFactor = 1e-37f;
constexpr float kNoReference = -1e30f;       // reference of a row that has seen no key: any visible key lies above it
constexpr int kJoinRows = 8;                 // rows a CTA of the join takes, a warp each

// One poll of a barrier, asleep for up to 20 us; a waiting warp that polls by itself takes issue slots from the working ones.
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(20000) : "memory");
    return ok != 0;
}
// Bounded wait of a whole warp with one verdict: false when the CTA is aborting (this wait or another one ran out).
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    for (uint32_t it = 0; it < (1u << 16); ++it) {
        if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
        if ((it & 15u) == 15u && __any_sync(0xffffffffu, *abort_flag != 0)) return false;
    }
    // as mbar_wait records it: the barrier's address and the thread
    atomicCAS(const_cast<int*>(abort_flag), 0, (int)((bar & 0xffffu) | (threadIdx.x << 16)) | 0x40000000);
    return false;
}

// TMEM accesses of 16 lanes x 256 (128) bits: thread t of the warp holds lanes t / 4 and t / 4 + 8.
// 256 bits: registers 4 b ... 4 b + 3 are columns 8 b + 2 (t % 4), + 1 of the first lane, then of the second; 128 bits:
// registers 2 w, 2 w + 1 are column 4 w + t % 4 of the two lanes.
__device__ __forceinline__ void tc_ld_16x256_x4(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_st_16x256_x4(uint32_t taddr, const float* v) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x4.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_ld_16x128_x4(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.16x128b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tc_st_16x128_x4(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
constexpr int kBW = 32;                       // keys a softmax warp works on at once
__device__ __forceinline__ void ld_scores(uint32_t taddr, float (&x)[kBW / 2]) {
#pragma unroll
    for (int i = 0; i < kBW / 32; ++i) tc_ld_16x256_x4(taddr + 32 * i, x + 16 * i);
}

template <int D> struct Shape {
    static constexpr int kTile = kBN * D * 2;                 // one FP16 tile of 128 rows
    static constexpr int kStages = D == 64 ? 3 : 2;           // K tiles
    static constexpr int kStagesV = D == 64 ? 3 : 1;          // V tiles: wanted a softmax later, and the space goes to the fetches
    static constexpr bool kOwnP = D == 64;                    // P has TMEM columns of its own
    static constexpr int kOffQ = 0, kOffK = kOffQ + 2 * kTile, kOffV = kOffK + kStages * kTile;
    static constexpr int kOffScale = kOffV + kStagesV * kTile; // kScaleStages x {a, b, 1/vs: 128 floats each, 4 words of landmarks}
    static constexpr int kScaleBytes = 3 * kBN * 4 + 16;
    static constexpr int kRaw = 32 * D;                       // bytes of a converting warp's share of a tile: the fetches run one tile ahead
    static constexpr int kOffRaw = kOffScale + kScaleStages * kScaleBytes;
    static constexpr int kOffSeg = kOffRaw + 8 * kRaw;
    static constexpr int kOffBar = kOffSeg + kSegStages * 64;
    static constexpr int kNumBars = 2 * (kStages + kStagesV) + 2 * kScaleStages + 2 * kSegStages + 5 * 2 + 1;
    static constexpr int kOffScan = kOffBar + kNumBars * 8;
    static constexpr int kSmem = kOffScan + 8 * (kChunkThreads / 32) + 1024;       // + alignment slack
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
// length of one head of a sequence on the line of work: its items' key tiles and kItemCost for each item; 0 when the
// sequence is not this kernel's
__device__ __forceinline__ long long seq_tiles(const ChunkArgs& a, int b) {
    const PagedSeq s = paged_seq(a.p, b);
    if (!s.ok || (long long)s.n * a.G <= a.min_rows) return 0;
    long long sum = 0;
    for (int r = 0; r < s.n * a.G; r += kChunkRows) sum += item_keys(a, s, r, min(kChunkRows, s.n * a.G - r)).tiles + kItemCost;
    return sum;
}

template <int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
paged_chunk_kernel(const __grid_constant__ ChunkArgs a) {
    using C = Shape<D>;
    constexpr int ST = C::kStages, SV = C::kStagesV;
    enum Bar { KFULL = 0, KEMPTY = KFULL + ST, VFULL = KEMPTY + ST, VEMPTY = VFULL + SV, SCFULL = VEMPTY + SV,
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
        for (int i = 0; i < ST; ++i) { mbar_init(bar(KFULL + i), 4); mbar_init(bar(KEMPTY + i), 2); }
        for (int i = 0; i < SV; ++i) { mbar_init(bar(VFULL + i), 4); mbar_init(bar(VEMPTY + i), 2); }
        for (int i = 0; i < kScaleStages; ++i) { mbar_init(bar(SCFULL + i), 4); mbar_init(bar(SCEMPTY + i), 16); }
        for (int i = 0; i < kSegStages; ++i) { mbar_init(bar(SEGFULL + i), 1); mbar_init(bar(SEGEMPTY + i), kSegReaders); }
        for (int g = 0; g < 2; ++g) {
            mbar_init(bar(SFULL + g), 1); mbar_init(bar(SEMPTY + g), 8); mbar_init(bar(PFULL + g), 8);
            mbar_init(bar(PVDONE + g), 1); mbar_init(bar(QREADY + g), 8);
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
            if (share < kItemCost + 2) share = kItemCost + 2;   // a shorter run costs more in joining than it saves
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
                            const int span = it.tiles + kItemCost;      // the item's stretch of the line: its cost, then its tiles
                            if (off >= span) { off -= span; continue; }
                            const long long left = my1 - at, rest = span - off;
                            const long long take = rest < left ? rest : left;
                            const int t0 = off > kItemCost ? (int)off - kItemCost : 0, t1 = (int)(off + take) - kItemCost;
                            const long long item0 = at - off;
                            at += take;
                            off = 0;
                            if (t1 <= t0) continue;                       // the share ends before the item's first tile
                            Segment g;
                            g.b = b; g.h = h; g.row0 = row0; g.n_rows = n_rows;
                            g.q0 = s.q0; g.n = s.n; g.kv = s.kv; g.begin = it.begin; g.end = it.end;
                            g.i0 = t0;
                            g.n_iter = t1 - t0;
                            const bool whole = t0 == 0 && t1 == it.tiles;
                            g.slot = whole ? -1 : (int)blockIdx.x * 2 + (n_seg > 0 ? 1 : 0);
                            if (t0 == 0 && !whole) {         // it goes on in the next CTAs: this one names it for the join
                                meta.parts = (int)((item0 + span - 1) / share - (item0 + kItemCost) / share) + 1;
                                meta.slot = g.slot; meta.b = b; meta.h = h; meta.row0 = row0; meta.n_rows = n_rows; meta.q0 = s.q0;
                            }
                            const int st = n_seg % kSegStages;
                            if (n_seg >= kSegStages && !mbar_wait(bar(SEGEMPTY + st), ((n_seg / kSegStages) - 1) & 1, abort_flag)) { ok = false; break; }
                            *reinterpret_cast<Segment*>(smem + C::kOffSeg + st * 64) = g;
                            mbar_arrive(bar(SEGFULL + st));
                            ++n_seg;
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
            auto wait_w = [&](uint32_t bb, uint32_t parity) { return wait_warp(bb, parity, abort_flag); };
            const uint32_t idesc_qk = instr_desc(a.is_f16 ? 0 : 1, a.is_f16 ? 0 : 1, 0, kBN);
            constexpr uint32_t idesc_pv = instr_desc(0, 0, 1 /* V is MN-major */, D);
            const uint32_t desc_hi = (uint32_t)(smem_desc(0) >> 32);
            // K-major: the leading offset is not used; MN-major: 64 channels are one swizzle atom, the next 64 lie 16 KiB on
            auto lo_of = [](uint32_t addr, uint32_t lead) { return ((addr >> 4) & 0x3FFFu) | ((lead >> 4) << 16); };
            auto desc = [&](uint32_t lo) { return ((uint64_t)desc_hi << 32) | lo; };
            const uint32_t q_lo = lo_of(sbase + C::kOffQ + g * C::kTile, 16), k_lo0 = lo_of(sbase + C::kOffK, 16), v_lo0 = lo_of(sbase + C::kOffV, 16384);
            const uint32_t d_s = tmem + (uint32_t)g * 128u, d_o = tmem + C::kColO + (uint32_t)(g * D);
            const uint32_t a_p = C::kOwnP ? tmem + C::kColP + (uint32_t)g * 64u : d_s + 64u;
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
                    const int st = nv % SV;
                    const bool on = i >= lo && i < hi;
                    if (on && !wait_w(bar(PFULL + g), s_pv & 1)) return false;
                    if (!wait_w(bar(VFULL + st), (nv / SV) & 1)) return false;
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
            for (uint32_t it = 0; it < (1u << 16) && !mbar_try(bar(DRAIN), 0); ++it) {}
        }
    } else if (warp >= kConvWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
        if (work) {
            // ================= K (warps 16-19) and V (20-23) to 16 bits =================
            // A warp takes 32 rows of every tile as pieces of 1 KiB (16 or 8 keys), which never cross a page.  A piece's bytes wait
            // in shared memory, each where the thread that fetched it will read it (no barrier); a piece that has been converted
            // makes room for the same piece of the next tile.
            constexpr int LR = D / 16, RI = 32 / LR;                 // lanes of a row, rows of a load
            constexpr int PR = 1024 / D, NP = PR / RI, PPT = 32 / PR;   // rows and loads of a piece, pieces of the warp's share of a tile
            const bool is_v = warp >= kConvWarp + 4;
            const int part = warp & 3, w32 = 32 * part;              // this warp's rows of the tile
            const int FULL = is_v ? VFULL : KFULL, EMPTY = is_v ? VEMPTY : KEMPTY;
            unsigned char* tiles = smem + (is_v ? C::kOffV : C::kOffK);
            const int8_t* src = is_v ? a.p.v : a.p.k;
            auto wait_w = [&](uint32_t bb, uint32_t parity) { return wait_warp(bb, parity, abort_flag); };
            auto arrive_w = [&](uint32_t bb) { __syncwarp(); if (lane == 0) mbar_arrive(bb); };
            const int c16 = lane % LR, r16 = lane / LR;              // 16 channels, first row of a piece
            unsigned char* raw = smem + C::kOffRaw + (warp - kConvWarp) * C::kRaw + lane * 16;
            const uint32_t raw_addr = smem_u32(raw);
            const int page_mask = (1 << a.p.page_shift) - 1;
            const int ch = 2 * (c16 & 3);
            const bool bf16 = !is_v && !a.is_f16;                    // K in the type of the queries, V in that of the weights
            int n_t = 0;
            bool ok = true;
            for (int n_seg = 0; ok; ++n_seg) {
                const int sst = n_seg % kSegStages;
                if (!wait_w(bar(SEGFULL + sst), (n_seg / kSegStages) & 1)) break;
                const Segment* seg = reinterpret_cast<const Segment*>(smem + C::kOffSeg + sst * 64);
                const int sb = seg->b, sh = seg->h, n_iter = seg->n_iter, key_first = seg->begin + seg->i0 * kBN + w32, end = seg->end;
                arrive_w(bar(SEGEMPTY + sst));
                if (n_iter == 0) break;
                // Table entries, 16 tiles at a time and the next 16 ahead: lane 2 i + j holds that of keys 16 j ... of this
                // warp's quarter of tile i (0 where there is no key).
                auto entries_from = [&](int i) {
                    const int key = key_first + (i + (lane >> 1)) * kBN + 16 * (lane & 1);
                    if (i + (lane >> 1) >= n_iter || key >= end) return 0;
                    return a.p.table[(size_t)sb * a.p.max_pages + (key >> a.p.page_shift)];
                };
                auto checked = [&](int page) {                       // -1: outside the cache
                    if ((unsigned)page < (unsigned)a.p.pages) return page;
                    report_batch(a.p.status, sb, true);
                    return -1;
                };
                int pg = checked(entries_from(0)), pg_next = entries_from(16);
                float ks = 0.0f, vs = 0.0f;                          // the scales of this thread's key of the tile
                bool there = false;
                // Where the thread's first bytes of the two 16-key halves of its share of tile i lie.  A page that is not there is read
                // as page 0: its keys weigh nothing, and no load waits for a test.
                const int8_t* at[2];
                auto locate = [&](int i) {
                    if ((i & 15) == 0 && i > 0) { pg = checked(pg_next); pg_next = entries_from(i + 16); }
                    const int key = key_first + i * kBN;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int page = max(__shfl_sync(0xffffffffu, pg, 2 * (i & 15) + j), 0);
                        at[j] = src + (size_t)(paged_row(a.p, page, sh) + ((key + 16 * j) & page_mask) + r16) * D + 16 * c16;
                    }
                };
                auto fetch = [&](int blk) {                          // piece blk of the located tile
#pragma unroll
                    for (int u = 0; u < NP; ++u)
                        cp_async16(raw_addr + blk * 1024 + u * 512, at[PR * blk >> 4] + ((PR * blk & 15) + u * RI) * D);
                };
                auto fetch_scales = [&](int i) {
                    if (is_v || i >= n_iter) return;
                    const int key = key_first + i * kBN + lane;
                    const int page = __shfl_sync(0xffffffffu, pg, 2 * (i & 15) + (lane >> 4));
                    there = (unsigned)page < (unsigned)a.p.pages && key < end;
                    const uint32_t row = paged_row(a.p, there ? page : 0, sh) + (key & page_mask);
                    ks = __ldg(a.p.ks + row);
                    vs = __ldg(a.p.vs + row);
                };
                locate(0);
                fetch_scales(0);
#pragma unroll
                for (int blk = 0; blk < PPT; ++blk) {
                    fetch(blk);
                    cp_async_commit();
                }
                for (int i = 0; ok && i < n_iter; ++i, ++n_t) {
                    if (!is_v) {
                        const int sc = n_t % kScaleStages;
                        if (n_t >= kScaleStages && !wait_w(bar(SCEMPTY + sc), ((n_t / kScaleStages) - 1) & 1)) { ok = false; break; }
                        float* sa = reinterpret_cast<float*>(smem + C::kOffScale + sc * C::kScaleBytes) + w32;
                        const float v = fmaxf(vs, kLeastScale);
                        // A key that is not there weighs 2^-inf.  The factor of a score is never 0, so that the -inf of a masked score
                        // stays one.
                        sa[lane] = there ? fmaxf(a.c * ks, kLeastFactor) : kLeastFactor;
                        sa[kBN + lane] = there ? fminf(__log2f(v), 3e38f) : -INFINITY;   // finite: a masked score keeps its -inf beside an infinite scale
                        sa[2 * kBN + lane] = there ? __fdividef(1.0f, v) : 0.0f;
                        if (a.stride > 0) {                                               // landmark bits of the warp's keys
                            const uint32_t m = __ballot_sync(0xffffffffu, (key_first + i * kBN + lane) % a.stride == 0);
                            if (lane == 0) reinterpret_cast<uint32_t*>(sa - w32 + 3 * kBN)[part] = m;
                        }
                        arrive_w(bar(SCFULL + sc));
                    }
                    if (i + 1 < n_iter) {
                        locate(i + 1);
                        fetch_scales(i + 1);
                    }
                    const int depth = is_v ? SV : ST, st = n_t % depth;
                    if (n_t >= depth && !wait_w(bar(EMPTY + st), ((n_t / depth) - 1) & 1)) { ok = false; break; }
                    unsigned char* tile = tiles + st * C::kTile + (c16 >> 2) * 16384 + (w32 + r16) * 128;
#pragma unroll
                    for (int blk = 0; blk < PPT; ++blk) {
                        cp_async_wait<PPT - 1>();
                        const unsigned char* in = raw + blk * 1024;
                        uint4 xs[NP];
#pragma unroll
                        for (int u = 0; u < NP; ++u) xs[u] = *reinterpret_cast<const uint4*>(in + u * 512);
#pragma unroll
                        for (int u = 0; u < NP; ++u) {
                            const uint4 x = xs[u];
                            unsigned char* row = tile + (PR * blk + RI * u) * 128;
                            const int sw = (RI * u + r16) & 7;        // PR blk and w32 are multiples of 8
                            uint4 y0, y1;
                            if (bf16) {
                                y0 = make_uint4(bytes_to_bf162(x.x, 0x4140), bytes_to_bf162(x.x, 0x4342), bytes_to_bf162(x.y, 0x4140), bytes_to_bf162(x.y, 0x4342));
                                y1 = make_uint4(bytes_to_bf162(x.z, 0x4140), bytes_to_bf162(x.z, 0x4342), bytes_to_bf162(x.w, 0x4140), bytes_to_bf162(x.w, 0x4342));
                            } else {
                                const uint32_t w[4] = {x.x ^ 0x80808080u, x.y ^ 0x80808080u, x.z ^ 0x80808080u, x.w ^ 0x80808080u};
                                y0 = make_uint4(bytes_to_half2(w[0], 0x4140), bytes_to_half2(w[0], 0x4342), bytes_to_half2(w[1], 0x4140), bytes_to_half2(w[1], 0x4342));
                                y1 = make_uint4(bytes_to_half2(w[2], 0x4140), bytes_to_half2(w[2], 0x4342), bytes_to_half2(w[3], 0x4140), bytes_to_half2(w[3], 0x4342));
                            }
                            *reinterpret_cast<uint4*>(row + ((ch ^ sw) << 4)) = y0;
                            *reinterpret_cast<uint4*>(row + (((ch + 1) ^ sw) << 4)) = y1;
                        }
                        if (i + 1 < n_iter) fetch(blk);
                        cp_async_commit();
                    }
                    fence_async_smem();
                    arrive_w(bar(FULL + st));
                }
                cp_async_wait<0>();                                   // nothing of this segment is left in flight
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        if (work) {
            // ================= softmax: 16 query rows a warp =================
            // A thread holds a quarter of two rows: slot q is row 8 q + lane / 4 of the warp, columns 2 (lane % 4), + 1 of every
            // eight.  So it needs the three numbers of a quarter of the keys (shared memory returns 128 bytes a clock, broadcast
            // or not), and four warps share a scheduler.
            const int g = warp >> 3, quad = lane >> 2, col = 2 * (lane & 3);
            const int wr = 32 * (warp & 3) + 16 * ((warp >> 2) & 1);         // the warp's first row of the tile, and TMEM lane
            const uint32_t lane_addr = (uint32_t)wr << 16;
            const uint32_t tmem_S = tmem + (uint32_t)g * 128u + lane_addr, tmem_O = tmem + C::kColO + (uint32_t)(g * D) + lane_addr;
            const uint32_t tmem_P = C::kOwnP ? tmem + C::kColP + (uint32_t)g * 64u + lane_addr : tmem_S + 64u;
            // the TMEM accesses below are the whole warp's: so are the verdicts of its waits, and its arrivals
            auto wait_w = [&](uint32_t bb, uint32_t parity) { return wait_warp(bb, parity, abort_flag); };
            auto arrive_w = [&](uint32_t bb) { __syncwarp(); if (lane == 0) mbar_arrive(bb); };
            int n_t = 0, s_run = 0;                   // key tiles seen, score tiles of this row tile taken
            bool ok = true;
            // The warp's query rows of segment n into shared memory as they are, half a row a thread.  The products of the segment
            // before are all done when its last scores have come.
            auto segment = [&](int n) { return reinterpret_cast<const volatile Segment*>(smem + C::kOffSeg + (n % kSegStages) * 64); };
            auto load_q = [&](int n) {
                if (!wait_w(bar(SEGFULL + n % kSegStages), (n / kSegStages) & 1)) return false;
                const volatile Segment* seg = segment(n);
                if (seg->n_iter == 0) return true;
                const int r = wr + (lane >> 1), row0 = seg->row0, row = row0 + 128 * g + r;
                const bool live = row < seg->n_rows;
                const int token = (live ? row : row0) / a.G, head = seg->h * a.G + (live ? row : row0) % a.G;
                const uint16_t* src = static_cast<const uint16_t*>(a.q) + (long long)(seg->q0 + token) * a.q_row + (long long)head * a.q_head;
                unsigned char* dst = smem + C::kOffQ + g * C::kTile + r * 128;
                constexpr int N = D / 16;
                const int i0 = (lane & 1) * N;
                uint4 w[N];
#pragma unroll
                for (int i = 0; i < N; ++i) w[i] = live ? *reinterpret_cast<const uint4*>(src + 8 * (i0 + i)) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < N; ++i) *reinterpret_cast<uint4*>(dst + ((i0 + i) >> 3) * 16384 + ((((i0 + i) & 7) ^ (r & 7)) << 4)) = w[i];
                fence_async_smem();
                arrive_w(bar(QREADY + g));
                return true;
            };
            ok = load_q(0);
            for (int n_seg = 0; ok; ++n_seg) {
                // The segment stays where it is, and its slot this warp's, until its output is written: its fields are read when they
                // are wanted and hold no registers meanwhile.
                const volatile Segment* seg = segment(n_seg);
                if (seg->n_iter == 0) break;
                int lo = 0, hi = 0;                   // tiles of the item that this row tile takes part in
                bool rows_here = false;               // some of the warp's 16 rows are query rows
                int e_hi = 0x7fffffff, e_lo = -0x7fffffff;   // a tile whose first key lies outside [e_lo, e_hi] is masked in part
                {
                    const int n_rows = seg->n_rows, r0 = seg->row0 + 128 * g;
                    rows_here = r0 + wr < n_rows;
                    if (r0 < n_rows) {
                        PagedSeq s; s.q0 = seg->q0; s.n = seg->n; s.kv = seg->kv; s.ok = true;
                        const int rows = min(128, n_rows - r0), begin = seg->begin;
                        const Item mine = item_keys(a, s, r0, rows);
                        lo = (mine.begin - begin) / kBN;
                        hi = (mine.end - begin + kBN - 1) / kBN;
                        const bool shun = shunyam_active(a.window, s.kv);
                        if (a.causal || shun) e_hi = s.kv - s.n + r0 / a.G - (kBN - 1);
                        if (shun) e_lo = s.kv - s.n + (r0 + rows - 1) / a.G - a.window;
                    }
                }
                float2 nm[2], l_run[2];               // minus the row's reference, twice; its sum over even and odd keys
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    nm[q] = make_float2(-kNoReference, -kNoReference);
                    l_run[q] = make_float2(0.0f, 0.0f);
                }
                bool first = true;                    // no tile taken yet
                int i = seg->i0;
                const int i_end = i + seg->n_iter;
                int k0 = seg->begin + i * kBN;
                for (; ok && i < i_end; ++i, ++n_t, k0 += kBN) {
                    const int sc = n_t % kScaleStages;
                    if (!wait_w(bar(SCFULL + sc), (n_t / kScaleStages) & 1)) { ok = false; break; }
                    if (i < lo || i >= hi) { arrive_w(bar(SCEMPTY + sc)); continue; }
                    const float* sa = reinterpret_cast<const float*>(smem + C::kOffScale + sc * C::kScaleBytes) + col;
                    if (!wait_w(bar(SFULL + g), s_run & 1)) { ok = false; break; }
                    tc_fence_after();
                    if (!rows_here) {                 // rows behind the last one: what P holds for them reaches no output
                        arrive_w(bar(SCEMPTY + sc));
                        if (C::kOwnP) {
                            arrive_w(bar(SEMPTY + g));
                            // not before the weights of the tile before have been taken: the others may still be writing those,
                            // and this arrival would count for them
                            if (!first && !wait_w(bar(PVDONE + g), (s_run - 1) & 1)) { ok = false; break; }
                        }
                        arrive_w(bar(PFULL + g));
                        ++s_run;
                        first = false;
                        continue;
                    }
                    if (k0 > e_hi || k0 < e_lo) {
                        // Some rows do not see some of the keys: -inf on their scores, in tensor memory, before the loop below.
                        // (Inside it the test and the code would cost every tile registers and instruction fetches.)
                        const uint32_t* marks = reinterpret_cast<const uint32_t*>(sa - col + 3 * kBN);
                        const int pos0 = seg->kv - seg->n, row = seg->row0 + 128 * g + wr + quad;
                        const int p0 = pos0 + row / a.G - k0 - col, p1 = pos0 + (row + 8) / a.G - k0 - col;
                        const bool shun = shunyam_active(a.window, seg->kv), bounded = a.causal || shun;
#pragma unroll 1
                        for (int cb = 0; cb < kBN / 32; ++cb) {
                            float y[16];
                            tc_ld_16x256_x4(tmem_S + 32 * cb, y);
                            tc_wait_ld();
                            const uint32_t m = a.stride > 0 ? marks[cb] >> col : 0u;
#pragma unroll
                            for (int w = 0; w < 4; ++w)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int c = 32 * cb + 8 * w + e;
                                    const bool mark = shun && ((m >> (8 * w + e)) & 1u);
                                    const bool v0 = (!bounded || c <= p0) && (!shun || c >= p0 - a.window), v1 = (!bounded || c <= p1) && (!shun || c >= p1 - a.window);
                                    if (!(v0 || (mark && (!a.causal || c <= p0)))) y[4 * w + e] = -INFINITY;
                                    if (!(v1 || (mark && (!a.causal || c <= p1)))) y[4 * w + 2 + e] = -INFINITY;
                                }
                            tc_st_16x256_x4(tmem_S + 32 * cb, y);
                        }
                        tc_wait_st();
                    }
                    bool pv_done = first || !C::kOwnP;       // without columns of its own, P's S came behind the last PV
                    // Blocks of kBW keys, highest first (P may lie on the S of the blocks before).  Nothing in the loop waits for a
                    // maximum: a weight's exponent is taken against the row's reference, and only when one passes 2^15 -- or the
                    // row has no reference yet -- does the warp turn aside to move it.
#pragma unroll
                    for (int cb = kBN / kBW - 1; cb >= 0; --cb) {
                        const float* sk = sa + kBW * cb;
                        float z[kBW / 2];             // [4 (key / 8) + 2 slot + column]
                        ld_scores(tmem_S + kBW * cb, z);   // (four warps a scheduler cover the wait; a block ahead costs 16 registers)
                        tc_wait_ld();
#pragma unroll
                        for (int w = 0; w < kBW / 8; ++w) {
                            const float2 ka = *reinterpret_cast<const float2*>(sk + 8 * w), kb = *reinterpret_cast<const float2*>(sk + kBN + 8 * w);
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const int at = 4 * w + 2 * q;
                                const float2 t = __ffma2_rn(make_float2(z[at], z[at + 1]), ka, __fadd2_rn(kb, nm[q]));
                                z[at] = t.x;
                                z[at + 1] = t.y;
                            }
                        }
                        float t0 = fmaxf(z[0], z[1]), t1 = fmaxf(z[2], z[3]);
#pragma unroll
                        for (int j = 4; j < kBW / 2; j += 4) {
                            t0 = fmaxf(fmaxf(t0, z[j]), z[j + 1]);
                            t1 = fmaxf(fmaxf(t1, z[j + 2]), z[j + 3]);
                        }
                        if (__builtin_expect(__any_sync(0xffffffffu, fmaxf(t0, t1) > kMoveMax), 0)) {
                            // Move the references of the rows that outgrew theirs to the largest exponent of the block, and scale
                            // what was summed against the old ones: l, O, and the blocks of P that this tile already has.
                            ld_scores(tmem_S + kBW * cb, z);           // the scores again: a reference of -1e30 has swallowed them
                            tc_wait_ld();
                            float top[2] = {-INFINITY, -INFINITY}, f[2];
#pragma unroll
                            for (int w = 0; w < kBW / 8; ++w) {
                                const float2 ka = *reinterpret_cast<const float2*>(sk + 8 * w), kb = *reinterpret_cast<const float2*>(sk + kBN + 8 * w);
#pragma unroll
                                for (int q = 0; q < 2; ++q) {
                                    const int at = 4 * w + 2 * q;
                                    const float2 t = __ffma2_rn(make_float2(z[at], z[at + 1]), ka, kb);
                                    z[at] = t.x;
                                    z[at + 1] = t.y;
                                    top[q] = fmaxf(top[q], fmaxf(t.x, t.y));
                                }
                            }
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                top[q] = fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 1));
                                // a whole number: the scaling by 2^-whole below is exact, in FP16 too
                                top[q] = ceilf(fmaxf(top[q], __shfl_xor_sync(0xffffffffu, top[q], 2)));
                                const bool move = top[q] + nm[q].x > kMoveMax;
                                f[q] = !move ? 1.0f : nm[q].x == -kNoReference ? 0.0f : ex2(-nm[q].x - top[q]);
                                if (move) nm[q] = make_float2(-top[q], -top[q]);
#pragma unroll
                                for (int w = 0; w < kBW / 8; ++w) {
                                    z[4 * w + 2 * q] += nm[q].x;
                                    z[4 * w + 2 * q + 1] += nm[q].x;
                                }
                                l_run[q] = __fmul2_rn(l_run[q], make_float2(f[q], f[q]));
                            }
                            if (!first) {
                                if (!pv_done && !wait_w(bar(PVDONE + g), (s_run - 1) & 1)) { ok = false; break; }
                                pv_done = true;
                                tc_fence_after();
                                float o[16];
#pragma unroll 1
                                for (int hc = 0; hc < D / 32; ++hc) {
                                    tc_ld_16x256_x4(tmem_O + 32 * hc, o);
                                    tc_wait_ld();
#pragma unroll
                                    for (int j = 0; j < 16; ++j) o[j] *= f[(j >> 1) & 1];
                                    tc_st_16x256_x4(tmem_O + 32 * hc, o);
                                }
                            }
                            tc_wait_st();
#pragma unroll 1
                            for (int done = (kBW / 32) * (cb + 1); done < kBN / 32; ++done) {
                                uint32_t pw[8];
                                tc_ld_16x128_x4(tmem_P + 16 * done, pw);
                                tc_wait_ld();
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&pw[j]), __float2half2_rn(f[j & 1]));
                                    pw[j] = *reinterpret_cast<const uint32_t*>(&h);
                                }
                                tc_st_16x128_x4(tmem_P + 16 * done, pw);
                            }
                            tc_wait_st();
                            tc_fence_before();
                        }
                        if (C::kOwnP && cb == 0) {    // all scores have left: the next ones may overwrite these columns
                            tc_fence_before();
                            arrive_w(bar(SEMPTY + g));
                        }
                        if (!pv_done) {               // the last PV still reads P's columns until it is done
                            if (!wait_w(bar(PVDONE + g), (s_run - 1) & 1)) { ok = false; break; }
                            pv_done = true;
                            tc_fence_after();
                        }
#pragma unroll
                        for (int part = kBW / 32 - 1; part >= 0; --part) {
                            uint32_t pk[8];
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                const float2 ci = *reinterpret_cast<const float2*>(sk + 2 * kBN + 32 * part + 8 * w);
#pragma unroll
                                for (int q = 0; q < 2; ++q) {
                                    const int at = 16 * part + 4 * w + 2 * q;
                                    const float2 pw = make_float2(ex2(z[at]), ex2(z[at + 1]));
                                    l_run[q] = __ffma2_rn(pw, ci, l_run[q]);
                                    pk[2 * w + q] = f32x2_to_16(pw.x, pw.y, true);
                                }
                            }
                            tc_st_16x128_x4(tmem_P + (kBW / 2) * cb + 16 * part, pk);
                        }
                    }
                    if (!ok) break;
                    arrive_w(bar(SCEMPTY + sc));
                    tc_wait_st();
                    tc_fence_before();
                    arrive_w(bar(PFULL + g));
                    ++s_run;
                    first = false;
                }
                if (!ok) break;
                // the next segment's queries first: its first scores are then computed under what follows
                if (!load_q(n_seg + 1)) break;
                // ---- the segment's result: output rows, or partial ones ----
                if (!first) {
                    if (!wait_w(bar(PVDONE + g), (s_run - 1) & 1)) break;
                    tc_fence_after();
                }
                const int slot = seg->slot;
                float inv[2];
                bool live[2], empty[2];
                size_t rec[2];
                uint16_t* dst[2];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    float l = l_run[q].x + l_run[q].y;
                    l += __shfl_xor_sync(0xffffffffu, l, 1);
                    l += __shfl_xor_sync(0xffffffffu, l, 2);
                    const float m = -nm[q].x;
                    empty[q] = first || (m == kNoReference && l == 0.0f);   // (scores that are all NaN leave l NaN)
                    inv[q] = empty[q] ? 0.0f : slot >= 0 ? 1.0f : 1.0f / l;
                    const int r = wr + 8 * q + quad, row = seg->row0 + 128 * g + r;
                    live[q] = row < seg->n_rows;
                    rec[q] = (size_t)(slot < 0 ? 0 : slot) * kChunkRows + 128 * g + r;
                    dst[q] = static_cast<uint16_t*>(a.o) + (long long)(seg->q0 + row / a.G) * a.o_row + (long long)(seg->h * a.G + row % a.G) * a.o_head + col;
                    if (slot >= 0 && live[q] && col == 0) a.stat[rec[q]] = make_float2(empty[q] ? -INFINITY : m, l);
                }
#pragma unroll 1
                for (int hc = 0; hc < D / 32; ++hc) {
                    float o[16];
                    __syncwarp();
                    if (!first) {                     // warp-uniform: the row tile took part
                        tc_ld_16x256_x4(tmem_O + 32 * hc, o);
                        tc_wait_ld();
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const float y0 = empty[q] ? 0.0f : o[4 * w + 2 * q] * inv[q], y1 = empty[q] ? 0.0f : o[4 * w + 2 * q + 1] * inv[q];
                            if (!live[q]) continue;
                            if (slot >= 0) *reinterpret_cast<float2*>(a.part + rec[q] * D + 32 * hc + 8 * w + col) = make_float2(y0, y1);
                            else *reinterpret_cast<uint32_t*>(dst[q] + 32 * hc + 8 * w) = f32x2_to_16(y0, y1, a.is_f16 != 0);
                        }
                }
                tc_fence_before();
                arrive_w(bar(SEGEMPTY + n_seg % kSegStages));
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

// Joins the items that were cut: CTA (c, y) takes rows [8 y, 8 y + 8) of the item that begins in CTA c of the chunk
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
