// Host-only checks of the paged entry points, run without a GPU: every refusal of the C ABI that stands before the
// first CUDA call, and the table arithmetic that the kernels share, on tables that hold anything.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "../logos_b200/csrc/paged.cuh"

static int failures = 0;
#define EXPECT(call, want)                                                                             \
    do {                                                                                               \
        int rc__ = (call);                                                                             \
        if (rc__ != (want)) {                                                                          \
            ++failures;                                                                                \
            std::printf("line %d: %s returned %d, expected %d (%s)\n", __LINE__, #call, rc__, (int)(want), ctx.err); \
        }                                                                                              \
    } while (0)

int main() {
    logos_ctx ctx;
    ctx.sm_count = 148;
    alignas(256) static char mem[4096];
    void* p = mem;
    float* f = reinterpret_cast<float*>(mem);
    int32_t* n = reinterpret_cast<int32_t*>(mem);
    int8_t* c8 = reinterpret_cast<int8_t*>(mem);
    const logos_paged_cache cache{c8, c8, f, f, 4, 64, 2, 64};
    const logos_paged_batch batch{n, n, n, 2, 4, 8, 3, 200};
    logos_attn_params prm{0.125f, 1, 0, 0, 0.0f, 0.0f, 1.0f, LOGOS_DIFFUSE_NONE};
    logos_rope rope{};
    rope.dims = 64;

    auto append = [&](const logos_paged_cache& c, const logos_paged_batch& b, int dt = LOGOS_BF16, const void* k = nullptr, const logos_row_strides* ks = nullptr) {
        return logos_paged_append(&ctx, dt, k ? k : p, p, ks, nullptr, &c, &b);
    };
    auto read = [&](const logos_paged_cache& c, const logos_paged_batch& b, const logos_row_strides* ks = nullptr) {
        return logos_paged_read(&ctx, LOGOS_F32, &c, &b, p, p, ks, nullptr);
    };
    auto attend = [&](const logos_paged_cache& c, const logos_paged_batch& b, int Hq = 4, int dt = LOGOS_BF16, const logos_row_strides* o = nullptr) {
        return logos_paged_attention(&ctx, dt, p, &c, &b, Hq, &prm, p, nullptr, o);
    };
    // cache and batch
    for (int which = 0; which < 3; ++which) {
        auto call = [&](const logos_paged_cache& c, const logos_paged_batch& b) { return which == 0 ? append(c, b) : which == 1 ? read(c, b) : attend(c, b); };
        logos_paged_cache c = cache;
        c.k = nullptr; EXPECT(call(c, batch), LOGOS_ERR_INVALID_ARG); c = cache;
        c.v_scale = nullptr; EXPECT(call(c, batch), LOGOS_ERR_INVALID_ARG); c = cache;
        c.pages = 0; EXPECT(call(c, batch), LOGOS_ERR_INVALID_ARG); c = cache;
        c.H = 0; EXPECT(call(c, batch), LOGOS_ERR_INVALID_ARG); c = cache;
        c.page_size = 48; EXPECT(call(c, batch), LOGOS_ERR_UNSUPPORTED); c = cache;
        c.page_size = 0; EXPECT(call(c, batch), LOGOS_ERR_UNSUPPORTED); c = cache;
        c.pages = INT_MAX; EXPECT(call(c, batch), LOGOS_ERR_UNSUPPORTED); c = cache;
        c.DH = 96; EXPECT(call(c, batch), LOGOS_ERR_UNSUPPORTED); c = cache;
        c.v += 8; EXPECT(call(c, batch), LOGOS_ERR_ALIGNMENT); c = cache;
        logos_paged_batch b = batch;
        b.rows = (1 << 30) + 1; EXPECT(call(c, b), LOGOS_ERR_UNSUPPORTED); b = batch;
        b.max_pages = INT_MAX; b.max_kv = (1 << 30) + 1; EXPECT(call(c, b), LOGOS_ERR_UNSUPPORTED); b = batch;
        b.B = -1; EXPECT(call(c, b), LOGOS_ERR_INVALID_ARG); b = batch;
        b.B = 65536; EXPECT(call(c, b), LOGOS_ERR_INVALID_ARG); b = batch;
        b.max_kv = 257; EXPECT(call(c, b), LOGOS_ERR_INVALID_ARG); b = batch;
        b.max_q = 201; EXPECT(call(c, b), LOGOS_ERR_INVALID_ARG); b = batch;
        b.max_pages = INT_MAX; b.max_kv = -1; EXPECT(call(c, b), LOGOS_ERR_INVALID_ARG); b = batch;
        b.cu_q = nullptr; EXPECT(call(c, b), LOGOS_ERR_INVALID_ARG); b = batch;
        b.page_table = nullptr; EXPECT(call(c, b), LOGOS_ERR_INVALID_ARG); b = batch;
        b.rows = 0; EXPECT(call(c, b), LOGOS_OK); b = batch;                        // nothing to do: no launch
        b.B = 0; EXPECT(call(c, b), LOGOS_OK); b = batch;
        b.max_q = 0; EXPECT(call(c, b), LOGOS_OK);
    }
    EXPECT(append(cache, batch, 7), LOGOS_ERR_INVALID_ARG);
    EXPECT(append(cache, batch, LOGOS_BF16, mem + 8), LOGOS_ERR_ALIGNMENT);
    const logos_row_strides odd{132, 64}, negative{-128, 64}, over{64, 64}, narrow{128, 32};
    EXPECT(append(cache, batch, LOGOS_BF16, nullptr, &odd), LOGOS_ERR_ALIGNMENT);
    EXPECT(append(cache, batch, LOGOS_BF16, nullptr, &negative), LOGOS_ERR_ALIGNMENT);
    EXPECT(read(cache, batch, &over), LOGOS_ERR_INVALID_ARG);
    EXPECT(read(cache, batch, &narrow), LOGOS_ERR_INVALID_ARG);
    EXPECT(logos_paged_append(&ctx, LOGOS_BF16, nullptr, p, nullptr, nullptr, &cache, &batch), LOGOS_ERR_INVALID_ARG);
    EXPECT(logos_paged_append(&ctx, LOGOS_BF16, p, p, nullptr, nullptr, nullptr, &batch), LOGOS_ERR_INVALID_ARG);
    EXPECT(logos_paged_append(nullptr, LOGOS_BF16, p, p, nullptr, nullptr, &cache, &batch), LOGOS_ERR_INVALID_ARG);
    // attention
    EXPECT(attend(cache, batch, 3), LOGOS_ERR_INVALID_ARG);
    EXPECT(attend(cache, batch, 0), LOGOS_ERR_INVALID_ARG);
    EXPECT(attend(cache, batch, 4, LOGOS_F32), LOGOS_ERR_UNSUPPORTED);
    EXPECT(attend(cache, batch, 4, 9), LOGOS_ERR_INVALID_ARG);
    EXPECT(attend(cache, batch, 4, LOGOS_F16, &over), LOGOS_ERR_INVALID_ARG);
    prm.ns_eta = 0.1f; EXPECT(attend(cache, batch), LOGOS_ERR_UNSUPPORTED); prm.ns_eta = 0.0f;
    prm.diffuse_mode = LOGOS_DIFFUSE_CAUSAL; prm.ns_nu = 0.05f; EXPECT(attend(cache, batch), LOGOS_ERR_UNSUPPORTED);
    prm.diffuse_mode = 9; EXPECT(attend(cache, batch), LOGOS_ERR_INVALID_ARG); prm.diffuse_mode = 0;
    prm.scale = 0.0f; EXPECT(attend(cache, batch), LOGOS_ERR_UNSUPPORTED);
    prm.scale = NAN; EXPECT(attend(cache, batch), LOGOS_ERR_UNSUPPORTED);
    prm.scale = INFINITY; EXPECT(attend(cache, batch), LOGOS_ERR_UNSUPPORTED); prm.scale = 0.125f;
    prm.window = -1; EXPECT(attend(cache, batch), LOGOS_ERR_INVALID_ARG); prm.window = 0;
    EXPECT(attend(cache, batch), LOGOS_ERR_WORKSPACE);                              // the context has none
    if (logos_paged_attention_workspace_bytes(&ctx, &cache, &batch, 4) <= logos::kWorkspaceCounterBytes ||
        logos_paged_attention_workspace_bytes(&ctx, &cache, &batch, 3) != 0 || logos_paged_attention_workspace_bytes(&ctx, nullptr, &batch, 4) != 0)
        ++failures, std::printf("workspace sizes\n");
    // norm and rotation
    auto rotate = [&](int dt, const logos_rope* r, float eps, int rows, int Hq, int Hk, int DH, const void* q = nullptr, const logos_row_strides* qo = nullptr) {
        return logos_qk_norm_rope(&ctx, dt, q ? q : p, p, f, f, n, r, eps, p, p, rows, Hq, Hk, DH, nullptr, nullptr, qo, nullptr);
    };
    EXPECT(rotate(5, &rope, 1e-6f, 4, 2, 2, 64), LOGOS_ERR_INVALID_ARG);
    EXPECT(rotate(LOGOS_BF16, nullptr, 1e-6f, 4, 2, 2, 64), LOGOS_ERR_INVALID_ARG);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, -1, 2, 2, 64), LOGOS_ERR_INVALID_ARG);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 0, 0, 64), LOGOS_ERR_INVALID_ARG);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, (1 << 30) + 1, 2, 2, 64), LOGOS_ERR_UNSUPPORTED);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 2, 2, 80), LOGOS_ERR_UNSUPPORTED);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 1025, 2, 64), LOGOS_ERR_UNSUPPORTED);
    EXPECT(rotate(LOGOS_BF16, &rope, -1.0f, 4, 2, 2, 64), LOGOS_ERR_INVALID_ARG);
    EXPECT(rotate(LOGOS_BF16, &rope, NAN, 4, 2, 2, 64), LOGOS_ERR_INVALID_ARG);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 2, 2, 64, mem + 4), LOGOS_ERR_ALIGNMENT);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 2, 2, 64, nullptr, &odd), LOGOS_ERR_ALIGNMENT);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 2, 2, 64, nullptr, &over), LOGOS_ERR_INVALID_ARG);
    EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 0, 2, 2, 64), LOGOS_OK);
    rope.dims = 24; EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 2, 2, 64), LOGOS_ERR_INVALID_ARG);
    rope.dims = 128; EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 2, 2, 64), LOGOS_ERR_INVALID_ARG);
    rope.dims = 64; rope.inv_freq[31] = INFINITY; EXPECT(rotate(LOGOS_BF16, &rope, 1e-6f, 4, 2, 2, 64), LOGOS_ERR_INVALID_ARG);
    rope.inv_freq[31] = 0.0;
    auto back = [&](float* dwq, float* dwk) {
        return logos_qk_norm_rope_bwd(&ctx, LOGOS_F16, p, p, p, p, f, nullptr, n, &rope, 1e-6f, p, p, dwq, dwk, 4, 2, 2, 64, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr);
    };
    EXPECT(back(nullptr, nullptr), LOGOS_ERR_INVALID_ARG);
    EXPECT(back(f, f), LOGOS_ERR_INVALID_ARG);
    EXPECT(back(f, nullptr), LOGOS_ERR_WORKSPACE);

    // the tables: whatever they hold, an accepted sequence's rows and positions stay inside the bounds, every table
    // index inside the table and every page row inside the cache
    std::mt19937 rng(7);
    auto wild = [&](int lo, int hi) {
        switch (rng() % 6) {
            case 0: return (int)rng();
            case 1: return rng() % 2 ? INT_MAX : INT_MIN;
            default: return lo + (int)(rng() % (unsigned)(hi - lo + 1));
        }
    };
    long accepted = 0, pages_in = 0;
    for (int round = 0; round < 20000; ++round) {
        logos_paged_cache c = cache;
        c.page_size = 16 << (rng() % 4);
        c.pages = 1 + rng() % 9;
        c.H = 1 + rng() % 3;
        logos_paged_batch b = batch;
        b.B = 1 + rng() % 4;
        b.max_pages = 1 + rng() % 5;
        b.max_kv = rng() % (b.max_pages * c.page_size + 1);
        b.max_q = rng() % (b.max_kv + 1);
        b.rows = rng() % 40;
        std::vector<int32_t> cu(b.B + 1), kv(b.B), table((size_t)b.B * b.max_pages);
        for (auto& x : cu) x = wild(0, b.rows + 2);
        if (rng() % 2) std::sort(cu.begin(), cu.end());
        for (auto& x : kv) x = wild(0, b.max_kv + 2);
        for (auto& x : table) x = wild(-2, c.pages + 1);
        b.cu_q = cu.data(); b.kv_len = kv.data(); b.page_table = table.data();
        if (logos::paged_check(&ctx, "check", &c, &b) != LOGOS_OK) { ++failures; std::printf("a valid batch was refused: %s\n", ctx.err); break; }
        const logos::PagedArgs a = logos::paged_args(&ctx, &c, &b);
        for (int i = 0; i < b.B; ++i) {
            const logos::PagedSeq s = logos::paged_seq(a, i);
            if (!s.ok) continue;
            ++accepted;
            if (s.q0 < 0 || s.n < 0 || s.n > b.max_q || s.q0 + s.n > b.rows || s.kv < s.n || s.kv > b.max_kv) ++failures;
            for (int pos = 0; pos < s.kv; ++pos) {
                const size_t at = (size_t)i * b.max_pages + (pos >> a.page_shift);
                if (at >= table.size()) { ++failures; continue; }
                const int page = logos::paged_page(a, i, pos);
                if (page < 0) { if (table[at] >= 0 && table[at] < c.pages) ++failures; continue; }
                ++pages_in;
                const size_t row = (size_t)logos::paged_row(a, page, c.H - 1) + (pos & (c.page_size - 1));
                if (row >= (size_t)c.pages * c.H * c.page_size) ++failures;
            }
        }
    }
    if (accepted < 1000 || pages_in < 1000) { ++failures; std::printf("the check saw %ld sequences, %ld pages\n", accepted, pages_in); }
    std::printf(failures ? "%d failures\n" : "ok\n", failures);
    return failures != 0;
}
