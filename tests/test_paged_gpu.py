"""The paged INT8 cache: quantising append and read back (bit for bit), attention of new tokens over the pages against a
64-bit restatement.

Tolerance of the attention.  The weights are rounded to FP16 once, off by at most 2^-11 of themselves; a score's
exponent (|x| < 64 or so, three fp32 roundings) adds below 2^-15.  So an output is off by at most
(2^-11 + 2^-13) sum w |v|.  A weight more than 2^14 below the row's reference is an FP16 denormal, off by 2^-25
absolutely: 2^-25 sum |v8| / l with l >= 1 / max(vs).  Then half a step of the output's type."""
import pytest
import torch

from logos_b200 import lib as L
from logos_b200.engine import Engine
from logos_b200.paged import PagedBatch, PagedKVCache, PagePool, Rope

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def view(x, layout):
    return x if layout == "tokens" else x.transpose(0, 1).contiguous().transpose(0, 1)


def tables(n_q, n_kv, page, extra_pages=2, seed=0, max_q=None, max_kv=None):
    per = [-(-x // page) for x in n_kv]
    pages = sum(per) + extra_pages
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(1, -(-max(max_kv or 0, *n_kv) // page))
    table = torch.full((len(n_q), width), -7, dtype=torch.int32)
    for b, n in enumerate(per):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    cu = torch.tensor([0] + n_q, dtype=torch.int32).cumsum(0).to(torch.int32)
    return pages, PagedBatch(cu.cuda(), torch.tensor(n_kv, dtype=torch.int32).cuda(), table.cuda(), max_q or max(n_q), max_kv or max(n_kv))


def fresh(pages, H, page, D):
    """Pages that nobody has written: every byte and every scale a value that must not get anywhere."""
    return PagedKVCache.over(torch.full((pages, H, page, D), -128, dtype=torch.int8, device="cuda"),
                             torch.full((pages, H, page, D), -128, dtype=torch.int8, device="cuda"),
                             torch.full((pages, H, page), float("nan"), device="cuda"),
                             torch.full((pages, H, page), float("inf"), device="cuda"))


def rows_of(batch, page):
    """(page, row) of every token row, host arithmetic."""
    cu, kv, table = batch.cu_q.cpu(), batch.kv_len.cpu(), batch.page_table.cpu()
    out = []
    for b in range(batch.B):
        n = int(cu[b + 1] - cu[b])
        for pos in range(int(kv[b]) - n, int(kv[b])):
            out.append((int(table[b, pos // page]), pos % page))
    return out


def quantise(x):
    """nikhilam_compress of each row in fp32 (true divisions: the divisor is a tensor)."""
    x = x.float()
    s = (x.abs().amax(-1) + torch.tensor(1e-8)) / torch.full(x.shape[:-1], 127.5)
    return torch.clamp(torch.round(x / s[..., None]), -127, 127).to(torch.int8), s


@pytest.mark.parametrize("n_q,n_kv,H,D,page,layout,dtype,pad", [
    ([1], [1], 1, 64, 16, "tokens", "bf16", 0),
    ([1] * 40, [1 + 37 * i for i in range(40)], 16, 64, 64, "tokens", "fp16", 3),
    ([5, 0, 130, 33], [5, 9, 200, 97], 3, 128, 32, "heads", "bf16", 0),
    ([700, 1, 258], [700, 300, 258], 8, 64, 128, "heads", "fp32", 19),
    ([2] * 300, [16] * 300, 2, 128, 16, "tokens", "fp32", 1),
])
def test_append_and_read(engine, n_q, n_kv, H, D, page, layout, dtype, pad):
    g = torch.Generator(device="cuda").manual_seed(len(n_q) + D)
    pages, batch = tables(n_q, n_kv, page)
    cache = fresh(pages, H, page, D)
    before = [t.clone() for t in (cache.k, cache.v, cache.ks, cache.vs)]
    rows = sum(n_q)
    K, V = (torch.randn((rows + pad, H, D), generator=g, device="cuda") * torch.logspace(-6, 4, rows + pad, device="cuda")[:, None, None]
            for _ in range(2))
    K, V = (view(x.clamp(-6e4, 6e4).to(DT[dtype]), layout) for x in (K, V))
    if rows > 2:
        K[1] = 0                                            # a row of zeros: scale 1e-8 / 127.5
    engine.paged_append(K, V, cache, batch)
    engine.synchronize()
    where = rows_of(batch, page)
    at, off = (torch.tensor([w[i] for w in where], dtype=torch.long) for i in range(2))
    written = torch.zeros((pages, page), dtype=torch.bool)
    written[at, off] = True
    for x, c8, cs, b8, bs in ((K, cache.k, cache.ks, before[0], before[2]), (V, cache.v, cache.vs, before[1], before[3])):
        q, s = quantise(x[:rows].cpu())
        c8, cs, b8, bs = c8.cpu(), cs.cpu(), b8.cpu(), bs.cpu()
        assert torch.equal(c8[at, :, off], q) and torch.equal(cs[at, :, off], s)
        rest = ~written
        assert torch.equal(c8.transpose(1, 2)[rest], b8.transpose(1, 2)[rest])
        assert torch.equal(cs.transpose(1, 2)[rest].view(torch.int32), bs.transpose(1, 2)[rest].view(torch.int32))
    for out_t in ("fp32", dtype):
        ko, vo = (view(torch.full((rows + pad, H, D), 7.0, device="cuda", dtype=DT[out_t]), layout) for _ in range(2))
        engine.paged_read(cache, batch, ko, vo)
        for x, y in ((K, ko), (V, vo)):
            q, s = quantise(x[:rows].cpu())
            assert torch.equal(y[:rows].cpu(), (q.float() * s[..., None]).to(DT[out_t]))
            assert torch.equal(y[rows:], torch.full_like(y[rows:], 7.0))


def test_append_rounds_as_the_division_does(engine):
    """Values on the border between two bytes, a step to either side of it, and rows with an infinity or a NaN: the bytes of
    the fp32 division, rounded half to even."""
    g = torch.Generator().manual_seed(6)
    rows, H, D = 512, 4, 64
    top = 10.0 ** (torch.rand((rows, H, 1), generator=g) * 12 - 8)
    scale = (top + torch.tensor(1e-8)) / torch.tensor(127.5)
    half = torch.randint(-127, 127, (rows, H, D), generator=g).float() + 0.5
    x = half * scale
    up = torch.rand(x.shape, generator=g)
    x = torch.where(up < 0.3, torch.nextafter(x, torch.tensor(float("inf"))), torch.where(up > 0.7, torch.nextafter(x, torch.tensor(0.0)), x))
    x[..., :1] = top                                        # the row's largest value
    x = torch.minimum(torch.maximum(x, -top), top)
    x[3, 1, 5], x[4, 2, 6], x[5, 0, :] = float("inf"), float("nan"), 0.0
    pages, batch = tables([rows], [rows], 64)
    cache = fresh(pages, H, 64, D)
    engine.paged_append(x.cuda(), x.cuda(), cache, batch)
    where = rows_of(batch, 64)
    at, off = (torch.tensor([w[i] for w in where], dtype=torch.long) for i in range(2))
    # the kernel's maximum passes over a NaN, and a quotient that is none counts as 0
    s = (x.abs().nan_to_num(nan=0.0, posinf=float("inf")).amax(-1) + torch.tensor(1e-8)) / torch.full((rows, H), 127.5)
    q = torch.clamp(torch.round((x / s[..., None]).nan_to_num(nan=0.0)), -127, 127).to(torch.int8)
    for c8, cs in ((cache.k, cache.ks), (cache.v, cache.vs)):
        assert torch.equal(c8.cpu()[at, :, off], q) and torch.equal(cs.cpu()[at, :, off], s)


def attend64(Q, cache, batch, params, page):
    """(output, sum w |v|, sum |v8| max vs) in 64 bits, row by row of the batch; zeros where nothing is seen."""
    cu, kv, table = batch.cu_q.tolist(), batch.kv_len.tolist(), batch.page_table
    rows, Hq, D = Q.shape
    G = Hq // cache.heads
    out, size, tiny = (torch.zeros((rows, Hq, D), dtype=torch.float64, device="cuda") for _ in range(3))
    for b in range(batch.B):
        n, L_ = cu[b + 1] - cu[b], kv[b]
        if n == 0:
            continue
        j = torch.arange(L_, device="cuda")
        at, off = table[b][j // page].long(), j % page
        k = (cache.k[at, :, off].double() * cache.ks[at, :, off].double()[..., None]).repeat_interleave(G, 1).permute(1, 0, 2)
        v8, vs = cache.v[at, :, off].double(), cache.vs[at, :, off].double()
        v = (v8 * vs[..., None]).repeat_interleave(G, 1).permute(1, 0, 2)
        i = torch.arange(L_ - n, L_, device="cuda")[:, None]
        ok = (j <= i) if params.causal else torch.ones((n, L_), dtype=torch.bool, device="cuda")
        if 0 < params.window < L_:
            near = (j >= i - params.window) & (j <= i)
            if params.stride > 0:
                near = near | (j % params.stride == 0)
            ok = ok & near
        s = (Q[cu[b]:cu[b + 1]].double().permute(1, 0, 2) @ k.transpose(1, 2)) * params.scale
        w = torch.softmax(s.masked_fill(~ok, float("-inf")), -1).nan_to_num(0.0)
        out[cu[b]:cu[b + 1]] = (w @ v).permute(1, 0, 2)
        size[cu[b]:cu[b + 1]] = (w @ v.abs()).permute(1, 0, 2)
        seen = ok.double() @ v8.abs().permute(1, 0, 2)                         # [H, n, D]
        tiny[cu[b]:cu[b + 1]] = (seen * vs.amax(0)[:, None, None]).repeat_interleave(G, 0).permute(1, 0, 2)
    return out, size, tiny


def check_attention(got, Q, cache, batch, params, page):
    want, size, tiny = attend64(Q, cache, batch, params, page)
    rows = int(batch.cu_q[-1])
    half = torch.finfo(Q.dtype).eps / 2
    bound = (2.0 ** -11 + 2.0 ** -13) * size + 2.0 ** -25 * tiny + half * want.abs() + 1e-7
    err = (got.double() - want).abs()
    assert torch.isfinite(got[:rows]).all()
    over = (err - bound)[:rows].max().item()
    assert over <= 0, f"{over} beyond the bound, largest error {err[:rows].max().item()}"


def filled(engine, n_q, n_kv, H, D, page, seed, dtype=torch.bfloat16, v_spread=1.0, **kw):
    """A cache that holds every sequence, appended through the engine, and the batch of the new tokens."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages, batch = tables(n_q, n_kv, page, seed=seed, **kw)
    cache = fresh(pages, H, page, D)
    whole = PagedBatch(torch.tensor([0] + n_kv, dtype=torch.int32).cumsum(0).to(torch.int32).cuda(), batch.kv_len, batch.page_table,
                       max(n_kv), batch.max_kv)
    K, V = (torch.randn((sum(n_kv), H, D), generator=g, device="cuda") for _ in range(2))
    if v_spread != 1.0:                                     # rows of very different scales
        V *= v_spread ** torch.randn((sum(n_kv), H, 1), generator=g, device="cuda")
    engine.paged_append(K.to(dtype), V.to(dtype), cache, whole)
    return cache, batch, g


ATTEND = [  # n_q, n_kv, H, G, D, page, window, stride, causal, layout, dtype
    ([1], [1], 1, 1, 64, 16, 0, 0, True, "tokens", "fp16"),
    ([1] * 5, [1, 2, 31, 257, 1000], 4, 1, 64, 64, 0, 0, True, "tokens", "bf16"),
    ([1] * 3, [700, 33, 5000], 2, 4, 128, 16, 0, 0, True, "tokens", "bf16"),
    ([1, 1], [9000, 4097], 1, 8, 64, 128, 0, 0, True, "heads", "fp16"),
    ([3, 5, 1], [3, 300, 129], 2, 3, 64, 32, 0, 0, True, "heads", "bf16"),
    ([17, 0, 64], [17, 40, 500], 2, 1, 128, 64, 0, 0, True, "tokens", "fp16"),
    ([200, 1, 33], [900, 650, 33], 3, 2, 64, 16, 0, 0, True, "heads", "bf16"),
    ([130, 1], [1500, 1500], 2, 1, 64, 64, 64, 0, True, "tokens", "bf16"),
    ([130, 2, 40], [1500, 64, 65], 2, 2, 128, 32, 64, 16, True, "tokens", "fp16"),
    ([1, 4], [3000, 2001], 1, 1, 128, 128, 100, 0, True, "tokens", "bf16"),
    ([37, 1, 6], [300, 90, 6], 2, 2, 64, 16, 0, 0, False, "tokens", "bf16"),
    ([40], [400], 1, 1, 64, 64, 50, 7, False, "tokens", "fp16"),
    ([300], [300], 4, 1, 128, 64, 0, 0, True, "heads", "bf16"),
    ([1000, 257], [2300, 257], 2, 1, 64, 64, 0, 0, True, "tokens", "bf16"),
    ([129, 513], [129, 4000], 1, 4, 128, 128, 0, 0, True, "tokens", "fp16"),
    ([600], [3000], 1, 2, 64, 32, 200, 0, True, "tokens", "bf16"),
    ([385], [1100], 1, 1, 128, 16, 90, 33, True, "heads", "bf16"),
    ([64, 65, 33], [700, 700, 33], 2, 1, 128, 32, 0, 0, True, "tokens", "fp16"),   # either side of the two kernels' border
    ([32, 33], [300, 4000], 2, 2, 64, 64, 0, 0, True, "heads", "bf16"),
    ([1000], [2000], 2, 1, 64, 64, 0, 0, True, "tokens", "bf16"),      # warps of the last row tile without a row
    ([300, 33, 140], [3000, 5000, 140], 4, 1, 64, 16, 0, 0, True, "heads", "fp16"),
    ([1, 3], [1000, 40], 1, 128, 64, 64, 0, 0, True, "tokens", "bf16"),            # many query heads over one: one token is a chunk
    ([1, 2, 1], [5000, 2, 1], 1, 71, 128, 16, 300, 9, True, "heads", "fp16"),
]


@pytest.mark.parametrize("n_q,n_kv,H,G,D,page,window,stride,causal,layout,dtype", ATTEND)
def test_attention(engine, n_q, n_kv, H, G, D, page, window, stride, causal, layout, dtype):
    cache, batch, g = filled(engine, n_q, n_kv, H, D, page, seed=sum(n_kv) + D)
    pad = 3
    Q = view(torch.randn((sum(n_q) + pad, H * G, D), generator=g, device="cuda").to(DT[dtype]), layout)
    out = view(torch.full((sum(n_q) + pad, H * G, D), 9.0, dtype=DT[dtype], device="cuda"), layout)
    params = L.Params.make(D ** -0.5, causal, window, stride)
    engine.paged_attention(Q, cache, batch, params, out=out)
    engine.synchronize()
    check_attention(out, Q, cache, batch, params, page)
    assert torch.equal(out[sum(n_q):], torch.full_like(out[sum(n_q):], 9.0))
    for _ in range(5):
        again = engine.paged_attention(Q, cache, batch, params)
        assert torch.equal(again[: sum(n_q)], out[: sum(n_q)])


@pytest.mark.parametrize("n_q,D", [(1, 64), (1, 128), (9, 64), (150, 64), (150, 128)])
def test_attention_hard_values(engine, n_q, D):
    """Scores in the hundreds (one key takes all), values whose scales differ by a factor of thousands, queries of one
    tiny and one huge row."""
    cache, batch, g = filled(engine, [n_q, n_q], [700, 1300], 2, D, 64, seed=5, v_spread=30.0)
    Q = 30.0 * torch.randn((2 * n_q, 4, D), generator=g, device="cuda")
    Q[0] *= 1e-30
    Q[-1] *= 1e30 / 30
    Q = Q.bfloat16()
    params = L.Params.make(D ** -0.5)
    got = engine.paged_attention(Q, cache, batch, params)
    # the huge row's scores pass fp32's range of exact steps: it is checked on its own, the key of the largest score wins
    rows = 2 * n_q
    want, size, tiny = attend64(Q, cache, batch, params, 64)
    # |x| goes up to a few thousand here: an fp32 score is off by 2^-24 |x| in each of its three roundings
    k = (cache.k.double() * cache.ks.double()[..., None]).nan_to_num(0.0)
    reach = (Q[:-1].double().abs().amax() * D * 30 * D ** -0.5 * 1.4427)
    slack = min(1.0, float(3 * 2.0 ** -24 * reach))
    bound = (2.0 ** -11 + 2.0 ** -13 + 2 * slack) * size + 2.0 ** -25 * tiny + 2.0 ** -8 * want.abs() + 1e-7
    assert torch.isfinite(got).all() and k.isfinite().all()
    assert ((got.double() - want).abs() - bound)[: rows - 1].max().item() <= 0
    assert ((got.double() - want).abs() - 2.0 ** -7 * want.abs() - 1e-6)[rows - 1].max().item() <= 0


@pytest.mark.parametrize("n_q,D", [(1, 64), (20, 128), (200, 64)])
def test_nan_and_infinity_stay_in_their_rows(engine, n_q, D):
    """A NaN query spoils its own row and no other; an infinity in a token that is masked for the rows before it does not
    reach them."""
    cache, batch, g = filled(engine, [n_q], [500], 2, D, 32, seed=8)
    Q = torch.randn((n_q, 2, D), generator=g, device="cuda").bfloat16()
    params = L.Params.make(D ** -0.5)
    clean = engine.paged_attention(Q, cache, batch, params).clone()
    Q2 = Q.clone()
    Q2[n_q // 2, 1, 3] = float("nan")
    got = engine.paged_attention(Q2, cache, batch, params)
    assert got[n_q // 2, 1].isnan().all()
    got[n_q // 2, 1] = clean[n_q // 2, 1]
    assert torch.equal(got, clean)
    if n_q > 1:
        last = batch.page_table[0, 499 // 32].item(), 499 % 32
        cache.ks[last[0], :, last[1]] = float("inf")
        cache.vs[last[0], :, last[1]] = float("inf")
        got = engine.paged_attention(Q, cache, batch, params)
        assert torch.equal(got[:-1], clean[:-1])


def test_results_do_not_depend_on_the_page_order(engine):
    """The same sequences behind another permutation of pages, and with other page sizes: the same bits."""
    outs = []
    for page, seed in ((16, 1), (16, 2), (64, 3), (128, 4)):
        g = torch.Generator(device="cuda").manual_seed(1)
        n_q, n_kv = [1, 30, 300], [600, 333, 1000]
        pages, batch = tables(n_q, n_kv, page, seed=seed)
        cache = fresh(pages, 2, page, 64)
        whole = PagedBatch(torch.tensor([0, 600, 933, 1933], dtype=torch.int32).cuda(), batch.kv_len, batch.page_table, 1000, 1000)
        K, V = (torch.randn((1933, 2, 64), generator=g, device="cuda").bfloat16() for _ in range(2))
        engine.paged_append(K, V, cache, whole)
        Q = torch.randn((331, 4, 64), generator=g, device="cuda").bfloat16()
        outs.append(engine.paged_attention(Q, cache, batch, L.Params.make(0.125)))
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


def test_bad_tables_are_reported_and_touch_nothing_else(engine):
    """A page outside the cache, a sequence outside its bounds: the others come out right, the next synchronize says so,
    and the engine goes on.  (The kernels turn every bad entry into a skipped access; the table arithmetic is checked on
    the host in test_paged_cpu.py.)"""
    for n_q in (1, 40, 200):
        cache, batch, g = filled(engine, [n_q] * 3, [300, 400, 500], 2, 64, 64, seed=3)
        Q = torch.randn((3 * n_q, 2, 64), generator=g, device="cuda").bfloat16()
        params = L.Params.make(0.125)
        clean = engine.paged_attention(Q, cache, batch, params).clone()
        engine.synchronize()
        keep = batch.page_table.clone()
        for entry in (-1, cache.pages, 2 ** 31 - 1):
            batch.page_table[1, 2] = entry
            got = engine.paged_attention(Q, cache, batch, params)
            with pytest.raises(L.LogosError) as e:
                engine.synchronize()
            assert e.value.status == L.ERR_BAD_BATCH and "sequence 1" in str(e.value) and "page" in str(e.value)
            assert torch.equal(got[:n_q], clean[:n_q]) and torch.equal(got[2 * n_q:], clean[2 * n_q:])
        batch.page_table.copy_(keep)
        # Without sequence 0 the work of the others may be cut at other keys, so their sums run in another order: either
        # result is within check_attention's bound of the exact one, the two within twice that of each other.
        want, size, tiny = attend64(Q, cache, batch, params, 64)
        bound = 2 * ((2.0 ** -11 + 2.0 ** -13) * size + 2.0 ** -25 * tiny + torch.finfo(Q.dtype).eps / 2 * want.abs() + 1e-7)
        kv = batch.kv_len.clone()
        for value in (501, -1, n_q - 1):
            batch.kv_len[0] = value
            got = torch.full_like(Q, 5.0)
            engine.paged_attention(Q, cache, batch, params, out=got)
            with pytest.raises(L.LogosError) as e:
                engine.synchronize()
            assert e.value.status == L.ERR_BAD_BATCH and "sequence 0" in str(e.value)
            assert ((got.double() - clean.double()).abs() - bound)[n_q:].max().item() <= 0
            assert torch.equal(got[:n_q], torch.full_like(got[:n_q], 5.0))
        batch.kv_len.copy_(kv)
        # append and read: a bad page leaves its rows alone
        before = cache.k.clone()
        batch.page_table[2].fill_(cache.pages + 3)
        K = torch.randn((3 * n_q, 2, 64), generator=g, device="cuda").bfloat16()
        engine.paged_append(K, K, cache, batch)
        with pytest.raises(L.LogosError):
            engine.synchronize()
        untouched = torch.ones(cache.pages, dtype=torch.bool, device="cuda")
        untouched[batch.page_table[:2].long().clamp(0, cache.pages - 1).flatten()] = False
        assert torch.equal(cache.k[untouched], before[untouched])
        ko, vo = torch.full_like(K, 3.0), torch.full_like(K, 3.0)
        engine.paged_read(cache, batch, ko, vo)
        with pytest.raises(L.LogosError):
            engine.synchronize()
        assert torch.equal(ko[2 * n_q:], torch.full_like(ko[2 * n_q:], 3.0))
        engine.synchronize()                                  # and the report is gone


def test_many_sequences_need_no_counters(engine):
    """More (sequence, head) pairs than the workspace has arrival counters: one chunk per pair."""
    n = 2100
    kv = [1 + (i * 7) % 40 for i in range(n)]
    cache, batch, g = filled(engine, [1] * n, kv, 8, 64, 16, seed=2)
    Q = torch.randn((n, 8, 64), generator=g, device="cuda").bfloat16()
    params = L.Params.make(0.125)
    check_attention(engine.paged_attention(Q, cache, batch, params), Q, cache, batch, params, 16)


def test_captured_step_replays_with_new_lengths(engine):
    """norm + rotation, append and attention captured once and replayed while the sequences grow: the same bits as the
    eager calls."""
    from logos_b200.engine import Engine
    H, D, page, steps = 4, 64, 16, 40
    rope, params = Rope(64), L.Params.make(0.125)
    w = torch.ones(D, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(12)
    data = torch.randn((steps, 3, 3, H, D), generator=g, device="cuda").bfloat16()      # step, (q, k, v), sequence

    def make():
        pool = PagePool(64, page)
        seqs = [pool.open() for _ in range(3)]
        pool.batch([(s, 5 + 9 * s) for s in seqs])
        first = pool.batch([(s, steps) for s in seqs])                                   # all pages taken ahead
        start = first.kv_len - steps
        batch = PagedBatch(torch.arange(4, dtype=torch.int32, device="cuda"), start.clone(), first.page_table, 1, first.max_kv)
        return PagedKVCache(64, page, H, D), batch

    def step(eng, cache, batch, q, k, v, pos, out):
        eng.qk_norm_rope(q, k, w, w, pos, rope, out_q=q, out_k=k)
        eng.paged_append(k, v, cache, batch)
        eng.paged_attention(q, cache, batch, params, out=out)

    cache, batch = make()
    eager = []
    for i in range(steps):
        batch.kv_len += 1
        q, k, v = (data[i, j].clone() for j in range(3))
        out = torch.empty_like(q)
        step(engine, cache, batch, q, k, v, batch.kv_len - 1, out)
        eager.append(out)
    cache, batch = make()
    stream = torch.cuda.Stream()
    eng = Engine(0)
    eng.use_stream(stream)
    buf = [torch.empty((3, H, D), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    pos = torch.empty(3, dtype=torch.int32, device="cuda")
    eng.reserve(eng.paged_attention_workspace_bytes(cache, batch, 3, H))
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for t in buf:
            t.zero_()
        pos.zero_()
        step(eng, cache, batch, *buf[:3], pos, buf[3])                                   # warm-up; its row is written again
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(eng, cache, batch, *buf[:3], pos, buf[3])
        for i in range(steps):
            batch.kv_len += 1
            for j in range(3):
                buf[j].copy_(data[i, j])
            pos.copy_(batch.kv_len - 1)
            graph.replay()
            assert torch.equal(buf[3], eager[i]), f"step {i}"
    eng.synchronize()
    del graph
    eng.close()


def test_chunks_and_steps_give_what_one_pass_gives(engine):
    """A prompt taken in chunks, then single tokens, each through norm + rotation, append and attention: every row as
    the 64-bit attention over the rows the cache holds has it."""
    H, G, D, page = 2, 2, 128, 32
    rope, params = Rope(128), L.Params.make(D ** -0.5)
    g = torch.Generator(device="cuda").manual_seed(21)
    wq, wk = (1 + 0.1 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    pool, cache = PagePool(40, page), PagedKVCache(40, page, H, D)
    a, b = pool.open(), pool.open()
    for take in ([(a, 150), (b, 1)], [(b, 70), (a, 33)], [(a, 1), (b, 1)], [(a, 300), (b, 1)], [(a, 1), (b, 1)]):
        batch = pool.batch(take)
        rows = sum(n for _, n in take)
        Q = torch.randn((rows, H * G, D), generator=g, device="cuda").bfloat16()
        K, V = (torch.randn((rows, H, D), generator=g, device="cuda").bfloat16() for _ in range(2))
        Q, K = engine.qk_norm_rope(Q, K, wq, wk, batch.positions(rows), rope)
        engine.paged_append(K, V, cache, batch)
        out = engine.paged_attention(Q, cache, batch, params)
        engine.synchronize()
        check_attention(out, Q, cache, batch, params, page)


def test_fork_then_diverge(engine):
    """Two sequences that share a prompt's pages and then write their own tokens do not see each other's."""
    H, D, page = 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(22)
    pool, cache = PagePool(20, page), PagedKVCache(20, page, H, D)
    params = L.Params.make(0.125)
    a = pool.open()
    K = torch.randn((40, H, D), generator=g, device="cuda").bfloat16()
    engine.paged_append(K, K, cache, pool.batch([(a, 40)]))
    b = pool.fork(a, [cache])
    batch = pool.batch([(a, 3), (b, 3)])
    K = torch.randn((6, H, D), generator=g, device="cuda").bfloat16()
    engine.paged_append(K, K, cache, batch)
    Q = torch.randn((6, H, D), generator=g, device="cuda").bfloat16()
    check_attention(engine.paged_attention(Q, cache, batch, params), Q, cache, batch, params, page)
    q, s = quantise(K.cpu())
    for row, (at, off) in enumerate(rows_of(batch, page)):
        assert torch.equal(cache.k[at, :, off].cpu(), q[row])


def test_another_current_device_or_stream(engine):
    """The engine's own stream is used whatever torch has current, and the caller's device stays current."""
    from logos_b200.engine import Engine
    cache, batch, g = filled(engine, [3], [200], 2, 64, 64, seed=30)
    Q = torch.randn((3, 2, 64), generator=g, device="cuda").bfloat16()
    params = L.Params.make(0.125)
    want = engine.paged_attention(Q, cache, batch, params).clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    eng = Engine(0)
    eng.use_stream(side)
    out = torch.zeros_like(Q)
    torch.cuda.synchronize()
    eng.paged_attention(Q, cache, batch, params, out=out)
    eng.synchronize()
    assert torch.equal(out, want) and torch.cuda.current_device() == 0
    eng.close()


def test_refusals(engine):
    cache, batch, g = filled(engine, [2], [20], 2, 64, 16, seed=1)
    Q = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    params = L.Params.make(0.125)
    for bad in (lambda: engine.paged_attention(Q[:, :, :32], cache, batch, params),
                lambda: engine.paged_attention(Q, cache, batch, params, out=Q.float()),
                lambda: engine.paged_attention(Q.cpu(), cache, batch, params),
                lambda: engine.paged_append(Q, Q[:, :1], cache, batch),
                lambda: engine.paged_append(Q[:, :1], Q[:, :1], cache, batch),
                lambda: engine.paged_append(Q.transpose(1, 2), Q, cache, batch),
                lambda: engine.paged_read(cache, batch, Q, Q.half())):
        with pytest.raises(ValueError):
            bad()
    for status, call in ((L.ERR_INVALID_ARG, lambda: engine.paged_attention(Q[:, :1].contiguous(), cache, batch, params)),
                         (L.ERR_UNSUPPORTED, lambda: engine.paged_attention(Q.float(), cache, batch, params)),
                         (L.ERR_UNSUPPORTED, lambda: engine.paged_attention(Q, cache, batch, L.Params.make(0.125, ns_eta=0.1))),
                         (L.ERR_INVALID_ARG, lambda: engine.paged_read(cache, batch, Q.expand(2, 2, 64)[:, :1].expand(2, 2, 64), Q))):
        with pytest.raises(L.LogosError) as e:
            call()
        assert e.value.status == status
    empty = torch.zeros((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    none = PagedBatch(torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda"),
                      torch.zeros((0, 1), dtype=torch.int32, device="cuda"), 0, 0)
    engine.paged_append(empty, empty, cache, none)
    assert engine.paged_attention(empty, cache, none, params).shape == empty.shape
    engine.synchronize()


@pytest.mark.parametrize("n_q,D,page", [(3, 64, 64), (70, 128, 16)])
def test_offsets_beyond_32_bits(engine, n_q, D, page):
    """Pages more than 2^32 bytes into the cache, token tensors whose heads lie more than 2^31 values apart."""
    H, kv, far = 2, 700, 2 ** 31 + 64
    pages = 2 ** 32 // (H * page * D) + 200
    cache = fresh(pages, H, page, D)
    n = -(-kv // page)
    table = torch.arange(pages - 1, pages - 1 - n, -1, dtype=torch.int32, device="cuda")[None].contiguous()
    cu = lambda m: torch.tensor([0, m], dtype=torch.int32, device="cuda")  # noqa: E731
    held = torch.tensor([kv], dtype=torch.int32, device="cuda")
    whole, batch = PagedBatch(cu(kv), held, table, kv, kv), PagedBatch(cu(n_q), held, table, n_q, kv)
    g = torch.Generator(device="cuda").manual_seed(5)
    store = torch.empty(far + kv * D, dtype=torch.bfloat16, device="cuda")
    apart = lambda m: store.as_strided((m, H, D), (D, far, 1))  # noqa: E731
    K, V, Q = (torch.randn((m, H, D), generator=g, device="cuda").bfloat16() for m in (kv, kv, n_q))
    apart(kv).copy_(K)
    engine.paged_append(apart(kv), V, cache, whole)
    k_far, v_far = apart(kv), torch.empty((kv, H, D), dtype=torch.bfloat16, device="cuda")
    store.zero_()
    engine.paged_read(cache, whole, k_far, v_far)
    for got, want in ((k_far, K), (v_far, V)):
        # half a step of the quantiser and half a step of BF16, each relative to the row's largest value
        top = want.double().abs().amax(-1, keepdim=True)
        assert ((got.double() - want.double()).abs() <= (0.5 / 127.5 + 2.0 ** -8) * 1.01 * top).all()
    params = L.Params.make(D ** -0.5)
    apart(n_q).copy_(Q)
    got = engine.paged_attention(apart(n_q), cache, batch, params)
    out = engine.paged_attention(Q, cache, batch, params, out=apart(n_q))
    engine.synchronize()
    check_attention(got, Q, cache, batch, params, page)
    assert torch.equal(out, got)
    pos = torch.arange(n_q, dtype=torch.int32, device="cuda")
    apart(n_q).copy_(Q)
    want, _ = engine.qk_norm_rope(Q, None, None, None, pos, Rope(D))
    there, _ = engine.qk_norm_rope(apart(n_q), None, None, None, pos, Rope(D), out_q=apart(n_q))
    assert torch.equal(there, want)


@pytest.mark.parametrize("n_q", [1, 90])
def test_two_contexts_at_once(engine, n_q):
    """Two engines on streams of their own read one cache at the same time, each with its workspace."""
    cache, batch, g = filled(engine, [n_q, n_q, 1], [3000, 700, 5000], 2, 64, 32, seed=8)
    Q = torch.randn((2 * n_q + 1, 4, 64), generator=g, device="cuda").bfloat16()
    params = L.Params.make(0.125)
    want = engine.paged_attention(Q, cache, batch, params)
    engine.synchronize()
    others = [Engine(0) for _ in range(2)]
    outs = [[torch.empty_like(Q) for _ in range(10)] for _ in others]
    for e in others:
        e.use_stream(torch.cuda.Stream())
        e.reserve(e.paged_attention_workspace_bytes(cache, batch, Q.shape[0], 4))
    torch.cuda.synchronize()
    for i in range(10):
        for e, o in zip(others, outs):
            e.paged_attention(Q, cache, batch, params, out=o[i])
    for e, os_ in zip(others, outs):
        e.synchronize()
        assert all(torch.equal(o, want) for o in os_)
        e.close()
