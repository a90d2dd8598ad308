"""Cases of the operators around the paged INT8 key/value cache.

  rope       per-head RMS norm and position rotation of queries and keys in one pass
  rope_grad  its backward pass: gradients of queries, keys and the two norm weights
  append     new tokens' keys and values quantised into their pages, and what the cache then holds for them read back
  read       sequences read back from their pages
  attend     attention of new tokens (one or many per sequence) over the paged cache

`run` computes a case in elementary torch operations where `own` is False, and through the engine where it is True.
"""
import math

import torch

own = False

_ENGINE = []
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decode step of 32 sequences: latency
        dict(name="rope_step", op="rope", tokens=32, hq=16, hk=16, d=64, dims=64, pair="halves", layout="tokens", dtype="bf16"),
        # the prompts of 32 x 2048 tokens, laid out as the projection writes them
        dict(name="rope_prompts", op="rope", tokens=65536, hq=16, hk=16, d=64, dims=64, pair="halves", layout="heads", dtype="bf16"),
        # a training batch, grouped heads
        dict(name="rope_grad_batch", op="rope_grad", tokens=16384, hq=32, hk=8, d=128, dims=128, pair="halves", layout="tokens", dtype="bf16"),
        # an odd short batch, rotation of half the channels in neighbouring pairs
        dict(name="rope_grad_odd", op="rope_grad", tokens=1237, hq=16, hk=16, d=64, dims=32, pair="neighbours", layout="heads", dtype="fp16"),
        # the new rows of one decode step of 64 sequences
        dict(name="append_step", op="append", seqs=64, q_min=1, q_max=1, kv_max=8192, h=16, d=64, page=64, layout="tokens", dtype="bf16", pad=0),
        # ragged prompts going into a cache, some rows of padding behind the last one
        dict(name="append_prompts", op="append", seqs=16, q_min=700, q_max=4001, kv_max=4200, h=16, d=64, page=64, layout="heads", dtype="bf16", pad=37),
        # a few short sequences taken out in 32 bits
        dict(name="read_short", op="read", seqs=3, q_min=50, q_max=413, kv_max=413, h=8, d=128, page=16, layout="tokens", dtype="fp32", pad=0),
        # a batch of sequences read back for another consumer
        dict(name="read_batch", op="read", seqs=32, q_min=900, q_max=4096, kv_max=4096, h=16, d=64, page=64, layout="heads", dtype="bf16", pad=0),
        # decode at 8192 cached tokens, 64 sequences x 16 heads
        dict(name="attend_step", op="attend", seqs=64, q_min=1, q_max=1, kv_min=8192, kv_max=8192, hq=16, hk=16, d=64, page=64, window=0, stride=0, layout="tokens", dtype="fp16", pad=0),
        # decode of a few sequences with grouped heads and uneven contexts: latency
        dict(name="attend_step_few", op="attend", seqs=4, q_min=1, q_max=1, kv_min=500, kv_max=9001, hq=32, hk=8, d=128, page=16, window=0, stride=0, layout="tokens", dtype="bf16", pad=0),
        # one long chunk of a prompt over what is cached already
        dict(name="attend_chunk", op="attend", seqs=1, q_min=2048, q_max=2048, kv_min=16384, kv_max=16384, hq=32, hk=8, d=128, page=64, window=0, stride=0, layout="tokens", dtype="bf16", pad=0),
        # chunks and single tokens of different requests in one call
        dict(name="attend_mixed", op="attend", seqs=12, q_min=1, q_max=517, kv_min=600, kv_max=6001, hq=16, hk=16, d=64, page=64, window=0, stride=0, layout="heads", dtype="bf16", pad=11),
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))

    op = rng.choice(["rope", "rope_grad", "append", "read", "attend", "attend"])
    d = rng.choice([64, 128])
    layout = rng.choice(["tokens", "heads"])
    if op in ("rope", "rope_grad"):
        hk = rng.choice([1, 2, 4, 8, 16])
        hq = hk * rng.choice([1, 2, 3, 4, 8] if hk <= 4 else [1, 2])
        most = (1 << 26 if op == "rope" else 1 << 25) // (d * (hq + hk))
        return dict(op=op, tokens=spread(1, min(most, 60000)), hq=hq, hk=hk, d=d, dims=rng.choice([d, d // 2, d // 4]),
                    pair=rng.choice(["halves", "neighbours"]), layout=layout, dtype=rng.choice(["bf16", "fp16", "fp32"]))
    page = rng.choice([16, 32, 64, 128])
    if op in ("append", "read"):
        h = rng.choice([1, 2, 4, 8, 16])
        seqs = spread(1, 64)
        q_max = spread(1, max(1, min(4000, (1 << 25) // (h * d * seqs))))
        kv_max = q_max + rng.choice([0, 1, spread(1, 2000)])
        return dict(op=op, seqs=seqs, q_min=min(q_max, spread(1, q_max)), q_max=q_max, kv_max=kv_max, h=h, d=d, page=page,
                    layout=layout, dtype=rng.choice(["bf16", "fp16", "fp32"]), pad=rng.choice([0, 1, 19]))
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 3, 4, 8])
    if rng.random() < 0.5:                       # single tokens (or the few of a speculative step)
        q_max = rng.choice([1, 1, 1, 2, 3, 5])
        seqs = spread(1, 64)
        kv_max = spread(q_max, min(32000, max(64, (1 << 27) // (seqs * hk * d))))
    else:                                        # chunks
        seqs = spread(1, 8)
        q_max = spread(2, 1500)
        kv_max = spread(q_max, max(q_max, min(12000, (1 << 28) // (seqs * hq * q_max))))
    window, stride = rng.choice([(0, 0), (0, 0), (spread(1, kv_max), 0), (spread(1, kv_max), rng.choice([3, 16, 64]))])
    return dict(op=op, seqs=seqs, q_min=min(q_max, spread(1, q_max)), q_max=q_max, kv_min=spread(q_max, kv_max), kv_max=kv_max,
                hq=hq, hk=hk, d=d, page=page, window=window, stride=stride, layout=layout, dtype=rng.choice(["bf16", "fp16"]),
                pad=rng.choice([0, 1, 19]))


def _lengths(case):
    """New tokens and cached tokens (the new ones included) of each sequence, host lists: part of the case, as its sizes are."""
    g = torch.Generator().manual_seed(17)
    n = case["seqs"]
    q = torch.randint(case["q_min"], case["q_max"] + 1, (n,), generator=g)
    q[-1] = case["q_max"]
    if case["op"] == "attend":
        kv = torch.maximum(torch.randint(case["kv_min"], case["kv_max"] + 1, (n,), generator=g), q)
        kv[-1] = case["kv_max"]
    elif case["op"] == "read":
        kv = torch.minimum(q + torch.randint(0, 40, (n,), generator=g), torch.tensor(case["kv_max"]))
    else:
        kv = q + torch.randint(0, case["kv_max"] - case["q_max"] + 1, (n,), generator=g)
    return q.tolist(), kv.tolist()


def _heads(x, layout):
    """The same values as a [tokens, heads, channels] view of a tensor that lies token by token or head by head."""
    return x if layout == "tokens" else x.transpose(0, 1).contiguous().transpose(0, 1)


def _noise(g, *shape):
    """Activations: normal, a few channels larger."""
    x = torch.randn(shape, generator=g, device="cuda")
    x[..., :: 29] *= 4.0
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    s = {"case": dict(case)}
    d = case["d"]
    if case["op"] in ("rope", "rope_grad"):
        t = case["tokens"]
        s["q"] = _heads(_noise(g, t, case["hq"], d).to(dt), case["layout"])
        s["k"] = _heads(_noise(g, t, case["hk"], d).to(dt), case["layout"])
        s["wq"] = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")
        s["wk"] = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")
        s["positions"] = torch.randint(0, 131072, (t,), generator=g, device="cuda", dtype=torch.int32)
        s["base"], s["eps"] = 10000.0, 1e-6
        k = torch.arange(case["dims"] // 2, dtype=torch.float64)
        s["freq"] = (s["base"] ** (-2.0 * k / case["dims"])).cuda()
        if case["op"] == "rope_grad":
            s["dq"] = _heads(torch.randn((t, case["hq"], d), generator=g, device="cuda").to(dt), case["layout"])
            s["dk"] = _heads(torch.randn((t, case["hk"], d), generator=g, device="cuda").to(dt), case["layout"])
        return s
    n_q, n_kv = _lengths(case)
    page, n = case["page"], case["seqs"]
    h = case["hk"] if case["op"] == "attend" else case["h"]
    per = [-(-x // page) for x in n_kv]
    total_pages = sum(per) + 3
    order = torch.randperm(total_pages, generator=torch.Generator().manual_seed(seed + 5)).tolist()
    table = torch.full((n, max(per)), -1, dtype=torch.int32)
    at = 0
    for b in range(n):
        table[b, : per[b]] = torch.tensor(order[at: at + per[b]], dtype=torch.int32)
        at += per[b]
    s["table"] = table.cuda()
    cu = [0]
    for x in n_q:
        cu.append(cu[-1] + x)
    s["cu_q"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    s["kv_len"] = torch.tensor(n_kv, dtype=torch.int32, device="cuda")
    s["rows"], s["total"], s["max_q"], s["max_kv"] = cu[-1], cu[-1] + case["pad"], max(n_q), max(n_kv)
    # sequence and position of every new token
    seq = torch.repeat_interleave(torch.arange(n), torch.tensor(n_q))
    idx = torch.arange(cu[-1]) - torch.tensor(cu)[seq]
    pos = torch.tensor(n_kv)[seq] - torch.tensor(n_q)[seq] + idx
    s["seq"], s["idx"], s["pos"] = seq.cuda(), idx.cuda(), pos.cuda()
    shape = (total_pages, h, page, d)
    s["k8"] = torch.zeros(shape, dtype=torch.int8, device="cuda")
    s["v8"] = torch.zeros(shape, dtype=torch.int8, device="cuda")
    s["ks"] = torch.full(shape[:3], 0.5, device="cuda")
    s["vs"] = torch.full(shape[:3], 0.25, device="cuda")
    if case["op"] != "append":                   # a cache that is in use
        for c8, cs in ((s["k8"], s["ks"]), (s["v8"], s["vs"])):
            x = _noise(g, *shape)
            cs.copy_((x.abs().amax(-1) + 1e-8) / 127.5)
            c8.copy_(torch.clamp(torch.round(x.div_(cs[..., None])), -127, 127))
            del x
    if case["op"] == "append":
        s["k"] = _heads(_noise(g, s["total"], h, d).to(dt), case["layout"])
        s["v"] = _heads(_noise(g, s["total"], h, d).to(dt), case["layout"])
    if case["op"] in ("append", "read"):
        s["k_out"] = _heads(torch.zeros((s["total"], h, d), dtype=dt, device="cuda"), case["layout"])
        s["v_out"] = _heads(torch.zeros((s["total"], h, d), dtype=dt, device="cuda"), case["layout"])
    if case["op"] == "attend":
        s["q"] = _heads(_noise(g, s["total"], case["hq"], d).to(dt), case["layout"])
        s["out"] = _heads(torch.zeros((s["total"], case["hq"], d), dtype=dt, device="cuda"), case["layout"])
        s["scale"] = d ** -0.5
    return s


# ---- the plain form ---------------------------------------------------------------------------------------------

def _pairs(x, dims, pair):
    """The two halves of every rotated pair, and the channels that are not rotated."""
    r = x[..., :dims]
    if pair == "halves":
        return r[..., : dims // 2], r[..., dims // 2:], x[..., dims:]
    return r[..., 0::2], r[..., 1::2], x[..., dims:]


def _unpair(a, b, rest, pair):
    r = torch.cat((a, b), -1) if pair == "halves" else torch.stack((a, b), -1).flatten(-2)
    return torch.cat((r, rest), -1)


def _angles(s):
    angle = s["positions"].double()[:, None, None] * s["freq"]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rope_plain(x, w, cos, sin, s):
    c = s["case"]
    f = x.float()
    n = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + s["eps"]) * w
    a, b, rest = _pairs(n, c["dims"], c["pair"])
    return _unpair(a * cos - b * sin, b * cos + a * sin, rest, c["pair"]).to(x.dtype)


def _rope_grad_plain(x, dy, w, cos, sin, s):
    c = s["case"]
    f, g = x.float(), dy.float()
    r = torch.rsqrt((f * f).mean(-1, keepdim=True) + s["eps"])
    a, b, rest = _pairs(g, c["dims"], c["pair"])
    g = _unpair(a * cos + b * sin, b * cos - a * sin, rest, c["pair"])
    dw = (g * f * r).sum((0, 1), dtype=torch.float64).float()
    h = g * w
    return (r * (h - f * r * r * (h * f).mean(-1, keepdim=True))).to(x.dtype), dw


def _slots(s):
    """Page and row in the page of every new token."""
    page = s["case"]["page"]
    return s["table"][s["seq"], s["pos"] // page].long(), s["pos"] % page


def _append_plain(s):
    page, off = _slots(s)
    steps = torch.full((), 127.5, device="cuda")
    for new, c8, cs in ((s["k"], s["k8"], s["ks"]), (s["v"], s["v8"], s["vs"])):
        x = new[: s["rows"]].float()
        scale = (x.abs().amax(-1) + 1e-8) / steps
        c8[page, :, off] = torch.clamp(torch.round(x / scale[..., None]), -127, 127).to(torch.int8)
        cs[page, :, off] = scale


def _read_plain(s):
    page, off = _slots(s)
    for out, c8, cs in ((s["k_out"], s["k8"], s["ks"]), (s["v_out"], s["v8"], s["vs"])):
        out[: s["rows"]] = (c8[page, :, off].float() * cs[page, :, off][..., None]).to(out.dtype)


def _attend_plain(s):
    c = s["case"]
    n, hk, d, page = c["seqs"], c["hk"], c["d"], c["page"]
    group = c["hq"] // hk
    j = torch.arange(s["max_kv"], device="cuda")
    i = torch.arange(s["max_q"], device="cuda")
    at, off = s["table"][:, j // page].clamp(min=0).long(), (j % page).expand(n, -1)
    n_q = s["cu_q"][1:] - s["cu_q"][:-1]
    pos = (s["kv_len"] - n_q)[:, None] + i                                      # [n, max_q]
    seen = (j <= pos[:, :, None]) & (j < s["kv_len"][:, None, None])
    if c["window"] > 0:
        near = j >= pos[:, :, None] - c["window"]
        if c["stride"] > 0:
            near = near | (j % c["stride"] == 0)
        seen = seen & (near | (s["kv_len"] <= c["window"])[:, None, None])
    rows = (s["cu_q"][:-1, None] + i).clamp(max=s["total"] - 1).long()
    q = s["q"][rows].float().view(n, s["max_q"], hk, group, d).permute(0, 2, 3, 1, 4).reshape(n, hk, group * s["max_q"], d)
    k = (s["k8"][at, :, off].float() * s["ks"][at, :, off][..., None]).permute(0, 2, 3, 1)     # [n, hk, d, max_kv]
    score = (torch.matmul(q, k) * s["scale"]).view(n, hk, group, s["max_q"], s["max_kv"])
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    score = torch.exp(score - top)
    total = score.sum(-1, keepdim=True).clamp(min=1e-30)
    v = (s["v8"][at, :, off].float() * s["vs"][at, :, off][..., None]).permute(0, 2, 1, 3)     # [n, hk, max_kv, d]
    o = torch.matmul(score.view(n, hk, group * s["max_q"], s["max_kv"]), v).view(n, hk, group, s["max_q"], d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s["max_q"], c["hq"], d)
    s["out"][: s["rows"]] = o[s["seq"], s["idx"]].to(s["out"].dtype)
    return s["out"]


# ---- the engine's calls -----------------------------------------------------------------------------------------

def _engine(s):
    """The engine, and the handles over this state's tensors that a serving loop keeps."""
    from logos_b200 import lib as L
    from logos_b200.engine import Engine
    from logos_b200.paged import PagedBatch, PagedKVCache, Rope

    if not _ENGINE:
        _ENGINE.append(Engine())
    if "handles" not in s:
        c = s["case"]
        if c["op"] in ("rope", "rope_grad"):
            s["handles"] = (Rope(c["dims"], s["base"], interleaved=c["pair"] == "neighbours"),)
        else:
            cache = PagedKVCache.over(s["k8"], s["v8"], s["ks"], s["vs"])
            batch = PagedBatch(s["cu_q"], s["kv_len"], s["table"], max_q=s["max_q"], max_kv=s["max_kv"])
            params = L.Params.make(s["scale"], True, c["window"], c["stride"]) if c["op"] == "attend" else None
            s["handles"] = (cache, batch, params)
    return _ENGINE[0], s["handles"]


def run(s):
    c = s["case"]
    if own:
        eng, handles = _engine(s)
        if c["op"] == "rope":
            return eng.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["positions"], handles[0], eps=s["eps"])
        if c["op"] == "rope_grad":
            return eng.qk_norm_rope_bwd(s["q"], s["k"], s["dq"], s["dk"], s["wq"], s["wk"], s["positions"], handles[0],
                                        eps=s["eps"])
        cache, batch, params = handles
        if c["op"] == "append":
            eng.paged_append(s["k"], s["v"], cache, batch)
            eng.paged_read(cache, batch, s["k_out"], s["v_out"])
            return s["k_out"], s["v_out"], s["ks"], s["vs"]
        if c["op"] == "read":
            eng.paged_read(cache, batch, s["k_out"], s["v_out"])
            return s["k_out"], s["v_out"]
        return eng.paged_attention(s["q"], cache, batch, params, out=s["out"])
    if c["op"] == "rope":
        cos, sin = _angles(s)
        return _rope_plain(s["q"], s["wq"], cos, sin, s), _rope_plain(s["k"], s["wk"], cos, sin, s)
    if c["op"] == "rope_grad":
        cos, sin = _angles(s)
        dq, dwq = _rope_grad_plain(s["q"], s["dq"], s["wq"], cos, sin, s)
        dk, dwk = _rope_grad_plain(s["k"], s["dk"], s["wk"], cos, sin, s)
        return dq, dk, dwq, dwk
    if c["op"] == "append":
        _append_plain(s)
        _read_plain(s)
        return s["k_out"], s["v_out"], s["ks"], s["vs"]
    if c["op"] == "read":
        _read_plain(s)
        return s["k_out"], s["v_out"]
    return _attend_plain(s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------

def _reach(case):
    """Sums over the sequences: cached tokens that some new token sees, (new token, cached token) pairs it sees, new tokens."""
    n_q, n_kv = _lengths(case)
    tokens = pairs = 0
    for q, kv in zip(n_q, n_kv):
        p = torch.arange(kv - q, kv, dtype=torch.int64)
        if 0 < case["window"] < kv:
            lo = (p - case["window"]).clamp(min=0)
            marks = torch.div(lo + case["stride"] - 1, case["stride"], rounding_mode="floor") if case["stride"] > 0 else lo * 0
            pairs += int((p - lo + 1 + marks).sum())
            tokens += kv - int(lo[0]) + int(marks[0])
        else:
            pairs += int((p + 1).sum())
            tokens += kv
    return tokens, pairs, sum(n_q)


def work(case):
    e = _DTYPES[case["dtype"]].itemsize
    d = case["d"]
    if case["op"] in ("rope", "rope_grad"):
        row = (case["hq"] + case["hk"]) * d
        n = case["tokens"] * row
        if case["op"] == "rope":
            return {"bytes": 2 * n * e + 4 * case["tokens"] + 8 * d, "flops": 7 * n}
        return {"bytes": 3 * n * e + 4 * case["tokens"] + 16 * d, "flops": 14 * n}
    if case["op"] in ("append", "read"):
        t = sum(_lengths(case)[0])
        n = 2 * t * case["h"]
        # append: the new rows in, the pages' rows and scales out and the values out; read: rows and scales in, values out
        return {"bytes": n * (d * (2 * e + 1) + 4) if case["op"] == "append" else n * (d * (e + 1) + 4), "flops": 2 * n * d}
    tokens, pairs, new = _reach(case)
    return {"bytes": tokens * case["hk"] * (2 * d + 8) + 2 * new * case["hq"] * d * e, "flops": 4 * pairs * case["hq"] * d}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------

def _rotate64(x, positions, freq, dims, pair, sign):
    out = x.clone()
    angle = positions.double().view(-1, 1) * freq.view(1, -1) * sign
    for k in range(dims // 2):
        i, j = (k, k + dims // 2) if pair == "halves" else (2 * k, 2 * k + 1)
        c, z = torch.cos(angle[:, k]).view(-1, 1), torch.sin(angle[:, k]).view(-1, 1)
        out[..., i] = x[..., i] * c - x[..., j] * z
        out[..., j] = x[..., i] * z + x[..., j] * c
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op, d = case["op"], case["d"]
    if op in ("rope", "rope_grad"):
        freq = torch.tensor([s["base"] ** (-2.0 * k / case["dims"]) for k in range(case["dims"] // 2)], dtype=torch.float64, device="cuda")
        outs, weights = [], []
        for x, w, dy in ((s["q"], s["wq"], s.get("dq")), (s["k"], s["wk"], s.get("dk"))):
            x, w = x.double(), w.double()
            norm = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / d + s["eps"])
            u = x / norm
            if op == "rope":
                outs.append(_rotate64(u * w, s["positions"], freq, case["dims"], case["pair"], 1.0))
            else:
                g = _rotate64(dy.double(), s["positions"], freq, case["dims"], case["pair"], -1.0)
                weights.append((g * u).sum(0).sum(0))
                gw = g * w
                outs.append((gw - u * (gw * u).sum(-1, keepdim=True) / d) / norm)
        return tuple(outs + weights)
    n_q, n_kv = _lengths(case)
    table = s["table"].cpu()
    page = case["page"]
    if op in ("append", "read"):
        k_out, v_out = torch.zeros_like(s["k_out"], dtype=torch.float64), torch.zeros_like(s["v_out"], dtype=torch.float64)
        ks, vs = s["ks"].double(), s["vs"].double()
        row = 0
        for b in range(case["seqs"]):
            p = torch.arange(n_kv[b] - n_q[b], n_kv[b])
            where, off = table[b][p // page].long().cuda(), (p % page).cuda()
            here = slice(row, row + n_q[b])
            row += n_q[b]
            for new, c8, cs, out in ((s.get("k"), s["k8"], ks, k_out), (s.get("v"), s["v8"], vs, v_out)):
                if op == "append":
                    x = new[here].double()
                    scale = (x.abs().max(-1).values + 1e-8) / 127.5
                    cs[where, :, off] = scale
                    out[here] = torch.round(x / scale.unsqueeze(-1)).clamp(-127, 127) * scale.unsqueeze(-1)
                else:
                    out[here] = c8[where, :, off].double() * cs[where, :, off].unsqueeze(-1)
        return (k_out, v_out, ks, vs) if op == "append" else (k_out, v_out)
    out = torch.zeros_like(s["out"], dtype=torch.float64)
    group = case["hq"] // case["hk"]
    row = 0
    for b in range(case["seqs"]):
        t, length = n_q[b], n_kv[b]
        p = torch.arange(length)
        where, off = table[b][p // page].long().cuda(), (p % page).cuda()
        k = s["k8"][where, :, off].double() * s["ks"][where, :, off].double().unsqueeze(-1)      # [length, hk, d]
        v = s["v8"][where, :, off].double() * s["vs"][where, :, off].double().unsqueeze(-1)
        i = torch.arange(length - t, length, device="cuda").view(-1, 1)
        j = torch.arange(length, device="cuda").view(1, -1)
        hidden = j > i
        if 0 < case["window"] < length:
            far = j < i - case["window"]
            hidden = hidden | (far & (j % case["stride"] != 0) if case["stride"] > 0 else far)
        for h in range(case["hq"]):
            q = s["q"][row: row + t, h].double()
            a = torch.softmax((q @ k[:, h // group].t() * s["scale"]).masked_fill(hidden, -math.inf), -1)
            out[row: row + t, h] = a @ v[:, h // group]
        row += t
    return out
