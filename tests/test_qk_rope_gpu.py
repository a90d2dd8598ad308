"""Norm and rotation of queries and keys, and the backward pass, against 64-bit restatements.

Tolerances.  A stored value is off by half a step of its type, finfo.eps / 2 of itself, plus what fp32 arithmetic does
before: the row's factor r (a sum of at most 128 squares, an rsqrt), three products, an angle of at most pi held to
2^-24 of itself and a sine good to 2^-22 -- together below 2^-20 of |n_a| + |n_b|, the two channels of a pair."""
import math

import pytest
import torch

from logos_b200 import lib as L
from logos_b200.paged import Rope

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def pairs(rope, D):
    """(index of a, index of b, frequency) of every pair."""
    n = rope.dims // 2
    return [((2 * k, 2 * k + 1) if rope.interleaved else (k, k + n)) + (rope.inv_freq[k],) for k in range(n)]


def rotate64(n, pos, rope, sign=1.0):
    y = n.clone()
    for a, b, f in pairs(rope, n.shape[-1]):
        ang = pos.double() * f * sign
        c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
        y[..., a] = n[..., a] * c - n[..., b] * s
        y[..., b] = n[..., b] * c + n[..., a] * s
    return y


def partner_abs(n, rope):
    """|n_a| + |n_b| of each channel's pair; |n| of a channel that is not rotated."""
    m = n.abs()
    out = m.clone()
    for a, b, _ in pairs(rope, n.shape[-1]):
        out[..., a] = out[..., b] = m[..., a] + m[..., b]
    return out


def fwd64(x, w, pos, rope, eps):
    x = x.double()
    n = x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    return rotate64(n, pos, rope), partner_abs(n, rope)


def half_step(dt, want):
    """Half a step of the type at `want`.  Below the smallest normal value the steps stay smallest_normal * eps wide
    (fp16: 2^-14 * 2^-10 = 2^-24, so values under 2^-14 are off by up to 2^-25 however small they are)."""
    f = torch.finfo(dt)
    return f.eps / 2 * want.abs().clamp(min=f.smallest_normal)


def check(got, want, bound, what):
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), what
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert worst <= 0, f"{what}: {worst} beyond the bound (largest error {err.max().item()})"


def make(rows, H, D, dt, layout, g):
    x = torch.randn((rows, H, D), generator=g, device="cuda").to(dt)
    return x if layout == "tokens" else x.transpose(0, 1).contiguous().transpose(0, 1)


CASES = [  # rows, Hq, Hk, D, dims, interleaved, layout, dtype
    (1, 1, 1, 64, 64, False, "tokens", "bf16"), (33, 16, 16, 64, 64, False, "heads", "bf16"),
    (7, 8, 2, 128, 128, True, "tokens", "fp16"), (65, 3, 1, 128, 32, False, "heads", "fp32"),
    (131, 5, 5, 64, 16, True, "heads", "fp32"), (257, 12, 4, 128, 128, False, "tokens", "bf16"),
    (1000, 32, 8, 64, 48, False, "tokens", "fp16"), (40, 2, 2, 64, 0, False, "tokens", "bf16"),
    (3000, 40, 24, 64, 64, False, "tokens", "bf16"),
]


@pytest.mark.parametrize("rows,Hq,Hk,D,dims,inter,layout,dtype", CASES)
def test_forward(engine, rows, Hq, Hk, D, dims, inter, layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + D)
    dt = DT[dtype]
    Q, K = make(rows, Hq, D, dt, layout, g), make(rows, Hk, D, dt, layout, g)
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda", dtype=torch.int32)
    rope = Rope(dims, 10000.0, inter)
    yq, yk = engine.qk_norm_rope(Q, K, wq, wk, pos, rope, eps=1e-5)
    engine.synchronize()
    for x, w, y in ((Q, wq, yq), (K, wk, yk)):
        want, pair = fwd64(x, w, pos, rope, 1e-5)
        check(y, want, half_step(dt, want) + 2.0 ** -20 * pair, "forward")
    # the same bits in place, on the same layout
    Q2, K2 = Q.clone(memory_format=torch.preserve_format), K.clone(memory_format=torch.preserve_format)
    engine.qk_norm_rope(Q2, K2, wq, wk, pos, rope, eps=1e-5, out_q=Q2, out_k=K2)
    assert torch.equal(Q2, yq) and torch.equal(K2, yk)


def test_far_positions_and_no_norm(engine):
    """Angles at the ends of the position range (2^31 - 1, negative ones) and at pairs that hardly turn; no weights."""
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 - 1, -5, -(2 ** 31)], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    Q = torch.randn((6, 2, 64), generator=g, device="cuda")
    rope = Rope(64, 500000.0)
    y, none = engine.qk_norm_rope(Q, None, None, None, pos, rope)
    assert none is None
    want, pair = fwd64(Q, None, pos, rope, 0.0)
    # the double oracle's own angle is off by up to 2^31 * 2^-53; the frequency's 64-bit fixed point by 2^31 * 2^-64 turns
    check(y, want, 2.0 ** -24 * want.abs() + 2.0 ** -20 * pair, "far positions")
    assert torch.equal(y[0], Q[0])                       # position 0 does not turn


def test_zero_rows_and_empty_batch(engine):
    g = torch.Generator(device="cuda").manual_seed(4)
    Q = torch.randn((5, 3, 128), generator=g, device="cuda").bfloat16()
    Q[2] = 0
    w = torch.ones(128, device="cuda")
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    y, _ = engine.qk_norm_rope(Q, None, w, None, pos, Rope(128))
    assert torch.equal(y[2], torch.zeros_like(y[2])) and torch.isfinite(y).all()
    e = torch.empty((0, 3, 128), dtype=torch.bfloat16, device="cuda")
    y, _ = engine.qk_norm_rope(e, None, w, None, pos[:0], Rope(128))
    assert y.shape == e.shape
    dq, _, dw, _ = engine.qk_norm_rope_bwd(e, None, e, None, w, None, pos[:0], Rope(128))
    assert dq.shape == e.shape and torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.parametrize("rows,Hq,Hk,D,dims,inter,layout,dtype", CASES)
def test_backward(engine, rows, Hq, Hk, D, dims, inter, layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + D + 1)
    dt = DT[dtype]
    Q, K, gq, gk = (make(rows, h, D, dt, layout, g) for h in (Hq, Hk, Hq, Hk))
    wq, wk = (1 + 0.3 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, device="cuda", dtype=torch.int32)
    rope, eps = Rope(dims, 10000.0, inter), 1e-5
    dQ, dK, dwq, dwk = engine.qk_norm_rope_bwd(Q, K, gq, gk, wq, wk, pos, rope, eps=eps)
    for x, go, w, dx, dw in ((Q, gq, wq, dQ, dwq), (K, gk, wk, dK, dwk)):
        x, go, w = x.double(), go.double(), w.double()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
        gr = rotate64(go, pos, rope, -1.0)
        h = gr * w
        want = r * (h - x * r * r * (h * x).mean(-1, keepdim=True))
        # terms of the two sums: |h| of the pair and |x| r^2 mean|h x|
        pair = partner_abs(go, rope) * w.abs()
        size = r * (pair + x.abs() * r * r * (pair * x.abs()).mean(-1, keepdim=True))
        check(dx, want, half_step(dt, want) + 2.0 ** -19 * size, "dx")
        terms = (gr * x * r).sum((0, 1))
        # a thread adds at most 64 terms before the tree of 5 + 3 + 6 + 5 levels: under 128 roundings on any path
        bound = 128 * 2.0 ** -24 * (partner_abs(go, rope) * x.abs() * r).sum((0, 1))
        check(dw, terms, bound + 1e-30, "dw")
    again = engine.qk_norm_rope_bwd(Q, K, gq, gk, wq, wk, pos, rope, eps=eps)
    for a, b in zip((dQ, dK, dwq, dwk), again):
        assert torch.equal(a, b)


def test_backward_against_differences(engine):
    """d/dt of sum(g * f(x + t e)) and of the weights, by central differences of the 64-bit forward: step 1e-5, the
    truncation error is O(1e-10), so the bound is the kernel's fp32 one."""
    g = torch.Generator(device="cuda").manual_seed(9)
    rows, H, D = 3, 2, 64
    Q, go, e = (torch.randn((rows, H, D), generator=g, device="cuda") for _ in range(3))
    w, ew = (torch.randn(D, generator=g, device="cuda") for _ in range(2))
    pos = torch.tensor([0, 5, 90000], dtype=torch.int32, device="cuda")
    rope, eps = Rope(32, 10000.0, True), 1e-5
    dQ, _, dw, _ = engine.qk_norm_rope_bwd(Q, None, go, None, w, None, pos, rope, eps=eps)

    def f(x, wt):
        n = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * wt
        return (go.double() * rotate64(n, pos, rope)).sum().item()

    t = 1e-5
    num = (f(Q.double() + t * e.double(), w.double()) - f(Q.double() - t * e.double(), w.double())) / (2 * t)
    assert math.isclose(num, (dQ.double() * e.double()).sum().item(), rel_tol=0, abs_tol=2.0 ** -17 * (dQ.abs() * e.abs()).sum().item())
    num = (f(Q.double(), w.double() + t * ew.double()) - f(Q.double(), w.double() - t * ew.double())) / (2 * t)
    assert math.isclose(num, (dw.double() * ew.double()).sum().item(), rel_tol=0, abs_tol=2.0 ** -15 * (dw.abs() * ew.abs()).sum().item())


def test_backward_without_a_norm_turns_back(engine):
    g = torch.Generator(device="cuda").manual_seed(10)
    K, gk = (torch.randn((50, 4, 64), generator=g, device="cuda") for _ in range(2))
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    rope = Rope(64)
    none, dK, dwq, dwk = engine.qk_norm_rope_bwd(None, K, None, gk, None, None, pos, rope)
    assert none is None and dwq is None and dwk is None
    check(dK, rotate64(gk.double(), pos, rope, -1.0), 2.0 ** -24 * gk.abs().double() + 2.0 ** -20 * partner_abs(gk.double(), rope), "dK")


def test_refusals(engine):
    Q = torch.zeros((4, 2, 64), device="cuda", dtype=torch.bfloat16)
    w, pos, rope = torch.ones(64, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda"), Rope(64)
    for bad in (lambda: engine.qk_norm_rope(Q, Q.float(), w, w, pos, rope),
                lambda: engine.qk_norm_rope(Q, None, w.half(), None, pos, rope),
                lambda: engine.qk_norm_rope(Q, None, w, None, pos.long(), rope),
                lambda: engine.qk_norm_rope(Q, None, w, None, pos[:3], rope),
                lambda: engine.qk_norm_rope(Q.cpu(), None, w, None, pos, rope),
                lambda: engine.qk_norm_rope(Q.transpose(1, 2), None, w, None, pos, rope),
                lambda: engine.qk_norm_rope(None, None, None, None, pos, rope),
                lambda: engine.qk_norm_rope(Q, None, w, None, pos, rope, out_q=torch.zeros_like(Q)[:, :1]),
                lambda: engine.qk_norm_rope_bwd(Q, None, Q[:, :1], None, w, None, pos, rope)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(L.LogosError) as e:
        engine.qk_norm_rope(Q, None, w, None, pos, Rope(128))
    assert e.value.status == L.ERR_INVALID_ARG
    with pytest.raises(L.LogosError) as e:
        engine.qk_norm_rope(torch.zeros((4, 2, 96), device="cuda"), None, None, None, pos, Rope(64))
    assert e.value.status == L.ERR_UNSUPPORTED
