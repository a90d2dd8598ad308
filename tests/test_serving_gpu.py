"""The paged stack: prompts in chunks, single tokens and forks of several requests in one step, against a plain
composition of the layers with a rounding wherever the device stores 16 bits."""
import math

import pytest
import torch

from logos_b200 import lib as L
from logos_b200.paged import Rope
from logos_b200.serving import PagedStack
from logos_b200.stack import StackConfig, make_weights

CFG = StackConfig(vocab_size=512, d_model=256, num_heads=3, num_layers=2, max_seq_len=700, shunyam=False, navier_stokes=False)


def weights(cfg, device):
    w = make_weights(cfg, seed=3, std=0.05, device=device)
    g = torch.Generator().manual_seed(4)
    w["q_norm"], w["k_norm"] = ((1 + 0.2 * torch.randn((cfg.num_layers, 64), generator=g)).to(device) for _ in range(2))
    return w


def plain(cfg, w, ids, rope, eps):
    """Logits of every position of one sequence, fp64 with a BF16 rounding at the device's stores and the cache's INT8."""
    r16 = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    H, n = cfg.num_heads, len(ids)
    x = r16(w["embed"][torch.tensor(ids, device=w["embed"].device)])
    pos = torch.arange(n, device=x.device).double()
    ang = pos[:, None] * torch.tensor(rope.inv_freq, dtype=torch.float64, device=x.device)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    half = rope.dims // 2

    def turn(t, g):
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + eps) * g.double()
        a, b = t[..., :half], t[..., half:2 * half]
        return r16(torch.cat((a * c - b * s, b * c + a * s, t[..., 2 * half:]), -1))

    def through_cache(t):
        sc = (t.abs().amax(-1, keepdim=True) + 1e-8) / 127.5
        return (t / sc).round().clamp(-127, 127) * sc

    for l in range(cfg.num_layers):
        m = x.mean(-1, keepdim=True)
        xn = r16((x - m) * torch.rsqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-5) * w["ln_gamma"][l].double() + w["ln_beta"][l].double())
        q, k, v = (r16(torch.einsum("td,hdc->thc", xn, r16(w[name][l]))) for name in ("W_Q", "W_K", "W_V"))
        q, k, v = turn(q, w["q_norm"][l]), through_cache(turn(k, w["k_norm"][l])), through_cache(v)
        sc = torch.einsum("thc,shc->hts", q, k) / 8.0
        i = torch.arange(n, device=x.device)
        hidden = i[None, :] > i[:, None]
        if cfg.shunyam and n > cfg.window:
            hidden = hidden | ((i[None, :] < i[:, None] - cfg.window) & (i[None, :] % cfg.stride != 0))
        o = r16(torch.einsum("hts,shc->thc", torch.softmax(sc.masked_fill(hidden, -math.inf), -1), v))
        y = r16(torch.einsum("thc,hcd->td", o, r16(w["W_O"][l])))
        x = r16(y @ r16(w["W_proj"][l]) + x)
    return x @ r16(w["lm_head"])


def near(got, want, what):
    """Two layers of seven BF16 roundings each on either side, 2^-9 / sqrt(3) rms a rounding: sqrt(28) * 1.1e-3 = 6e-3 of
    the norm between the two sides if none is damped; three times that is the limit."""
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert rel < 2e-2, f"{what}: {rel}"


def test_refusals_without_a_device():
    with pytest.raises(ValueError):
        PagedStack(None, StackConfig(), {}, 4)
    with pytest.raises(ValueError):
        PagedStack(None, CFG, {}, 4, dtype=torch.float32)


def test_a_refused_step_takes_nothing():
    """Every refusal stands before the pages are taken and before the first kernel."""
    st = PagedStack(None, CFG, weights(CFG, "cpu"), 4)
    a, b = st.open(), st.open()
    for bad in ([(a, [1, CFG.vocab_size])], [(a, [1]), (b, [-1])], [(a, [])], [], [(a, [1]), (a, [2])], [(a, [1] * 701)]):
        with pytest.raises(ValueError):
            st.step(bad)
    with pytest.raises(MemoryError):
        st.step([(a, [1] * 200), (b, [2] * 100)])
    with pytest.raises(KeyError):
        st.step([(a, [1]), (77, [2])])
    assert st.pool.free_pages == 4 and st.pool.length(a) == st.pool.length(b) == 0


@pytest.mark.gpu
def test_chunks_steps_and_forks(engine):
    w = weights(CFG, "cuda")
    rope = Rope(64)
    st = PagedStack(engine, CFG, w, pages=45, page_size=16, rope=rope)
    g = torch.Generator().manual_seed(9)
    text = torch.randint(0, CFG.vocab_size, (600,), generator=g).tolist()
    a, b = st.open(), st.open()
    A, B = text[:150], text[200:241]
    got = st.step([(a, A), (b, B[:1])])                                # a prompt beside a first token
    wa, wb = plain(CFG, w, A, rope, st.eps), plain(CFG, w, B, rope, st.eps)
    near(got[0], wa[-1], "prompt")
    near(got[1], wb[0], "first token")
    near(st.step([(b, B[1:])])[0], wb[-1], "second chunk")
    c = st.fork(a)
    C = A + text[300:303]
    A = A + text[400:402]
    got = st.step([(c, C[150:]), (a, A[150:151]), (b, text[500:533])])  # three requests of three lengths
    near(got[0], plain(CFG, w, C, rope, st.eps)[-1], "fork")
    near(got[1], plain(CFG, w, A, rope, st.eps)[150], "original")
    near(got[2], plain(CFG, w, B + text[500:533], rope, st.eps)[-1], "other")
    near(st.step([(a, A[151:])])[0], plain(CFG, w, A, rope, st.eps)[-1], "one token")
    d = st.open()
    assert 16 * st.pool.free_pages < len(text) <= CFG.max_seq_len
    with pytest.raises(MemoryError):
        st.step([(d, text)])
    assert st.pool.length(d) == 0
    st.close(d)
    with pytest.raises(ValueError):
        st.step([(a, [])])
    with pytest.raises(ValueError):
        st.step([(a, text)])
    for s in (a, b, c):
        st.close(s)
    assert st.pool.free_pages == 45
    engine.synchronize()


@pytest.mark.gpu
def test_window_and_landmarks(engine):
    cfg = StackConfig(vocab_size=512, d_model=256, num_heads=3, num_layers=2, max_seq_len=700, shunyam=True, window=40, stride=16,
                      navier_stokes=False)
    w = weights(cfg, "cuda")
    rope = Rope(32, base=500.0)
    st = PagedStack(engine, cfg, w, pages=20, page_size=32, rope=rope)
    ids = torch.randint(0, cfg.vocab_size, (300,), generator=torch.Generator().manual_seed(2)).tolist()
    s = st.open()
    near(st.step([(s, ids[:260])])[0], plain(cfg, w, ids[:260], rope, st.eps)[-1], "prompt")
    # the window rule looks at the length so far: the later rows stand in a longer sequence, where nothing changes for them
    near(st.step([(s, ids[260:])])[0], plain(cfg, w, ids, rope, st.eps)[-1], "chunk")
    assert L.load_library() is engine.lib
