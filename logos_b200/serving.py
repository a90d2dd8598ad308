"""The attention stack over pages: requests of any length, several new tokens per sequence and step.

`AttentionStack` (stack.py) decodes a fixed batch, one token per sequence, from one contiguous cache; its sequences all have
a slot of the longest length.  Here sequences come and go, share prompts, take prompts in chunks, and one step
holds chunks and single tokens of different requests side by side; memory is taken page by page.  Per layer, for
all the step's rows at once: LayerNorm, the fused Q/K/V projection, norm and rotation of queries and keys in place, the
quantising append, attention over the pages, W_O read from the head-major output, W_proj with the residual.

Positions enter by rotation (the reference adds them to the embedding, cuda/ModelGPU.cu:743-771); the Navier-Stokes
terms are not offered over pages.  One GPU.
"""
from __future__ import annotations

import math

import torch

from . import lib as L
from .engine import Engine
from .paged import PagedKVCache, PagePool, Rope
from .stack import StackConfig


class PagedStack:
    """weights: as make_weights (stack.py) lays them out, with optional "q_norm" and "k_norm" ([layers, 64] fp32)."""

    def __init__(self, engine: Engine, cfg: StackConfig, weights: dict, pages: int, page_size: int = 64,
                 rope: Rope | None = None, eps: float = 1e-6, dtype=torch.bfloat16):
        if cfg.navier_stokes:
            raise ValueError("PagedStack: the Navier-Stokes terms are not offered over pages (StackConfig.navier_stokes)")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"PagedStack: {dtype} (BF16 or FP16)")
        self.eng, self.cfg, self.dtype, self.eps = engine, cfg, dtype, eps
        H, D = cfg.num_heads, cfg.d_model
        w, sh = weights, lambda t: t.to(dtype).contiguous()
        self.Wt_qkv = [sh(torch.cat([w[k][l].transpose(1, 2).reshape(H * 64, D) for k in ("W_Q", "W_K", "W_V")]))
                       for l in range(cfg.num_layers)]
        self.Wt_o = [sh(w["W_O"][l].reshape(H * 64, D).t()) for l in range(cfg.num_layers)]
        self.Wt_proj = [sh(w["W_proj"][l].t()) for l in range(cfg.num_layers)]
        self.Wt_lm = sh(w["lm_head"].t())
        self.embed = w["embed"].to(dtype)
        self.ln_g, self.ln_b = w["ln_gamma"].float(), w["ln_beta"].float()
        norm = lambda k, l: w[k][l].float().contiguous() if k in w else None  # noqa: E731
        self.q_norm = [norm("q_norm", l) for l in range(cfg.num_layers)]
        self.k_norm = [norm("k_norm", l) for l in range(cfg.num_layers)]
        self.rope = Rope(64) if rope is None else rope
        self.pool = PagePool(pages, page_size)
        self.caches = [PagedKVCache(pages, page_size, H, 64, device=self.embed.device) for _ in range(cfg.num_layers)]
        self.params = L.Params.make(1.0 / math.sqrt(64.0), True, cfg.window if cfg.shunyam else 0, cfg.stride)

    def open(self) -> int:
        return self.pool.open()

    def fork(self, seq: int) -> int:
        """A new sequence that starts with `seq`'s tokens (full pages shared, the open one copied)."""
        return self.pool.fork(seq, self.caches)

    def close(self, seq: int):
        self.pool.close(seq)

    def step(self, requests) -> torch.Tensor:
        """requests: (sequence, its new token ids) pairs, at least one token each -> logits of every sequence's last token,
        [len(requests), vocabulary] fp32.  Raises MemoryError, with nothing changed, when the pages do not suffice."""
        requests = [(seq, list(ids)) for seq, ids in requests]
        if not requests or any(not ids for _, ids in requests):
            raise ValueError("PagedStack.step: every request brings at least one token")
        tokens = [int(t) for _, ids in requests for t in ids]
        if min(tokens) < 0 or max(tokens) >= self.embed.shape[0]:
            raise ValueError(f"PagedStack.step: a token outside the vocabulary of {self.embed.shape[0]}")
        longest = max(self.pool.length(seq) + len(ids) for seq, ids in requests)
        if longest > self.cfg.max_seq_len:
            raise ValueError(f"PagedStack.step: {longest} tokens in a sequence, the model takes {self.cfg.max_seq_len}")
        cfg, eng, dev = self.cfg, self.eng, self.embed.device
        batch = self.pool.batch([(seq, len(ids)) for seq, ids in requests], device=dev)
        rows = len(tokens)
        positions = batch.positions(rows)
        x = self.embed[torch.tensor(tokens, dtype=torch.long, device=dev)]
        heads = torch.empty((1, cfg.num_heads, rows, 64), dtype=self.dtype, device=dev)
        for l in range(cfg.num_layers):
            xn = eng.layer_norm(x, self.ln_g[l], self.ln_b[l], 1e-5)
            q, k, v = (t[0].transpose(0, 1) for t in eng.qkv_project(xn, self.Wt_qkv[l], 1, rows, cfg.num_heads))   # [rows, H, 64]
            eng.qk_norm_rope(q, k, self.q_norm[l], self.k_norm[l], positions, self.rope, eps=self.eps, out_q=q, out_k=k)
            eng.paged_append(k, v, self.caches[l], batch)
            eng.paged_attention(q, self.caches[l], batch, self.params, out=heads[0].transpose(0, 1))
            y = eng.project_heads(heads, self.Wt_o[l])
            x = eng.project(y, self.Wt_proj[l], residual=x)
        last = x[(batch.cu_q[1:] - 1).long()]
        return eng.project(last.contiguous(), self.Wt_lm, out_dtype=torch.float32)
