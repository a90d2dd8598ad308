"""Pages of INT8 keys and values that sequences of any length share, and the handles over them.

    PagedKVCache   one layer's pages: int8 [pages][H][page_size][DH] for K and for V, one fp32 scale per row
    PagePool       host-side bookkeeping: which pages a sequence holds, prompts shared between sequences
    PagedBatch     the new tokens of a batch of sequences, as the engine's paged calls take them
    Rope           frequencies of the position rotation

The reference keeps one contiguous INT8 tensor per head and re-makes it every forward (HeadCache,
cuda/ModelGPU.cuh:15-49); it has no pages.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import lib as L

PAGE_SIZES = (16, 32, 64, 128)


class Rope:
    """Rotation of the first `dims` channels of a head: frequency of pair k = base^(-2k/dims) / factor, or the `inv_freq`
    given.  interleaved: pairs (2k, 2k + 1) instead of (k, k + dims/2)."""

    def __init__(self, dims: int, base: float = 10000.0, interleaved: bool = False, factor: float = 1.0, inv_freq=None):
        if dims < 0 or dims % 16 or dims > 2 * L.ROPE_MAX_PAIRS:
            raise ValueError(f"Rope: dims = {dims} (a multiple of 16 up to {2 * L.ROPE_MAX_PAIRS})")
        f = [base ** (-2.0 * k / dims) / factor for k in range(dims // 2)] if inv_freq is None else [float(x) for x in inv_freq]
        if len(f) != dims // 2:
            raise ValueError(f"Rope: {len(f)} frequencies for {dims // 2} pairs")
        self.dims, self.interleaved, self.inv_freq = dims, bool(interleaved), tuple(f)
        self.desc = L.Rope(dims, int(bool(interleaved)), (C.c_double * L.ROPE_MAX_PAIRS)(*f))
        self.address = C.addressof(self.desc)


def _need(t: torch.Tensor, dtype, what: str):
    if t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous {dtype} tensor is needed, got {t.dtype} with strides {t.stride()}")


class PagedKVCache:
    """One layer's pages.  Rows are undefined until they are appended."""

    def __init__(self, pages: int, page_size: int, heads: int, dh: int, device="cuda"):
        if min(pages, heads) <= 0 or page_size not in PAGE_SIZES or dh not in (64, 128):
            raise ValueError(f"PagedKVCache: {pages} pages of {page_size} tokens, {heads} heads of {dh} "
                             f"(page size one of {PAGE_SIZES}, DH 64 or 128)")
        shape = (pages, heads, page_size, dh)
        self._over(torch.zeros(shape, dtype=torch.int8, device=device), torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.ones(shape[:3], dtype=torch.float32, device=device),
                   torch.ones(shape[:3], dtype=torch.float32, device=device))

    @classmethod
    def over(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> "PagedKVCache":
        """The cache over tensors the caller owns: int8 [pages, H, page_size, DH] twice, float32 [pages, H, page_size] twice."""
        c = cls.__new__(cls)
        c._over(k, v, k_scale, v_scale)
        return c

    def _over(self, k, v, ks, vs):
        for t, dt in ((k, torch.int8), (v, torch.int8), (ks, torch.float32), (vs, torch.float32)):
            _need(t, dt, "PagedKVCache")
        if k.dim() != 4 or k.shape != v.shape or ks.shape != k.shape[:3] or vs.shape != k.shape[:3]:
            raise ValueError(f"PagedKVCache: K {tuple(k.shape)}, V {tuple(v.shape)}, scales {tuple(ks.shape)}, {tuple(vs.shape)}")
        if len({t.device for t in (k, v, ks, vs)}) != 1:
            raise ValueError("PagedKVCache: tensors on several devices")
        self.k, self.v, self.ks, self.vs = k, v, ks, vs
        self.pages, self.heads, self.page_size, self.dh = k.shape
        self.desc = L.PagedCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), self.pages, self.page_size,
                                 self.heads, self.dh)
        self.address, self.device_index = C.addressof(self.desc), k.get_device()

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k, self.v, self.ks, self.vs))

    def copy_pages(self, src, dst):
        """Page src[i] -> page dst[i] (lists of page numbers); a shared page gets a copy of its own this way."""
        i = torch.as_tensor(src, dtype=torch.long, device=self.k.device)
        o = torch.as_tensor(dst, dtype=torch.long, device=self.k.device)
        for t in (self.k, self.v, self.ks, self.vs):
            t[o] = t[i]


class PagedBatch:
    """The device tables of a batch (int32: cu_q [B + 1], kv_len [B], page_table [B, max_pages]) with the bounds that
    size the launches: most new tokens and most held tokens of a sequence.  A captured graph may be replayed with
    new contents of the same tensors inside the same bounds."""

    def __init__(self, cu_q: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor, max_q: int, max_kv: int):
        for t in (cu_q, kv_len, page_table):
            _need(t, torch.int32, "PagedBatch")
        B = kv_len.numel()
        if cu_q.numel() != B + 1 or page_table.dim() != 2 or page_table.shape[0] != B:
            raise ValueError(f"PagedBatch: {B} sequences, cu_q of {cu_q.numel()}, page table {tuple(page_table.shape)}")
        if len({t.device for t in (cu_q, kv_len, page_table)}) != 1:
            raise ValueError("PagedBatch: tensors on several devices")
        self.cu_q, self.kv_len, self.page_table = cu_q, kv_len, page_table
        self.B, self.max_q, self.max_kv = B, int(max_q), int(max_kv)
        self.device_index = cu_q.get_device()
        self._over = (-1, None)

    def over(self, rows: int):
        """logos_paged_batch for token tensors of `rows` rows, by reference.  Another number of rows takes another descriptor:
        the one that a call on another thread holds stays as it is."""
        held, desc = self._over
        if held != rows:
            desc = C.byref(L.PagedBatch(self.cu_q.data_ptr(), self.kv_len.data_ptr(), self.page_table.data_ptr(), self.B,
                                        self.page_table.shape[1], rows, self.max_q, self.max_kv))
            self._over = (rows, desc)
        return desc

    def positions(self, rows: int) -> torch.Tensor:
        """int32 [rows]: the position of every token row (0 for rows behind the last sequence)."""
        r = torch.arange(rows, device=self.cu_q.device, dtype=torch.int32)
        if self.B == 0:
            return torch.zeros_like(r)
        b = torch.searchsorted(self.cu_q[1:], r, right=True).clamp(max=self.B - 1)
        p = self.kv_len[b] - self.cu_q[b + 1] + r
        return torch.where(r < self.cu_q[-1], p, 0).to(torch.int32)


class PagePool:
    """Which pages a sequence holds.  The page numbers hold for every layer's PagedKVCache alike."""

    def __init__(self, pages: int, page_size: int):
        if pages <= 0 or page_size not in PAGE_SIZES:
            raise ValueError(f"PagePool: {pages} pages of {page_size} tokens")
        self.page_size = page_size
        self._free = list(range(pages - 1, -1, -1))
        self._users = [0] * pages
        self._seqs: dict[int, list[int]] = {}
        self._len: dict[int, int] = {}
        self._next = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq: int) -> int:
        return self._len[seq]

    def pages_of(self, seq: int) -> list[int]:
        return list(self._seqs[seq])

    def open(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._seqs[seq], self._len[seq] = [], 0
        return seq

    def close(self, seq: int):
        for p in self._seqs.pop(seq):
            self._users[p] -= 1
            if self._users[p] == 0:
                self._free.append(p)
        del self._len[seq]

    def _take(self) -> int:
        p = self._free.pop()
        self._users[p] = 1
        return p

    def fork(self, seq: int, caches) -> int:
        """A new sequence that starts with `seq`'s tokens.  Full pages are shared; a page that is still being filled is
        copied in every one of `caches` (the layers' PagedKVCache), so that no two sequences ever write one page."""
        held, n = self._seqs[seq], self._len[seq]
        partial = n % self.page_size != 0
        if partial and not self._free:
            raise MemoryError("PagePool: no page left for the copy of a page that is being filled")
        new = self.open()
        full = held[: n // self.page_size]
        for p in full:
            self._users[p] += 1
        self._seqs[new] = list(full)
        if partial:
            p = self._take()
            for c in caches:
                c.copy_pages([held[n // self.page_size]], [p])
            self._seqs[new].append(p)
        self._len[new] = n
        return new

    def batch(self, new_tokens, device="cuda", max_q: int = 0, max_kv: int = 0) -> PagedBatch:
        """new_tokens: (sequence, count) pairs in the order of the token rows.  Takes the pages that the new tokens
        need and returns the batch, lengths after the append.  max_q / max_kv: larger bounds than this batch's own.
        Nothing is taken when the pool is too small for the whole batch (MemoryError)."""
        pairs = [(int(s), int(n)) for s, n in new_tokens]
        if len({s for s, _ in pairs}) != len(pairs):
            raise ValueError("PagePool.batch: a sequence is named twice")
        if any(n < 0 for _, n in pairs):
            raise ValueError("PagePool.batch: a negative number of tokens")
        grow = [-(-(self._len[s] + n) // self.page_size) - len(self._seqs[s]) for s, n in pairs]
        if sum(grow) > len(self._free):
            raise MemoryError(f"PagePool: {sum(grow)} pages wanted, {len(self._free)} free")
        cu, kv = [0], []
        for (s, n), more in zip(pairs, grow):
            self._seqs[s].extend(self._take() for _ in range(more))
            self._len[s] += n
            cu.append(cu[-1] + n)
            kv.append(self._len[s])
        max_kv = max([max_kv] + kv)
        max_q = max([max_q] + [n for _, n in pairs])
        width = max(1, -(-max_kv // self.page_size))
        table = torch.zeros((len(pairs), width), dtype=torch.int32)
        for i, (s, _) in enumerate(pairs):
            table[i, : len(self._seqs[s])] = torch.tensor(self._seqs[s], dtype=torch.int32)
        to = lambda x: torch.as_tensor(x, dtype=torch.int32).to(device)  # noqa: E731
        return PagedBatch(to(cu), to(kv), table.to(device), max_q, max_kv)
