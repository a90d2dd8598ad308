"""The paged cache without a GPU: refusals of the C ABI and the kernels' table arithmetic (compiled as host code), the
page pool, the handles."""
import os
import subprocess

import pytest
import torch

from logos_b200 import lib as L
from logos_b200.paged import PagedBatch, PagedKVCache, PagePool, Rope

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


def test_refusals_and_table_arithmetic(tmp_path):
    """Every refusal stands before the first CUDA call, and tables that hold anything never lead outside the tensors."""
    from logos_b200.build import PKG, build
    build()
    exe = str(tmp_path / "paged_host_check")
    subprocess.run(["nvcc", "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "--cudart", "static",
                    "-o", exe, os.path.join(ROOT, "tests", "paged_host_check.cu"), "-L" + PKG, "-llogos_attn",
                    "-Xlinker", "-rpath=" + PKG], check=True, capture_output=True, text=True)
    r = subprocess.run([exe], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_pool_takes_and_returns_pages():
    pool = PagePool(6, 16)
    a, b = pool.open(), pool.open()
    batch = pool.batch([(a, 17), (b, 16)], device="cpu")
    assert batch.cu_q.tolist() == [0, 17, 33] and batch.kv_len.tolist() == [17, 16]
    assert (batch.max_q, batch.max_kv) == (17, 17) and batch.page_table.shape == (2, 2)
    assert pool.free_pages == 3 and len(pool.pages_of(a)) == 2 and len(pool.pages_of(b)) == 1
    assert not set(pool.pages_of(a)) & set(pool.pages_of(b))
    batch = pool.batch([(b, 1), (a, 0)], device="cpu", max_q=4, max_kv=64)
    assert batch.kv_len.tolist() == [17, 17] and batch.max_q == 4 and batch.page_table.shape == (2, 4)
    with pytest.raises(MemoryError):
        pool.batch([(a, 16), (b, 33)], device="cpu")
    assert pool.length(a) == 17 and pool.free_pages == 2          # nothing was taken
    with pytest.raises(ValueError):
        pool.batch([(a, 1), (a, 1)], device="cpu")
    with pytest.raises(ValueError):
        pool.batch([(a, -1)], device="cpu")
    pool.close(a)
    assert pool.free_pages == 4
    pool.close(b)
    assert pool.free_pages == 6


def test_pool_fork_shares_full_pages_and_copies_the_open_one():
    pool, caches = PagePool(8, 16), [PagedKVCache(8, 16, 2, 64, device="cpu") for _ in range(2)]
    a = pool.open()
    pool.batch([(a, 40)], device="cpu")
    for i, c in enumerate(caches):
        c.k.copy_(torch.arange(c.k.numel()).view(c.k.shape) % 120 + i)
        c.vs.copy_(torch.arange(c.vs.numel()).view(c.vs.shape))
    b = pool.fork(a, caches)
    pa, pb = pool.pages_of(a), pool.pages_of(b)
    assert pa[:2] == pb[:2] and pa[2] != pb[2] and pool.length(b) == 40 and pool.free_pages == 4
    for c in caches:
        for t in (c.k, c.v, c.ks, c.vs):
            assert torch.equal(t[pa[2]], t[pb[2]])
    pool.batch([(a, 8), (b, 8)], device="cpu")                    # both fill their own third page
    assert pool.pages_of(a) == pa and pool.pages_of(b) == pb
    pool.close(a)
    assert pool.free_pages == 5                                    # the shared pages are still b's
    c = pool.fork(b, caches)                                       # 48 tokens: no page is open
    assert pool.pages_of(c) == pb and pool.free_pages == 5
    pool.close(b)
    pool.close(c)
    assert pool.free_pages == 8
    d = pool.open()
    pool.batch([(d, 120)], device="cpu")
    with pytest.raises(MemoryError):
        pool.fork(d, caches)
    assert pool.free_pages == 0 and pool.length(d) == 120


def test_batch_positions():
    batch = PagedBatch(torch.tensor([0, 3, 3, 5], dtype=torch.int32), torch.tensor([10, 4, 2], dtype=torch.int32),
                       torch.zeros((3, 1), dtype=torch.int32), 3, 10)
    assert batch.positions(7).tolist() == [7, 8, 9, 0, 1, 0, 0]


def test_handles_refuse_what_does_not_fit():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError):
        PagedKVCache(4, 48, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(4, 16, 2, 96, device="cpu")
    k, s = torch.zeros((4, 2, 16, 64), dtype=torch.int8), torch.zeros((4, 2, 16))
    with pytest.raises(ValueError):
        PagedKVCache.over(k, k, s, s.double())
    with pytest.raises(ValueError):
        PagedKVCache.over(k, k.transpose(0, 1), s, s)
    with pytest.raises(ValueError):
        PagedKVCache.over(k, k, s, s[:3].contiguous())
    assert PagedKVCache.over(k, k, s, s).nbytes() == 2 * (k.numel() + 4 * s.numel())
    with pytest.raises(ValueError):
        PagedBatch(i32(2), i32(2), i32(2, 1), 1, 1)
    with pytest.raises(ValueError):
        PagedBatch(i32(3), i32(2).long(), i32(2, 1), 1, 1)
    with pytest.raises(ValueError):
        PagedBatch(i32(3), i32(2), i32(3, 1), 1, 1)
    for bad in (-16, 24, 144):
        with pytest.raises(ValueError):
            Rope(bad)
    with pytest.raises(ValueError):
        Rope(32, inv_freq=[1.0] * 15)
    r = Rope(32, 500.0, True)
    assert r.desc.dims == 32 and r.desc.interleaved == 1 and list(r.desc.inv_freq)[:2] == [1.0, 500.0 ** (-1 / 16)]
    assert L.load_library().logos_status_string(L.ERR_BAD_BATCH) != b"unknown status"


def test_descriptors_outlive_the_stores_they_came_from():
    """A call holds several strides and a batch's descriptor at once, and others may be made meanwhile."""
    from logos_b200.engine import _strides
    held = [_strides(3 * i + 64, 128 * i) for i in range(4)]
    for i in range(10000):
        _strides(64 * i, 7)
    assert [(d._obj.row, d._obj.head) for d in held] == [(3 * i + 64, 128 * i) for i in range(4)]
    batch = PagedBatch(torch.tensor([0, 3], dtype=torch.int32), torch.tensor([10], dtype=torch.int32),
                       torch.zeros((1, 1), dtype=torch.int32), 3, 10)
    few, many = batch.over(3), batch.over(9)
    assert (few._obj.rows, many._obj.rows, batch.over(9)._obj.max_kv) == (3, 9, 10)
