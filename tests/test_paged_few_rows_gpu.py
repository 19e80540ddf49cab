"""Paged attention of sequences that bring few rows a key head: the kernel that has keys as rows, on its own, beside longer
chunks in one call, and where the running maximum moves."""
import pytest
import torch

import dtb200
from paged_reference import Batch, attention
from test_paged_attention_gpu import _check

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _compare(batch, q, **how):
    out, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **how, **batch.where)
    dtb200.check_device_status()
    want, want_lse, tol, lse_tol = attention(batch, q, causal=how.get("causal", True), window=how.get("window") or 0)
    _check(out, want, tol)
    _check(lse, want_lse, lse_tol)
    return out


@pytest.mark.parametrize("new, kv, Hq, Hkv, D, page, dtype, layout, causal, window", [
    ([1], [1], 1, 1, 128, 16, BF, "hnd", True, 0),
    ([1, 1], [127, 4097], 16, 1, 128, 128, BF, "hnd", True, 0),            # all 16 columns
    ([1, 1, 1], [5, 640, 129], 9, 1, 64, 16, HF, "nhd", True, 0),          # nine of them
    ([2, 1, 2], [3000, 1, 2], 16, 2, 128, 64, HF, "hnd", True, 0),         # two tokens of eight heads
    ([16, 1, 0, 16], [900, 33, 70, 16], 3, 3, 64, 8, BF, "hnd", True, 0),
    ([5, 3, 4], [1000, 130, 4], 6, 2, 128, 32, BF, "nhd", False, 0),
    ([5, 3, 4], [1000, 130, 260], 6, 2, 128, 32, HF, "hnd", True, 7),
    ([4, 1], [2500, 2500], 12, 3, 64, 256, BF, "hnd", True, 1),
    ([4, 1], [2500, 2500], 12, 3, 128, 256, BF, "hnd", True, 131),
    ([3, 9], [2, 5], 2, 2, 128, 16, BF, "hnd", True, 0),                   # more new tokens than the sequence has
    ([1] * 33, [1 + 211 * i % 1900 for i in range(33)], 5, 1, 128, 16, BF, "hnd", True, 0),
    ([1], [90000], 5, 1, 128, 64, BF, "nhd", True, 0),                     # one sequence in pieces over all blocks
])
def test_few_rows(new, kv, Hq, Hkv, D, page, dtype, layout, causal, window):
    batch = Batch(new, kv, Hkv=Hkv, D=D, page=page, dtype=dtype, layout=layout, seed=1)
    assert batch.tokens * (Hq // Hkv) <= 16 * len(new)       # what the launch goes by
    q = batch.queries(Hq, 2, sharp=2.0)
    out = _compare(batch, q, causal=causal, window=window or None)
    again = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, causal=causal, window=window or None, **batch.where)
    assert torch.equal(out, again)


@pytest.mark.parametrize("D, dtype", [(128, BF), (64, HF)])
def test_beside_chunks_of_two_query_tiles(D, dtype):
    """A block sweeps units of both kinds one after the other, in both orders: what one keeps in the second query tile's memory,
    the other copies queries to."""
    new = [300 if i % 24 == 5 else 1 + i % 3 for i in range(240)]
    kv = [max(n, 17 * i % 700) for i, n in enumerate(new)]
    batch = Batch(new, kv, Hkv=4, D=D, page=16, dtype=dtype, seed=3)
    assert batch.tokens <= 16 * len(new)
    q = batch.queries(4, 4, sharp=2.0)
    first = _compare(batch, q)
    for _ in range(20):
        assert torch.equal(first, dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("down", [False, True])
def test_maximum_that_moves(dtype, down):
    """Keys that grow, or shrink, by a factor of 40 along the sequence: logits' maxima from tile to tile differ by far more
    than 2^8, in some columns and not in others."""
    batch = Batch([1, 2], [3000, 1500], Hkv=2, D=128, page=16, dtype=dtype, seed=5)
    for b, n in enumerate(batch.kv):
        for i in range(-(-n // 16)):
            part = i * 16 / n
            batch.key_cache[int(batch.page_table[b, i])] *= 1 + 39 * (1 - part if down else part)
    q = batch.queries(8, 6)
    q[:, 1::2] *= 0.01
    _compare(batch, q)


def test_not_a_number_reaches_the_rows_that_see_it():
    batch = Batch([1, 2], [300, 260], Hkv=2, D=128, page=16, dtype=BF, seed=7)
    q = batch.queries(8, 8)
    page, row = int(batch.page_table[0, 100 // 16]), 100 % 16
    batch.key_cache[page, 1, row, 3] = float("nan")
    page, row = int(batch.page_table[1, 259 // 16]), 259 % 16            # the last token's own key: the one before does not see it
    batch.key_cache[page, 0, row, 0] = float("nan")
    out = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where)
    dtb200.check_device_status()
    bad = torch.zeros(3, 8, dtype=torch.bool, device="cuda")
    bad[0, 4:] = True
    bad[2, :4] = True
    assert torch.equal(out.isnan().any(-1), bad)
    assert torch.equal(out.isnan().all(-1), bad)


def test_first_call_of_a_device_is_a_captured_one(monkeypatch):
    from dtb200 import ops, paged

    batch = Batch([1, 2], [300, 260], Hkv=2, D=128, page=16, dtype=BF, seed=9)
    q = batch.queries(4, 10)
    want = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where)
    monkeypatch.setattr(paged, "_status_ptrs", {})
    monkeypatch.setattr(paged, "_workspaces", {})
    bufs = dict(ops._status_bufs)
    ops._status_bufs.clear()
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **batch.where)
            mass = dtb200.paged_key_weights(q, batch.key_cache, lse, **batch.where)
        assert not ops._status_bufs
        graph.replay()
        dtb200.check_device_status()
        assert torch.equal(out, want) and bool(mass.isfinite().all())
        after = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where)
        dtb200.check_device_status()
        assert ops._status_bufs and torch.equal(after, want)
    finally:
        ops._status_bufs.clear()
        ops._status_bufs.update(bufs)
