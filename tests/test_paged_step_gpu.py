"""A whole step over the cache, captured and replayed, and calls from several threads on one stream."""
import threading

import pytest
import torch

import dtb200
from paged_reference import Batch

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _step(state, caches):
    where = {k: state[k] for k in ("page_table", "query_start", "kv_len")}
    q = dtb200.paged_append_(*caches, state["k"], state["v"], query=state["q"], table=state["rope"], **where)
    o, lse = dtb200.paged_attention(q, *caches, return_lse=True, **where)
    mass = dtb200.paged_key_weights(q, caches[0], lse, prior=state["prior"], **where)
    kept, mass_kept, kv_len = dtb200.paged_evict(*caches, mass, page_table=state["page_table"], out_table=state["out_table"], kv_len=state["kv_len"],
                                                 keep=200, recent=30)
    return q, o, lse, mass, kept, mass_kept, kv_len


def test_a_captured_step_follows_other_lengths_and_pages():
    kv, new = [900, 2600, 150], [40, 1, 3]
    batch = Batch(new, kv, Hkv=2, D=128, page=16, extra_width=4, spare=60)
    g = torch.Generator("cuda").manual_seed(0)
    caches = [torch.randn(c.shape, generator=g, device="cuda").to(BF) for c in (batch.key_cache, batch.value_cache)]
    q, k, v = (torch.randn(44, h, 128, generator=g, device="cuda").to(BF) for h in (8, 2, 2))
    slots = batch.page_table.shape[1] * 16
    state = {**batch.where, "q": q, "k": k, "v": v, "rope": dtb200.make_rotary_table(128), "prior": torch.rand(3, 2, slots, generator=g, device="cuda"),
             "out_table": torch.arange(batch.pages - 39, batch.pages, dtype=torch.int32, device="cuda").view(3, 13)}
    used = torch.randperm(batch.pages - 39, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    copy = [c.clone() for c in caches]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _step(state, copy)
    side = torch.cuda.Stream()
    for lens, order in (([900, 2600, 150], used), ([41, 1000, 2550], used.flip(0)), ([700, 3, 90], used.roll(7))):
        at = 0
        for b, n in enumerate(lens):
            pages = -(-n // 16)
            state["page_table"][b] = -1
            state["page_table"][b, :pages] = order[at:at + pages]
            at += pages
        state["kv_len"].copy_(torch.tensor(lens))
        plain = [c.clone() for c in caches]
        want = _step(state, plain)
        for c, now in zip(caches, copy):
            now.copy_(c)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((*want, *plain), (*captured, *copy)):
            assert torch.equal(a, b)
    dtb200.check_device_status()


def test_threads_on_one_stream():
    """Each with another batch, cut into pieces, and other sizes of workspace."""
    jobs = []
    for i, (D, n) in enumerate(((64, 30), (128, 70), (128, 1), (64, 200))):
        batch = Batch([n, 1], [30000 + 1000 * i, 9000], Hkv=1, D=D, page=64, seed=i)
        q = batch.queries(5, i)
        jobs.append((batch, q, dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **batch.where)))
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(len(jobs))

    def work(batch, q, want):
        start.wait()
        for _ in range(60):
            got = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **batch.where)
            if not all(torch.equal(a, b) for a, b in zip(got, want)):
                wrong.append(q.shape)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    dtb200.check_device_status()


def test_attention_of_threads_on_one_stream_and_of_two_graphs():
    """The calls of ``attention`` that go through a workspace, alike."""
    jobs = []
    for i, (heads, keys) in enumerate(((2, 9000), (5, 3000), (3, 20000))):
        g = torch.Generator("cuda").manual_seed(i)
        q, k, v = (torch.randn(1, heads, n, 128, generator=g, device="cuda").to(BF) for n in (256, keys, keys))
        jobs.append((q, k, v, dtb200.attention(q, k, v)))
    torch.cuda.synchronize()
    wrong = []

    def work(q, k, v, want):
        for _ in range(60):
            if not torch.equal(dtb200.attention(q, k, v), want):
                wrong.append(q.shape)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    graphs = []
    for q, k, v, want in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = dtb200.attention(q, k, v)
        graphs.append((graph, out, want, torch.cuda.Stream()))
    for _ in range(20):
        for graph, _, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert not wrong and all(torch.equal(out, want) for _, out, want, _ in graphs)
    dtb200.check_device_status()
