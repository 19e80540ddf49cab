"""Eviction by accumulated weight: which tokens stay is decided exactly, and their rows are copied bit for bit."""
import pytest
import torch

import dtb200
from paged_reference import Batch, attention

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _choose(w, keep, recent):
    """Slots kept of one head: stable order by falling weight, NaN first, equal weights by slot."""
    n = len(w)
    if n <= keep:
        return list(range(n))
    old = n - recent
    rank = [float("inf") if x != x else x for x in w[:old]]
    first = [1 if x != x else 0 for x in w[:old]]
    order = sorted(range(old), key=lambda i: (-first[i], -rank[i], i))
    return sorted(order[:keep - recent]) + list(range(old, n))


def _evict_and_check(batch, weights, keep, recent, extra_out=0):
    B, page = len(batch.kv), batch.page
    width = -(-keep // page) + extra_out
    free = torch.arange(batch.pages, batch.pages + B * width, dtype=torch.int32, device="cuda")
    out_table = free[torch.randperm(B * width, generator=torch.Generator().manual_seed(3)).cuda()].view(B, width)

    def grown(c):
        extra = torch.full((B * width, *c.shape[1:]), 77.0, dtype=c.dtype, device="cuda")
        x = torch.cat([c, extra])
        return x if c.stride(1) >= c.stride(2) else x.transpose(1, 2).contiguous().transpose(1, 2)

    kc, vc = grown(batch.key_cache), grown(batch.value_cache)
    before = kc.clone(), vc.clone()
    kept, w_out, kv_len = dtb200.paged_evict(kc, vc, weights, page_table=batch.page_table, out_table=out_table, kv_len=batch.kv_len,
                                             keep=keep, recent=recent)
    cpu, table, to = weights.cpu(), batch.page_table.tolist(), out_table.tolist()
    for b, n in enumerate(batch.kv):
        m = min(n, keep)
        assert int(kv_len[b]) == m
        for h in range(batch.Hkv):
            want = _choose(cpu[b, h, :n].tolist(), keep, recent)
            assert kept[b, h, :m].tolist() == want and (kept[b, h, m:] == -1).all()
            assert torch.equal(w_out[b, h, :m].cpu().nan_to_num(-5.0), cpu[b, h, want].nan_to_num(-5.0)) and not w_out[b, h, m:].any()
            for c, old in ((kc, before[0]), (vc, before[1])):
                if want:
                    src = old[torch.tensor([table[b][s // page] for s in want]), h, torch.tensor([s % page for s in want])]
                    dst = torch.tensor([to[b][i // page] for i in range(m)]), h, torch.tensor([i % page for i in range(m)])
                    assert torch.equal(c[dst], src)
    # nothing else is written
    for c, old in ((kc, before[0]), (vc, before[1])):
        assert torch.equal(c[:batch.pages].nan_to_num(9.0), old[:batch.pages].nan_to_num(9.0))
        for b, n in enumerate(batch.kv):
            for i in range(min(n, keep), width * page):
                assert (c[to[b][i // page], :, i % page] == 77.0).all()
    return kept, w_out, kv_len, kc, vc, out_table


@pytest.mark.parametrize("kv,keep,recent,Hkv,D,page,dtype,layout", [
    ([1], 1, 0, 1, 128, 16, BF, "hnd"),
    ([100, 3, 0, 64], 64, 16, 2, 128, 16, BF, "hnd"),
    ([1000, 2500], 700, 0, 3, 64, 32, HF, "nhd"),
    ([1025, 1024, 1023], 1024, 1024, 1, 128, 64, BF, "nhd"),
    ([5000], 4999, 10, 2, 128, 256, BF, "hnd"),
    ([3000], 1, 1, 2, 40, 5, BF, "hnd"),
    ([3000], 1, 0, 2, 128, 128, BF, "hnd"),
])
@pytest.mark.parametrize("ties", [False, True])
def test_evict(kv, keep, recent, Hkv, D, page, dtype, layout, ties):
    batch = Batch([0] * len(kv), kv, Hkv=Hkv, D=D, page=page, dtype=dtype, layout=layout)
    slots = batch.page_table.shape[1] * page
    g = torch.Generator("cuda").manual_seed(keep)
    weights = torch.randn(len(kv), Hkv, slots, generator=g, device="cuda")
    if ties:
        weights = (weights * 2).round()          # signs, zeros of both signs among them
    _evict_and_check(batch, weights, keep, recent, extra_out=1)


def test_odd_weights():
    batch = Batch([0], [600], Hkv=2, D=128, page=16)
    slots = batch.page_table.shape[1] * 16
    w = torch.randn(1, 2, slots, device="cuda", generator=torch.Generator("cuda").manual_seed(0))
    w[0, 0, ::7] = float("nan")
    w[0, 0, 1::7] = float("inf")
    w[0, 0, 2::7] = -float("inf")
    w[0, 1] = 0.0
    w[0, 1, ::2] = -0.0
    w[0, 1, 5::11] = 1e-40
    for keep, recent in ((100, 10), (300, 0), (30, 30)):
        _evict_and_check(batch, w, keep, recent)


def test_pages_that_do_not_exist():
    batch = Batch([0, 0], [100, 90], Hkv=1, D=64, page=16, dtype=HF)
    batch.page_table[0, 2] = -7
    out_table = torch.tensor([[batch.pages - 1, batch.pages], [2 ** 30, -1]], dtype=torch.int32, device="cuda")
    w = torch.rand(2, 1, batch.page_table.shape[1] * 16, device="cuda")
    dtb200.paged_evict(batch.key_cache, batch.value_cache, w, page_table=batch.page_table, out_table=out_table, kv_len=batch.kv_len, keep=30)
    batch.kv_len[1] = 10 ** 9
    dtb200.paged_evict(batch.key_cache, batch.value_cache, w, page_table=batch.page_table, out_table=out_table, kv_len=batch.kv_len, keep=30)
    torch.cuda.synchronize()


def test_a_rollout_appends_attends_counts_and_evicts():
    """The operators in the order a rollout calls them, step by step against attention over the rows that should be there."""
    Hq, Hkv, D, page, keep, recent = 6, 2, 128, 16, 48, 24
    g = torch.Generator("cuda").manual_seed(0)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(BF)

    B, pages = 2, 64
    kc, vc = (torch.full((pages, Hkv, page, D), float("nan"), dtype=BF, device="cuda") for _ in range(2))
    free = list(range(pages))
    table = torch.tensor([[free.pop() for _ in range(8)] for _ in range(B)], dtype=torch.int32, device="cuda")
    rope = dtb200.make_rotary_table(D)
    lens, weights = [0, 0], torch.zeros(B, Hkv, 8 * page, device="cuda")
    held = [(torch.empty(Hkv, 0, D, device="cuda", dtype=BF),) * 2 for _ in range(B)]
    seen = [0, 0]                                  # tokens so far, evicted ones included: the positions of new ones
    for new in ([30, 40], [20, 1], [1, 25], [16, 16], [1, 1]):
        T = sum(new)
        q, k, v = normal(T, Hq, D), normal(T, Hkv, D), normal(T, Hkv, D)
        lens = [a + n for a, n in zip(lens, new)]
        positions = torch.cat([torch.arange(s, s + n, device="cuda") for s, n in zip(seen, new)])
        seen = [s + n for s, n in zip(seen, new)]
        where = {"page_table": table, "query_start": torch.tensor([0, new[0], T], dtype=torch.int32, device="cuda"),
                 "kv_len": torch.tensor(lens, dtype=torch.int32, device="cuda")}
        turned = dtb200.paged_append_(kc, vc, k, v, table=rope, positions=positions, query=q, **where)
        kt = dtb200.rotary(k, table=rope, positions=positions)
        o, lse = dtb200.paged_attention(turned, kc, vc, return_lse=True, **where)
        dtb200.paged_key_weights(turned, kc, lse, prior=weights, out=weights, **where)
        batch = Batch(new, lens, Hkv=Hkv, D=D, page=page)
        batch.page_table, batch.key_cache, batch.value_cache = table, kc, vc
        at = 0
        for b, n in enumerate(new):
            held[b] = tuple(torch.cat([x, y[at:at + n].transpose(0, 1)], 1) for x, y in zip(held[b], (kt, v)))
            at += n
            assert torch.equal(batch.gather(kc, b), held[b][0].double()) and torch.equal(batch.gather(vc, b), held[b][1].double())
        want, _, tol, _ = attention(batch, turned)
        assert ((o.double() - want).abs() <= tol).all()
        if max(lens) > keep + 16:
            fresh = torch.tensor([[free.pop(0) for _ in range(8)] for _ in range(B)], dtype=torch.int32, device="cuda")
            kept, weights, kv_len = dtb200.paged_evict(kc, vc, weights, page_table=table, out_table=fresh, kv_len=where["kv_len"], keep=keep, recent=recent)
            free += table.flatten().tolist()
            table, lens = fresh, kv_len.tolist()
            for b in range(B):
                index = kept[b, :, :lens[b]].long()[..., None].expand(-1, -1, D)
                held[b] = tuple(x.gather(1, index) for x in held[b])
    dtb200.check_device_status()
    assert max(lens) <= keep + 16
