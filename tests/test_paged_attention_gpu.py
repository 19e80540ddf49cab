"""Paged attention and key weights against their definitions in 64 bits."""
import pytest
import torch

import dtb200
from paged_reference import Batch, attention, key_weights

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _check(got, want, tol, rows=None):
    got, want, tol = (x if rows is None else x[rows] for x in (got.double(), want, tol))
    over = (got - want).abs() - tol
    over = torch.where(got == want, torch.zeros_like(over), over)       # infinities
    assert not over.isnan().any(), "NaN"
    assert over.max().item() <= 0, f"beyond the bound by {over.max().item():.3e}, worst ratio {((got - want).abs() / tol).nan_to_num().max().item():.2f}"


SHAPES = [  # new, kv, Hq, Hkv, D, page, dtype, layout, causal, window
    ([1], [1], 1, 1, 128, 16, BF, "hnd", True, 0),
    ([1, 1, 1], [7, 128, 129], 8, 2, 128, 16, BF, "hnd", True, 0),
    ([1, 1, 1, 1], [900, 1, 333, 2000], 24, 8, 128, 32, BF, "nhd", True, 0),
    ([1, 0, 5, 0, 3], [0, 40, 5, 0, 200], 6, 3, 128, 16, HF, "hnd", True, 0),
    ([17], [17], 4, 4, 128, 8, BF, "hnd", True, 0),
    ([300], [300], 4, 1, 128, 64, BF, "nhd", True, 0),
    ([257], [1000], 2, 2, 128, 128, HF, "hnd", True, 0),
    ([130, 1, 77], [1500, 3000, 77], 10, 2, 128, 64, BF, "hnd", True, 0),
    ([130, 1, 77], [1500, 3000, 77], 10, 2, 128, 64, BF, "hnd", False, 0),
    ([64, 3], [700, 650], 14, 2, 64, 16, BF, "nhd", True, 0),
    ([1, 1], [4000, 123], 16, 2, 64, 256, HF, "hnd", True, 0),
    ([200, 1, 9], [600, 2500, 9], 6, 2, 128, 32, BF, "hnd", True, 100),
    ([200, 1, 9], [600, 2500, 9], 6, 2, 64, 32, HF, "nhd", True, 1),
    ([500], [1500], 3, 1, 128, 16, BF, "hnd", True, 777),
    ([1], [5000], 128, 1, 128, 64, BF, "hnd", True, 0),
    ([3], [2000], 100, 1, 128, 64, BF, "hnd", True, 0),
    ([40, 50], [30, 50], 4, 2, 128, 16, BF, "hnd", True, 0),       # more new tokens than the sequence has
    ([40, 50], [30, 50], 4, 2, 128, 16, BF, "hnd", False, 0),
    ([1] * 70, [13 * i % 900 for i in range(70)], 8, 4, 128, 16, BF, "hnd", True, 0),
    ([600, 600], [8000, 700], 5, 1, 128, 384, BF, "nhd", True, 0),
]


def _make(shape, seed=0, **more):
    new, kv, Hq, Hkv, D, page, dtype, layout, causal, window = shape
    batch = Batch(new, kv, Hkv=Hkv, D=D, page=page, dtype=dtype, layout=layout, seed=seed, **more)
    return batch, batch.queries(Hq, seed + 1, sharp=2.0), {"causal": causal, "window": window or None}


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{'_'.join(map(str, s[0][:4]))}of{'_'.join(map(str, s[1][:4]))}")
def test_attention(shape):
    batch, q, how = _make(shape)
    out, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **how, **batch.where)
    dtb200.check_device_status()
    want, want_lse, tol, lse_tol = attention(batch, q, causal=how["causal"], window=how["window"] or 0)
    _check(out, want, tol)
    _check(lse, want_lse, lse_tol)
    again = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **how, **batch.where)
    assert torch.equal(out, again)


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{'_'.join(map(str, s[0][:4]))}of{'_'.join(map(str, s[1][:4]))}")
def test_key_weights(shape):
    batch, q, how = _make(shape, seed=5)
    window = how["window"] or 0
    _, lse, _, _ = attention(batch, q, causal=how["causal"], window=window)
    lse = lse.float()
    slots = batch.page_table.shape[1] * batch.page
    prior = torch.rand(len(batch.new), batch.Hkv, slots, device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    for pr in (None, prior):
        want, tol = key_weights(batch, q, lse, pr, causal=how["causal"], window=window)
        got = dtb200.paged_key_weights(q, batch.key_cache, lse, prior=pr, **how, **batch.where)
        dtb200.check_device_status()
        _check(got, want, tol)
    same = dtb200.paged_key_weights(q, batch.key_cache, lse, prior=prior, out=prior, **how, **batch.where)
    assert same is prior and torch.equal(prior, got)


def test_weights_of_a_step_add_up_to_the_rows_that_see_something():
    batch, q, how = _make(SHAPES[7], seed=3)
    _, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **how, **batch.where)
    got = dtb200.paged_key_weights(q, batch.key_cache, lse, **how, **batch.where).double().sum(-1)
    want = torch.tensor(batch.new, device="cuda", dtype=torch.float64)[:, None].expand_as(got) * 5
    # each row's weights add up to 1 but for f32's logits (|logit| below 64) and exponentials
    assert ((got - want).abs() <= want * 2.0 ** -14).all()


def test_scale_and_out_and_rows_of_no_sequence():
    batch, _, _ = _make(SHAPES[2], seed=2, tail=5)
    wide = torch.randn(batch.tokens, 2, 24, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(BF)
    q = wide[:, 0]                                                   # strided heads
    out = torch.full((24, batch.tokens, 128), 7.0, dtype=BF, device="cuda").transpose(0, 1)
    got = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, scale=0.2, out=out, **batch.where)
    assert got is out
    want, _, tol, _ = attention(batch, q, scale=0.2)
    n = sum(batch.new)
    _check(out, want, tol, slice(0, n))
    assert (out[n:] == 7.0).all()
    odd = torch.empty(batch.tokens, 24, 132, dtype=BF, device="cuda")[..., 1:129]     # rows off 16-byte boundaries
    odd.fill_(7.0)
    dtb200.paged_attention(q, batch.key_cache, batch.value_cache, scale=0.2, out=odd, **batch.where)
    assert torch.equal(odd, out)


def test_pages_that_do_not_exist_read_as_zeros():
    batch, q, how = _make(SHAPES[7], seed=4)
    batch.page_table[0, 3] = -1
    batch.page_table[1, 0] = batch.pages
    batch.page_table[1, 7] = 2 ** 31 - 1
    batch.page_table[2, 1] = -(2 ** 31)
    out, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **how, **batch.where)
    want, want_lse, tol, lse_tol = attention(batch, q)
    _check(out, want, tol)
    _check(lse, want_lse, lse_tol)
    got = dtb200.paged_key_weights(q, batch.key_cache, want_lse.float(), **batch.where)
    _check(got, *key_weights(batch, q, want_lse.float()))
    dtb200.check_device_status()


def test_lengths_past_the_table_end_at_it():
    batch, q, how = _make(([4, 4], [64, 50], 2, 2, 128, 16, BF, "hnd", True, 0), extra_width=0)
    batch.kv_len[0] = 2 ** 31 - 1
    out = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where)
    want, _, tol, _ = attention(batch, q)
    _check(out, want, tol)


@pytest.mark.parametrize("starts", [[0, 5, 3, 9], [-4, 2, 100, 6], [9, 9, 9, 9]])
def test_starts_out_of_order_stay_in_bounds(starts):
    batch, q, how = _make(([3, 3, 3], [40, 50, 60], 2, 2, 128, 16, BF, "hnd", True, 0))
    batch.query_start.copy_(torch.tensor(starts))
    out = torch.zeros_like(q)
    dtb200.paged_attention(q, batch.key_cache, batch.value_cache, out=out, **batch.where)
    lse = torch.zeros(9, 2, device="cuda")
    dtb200.paged_key_weights(q, batch.key_cache, lse, **batch.where)
    dtb200.check_device_status()


def test_not_a_number_and_infinities_reach_the_rows_that_see_them():
    batch, q, how = _make(([1, 40], [300, 260], 4, 2, 128, 16, BF, "hnd", True, 0))
    page, row = int(batch.page_table[0, 100 // 16]), 100 % 16
    batch.key_cache[page, 1, row, 3] = float("nan")
    page, row = int(batch.page_table[1, 240 // 16]), 240 % 16
    batch.key_cache[page, 0, row, 0] = 3e38
    q[1:, :2, 0] = torch.where(torch.arange(40, device="cuda") % 2 == 0, 2.0, -2.0).to(BF)[:, None]
    out = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where)
    dtb200.check_device_status()
    rows = torch.arange(40, device="cuda")
    bad = torch.zeros(41, 4, dtype=torch.bool, device="cuda")
    bad[0, 2:] = True
    bad[1:, :2] = ((rows % 2 == 0) & (rows >= 20))[:, None]          # token 220 + i sees slot 240; logits of +inf only
    assert torch.equal(out.isnan().any(-1), bad)


def test_another_stream_and_replays_with_other_lengths():
    shape = ([1, 1, 30], [500, 1200, 700], 8, 2, 128, 32, BF, "hnd", True, 0)
    batch, q, how = _make(shape)
    plain = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where)
    side.synchronize()
    assert torch.equal(plain, other)
    graphs, outs, lses = [], [], []
    for _ in range(2):                       # two graphs that may run at the same time
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            o, l = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **batch.where)
            w = dtb200.paged_key_weights(q, batch.key_cache, l, **batch.where)
        outs.append((o, l, w))
    streams = [torch.cuda.Stream() for _ in graphs]
    for kv in ([500, 1200, 700], [37, 1100, 699], [1, 1, 30]):
        batch.kv = kv
        batch.kv_len.copy_(torch.tensor(kv))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        want, want_lse, tol, lse_tol = attention(batch, q)
        for o, l, w in outs:
            _check(o, want, tol)
            _check(l, want_lse, lse_tol)
            _check(w, *key_weights(batch, q, l))
    dtb200.check_device_status()


def test_nothing_to_do():
    batch, q, how = _make(([0, 0], [50, 0], 4, 2, 128, 16, BF, "hnd", True, 0))
    out, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **batch.where)
    assert out.shape == (0, 4, 128) and lse.shape == (0, 4)
    prior = torch.rand(2, 2, batch.page_table.shape[1] * 16, device="cuda")
    got = dtb200.paged_key_weights(q, batch.key_cache, lse, prior=prior, **batch.where)
    assert torch.equal(got[0, :, :50], prior[0, :, :50]) and not got[0, :, 50:].any() and not got[1].any()
    none = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, page_table=batch.page_table[:0], query_start=batch.query_start[:1],
                                  kv_len=batch.kv_len[:0])
    assert none.shape == (0, 4, 128)


def test_empty_caches_read_as_zeros():
    q = torch.randn(3, 4, 128, device="cuda").to(BF)
    cache = torch.empty(0, 2, 16, 128, dtype=BF, device="cuda")
    where = {"page_table": torch.zeros(1, 2, dtype=torch.int32, device="cuda"), "query_start": torch.tensor([0, 3], dtype=torch.int32, device="cuda"),
             "kv_len": torch.tensor([20], dtype=torch.int32, device="cuda")}
    out, lse = dtb200.paged_attention(q, cache, cache, return_lse=True, **where)
    assert not out.any()
    want = torch.tensor([18.0, 19.0, 20.0], device="cuda").log2()[:, None].expand(3, 4)
    assert ((lse - want).abs() <= 2.0 ** -18).all()


def test_slots_past_32_bits_of_elements():
    """A page more than 2^32 elements into its cache."""
    page, Hkv = 16, 1
    pages = 2 ** 32 // (page * 128) + 3
    cache = torch.empty(pages, Hkv, page, 128, dtype=BF, device="cuda")       # 8.6 GB, for keys and values alike
    batch, q, _ = _make(([2], [40], 2, 1, 128, page, BF, "hnd", True, 0))
    for i, far in enumerate((pages - 1, 3, pages - 2)):
        cache[far] = batch.key_cache[int(batch.page_table[0, i])]
        batch.page_table[0, i] = far
    batch.key_cache = batch.value_cache = cache
    batch.pages = pages
    out = dtb200.paged_attention(q, cache, cache, **batch.where)
    want, _, tol, _ = attention(batch, q)
    _check(out, want, tol)


def test_refusals():
    batch, q, _ = _make(SHAPES[1])
    kc, vc, w = batch.key_cache, batch.value_cache, batch.where
    call = dtb200.paged_attention
    for error, f in [
        (NotImplementedError, lambda: call(q.float(), kc.float(), vc.float(), **w)),
        (ValueError, lambda: call(q[..., :64], kc, vc, **w)),
        (ValueError, lambda: call(q[:, :7], kc, vc, **w)),
        (ValueError, lambda: call(q, kc, vc[:1], **w)),
        (ValueError, lambda: call(q, kc.transpose(2, 3), vc, **w)),
        (ValueError, lambda: call(q, kc, vc, scale=0.0, **w)),
        (ValueError, lambda: call(q, kc, vc, scale=float("nan"), **w)),
        (ValueError, lambda: call(q, kc, vc, window=0, **w)),
        (ValueError, lambda: call(q, kc, vc, window=4, causal=False, **w)),
        (ValueError, lambda: call(q, kc, vc, out=q[:1], **w)),
        (ValueError, lambda: call(q, kc.half(), vc.half(), **w)),
        (NotImplementedError, lambda: call(q, kc, vc, **{**w, "kv_len": batch.kv_len.long()})),
        (ValueError, lambda: call(q, kc, vc, **{**w, "kv_len": batch.kv_len[:2]})),
        (ValueError, lambda: call(q, kc, vc, **{**w, "query_start": batch.query_start[:3]})),
        (RuntimeError, lambda: call(q, kc, vc, **{**w, "page_table": batch.page_table.cpu()})),
        (NotImplementedError, lambda: call(q, kc[:, :, :12], vc[:, :, :12], **w)),
        (ValueError, lambda: dtb200.paged_key_weights(q, kc, torch.zeros(3, 7, device="cuda"), **w)),
        (ValueError, lambda: dtb200.paged_key_weights(q, kc, torch.zeros(3, 8, device="cuda"), prior=torch.zeros(3, 2, 5, device="cuda"), **w)),
    ]:
        with pytest.raises(error):
            f()
