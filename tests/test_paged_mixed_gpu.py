"""Paged attention of batches whose sequences bring few rows, nothing, rows without keys and chunks, in orders that one block sweeps."""
import math

import pytest
import torch

import dtb200
from paged_reference import Batch
from test_paged_attention_gpu import _check

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _attention(batch, q):
    """As ``paged_reference.attention`` of causal batches, all heads of a sequence at once."""
    T, Hq, D = q.shape
    o, lse, tol, lse_tol = (torch.zeros(T, Hq, *x, dtype=torch.float64, device=q.device) for x in ((D,), (), (D,), ()))
    half = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate(batch.new):
        m, rows = batch.kv[b], batch.rows(b)
        if n == 0 or m == 0:
            lse[rows] = -math.inf
            continue
        k, v = (batch.gather(c, b).repeat_interleave(Hq // batch.Hkv, 0) for c in (batch.key_cache, batch.value_cache))
        x = q[rows].double().transpose(0, 1)
        seen = torch.arange(m, device=q.device) <= torch.arange(m - n, m, device=q.device)[:, None]
        s = (x @ k.mT * D ** -0.5).masked_fill(~seen, -math.inf)
        z = torch.logsumexp(s, -1, keepdim=True)
        p = torch.exp(s - z)
        delta = (D + 8) * 2.0 ** -24 * (x.abs() @ k.abs().mT * D ** -0.5).amax(-1, keepdim=True)
        out = p @ v
        o[rows], lse[rows] = out.transpose(0, 1), (z[..., 0] / math.log(2)).T
        tol[rows] = (half * out.abs() + (half * (1 + half) + 2 * delta + 2.0 ** -18) * (p @ v.abs()) + torch.finfo(q.dtype).tiny).transpose(0, 1)
        lse_tol[rows] = (2 * delta[..., 0] / math.log(2) + 2.0 ** -18).T + 2.0 ** -22 * lse[rows].abs()
    return o, lse, tol, lse_tol


def _compare(batch, q):
    out, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **batch.where)
    dtb200.check_device_status()
    want, want_lse, tol, lse_tol = _attention(batch, q)
    _check(out, want, tol)
    _check(lse, want_lse, lse_tol)
    for _ in range(10):
        assert torch.equal(out, dtb200.paged_attention(q, batch.key_cache, batch.value_cache, **batch.where))
    dtb200.check_device_status()


@pytest.mark.parametrize("empty, nothing", [(3, 0), (2, 0), (0, 3), (2, 40), (0, 200)])
@pytest.mark.parametrize("D, dtype", [(128, BF), (64, HF)])
def test_few_rows_then_units_without_keys_then_a_chunk(empty, nothing, D, dtype):
    """Eight units a sequence, 32 or so a block: 16 and 24 of them without a key tile between few rows and two query tiles, and
    sequences that bring nothing in the way of the warp that describes the units."""
    new, kv = [], []
    for i in range(25 if nothing < 100 else 12):
        few = 20 - empty
        new += [1 + (i + j) % 2 * (j == few - 1) for j in range(few)] + [1] * empty + [0] * nothing + [17 + i % 4]
        kv += [50 + 13 * (i + j) % 170 for j in range(few)] + [0] * empty + [j % 60 for j in range(nothing)] + [17 + i % 4 + 31 * i % 200]
    batch = Batch(new, kv, Hkv=8, D=D, page=16, dtype=dtype, seed=3)
    assert batch.tokens * 8 <= 16 * len(new)                 # what the launch goes by
    _compare(batch, batch.queries(64, 4, sharp=2.0))


def test_padded_slots_in_front_of_a_chunk():
    new = [1] * 48 + [1, 1, 1] + [64]
    kv = [100 + 37 * i for i in range(48)] + [0, 0, 0] + [900]
    batch = Batch(new, kv, Hkv=8, D=128, page=32, dtype=BF, seed=5)
    _compare(batch, batch.queries(8, 6, sharp=2.0))


@pytest.mark.parametrize("pages, width", [(0, 4), (5, 0)])
def test_append_of_single_tokens_without_pages_turns_their_queries(pages, width):
    B = 64
    g = torch.Generator("cuda").manual_seed(0)
    q, k = (torch.randn(B, h, 128, generator=g, device="cuda").to(BF) for h in (8, 2))
    cache = torch.full((pages, 2, 16, 128), 3.0, dtype=BF, device="cuda")
    rope = dtb200.make_rotary_table(128)
    lens = torch.arange(1, B + 1, dtype=torch.int32, device="cuda")
    got = dtb200.paged_append_(cache, cache.clone(), k, k, query=q, table=rope, page_table=torch.zeros(B, width, dtype=torch.int32, device="cuda"),
                               query_start=torch.arange(B + 1, dtype=torch.int32, device="cuda"), kv_len=lens)
    assert torch.equal(got, dtb200.rotary(q, table=rope, positions=lens - 1)) and (cache == 3.0).all()


def test_a_single_token_cut_out_of_a_wider_row():
    batch = Batch([1], [300], Hkv=2, D=128, page=16, dtype=BF)
    q = batch.queries(8, 1)
    wide = torch.zeros(3, 8 * 128 + 4, dtype=BF, device="cuda")
    view = wide[:, :1024].view(3, 8, 128)[:1]
    view.copy_(q)
    assert view.stride(0) % 8 and view.is_contiguous()
    want, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, return_lse=True, **batch.where)
    out = torch.zeros_like(wide)[:, :1024].view(3, 8, 128)[:1]
    assert torch.equal(dtb200.paged_attention(view, batch.key_cache, batch.value_cache, out=out, **batch.where), want)
    got, same = (dtb200.paged_key_weights(x, batch.key_cache, lse, **batch.where) for x in (view, q))
    assert torch.equal(got, same)
