"""Append, attention and key weights agree on where new tokens lie when a sequence is longer than its page table can name."""
import math

import pytest
import torch

import dtb200
from paged_reference import Batch
from test_paged_attention_gpu import _check

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("new, over, Hq, Hkv, D, dtype, window", [
    ([10, 3], [6, 0], 4, 2, 128, BF, 0),              # few rows: slots 60-69 and 61-63 of 64
    ([10, 3], [6, 0], 8, 2, 64, HF, 5),               # the last two tokens see nothing, their window behind the table's end
    ([150, 1, 40], [100, 1, 39], 4, 2, 128, BF, 0),   # a single token behind the end; one slot left for the others of the last
    ([150, 2, 40], [100, 1, 20], 4, 1, 128, BF, 30),
])
def test_tokens_see_themselves(new, over, Hq, Hkv, D, dtype, window):
    page = 16
    capacity = -(-max(n - o for n, o in zip(new, over)) // page) * page + (16 if len(new) == 3 else 48)
    kv = [capacity + o for o in over]
    batch = Batch([0] * len(new), [min(m, capacity) for m in kv], Hkv=Hkv, D=D, page=page, dtype=dtype, extra_width=0)
    g = torch.Generator("cuda").manual_seed(1)
    T = sum(new)
    q, k, v = (torch.randn(T, h, D, generator=g, device="cuda").to(dtype) for h in (Hq, Hkv, Hkv))
    starts = [sum(new[:b]) for b in range(len(new) + 1)]
    where = {"page_table": batch.page_table, "query_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
             "kv_len": torch.tensor(kv, dtype=torch.int32, device="cuda")}
    dtb200.paged_append_(batch.key_cache, batch.value_cache, k, v, **where)
    out, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, window=window or None, return_lse=True, **where)
    got = dtb200.paged_key_weights(q, batch.key_cache, lse, window=window or None, **where)
    dtb200.check_device_status()
    half, total = torch.finfo(dtype).eps / 2, torch.zeros_like(got, dtype=torch.float64)
    weight_tol = torch.zeros_like(total)
    for b, n in enumerate(new):
        keys, values = batch.gather(batch.key_cache, b), batch.gather(batch.value_cache, b)
        slot = torch.arange(kv[b] - n, kv[b], device="cuda")
        if slot[0] >= capacity:                        # none of them has a slot: they count as the last ones
            slot -= slot[-1] + 1 - capacity
        else:
            own = slot < capacity                      # what was appended is there
            assert torch.equal(keys[:, slot[own]], k[starts[b]:starts[b + 1]][own].transpose(0, 1).double())
        key = torch.arange(capacity, device="cuda")
        seen = (key <= slot[:, None]) & ((key > slot[:, None] - window) if window else True)
        some = seen.any(-1)
        for h in range(Hq):
            x, hk = q[starts[b]:starts[b + 1], h].double(), h // (Hq // Hkv)
            s = (x @ keys[hk].T * D ** -0.5).masked_fill(~seen, -math.inf)
            z = torch.logsumexp(s, -1, keepdim=True)
            p = torch.where(some[:, None], torch.exp(s - z), 0.0)
            delta = (D + 8) * 2.0 ** -24 * (x.abs() @ keys[hk].abs().T * D ** -0.5).amax(-1, keepdim=True)
            want = p @ values[hk]
            rows = slice(starts[b], starts[b + 1])
            _check(out[rows, h], want, half * want.abs() + (half * (1 + half) + 2 * delta + 2.0 ** -18) * (p @ values[hk].abs()) + torch.finfo(dtype).tiny)
            log = z[:, 0] / math.log(2)
            _check(lse[rows, h], log, 2 * delta[:, 0] / math.log(2) + 2.0 ** -18 + 2.0 ** -22 * log.abs().nan_to_num(0, 0, 0))
            total[b, hk] += p.sum(0)
            # the logit and lse, each off by what _check allows, the difference of the two in f32, and the exponential
            weight_tol[b, hk] += (p * (4 * delta + 2.0 ** -17 + 2.0 ** -21 * log.abs().nan_to_num(0, 0, 0)[:, None])).sum(0)
    _check(got, total, weight_tol + (max(new) * Hq // Hkv + 2) * 2.0 ** -24 * total + 1e-30)
