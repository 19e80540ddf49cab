"""Paged attention of prompts that are long enough for each block to be dealt many whole units, at sampled rows of every query block."""
import math

import pytest
import torch

import dtb200
from paged_reference import Batch
from test_paged_attention_gpu import _check

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _sampled(batch, q, rows, window):
    """As ``paged_reference.attention``, of some rows of causal sequences: (o, lse, bounds on both)."""
    D, G = q.shape[-1], q.shape[1] // batch.Hkv
    half = torch.finfo(q.dtype).eps / 2
    parts = []
    for b, n in enumerate(batch.new):
        own = [r - batch.rows(b).start for r in rows if batch.rows(b).start <= r < batch.rows(b).stop]
        at = torch.tensor(own, device=q.device) + batch.kv[b] - n
        x = q[batch.rows(b)][own].double()
        k, v = batch.gather(batch.key_cache, b), batch.gather(batch.value_cache, b)
        key = torch.arange(batch.kv[b], device=q.device)
        seen = (key <= at[:, None]) & (key > at[:, None] - window if window else True)
        o, lse, tol, lse_tol = (torch.empty(len(own), *s, dtype=torch.float64, device=q.device)
                                for s in ((q.shape[1], D), (q.shape[1],), (q.shape[1], D), (q.shape[1],)))
        for h in range(q.shape[1]):
            s = (x[:, h] @ k[h // G].T * D ** -0.5).masked_fill(~seen, -math.inf)
            z = torch.logsumexp(s, -1, keepdim=True)
            p = torch.exp(s - z)
            o[:, h], lse[:, h] = p @ v[h // G], z[:, 0] / math.log(2)
            delta = (D + 8) * 2.0 ** -24 * (x[:, h].abs() @ k[h // G].abs().T * D ** -0.5).amax(-1, keepdim=True)
            tol[:, h] = half * o[:, h].abs() + (half * (1 + half) + 2 * delta + 2.0 ** -18) * (p @ v[h // G].abs()) + torch.finfo(q.dtype).tiny
            lse_tol[:, h] = 2 * delta[:, 0] / math.log(2) + 2.0 ** -18 + 2.0 ** -22 * lse[:, h].abs()
        parts.append((o, lse, tol, lse_tol))
    return [torch.cat(x) for x in zip(*parts)]


@pytest.mark.parametrize("new, kv, Hq, Hkv, D, page, dtype, window", [
    ([16384], [16384], 40, 8, 128, 64, BF, 0),              # 50 tokens a query block: 17 whole units a block, and cut ones behind
    ([8192] * 3, [8192] * 3, 20, 4, 64, 128, HF, 0),
    ([7000, 13000], [9000, 20000], 16, 8, 128, 16, BF, 9000),
])
def test_many_rounds(new, kv, Hq, Hkv, D, page, dtype, window):
    batch = Batch(new, kv, Hkv=Hkv, D=D, page=page, dtype=dtype, seed=1)
    q = batch.queries(Hq, 2, sharp=2.0)
    # a call before it that leaves other states in the workspace
    dtb200.paged_attention(-q, batch.key_cache, batch.value_cache, causal=False, **batch.where)
    out, lse = dtb200.paged_attention(q, batch.key_cache, batch.value_cache, window=window or None, return_lse=True, **batch.where)
    dtb200.check_device_status()
    rows = sorted({*range(0, batch.tokens, 37), *range(batch.tokens - 3, batch.tokens)})
    want, want_lse, tol, lse_tol = _sampled(batch, q, rows, window)
    _check(out[rows], want, tol)
    _check(lse[rows], want_lse, lse_tol)
