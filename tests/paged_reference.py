"""The paged-cache operators from their definitions in 64 bits, and the caches that their tests run on."""
import math

import torch

F64 = torch.float64


class Batch:
    """Sequences of ``new[b]`` new tokens and ``kv[b]`` in all, over pages dealt out in random order; whatever is not a
    counted token's row is NaN."""

    def __init__(self, new, kv, *, Hkv, D, page, dtype=torch.bfloat16, layout="hnd", seed=0, device="cuda", spare=2, extra_width=1, tail=0):
        g = torch.Generator().manual_seed(seed)
        self.new, self.kv, self.page, self.Hkv, self.D, self.dtype = list(new), list(kv), page, Hkv, D, dtype
        B = len(new)
        used = [-(-n // page) for n in kv]
        self.pages = sum(used) + spare
        order = torch.randperm(self.pages, generator=g, dtype=torch.int64).to(torch.int32)
        width = max(used + [0]) + extra_width
        # entries behind a sequence's pages name whatever: other sequences' pages, none, and pages that do not exist
        table = torch.randint(-5, self.pages + 5, (B, width), generator=g, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n]
            at += n
        self.page_table = table.to(device)
        self.query_start = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=device)
        self.kv_len = torch.tensor(kv, dtype=torch.int32, device=device)
        self.tokens = sum(new) + tail          # rows of no sequence behind
        self.where = {"page_table": self.page_table, "query_start": self.query_start, "kv_len": self.kv_len}

        def cache():
            x = torch.full((self.pages, Hkv, page, D), float("nan"))
            for b, n in enumerate(kv):
                for i in range(used[b]):
                    rows = min(page, n - i * page)
                    x[table[b, i], :, :rows] = torch.randn(Hkv, rows, D, generator=g)
            x = x.to(dtype).to(device)
            return x if layout == "hnd" else x.transpose(1, 2).contiguous().transpose(1, 2)

        self.key_cache, self.value_cache = cache(), cache()

    def rows(self, b):
        lo = sum(self.new[:b])
        return slice(lo, lo + self.new[b])

    def gather(self, cache, b, n=None):
        """[Hkv, kv, D] in 64 bits; zeros where a page does not exist."""
        n = self.kv[b] if n is None else n
        out = torch.zeros(self.Hkv, n, self.D, dtype=F64, device=cache.device)
        for i in range(-(-n // self.page)):
            rows = min(self.page, n - i * self.page)
            page = int(self.page_table[b, i])
            if 0 <= page < cache.shape[0]:
                out[:, i * self.page:i * self.page + rows] = cache[page, :, :rows].to(F64)
        return out

    def queries(self, Hq, seed=1, sharp=1.0):
        g = torch.Generator().manual_seed(seed)
        return (torch.randn(self.tokens, Hq, self.D, generator=g) * sharp).to(self.dtype).to(self.key_cache.device)


def visible(n, kv, causal, window, device):
    if not causal:
        return torch.ones(n, kv, dtype=torch.bool, device=device)
    at = torch.arange(n, device=device)[:, None] + (kv - n)
    key = torch.arange(kv, device=device)[None]
    seen = key <= at
    return seen & (key > at - window) if window else seen


def attention(batch, q, *, scale=None, causal=True, window=0):
    """(o, lse in powers of two, bound on |o - computed|) per row, NaN where no sequence has the row."""
    T, Hq, D = q.shape
    G = Hq // batch.Hkv
    scale = D ** -0.5 if scale is None else scale
    o = torch.full((T, Hq, D), float("nan"), dtype=F64, device=q.device)
    lse = torch.full((T, Hq), float("nan"), dtype=F64, device=q.device)
    tol, lse_tol = torch.zeros_like(o), torch.zeros_like(lse)
    half = torch.finfo(q.dtype).eps / 2
    for b, n in enumerate(batch.new):
        k, v = batch.gather(batch.key_cache, b), batch.gather(batch.value_cache, b)
        seen = visible(n, batch.kv[b], causal, window, q.device)
        some = seen.any(-1)
        for h in range(Hq):
            x = q[batch.rows(b), h].to(F64)
            if batch.kv[b] == 0:
                o[batch.rows(b), h], lse[batch.rows(b), h] = 0.0, -math.inf
                continue
            s = (x @ k[h // G].T * scale).masked_fill(~seen, -math.inf)
            z = torch.logsumexp(s, -1, keepdim=True)
            p = torch.where(some[:, None], torch.exp(s - z), 0.0)
            out = p @ v[h // G]
            o[batch.rows(b), h] = out
            lse[batch.rows(b), h] = z[:, 0] / math.log(2)
            # f32 sums of D products of exact factors, then the scaling and the subtraction of the maximum, move a logit by
            # delta at most, and with it a probability and their sum; probabilities are rounded to the inputs' type once and
            # results once; exponentials and sums of the f32 parts stay below 2^-18 together
            size = (x.abs() @ k[h // G].abs().T * scale).amax(-1, keepdim=True)
            delta = (D + 8) * 2.0 ** -24 * size
            mass = p @ v[h // G].abs()
            tol[batch.rows(b), h] = half * out.abs() + (half * (1 + half) + 2 * delta + 2.0 ** -18) * mass + torch.finfo(q.dtype).tiny
            lse_tol[batch.rows(b), h] = (2 * delta[:, 0] / math.log(2) + 2.0 ** -18 + 2.0 ** -22 * lse[batch.rows(b), h].abs().nan_to_num(0, 0, 0))
    return o, lse, tol, lse_tol


def key_weights(batch, q, lse, prior=None, *, scale=None, causal=True, window=0):
    """(weights, bound) from the given lse."""
    T, Hq, D = q.shape
    G = Hq // batch.Hkv
    scale = D ** -0.5 if scale is None else scale
    slots = batch.page_table.shape[1] * batch.page
    out = torch.zeros(len(batch.new), batch.Hkv, slots, dtype=F64, device=q.device)
    tol = torch.zeros_like(out)
    for b, n in enumerate(batch.new):
        kv = batch.kv[b]
        k = batch.gather(batch.key_cache, b)
        seen = visible(n, kv, causal, window, q.device)
        for hk in range(batch.Hkv):
            total = torch.zeros(kv, dtype=F64, device=q.device)
            off = torch.zeros_like(total)
            for h in range(hk * G, hk * G + G):
                x = q[batch.rows(b), h].to(F64)
                s = x @ k[hk].T * scale
                z = lse[batch.rows(b), h, None].to(F64) * math.log(2)
                p = torch.where(seen, torch.exp(s - z), 0.0)
                # a logit and its distance to lse in f32, and the exponential's own error
                delta = (D + 8) * 2.0 ** -24 * (x.abs() @ k[hk].abs().T * scale) + 2.0 ** -22 * (s.abs() + z.abs().nan_to_num(0, 0, 0)) + 2.0 ** -20
                total += p.sum(0)
                off += torch.where(seen, p * delta, 0.0).sum(0)
            if prior is not None:
                total += prior[b, hk, :kv].to(F64)
            out[b, hk, :kv] = total
            tol[b, hk, :kv] = off + (n * G + 2) * 2.0 ** -24 * total.abs() + 1e-30
    return out, tol


def turn(x, positions, freq, interleaved, amplitude=1.0, transpose=False, axis=None):
    """Each pair of channels as a complex number; ``positions`` [.., tokens] with axes in front where ``axis`` is given."""
    y = x.to(F64).clone()
    n = len(freq)
    for i in range(n):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
        t = (positions if axis is None else positions[axis[i]]).to(F64) * freq[i]
        z = torch.polar(torch.full_like(t, amplitude), -t if transpose else t)[..., None]
        w = torch.complex(x[..., a].to(F64), x[..., b].to(F64)) * z
        y[..., a], y[..., b] = w.real, w.imag
    return y
