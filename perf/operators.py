"""The paged key/value cache of dtb200 and the operators around it, as a program calls them, for timing.

A rollout that makes a video chunk by chunk, or a text tower that reads a prompt, keeps the keys and values of earlier
tokens in pages ``[pages, kv heads, page size, head dim]``.  The new tokens of all sequences lie one after the other
(``query_start`` says where each sequence's begin), a sequence's page table names its pages in order, and its length
``kv_len`` counts its new tokens too.  A case is one of:

  rotary     queries and keys turned by their positions: ``dtb200.rotary``
  append     new keys turned and written, with the values, into their pages, and the queries turned: ``dtb200.paged_append_``
  attention  the new tokens against the pages of their sequence: ``dtb200.paged_attention``
  weights    what each key got of the new tokens' attention, summed: ``dtb200.paged_key_weights``
  evict      the heaviest and the latest tokens of each head copied to fresh pages: ``dtb200.paged_evict``
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BITS = {"bf16": 16, "fp16": 16, "fp32": 32}


def _dtb200():
    path = os.path.join(os.getcwd(), "diffusers-tpu_b200")
    if path not in sys.path:
        sys.path.insert(1, path)
    import dtb200

    return dtb200


# ----------------------------------------------------------------------------------------------------------------------
# cases
# ----------------------------------------------------------------------------------------------------------------------
def _cache_case(op, B, Hq, Hkv, kv, new, *, D=128, page=64, dtype="bf16", layout="hnd", chunks=None, lens=0, **more):
    """``B`` sequences of ``kv[0]`` to ``kv[1]`` tokens, of which ``new[0]`` to ``new[1]`` are new; where ``chunks`` is
    given only that many sequences have so many, and the others one."""
    return {"op": op, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "dtype": dtype, "layout": layout,
            "kv_lo": kv[0], "kv_hi": kv[1], "new_lo": new[0], "new_hi": new[1], "chunks": B if chunks is None else chunks,
            "lens": lens, **more}


def _rotary_case(tokens, Hq, Hkv, D, rotary, *, dtype="bf16", layout="half", axes=1, scaling="none", factor=1.0, far=0,
                 transpose=False):
    return {"op": "rotary", "tokens": tokens, "Hq": Hq, "Hkv": Hkv, "D": D, "rotary": rotary, "dtype": dtype,
            "layout": layout, "axes": axes, "scaling": scaling, "factor": factor, "far": far, "transpose": transpose}


def _attention_case(*args, causal=True, window=0, lse=False, **more):
    return _cache_case("attention", *args, causal=causal, window=window, lse=lse, **more)


def listed():
    cases = {
        # one new token of 16 sequences, far into a context stretched four times: all latency
        "rotary_step": _rotary_case(16, 24, 8, 128, 64, scaling="yarn", factor=4.0, far=100_000),
        # a layer's queries and keys of two 2048 x 2048 images, time, row and column as axes, neighbours as pairs
        "rotary_image": _rotary_case(2 * 16896, 24, 24, 128, 128, layout="interleaved", axes=3),
        # one new token of 64 sequences goes into the cache
        "append_step": _cache_case("append", 64, 24, 8, (65, 1000), (1, 1), page=16, rotary=128, rope="half"),
        # a prefill of four ragged prompts, cache stored token by token
        "append_prompts": _cache_case("append", 4, 40, 8, (2000, 9000), (2000, 9000), page=64, layout="nhd", rotary=128, rope="half"),
        # single tokens of a few short sequences: the smallest call of a text tower, all latency
        "decode_small": _attention_case(4, 24, 8, (200, 1000), (1, 1), page=16),
        # single tokens of many long sequences: the keys and values are read once, and that is all
        "decode_batch": _attention_case(48, 40, 8, (2000, 32768), (1, 1), page=32, lse=True),
        # a chunk of a long prompt: later chunks see the earlier ones
        "prefill_chunk": _attention_case(1, 40, 8, (61234, 61234), (2048, 2048), page=64, layout="nhd"),
        # the next six latent frames of a 480p clip against all frames so far, every frame of the chunk seeing the whole chunk
        "video_chunk": _attention_case(1, 40, 40, (48872, 48872), (9360, 9360), page=128, causal=False),
        # a decode step's attention added to what the keys of long sequences have got so far
        "weights_step": _cache_case("weights", 8, 40, 8, (4000, 32768), (1, 1), page=32),
        # the last 64 tokens of long prompts vote on which keys to keep
        "weights_vote": _cache_case("weights", 2, 24, 8, (30000, 60000), (64, 64), page=64, layout="nhd"),
        # a short sequence is halved
        "evict_small": _cache_case("evict", 1, 24, 8, (1000, 1000), (1, 1), page=16, keep=512, recent=64),
        # four clips keep a quarter of what they have seen
        "evict_long": _cache_case("evict", 4, 24, 8, (50000, 65536), (1, 1), page=64, keep=16000, recent=3120),
    }
    return [{"name": name, **case} for name, case in cases.items()]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rotary", "append", "attention", "attention", "attention", "weights", "evict"])
    Hkv = rng.choice([1, 2, 4, 5, 8, 10, 24])
    Hq = Hkv * rng.choice([1, 2, 3, 4, 5, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rotary":
        D = rng.choice([40, 64, 80, 96, 128, 128, 128, 256])
        rotary = rng.choice([D, D, D // 2])
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        axes = rng.choice([1, 1, 3]) if rotary >= 32 else 1
        scaling = rng.choice(["none", "linear", "ntk", "yarn"]) if axes == 1 else "none"
        tokens = min(spread(1, 33792), 830_000_000 // ((Hq + Hkv) * D * BITS[dtype] // 4))
        return _rotary_case(tokens, Hq, Hkv, D, rotary, dtype=dtype, layout=rng.choice(["half", "interleaved"]), axes=axes,
                            scaling=scaling, factor=rng.choice([2.0, 4.0, 8.0]) if scaling != "none" else 1.0,
                            far=rng.choice([0, 1000, 1_000_000]), transpose=rng.random() < 0.4)
    shape = {"D": rng.choice([64, 128, 128]), "page": rng.choice([16, 32, 64, 128, 256]), "dtype": dtype,
             "layout": rng.choice(["hnd", "nhd"]), "lens": rng.randrange(1 << 20)}
    B = spread(1, 64)
    tokens = 400_000_000 // (Hkv * shape["D"])          # of the whole cache
    longest = max(min(spread(64, 65536), tokens // B), 1)
    shortest = max(longest // rng.choice([1, 4, 50]), 1)
    if op == "append":
        shape.update(rotary=shape["D"], rope=rng.choice(["half", "interleaved"]))
        longest = min(longest, 300)
        shortest = min(shortest, longest)
        new = (1, 1) if rng.random() < 0.4 else (1, longest)
        return _cache_case("append", B, Hq, Hkv, (shortest, longest), new, **shape)
    if op == "weights":
        longest = max(longest // 4, 1)
        shortest = min(shortest, longest)
        return _cache_case("weights", min(B, 16), Hq, Hkv, (shortest, longest), (1, rng.choice([1, 4, 64])), **shape)
    if op == "evict":
        keep = max(min(spread(16, 65536), longest * rng.choice([1, 2, 3]) // 4, 60_000_000 // (min(B, 8) * Hkv * shape["D"])), 1)
        return _cache_case("evict", min(B, 8), Hq, Hkv, (shortest, longest), (1, 1), keep=keep, recent=rng.randint(0, keep), **shape)
    kind = rng.choice(["step", "step", "chunk", "mixed", "prompt"])
    more = {"window": spread(100, 10000)} if rng.random() < 0.2 else {}
    if kind == "step":
        new, chunks = (1, rng.choice([1, 1, 4])), B
    elif kind == "mixed":
        new, chunks = (1, spread(16, 1024)), 1
    else:
        B = min(B, 6)
        longest = min(longest, 40000 // B)
        shortest = longest if kind == "prompt" else min(shortest, longest)
        new, chunks = (1, spread(2, 2048) if kind == "chunk" else min(longest, 6000)), B
        new = (1, max(min(new[1], 15_000_000_000 // (B * Hq * longest)), 1))
    if not more and kind == "chunk":
        more["causal"] = rng.random() < 0.5
    return _attention_case(B, Hq, Hkv, (shortest, longest), new, chunks=chunks, lse=rng.random() < 0.5, **more, **shape)


def _lengths(case):
    """New tokens and whole length of each sequence."""
    rng = random.Random(1000 + case["lens"])
    new, kv = [], []
    for b in range(case["B"]):
        n = int(round(math.exp(rng.uniform(math.log(case["kv_lo"]), math.log(case["kv_hi"])))))
        m = rng.randint(case["new_lo"], case["new_hi"]) if b < case["chunks"] else 1
        kv.append(n)
        new.append(min(m, n))
    if case["op"] == "append" and case["new_lo"] > 1:      # whole prompts
        new = list(kv)
    return new, kv


def _visible(case, n, length):
    """(query, key) pairs of one head of a sequence, and the keys that any of them sees."""
    if not case.get("causal", True):
        return n * length, length
    first = length - n                     # position of the first new token
    window = case.get("window", 0)
    if not window:
        return n * first + n * (n + 1) // 2, length
    full = sum(min(first + i + 1, window) for i in range(n))
    return full, min(length, window + n - 1)


# ----------------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ----------------------------------------------------------------------------------------------------------------------
def _axis_pairs(case):
    pairs = case["rotary"] // 2
    if case["axes"] == 1:
        return [pairs]
    side = 3 * pairs // 8                  # rows and columns get more pairs than time
    return [pairs - 2 * side, side, side]


def _frequencies(pairs, base, scaling, factor, original):
    """64-bit angle per position of each pair of one axis, and the factor on the result."""
    j = torch.arange(pairs, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (pairs / (pairs - 1)) if pairs > 1 else base
    freq = base ** (-j / pairs)
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "yarn":
        def pair_of(turns):                # the pair that makes so many turns over the original length
            return pairs * math.log(original / (turns * 2 * math.pi)) / math.log(base)

        low, high = max(math.floor(pair_of(32.0)), 0), min(math.ceil(pair_of(1.0)), pairs - 1)
        ramp = ((j - low) / max(high - low, 1e-3)).clamp(0, 1)
        return freq / factor * ramp + freq * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


_BASE, _ORIGINAL = 10000.0, 8192


def _rotary_state(case, device):
    axes = _axis_pairs(case)
    if own:
        table = _dtb200().make_rotary_table(
            case["rotary"], base=_BASE, layout=case["layout"], axes=axes if len(axes) > 1 else None,
            scaling=None if case["scaling"] == "none" else case["scaling"], factor=case["factor"], original_length=_ORIGINAL, device=device)
        return {"table": table}
    parts = [_frequencies(p, _BASE, case["scaling"], case["factor"], _ORIGINAL) for p in axes]
    axis = torch.cat([torch.full((p,), a, dtype=torch.int64) for a, p in enumerate(axes)])
    return {"freq": torch.cat([f for f, _ in parts]).to(device), "axis": axis.to(device), "amplitude": parts[0][1],
            "half": case["layout"] == "half"}


def _prepare_rotary(case, g):
    T, dtype = case["tokens"], DTYPES[case["dtype"]]
    state = {"case": case, "rope": _rotary_state(case, "cuda")}
    state["q"], state["k"] = (torch.randn(T, h, case["D"], generator=g, device="cuda", dtype=dtype) for h in (case["Hq"], case["Hkv"]))
    positions = torch.arange(T, device="cuda")
    if case["axes"] == 3:                  # frame, row and column of a latent of 64 x 64
        positions = torch.stack([positions // 4096, positions // 64 % 64, positions % 64])
    elif case["far"]:
        positions = torch.randint(0, case["far"], (T,), generator=g, device="cuda")
    state["positions"] = positions.to(torch.int32)
    return state


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "rotary":
        return _prepare_rotary(case, g)
    B, Hq, Hkv, D, page, dtype = (case[k] for k in ("B", "Hq", "Hkv", "D", "page", "dtype"))
    dtype = DTYPES[dtype]
    new, kv = _lengths(case)
    used = [-(-n // page) for n in kv]
    kept = [-(-min(n, case["keep"]) // page) for n in kv] if case["op"] == "evict" else []
    pages = sum(used) + sum(kept) + 3      # a few belong to others
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)

    def table_of(counts, at):
        table = torch.full((B, max(counts)), -1, dtype=torch.int32, device="cuda")
        for b, n in enumerate(counts):
            table[b, :n] = order[at:at + n]
            at += n
        return table, at

    state = {"case": case, "new": new, "kv": kv}
    state["page_table"], at = table_of(used, 0)
    if kept:
        state["out_table"], at = table_of(kept, at)
    state["kv_len"] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["query_start"] = torch.tensor(starts, dtype=torch.int32, device="cuda")

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def cache():
        return normal(pages, Hkv, page, D) if case["layout"] == "hnd" else normal(pages, page, Hkv, D).transpose(1, 2)

    state["key_cache"] = cache()
    if case["op"] != "weights":
        state["value_cache"] = cache()
    T = starts[-1]
    if case["op"] == "append":
        state["q"], state["k"], state["v"] = normal(T, Hq, D), normal(T, Hkv, D), normal(T, Hkv, D)
        state["rope"] = _rotary_state({"rotary": case["rotary"], "layout": case["rope"], "axes": 1, "scaling": "none", "factor": 1.0}, "cuda")
    elif case["op"] == "evict":
        width = state["page_table"].shape[1] * page
        # few keys get much, most get little
        state["weights"] = torch.randn(B, Hkv, width, generator=g, device="cuda").mul_(2.0).exp_()
    else:
        state["q"] = normal(T, Hq, D).mul_(2.0)
    if case["op"] == "weights":
        width = state["page_table"].shape[1] * page
        state["prior"] = torch.rand(B, Hkv, width, generator=g, device="cuda")
        lse = torch.empty(T, Hq, device="cuda")
        for b, rows, q in _sequences(state):
            keys = _gather(state, "key_cache", b).float()
            for h, s in _scores(case, q.float(), keys, new[b], kv[b], D ** -0.5):
                lse[rows, h] = (torch.logsumexp(s, -1) / math.log(2)).view(new[b], -1)
        state["lse"] = lse                 # in units of powers of two
    return state


# ----------------------------------------------------------------------------------------------------------------------
# plain forms
# ----------------------------------------------------------------------------------------------------------------------
def _sequences(state):
    """Each sequence's number, its rows among the new tokens, and its queries."""
    at = 0
    for b, n in enumerate(state["new"]):
        yield b, slice(at, at + n), state["q"][at:at + n]
        at += n


def _gather(state, which, b):
    """Keys or values of a sequence, ``[kv heads, length, D]``."""
    page, n = state["case"]["page"], state["kv"][b]
    ids = state["page_table"][b, :-(-n // page)].long()
    x = state[which][ids].transpose(0, 1)
    return x.reshape(x.shape[0], -1, x.shape[-1])[:, :n]


def _mask(case, n, length, device):
    """What each new token sees of the keys, or None where that is all of them."""
    if not case.get("causal", True):
        return None
    at = torch.arange(length - n, length, device=device)[:, None]
    key = torch.arange(length, device=device)[None, :]
    seen = key <= at
    if case.get("window", 0):
        seen &= key > at - case["window"]
    return seen


def _scores(case, q, keys, n, length, scale):
    """Query heads of a key head, and their masked logits ``[new tokens * heads of the group, length]``."""
    seen = _mask(case, n, length, q.device)
    G = case["Hq"] // case["Hkv"]
    for hk in range(case["Hkv"]):
        heads = slice(hk * G, hk * G + G)
        s = (q[:, heads].reshape(n * G, -1) @ keys[hk].T).mul_(scale)
        if seen is not None and n > 1:
            s.view(n, G, length).masked_fill_(~seen[:, None], -math.inf)
        elif case.get("window", 0):
            s.masked_fill_(~seen, -math.inf)
        yield heads, s


def _plain_attention(state):
    case, q = state["case"], state["q"]
    T, Hq, D = q.shape
    out, lse = torch.empty_like(q), torch.empty(T, Hq, device=q.device)
    for b, rows, qb in _sequences(state):
        keys, values = _gather(state, "key_cache", b).float(), _gather(state, "value_cache", b).float()
        n = state["new"][b]
        for heads, s in _scores(case, qb.float(), keys, n, state["kv"][b], D ** -0.5):
            top = s.amax(-1, keepdim=True)
            p = s.sub_(top).exp_()
            total = p.sum(-1, keepdim=True)
            hk = heads.start // (Hq // case["Hkv"])
            out[rows, heads] = ((p @ values[hk]) / total).view(n, -1, D).to(q.dtype)
            lse[rows, heads] = ((top + total.log()) / math.log(2)).view(n, -1)
    return (out, lse) if case["lse"] else out


def _plain_rotate(x, positions, rope, transpose):
    """``positions`` [tokens] or [axes, tokens]; angles in 64 bits, for far positions."""
    where = positions[rope["axis"]] if positions.dim() == 2 else positions[None].expand(rope["freq"].numel(), -1)
    angle = (where.double() * rope["freq"][:, None]).T[:, None, :]
    cos, sin = (angle.cos() * rope["amplitude"]).float(), (angle.sin() * rope["amplitude"]).float()
    if transpose:
        sin = -sin
    pairs = rope["freq"].numel()
    y = x.float()
    turned, rest = y[..., :2 * pairs], y[..., 2 * pairs:]
    a, b = (turned[..., :pairs], turned[..., pairs:]) if rope["half"] else (turned[..., 0::2], turned[..., 1::2])
    c, d = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([c, d], -1) if rope["half"] else torch.stack([c, d], -1).flatten(-2)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _slots(state):
    """Page, and row of the page, of each new token, and its position."""
    page = state["case"]["page"]
    where, at = [], []
    for b, n in enumerate(state["new"]):
        pos = torch.arange(state["kv"][b] - n, state["kv"][b], device="cuda")
        where.append(state["page_table"][b, pos // page].long())
        at.append(pos)
    at = torch.cat(at)
    return torch.cat(where), at % page, at


def _plain_append(state):
    ids, row, at = _slots(state)
    state["key_cache"][ids, :, row] = _plain_rotate(state["k"], at, state["rope"], False)
    state["value_cache"][ids, :, row] = state["v"]
    return _plain_rotate(state["q"], at, state["rope"], False), state["key_cache"], state["value_cache"]


def _plain_weights(state):
    case, q = state["case"], state["q"]
    out = torch.zeros_like(state["prior"])
    for b, rows, qb in _sequences(state):
        n, length = state["new"][b], state["kv"][b]
        keys = _gather(state, "key_cache", b).float()
        for heads, s in _scores(case, qb.float(), keys, n, length, q.shape[-1] ** -0.5):
            hk = heads.start // (case["Hq"] // case["Hkv"])
            lse = state["lse"][rows, heads].reshape(-1, 1)
            out[b, hk, :length] = state["prior"][b, hk, :length] + (s / math.log(2) - lse).exp2().sum(0)
    return out


def _plain_evict(state):
    case, keep, recent = state["case"], state["case"]["keep"], state["case"]["recent"]
    B, Hkv, page = case["B"], case["Hkv"], case["page"]
    device = state["weights"].device
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32, device=device)
    weights = torch.zeros(B, Hkv, state["out_table"].shape[1] * page, device=device)
    heads = torch.arange(Hkv, device=device)[:, None]
    for b, length in enumerate(state["kv"]):
        n = min(length, keep)
        if length > keep:
            old = length - recent
            order = state["weights"][b, :, :old].sort(dim=-1, descending=True, stable=True).indices[:, :keep - recent]
            last = torch.arange(old, length, device=device).expand(Hkv, -1)
            index = torch.cat([order.sort(dim=-1).values, last], -1)
        else:
            index = torch.arange(length, device=device).expand(Hkv, -1)
        kept[b, :, :n] = index.to(torch.int32)
        weights[b, :, :n] = state["weights"][b].gather(-1, index)
        src = state["page_table"][b].long()[index // page]
        at = torch.arange(n, device=device)
        dst = state["out_table"][b].long()[at // page][None].expand(Hkv, -1)
        for which in ("key_cache", "value_cache"):
            state[which][dst, heads, (at % page)[None].expand(Hkv, -1)] = state[which][src, heads, index % page]
    return kept, weights, state["kv_len"].clamp(max=keep), state["key_cache"], state["value_cache"]


# ----------------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        if op == "rotary":
            return tuple(_plain_rotate(state[x], state["positions"], state["rope"], case["transpose"]) for x in "qk")
        return {"append": _plain_append, "attention": _plain_attention, "weights": _plain_weights, "evict": _plain_evict}[op](state)
    dtb200 = _dtb200()
    if op == "rotary":
        return dtb200.rotary(state["q"], state["k"], table=state["rope"]["table"], positions=state["positions"], transpose=case["transpose"])
    if op == "evict":
        kept, weights, kv_len = dtb200.paged_evict(state["key_cache"], state["value_cache"], state["weights"], page_table=state["page_table"],
                                                   out_table=state["out_table"], kv_len=state["kv_len"], keep=case["keep"], recent=case["recent"])
        return kept, weights, kv_len, state["key_cache"], state["value_cache"]
    where = {"page_table": state["page_table"], "query_start": state["query_start"], "kv_len": state["kv_len"]}
    if op == "append":
        q = dtb200.paged_append_(state["key_cache"], state["value_cache"], state["k"], state["v"], query=state["q"],
                                 table=state["rope"]["table"], **where)
        return q, state["key_cache"], state["value_cache"]
    if op == "weights":
        return dtb200.paged_key_weights(state["q"], state["key_cache"], state["lse"], prior=state["prior"], **where)
    return dtb200.paged_attention(state["q"], state["key_cache"], state["value_cache"], causal=case["causal"],
                                  window=case["window"] or None, return_lse=case["lse"], **where)


def work(case):
    """Each row that a pass needs read once and each that it makes written once; products for visible pairs only."""
    op, wide = case["op"], BITS[case["dtype"]] // 8
    if op == "rotary":
        rows = case["tokens"] * (case["Hq"] + case["Hkv"])
        return {"bytes": 2.0 * rows * case["D"] * wide + 4.0 * case["tokens"] * case["axes"], "flops": 3.0 * rows * case["rotary"]}
    new, kv = _lengths(case)
    Hq, Hkv, D, T = case["Hq"], case["Hkv"], case["D"], sum(new)
    tables = sum(4.0 * -(-n // case["page"]) for n in kv)
    if op == "append":
        return {"bytes": 2.0 * T * (Hq + 2 * Hkv) * D * wide, "flops": 3.0 * T * (Hq + Hkv) * case["rotary"]}
    if op == "evict":
        kept = sum(min(n, case["keep"]) for n in kv)
        return {"bytes": Hkv * (4.0 * sum(kv) + kept * (4.0 * D * wide + 8.0)) + tables, "flops": 0.0}
    pairs, keys = (sum(x) for x in zip(*(_visible(case, n, length) for n, length in zip(new, kv))))
    if op == "weights":
        return {"bytes": T * Hq * (D * wide + 4.0) + keys * Hkv * (D * wide + 8.0) + tables, "flops": 2.0 * Hq * D * pairs}
    return {"bytes": 2.0 * T * Hq * D * wide + 2.0 * keys * Hkv * D * wide + tables, "flops": 4.0 * Hq * D * pairs}


# ----------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ----------------------------------------------------------------------------------------------------------------------
_EXACT_PAIRS = 3e10          # (query, key) pairs over all heads; more take too long


def _exact_rows(state, name, b, hk):
    """Rows of one head of a sequence's keys or values in 64 bits, page by page through its table."""
    n, page = state["kv"][b], state["case"]["page"]
    at = torch.arange(n, device="cuda")
    return state[name][state["page_table"][b].long()[at // page], hk, at % page].double()


def _exact_turn(x, at, case, transpose=False):
    """Each pair as a complex number times exp(i angle)."""
    axes = _axis_pairs(case)
    freq, axis, gain = [], [], 1.0
    for a, pairs in enumerate(axes):
        f, gain = _frequencies(pairs, _BASE, case["scaling"], case["factor"], _ORIGINAL)
        freq += f.tolist()
        axis += [a] * pairs
    y, half = x.double().clone(), len(freq)
    for i in range(half):
        a, b = (i, i + half) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        t = (at[axis[i]] if at.dim() == 2 else at).double() * freq[i]
        z = torch.complex(x[..., a].double(), x[..., b].double()) * torch.polar(torch.full_like(t, gain), -t if transpose else t)[:, None]
        y[..., a], y[..., b] = z.real, z.imag
    return y


def exact(case, seed):
    op = case["op"]
    if op in ("attention", "weights"):
        new, kv = _lengths(case)
        if case["Hq"] * float(sum(n * m for n, m in zip(new, kv))) > _EXACT_PAIRS:
            return None
    state = prepare(case, seed)
    if op == "rotary":
        return tuple(_exact_turn(state[x], state["positions"], case, case["transpose"]) for x in "qk")
    new, kv = state["new"], state["kv"]
    if op == "evict":                      # chosen by counting what is heavier, and copied
        kept = torch.full((case["B"], case["Hkv"], case["keep"]), -1, dtype=torch.int32)
        mass = torch.zeros(case["B"], case["Hkv"], state["out_table"].shape[1] * case["page"], dtype=torch.float64)
        for b, m in enumerate(kv):
            for hk in range(case["Hkv"]):
                w = state["weights"][b, hk, :m].cpu().double()
                late = list(range(max(m - case["recent"], 0), m)) if m > case["keep"] else list(range(m))
                early = sorted(range(m - len(late)), key=w.tolist().__getitem__, reverse=True)    # stable: ties in order
                index = torch.tensor(sorted(early[:min(m, case["keep"]) - len(late)]) + late)
                kept[b, hk, :len(index)] = index.int()
                mass[b, hk, :len(index)] = w[index]
        return kept.cuda(), mass.cuda(), torch.tensor([min(m, case["keep"]) for m in kv], dtype=torch.int32, device="cuda"), None, None
    if op == "append":
        at = torch.cat([torch.arange(m - n, m, device="cuda") for n, m in zip(new, kv)])
        shape = {"rotary": case["rotary"], "layout": case["rope"], "axes": 1, "scaling": "none", "factor": 1.0}
        return _exact_turn(state["q"], at, shape), None, None
    q, G = state["q"], case["Hq"] // case["Hkv"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    logs = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    mass = torch.zeros(state["prior"].shape, dtype=torch.float64, device="cuda") if op == "weights" else None
    first = 0
    for b, (n, m) in enumerate(zip(new, kv)):
        for hk in range(case["Hkv"]):
            k = _exact_rows(state, "key_cache", b, hk)
            v = _exact_rows(state, "value_cache", b, hk) if op == "attention" else None
            if op == "weights":
                mass[b, hk, :m] = state["prior"][b, hk, :m].double()
            for h in range(hk * G, hk * G + G):
                step = max(1, int(4e8) // m)
                for lo in range(0, n, step):
                    hi = min(lo + step, n)
                    s = q[first + lo:first + hi, h].double() @ k.T * case["D"] ** -0.5
                    if case.get("causal", True):
                        gap = torch.arange(m - n + lo, m - n + hi, device="cuda")[:, None] - torch.arange(m, device="cuda")
                        hidden = gap < 0
                        if case.get("window", 0):
                            hidden |= gap >= case["window"]
                        s[hidden] = -math.inf
                    if op == "weights":
                        mass[b, hk, :m] += torch.exp(s - state["lse"][first + lo:first + hi, h, None].double() * math.log(2)).sum(0)
                        continue
                    z = torch.logsumexp(s, -1, keepdim=True)
                    out[first + lo:first + hi, h] = torch.exp(s - z) @ v
                    logs[first + lo:first + hi, h] = z[:, 0] / math.log(2)
        first += n
    if op == "weights":
        return mass
    return (out, logs) if case["lse"] else out
