"""Rotary positions and a paged key/value cache: the operators of a model that attends to what earlier calls left behind.

A cache is two tensors ``[pages, heads_kv, page_size, dim]`` (bf16 or fp16, any strides with a contiguous last axis, so
``[pages, page_size, heads_kv, dim]`` storage is passed as its ``transpose(1, 2)``).  The new tokens of all sequences lie one
after the other in ``[tokens, heads, dim]`` tensors: those of sequence ``b`` are rows ``query_start[b]`` to
``query_start[b + 1]``.  ``page_table[b]`` names the pages of a sequence in order and ``kv_len[b]`` counts its tokens, the
new ones included, so a step is

    q = paged_append_(key_cache, value_cache, k, v, query=q, table=rope, **where)   # rotate, write k and v
    o = paged_attention(q, key_cache, value_cache, **where)                          # attend

with ``where = dict(page_table=..., query_start=..., kv_len=...)``, int32 tensors on the device that the calls never read
on the host: a captured step replays with other lengths and pages.  :func:`paged_key_weights` sums what each key got of the
attention, and :func:`paged_evict` cuts sequences to their heaviest and latest tokens by it.

The reference keeps no cache; its rotary embedding takes precomputed tables (``diffusers_tpu/models/minimax_h3/jax_dit.py:251-262``).
All compute goes through the C ABI in ``libdtb200_attn.so``; nothing here falls back to PyTorch.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .ops import _on_device, _status_buffer, _stream_ptr

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


class RotaryTable:
    """What :func:`make_rotary_table` builds and :func:`rotary` and :func:`paged_append_` take: how far each pair of channels
    turns per position, on the device in 64 bits, which row of the positions turns it, and the factor on the result."""

    def __init__(self, turns: torch.Tensor, axis: Optional[torch.Tensor], n_axes: int, interleaved: bool, amplitude: float):
        self.turns, self.axis, self.n_axes, self.interleaved, self.amplitude = turns, axis, n_axes, interleaved, amplitude
        self.rotary = 2 * turns.numel()
        self.device = turns.device
        self._ptrs = (turns.data_ptr(), axis.data_ptr() if axis is not None else None)


def make_rotary_table(rotary: int, *, base: float = 10000.0, layout: str = "half", axes: Optional[Sequence[int]] = None,
                      scaling: Optional[str] = None, factor: float = 1.0, original_length: int = 8192, fast_turns: float = 32.0,
                      slow_turns: float = 1.0, device: Union[torch.device, str] = "cuda") -> RotaryTable:
    """Angles of a rotary embedding over the leading ``rotary`` channels of a head.

    Pair ``j`` of ``n`` turns by ``base ** (-j / n)`` per position.  ``layout="half"`` pairs channel ``i`` with
    ``i + rotary / 2``, ``"interleaved"`` neighbours.  ``axes`` gives the number of pairs that each of several position
    axes turns (time, row and column of a video token, say), each with a ladder of its own.  For contexts longer than a
    model was trained on, ``scaling`` is ``"linear"`` (positions divided by ``factor``), ``"ntk"`` (base raised so that the
    slowest pair slows by ``factor`` and the fastest not at all) or ``"yarn"`` (pairs of fewer than ``slow_turns`` turns over
    ``original_length`` positions slow by ``factor``, those of more than ``fast_turns`` keep their speed, a ramp between, and
    queries and keys are multiplied by ``0.1 ln(factor) + 1``).
    """
    if rotary <= 0 or rotary % 2:
        raise ValueError(f"rotary must be a positive even number of channels, got {rotary}")
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    if not (base > 1.0 and math.isfinite(base)) or not (factor > 0.0 and math.isfinite(factor)):
        raise ValueError("base must be above 1 and factor above 0")
    counts = [rotary // 2] if axes is None else [int(n) for n in axes]
    if any(n <= 0 for n in counts) or sum(counts) != rotary // 2:
        raise ValueError(f"axes must be positive numbers of pairs that add up to {rotary // 2}, got {counts}")
    amplitude = 1.0
    turns, axis = [], []
    for a, n in enumerate(counts):
        b = base
        if scaling == "ntk" and n > 1:
            b = base * factor ** (n / (n - 1))
        ladder = [b ** (-j / n) for j in range(n)]
        if scaling == "linear":
            ladder = [f / factor for f in ladder]
        elif scaling == "yarn":
            def pair_of(t):
                return n * math.log(original_length / (t * 2 * math.pi)) / math.log(base)

            low, high = max(math.floor(pair_of(fast_turns)), 0), min(math.ceil(pair_of(slow_turns)), n - 1)
            for j in range(n):
                ramp = min(max((j - low) / max(high - low, 1e-3), 0.0), 1.0)
                ladder[j] = ladder[j] / factor * ramp + ladder[j] * (1.0 - ramp)
            amplitude = 0.1 * math.log(factor) + 1.0
        turns += [f / (2 * math.pi) for f in ladder]
        axis += [a] * n
    device = torch.device(device)
    return RotaryTable(torch.tensor(turns, dtype=torch.float64, device=device),
                       torch.tensor(axis, dtype=torch.int32, device=device) if len(counts) > 1 else None,
                       len(counts), layout == "interleaved", amplitude)


def _need_cuda(name: str, t: torch.Tensor, device: Optional[torch.device] = None) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: dtb200 has no CPU path")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")


def _rows(name: str, t: torch.Tensor) -> torch.Tensor:
    """``t`` where the kernels can address it (contiguous channels, no broadcast axis), else a copy."""
    st, sh = t.stride(), t.shape
    if st[-1] == 1 or sh[-1] == 1:
        for i in range(len(sh) - 1):
            if st[i] <= 0 and sh[i] > 1:
                return t.contiguous()
        return t
    return t.contiguous()


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """As :func:`_rows`, with pointer and strides multiples of 16 bytes."""
    st, sh = t.stride(), t.shape
    if st[-1] == 1 and t.data_ptr() % 16 == 0 and all(sh[i] == 1 or (st[i] > 0 and st[i] % 8 == 0) for i in range(len(sh) - 1)):
        return t
    return t.contiguous()


def _stride(t: torch.Tensor, i: int) -> int:
    """Element stride of an axis; of one with a single entry, which torch may give any stride, one that is harmless."""
    return t.stride(i) if t.shape[i] != 1 else 0


def _need_out(name: str, out: torch.Tensor, like: torch.Tensor) -> None:
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    if out.shape[-1] > 1 and out.stride(-1) != 1 or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{name} must have contiguous channels and no broadcast axis")


def _positions(positions: torch.Tensor, table: RotaryTable, batch: int, tokens: int, device: torch.device):
    """Checked positions and their (axis, batch, token) strides."""
    if not isinstance(positions, torch.Tensor):
        raise TypeError("positions must be a tensor")
    _need_cuda("positions", positions, device)
    if positions.dtype not in _POSITION_TYPES:
        raise NotImplementedError(f"positions must be int32, int64 or float32, got {positions.dtype}")
    shape, strides = tuple(positions.shape), positions.stride()
    sa = 0
    if table.n_axes > 1:
        if not shape or shape[0] != table.n_axes:
            raise ValueError(f"positions must start with the table's {table.n_axes} axes, got {shape}")
        sa, shape, strides = strides[0], shape[1:], strides[1:]
    if shape == (tokens,):
        return positions, sa, 0, strides[0]
    if shape == (batch, tokens):
        return positions, sa, strides[0], strides[1]
    raise ValueError(f"positions must be [{tokens}] or [{batch}, {tokens}] (behind the axes), got {tuple(positions.shape)}")


def rotary(query: torch.Tensor, key: Optional[torch.Tensor] = None, *, table: RotaryTable, positions: torch.Tensor,
           transpose: bool = False, out: Optional[torch.Tensor] = None, key_out: Optional[torch.Tensor] = None):
    """Queries, and keys if given, turned by their positions: ``[tokens, heads, dim]`` or ``[B, tokens, heads, dim]`` (pass
    ``[B, heads, tokens, dim]`` as its ``transpose(1, 2)``), bf16, fp16 or f32, any even number of rotated channels.

    ``positions`` is ``[tokens]`` or ``[B, tokens]``, int32, int64 or f32, with the table's axes in front where it has several.
    Angles are reduced in 64 bits, products are f32, results are rounded once; channels past ``table.rotary`` are copied.
    ``transpose=True`` applies the transposed map: the gradient of the inputs from that of the results (and the inverse,
    where the table does not scale).  ``out`` and ``key_out`` may be the inputs.  Returns the turned query, or (query, key).
    """
    _need_cuda("query", query)
    dev = query.device
    if query.dtype not in _DTYPES:
        raise NotImplementedError(f"rotary takes bf16, fp16 or f32, got {query.dtype}")
    if query.dim() not in (3, 4):
        raise ValueError(f"query must be [tokens, heads, dim] or [B, tokens, heads, dim], got {tuple(query.shape)}")
    if table.device != dev:
        raise ValueError(f"the rotary table is on {table.device}, not on {dev}")
    D = query.shape[-1]
    if table.rotary > D:
        raise ValueError(f"the table turns {table.rotary} channels, heads have {D}")
    if D > 512:
        raise NotImplementedError("heads of more than 512 channels")
    four = query.dim() == 4
    batch, tokens = (query.shape[0] if four else 1), query.shape[-3]
    if key is not None:
        _need_cuda("key", key, dev)
        if key.dtype != query.dtype or key.dim() != query.dim() or key.shape[:-2] != query.shape[:-2] or key.shape[-1] != D:
            raise ValueError(f"key {tuple(key.shape)} {key.dtype} does not go with query {tuple(query.shape)} {query.dtype}")
    elif key_out is not None:
        raise ValueError("key_out without key")
    positions, pa, pb, ps = _positions(positions, table, batch, tokens, dev)
    if out is None:
        out = torch.empty_like(query)
    else:
        _need_out("out", out, query)
    if key is not None:
        if key_out is None:
            key_out = torch.empty_like(key)
        else:
            _need_out("key_out", key_out, key)
    if batch and tokens and (query.shape[-2] or (key is not None and key.shape[-2])):
        q, k = _rows("query", query), (_rows("key", key) if key is not None else None)
        qo, ko = out, key_out
        if not query.shape[-2]:
            q, qo, k, ko = k, ko, None, None
        elif k is not None and not key.shape[-2]:
            k = ko = None
        # empty_like of a view may not keep its channels contiguous
        fix = [t if t is None or t.stride(-1) == 1 or D == 1 else torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (qo, ko)]

        def strides(t):
            return (0, 0, 0) if t is None else (_stride(t, 0) if four else 0, _stride(t, -3), _stride(t, -2))

        p = _lib.RotaryParams(q.data_ptr(), fix[0].data_ptr(), k.data_ptr() if k is not None else None,
                              fix[1].data_ptr() if fix[1] is not None else None, *table._ptrs, positions.data_ptr(),
                              *strides(q), *strides(fix[0]), *strides(k), *strides(fix[1]), pa, pb, ps,
                              _POSITION_TYPES[positions.dtype], batch, tokens, q.shape[-2], k.shape[-2] if k is not None else 0, D,
                              table.rotary, table.n_axes, table.interleaved, bool(transpose), _DTYPES[query.dtype], table.amplitude)
        with _on_device(dev):
            st = _lib.load().dtb_rotary(ctypes.byref(p), _stream_ptr(dev))
        _lib.check(st, "dtb_rotary")
        if fix[0] is not qo:
            qo.copy_(fix[0])
        if fix[1] is not ko:
            ko.copy_(fix[1])
    return out if key is None else (out, key_out)


def _check_cache(name: str, cache: torch.Tensor, device: torch.device, dtype: Optional[torch.dtype] = None) -> None:
    _need_cuda(name, cache, device)
    if cache.dtype != torch.bfloat16 and cache.dtype != torch.float16:
        raise NotImplementedError(f"{name} must be bf16 or fp16, got {cache.dtype}")
    if dtype is not None and cache.dtype != dtype:
        raise ValueError(f"{name} is {cache.dtype}, the new tokens are {dtype}")
    if cache.dim() != 4:
        raise ValueError(f"{name} must be [pages, heads_kv, page_size, dim], got {tuple(cache.shape)}")
    st, sh = cache.stride(), cache.shape
    # a cache is never copied to make it fit
    if st[3] != 1 or cache.data_ptr() % 16 or any(n > 1 and (s <= 0 or s % 8) for s, n in zip(st[:3], sh[:3])):
        raise ValueError(f"{name} needs contiguous channels, positive strides and rows on 16-byte boundaries, got strides {st}")


def _check_where(page_table: torch.Tensor, query_start: Optional[torch.Tensor], kv_len: torch.Tensor, device: torch.device) -> int:
    batch = kv_len.shape[0] if kv_len.dim() == 1 else -1
    for name, t, shape in (("kv_len", kv_len, (batch,)), ("page_table", page_table, (batch, page_table.shape[-1] if page_table.dim() else 0)),
                           ("query_start", query_start, (batch + 1,))):
        if t is None:
            continue
        _need_cuda(name, t, device)
        if t.dtype != torch.int32:
            raise NotImplementedError(f"{name} must be int32, got {t.dtype}")
        if tuple(t.shape) != shape or batch < 0:
            raise ValueError(f"{name} has shape {tuple(t.shape)}: kv_len is [B], query_start [B + 1], page_table [B, pages of a sequence]")
        if shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous in its last axis")
    return batch


def _check_heads(query: torch.Tensor, cache: torch.Tensor) -> None:
    _need_cuda("query", query)
    if query.dim() != 3:
        raise ValueError(f"query must be [tokens, heads, dim], got {tuple(query.shape)}")
    if cache.dim() == 4 and query.shape[2] != cache.shape[3]:
        raise ValueError(f"query heads have {query.shape[2]} channels, the cache's {cache.shape[3]}")
    if cache.dim() == 4 and (not cache.shape[1] or not query.shape[1] or query.shape[1] % cache.shape[1]):
        raise ValueError("query heads must be a multiple of key/value heads")


def _check_scale(scale: Optional[float]) -> float:
    if scale is None:
        return 0.0
    scale = float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _check_window(causal: bool, window: Optional[int]) -> int:
    if window is None:
        return 0
    if window <= 0:
        raise ValueError(f"window must be positive, got {window}")
    if not causal:
        raise ValueError("a window needs causal=True")
    return min(int(window), 0x7fffffff)


def paged_append_(key_cache: torch.Tensor, value_cache: torch.Tensor, key: torch.Tensor, value: torch.Tensor, *,
                  page_table: torch.Tensor, query_start: torch.Tensor, kv_len: torch.Tensor, table: Optional[RotaryTable] = None,
                  positions: Optional[torch.Tensor] = None, query: Optional[torch.Tensor] = None,
                  query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Writes the new keys and values ``[tokens, heads_kv, dim]`` into the pages of their sequences, in place, and returns the
    query (``[tokens, heads, dim]``, optional): the step in front of :func:`paged_attention`, in one launch.

    With a ``table`` keys and queries are turned on the way (:func:`rotary`), by ``positions`` (``[tokens]``, with the table's
    axes in front where it has several) or, without them, by each token's place in its sequence.  ``query_out`` may be
    ``query``.  Rows of no sequence are left as they were, in ``query_out`` too; tokens that their page table has no page for
    are dropped.  No two sequences that append may share the page that they append to.
    """
    _need_cuda("key", key)
    dev, dtype = key.device, key.dtype
    _check_cache("key_cache", key_cache, dev, dtype)
    _check_cache("value_cache", value_cache, dev, dtype)
    if key.dim() != 3 or value.shape != key.shape or value.dtype != dtype or value.device != dev:
        raise ValueError(f"key and value must both be [tokens, heads_kv, dim], got {tuple(key.shape)} and {tuple(value.shape)} {value.dtype}")
    if key_cache.shape != value_cache.shape or key.shape[1:] != (key_cache.shape[1], key_cache.shape[3]):
        raise ValueError(f"key {tuple(key.shape)} does not go with caches {tuple(key_cache.shape)} and {tuple(value_cache.shape)}")
    batch = _check_where(page_table, query_start, kv_len, dev)
    T, Hkv, D = key.shape
    if table is not None:
        if table.device != dev:
            raise ValueError(f"the rotary table is on {table.device}, not on {dev}")
        if table.rotary > D:
            raise ValueError(f"the table turns {table.rotary} channels, heads have {D}")
        if table.n_axes > 1 and positions is None:
            raise ValueError(f"a table of {table.n_axes} axes needs positions")
    elif positions is not None:
        raise ValueError("positions without a table")
    if D > 512:
        raise NotImplementedError("heads of more than 512 channels")
    pa = ps = 0
    if positions is not None:
        positions, pa, _, ps = _positions(positions, table, 1, T, dev)
    if query is not None:
        _need_cuda("query", query, dev)
        if query.dim() != 3 or query.shape[0] != T or query.shape[2] != D or query.dtype != dtype:
            raise ValueError(f"query {tuple(query.shape)} {query.dtype} does not go with key {tuple(key.shape)} {dtype}")
        if query_out is None:
            query_out = torch.empty(query.shape, dtype=dtype, device=dev)
        else:
            _need_out("query_out", query_out, query)
    elif query_out is not None:
        raise ValueError("query_out without query")
    if not T or not batch or not Hkv:
        return query_out
    k, v = _rows("key", key), _rows("value", value)
    q = _rows("query", query) if query is not None and query.shape[1] else None
    qs = (_stride(q, 0), _stride(q, 1), _stride(query_out, 0), _stride(query_out, 1)) if q is not None else (0, 0, 0, 0)
    t_ptr, a_ptr = table._ptrs if table is not None else (None, None)
    kc, vc = key_cache, value_cache
    p = _lib.PagedAppendParams(
        k.data_ptr(), v.data_ptr(), q.data_ptr() if q is not None else None, query_out.data_ptr() if q is not None else None,
        kc.data_ptr(), vc.data_ptr(), page_table.data_ptr(), query_start.data_ptr(), kv_len.data_ptr(), t_ptr, a_ptr,
        positions.data_ptr() if positions is not None else None,
        _stride(k, 0), _stride(k, 1), _stride(v, 0), _stride(v, 1), *qs,
        _stride(kc, 0), _stride(kc, 1), _stride(kc, 2), _stride(vc, 0), _stride(vc, 1), _stride(vc, 2), page_table.stride(0), pa, ps,
        page_table.shape[1], batch, T, q.shape[1] if q is not None else 0, Hkv, D, kc.shape[0], kc.shape[2], _DTYPES[dtype],
        _POSITION_TYPES[positions.dtype] if positions is not None else 0, table.rotary if table is not None else 0,
        table.n_axes if table is not None else 1, table.interleaved if table is not None else 0, table.amplitude if table is not None else 1.0)
    if not kc.numel() or not page_table.numel():
        if q is None:
            return query_out
        p.pages = 0                      # nothing to write to: the queries are still turned
        p.key_cache = p.value_cache = p.page_table = query_start.data_ptr() & ~15
    with _on_device(dev):
        st = _lib.load().dtb_paged_append(ctypes.byref(p), _stream_ptr(dev))
    _lib.check(st, "dtb_paged_append")
    return query_out


def paged_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, *, page_table: torch.Tensor,
                    query_start: torch.Tensor, kv_len: torch.Tensor, scale: Optional[float] = None, causal: bool = True,
                    window: Optional[int] = None, out: Optional[torch.Tensor] = None,
                    return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the new tokens ``[tokens, heads, dim]`` over the pages of their sequences, ``[tokens, heads, dim]``.

    Sequences may bring chunks, single tokens and nothing, mixed in one call; ``heads`` is a multiple of the cache's heads
    (at most 128 times), ``dim`` 64 or 128, ``page_size`` 8, 16, 32, 64 or a multiple of 128.  With ``causal`` a token sees the
    tokens up to itself, and with ``window`` only the last so many of those; without, all ``kv_len`` tokens of its sequence, the
    whole chunk among them.  ``scale=None`` means ``1 / sqrt(dim)``.  What lies in pages past a sequence's length is never used,
    NaN or not.  (A NaN or an infinity among the values of a token that counts reaches, besides the rows that see it, those up
    to 255 rows before it that do not, as it does through a masked softmax and a matrix product.)

    Rows that see nothing come out as zeros; rows of no sequence are not written.  With ``return_lse`` also returns f32
    ``[tokens, heads]``, the base-2 logarithm of the sum of exponentials of the scaled logits (``m + log2(l)`` of
    :class:`ResidualState`), -inf for rows that see nothing.
    """
    _check_heads(query, key_cache)
    dev, dtype = query.device, query.dtype
    _check_cache("key_cache", key_cache, dev, dtype)
    _check_cache("value_cache", value_cache, dev, dtype)
    if key_cache.shape != value_cache.shape:
        raise ValueError("the caches must have the same shape")
    batch = _check_where(page_table, query_start, kv_len, dev)
    scale, window = _check_scale(scale), _check_window(causal, window)
    T, Hq, D = query.shape
    if out is None:
        out = torch.empty(query.shape, dtype=dtype, device=dev)
        o = out
    else:
        _need_out("out", out, query)
        o = out if _rows16(out) is out else torch.empty(query.shape, dtype=dtype, device=dev)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    q = _rows16(query)
    kc, vc = key_cache, value_cache
    if o is not out:
        o.copy_(out)                     # rows of no sequence stay
    # an empty cache has no address: its pages are never read
    kp, vp, tp = kc.data_ptr() or 4096, vc.data_ptr() or 4096, page_table.data_ptr() or 4096
    p = _lib.PagedAttnParams(
        q.data_ptr(), kp, vp, o.data_ptr(), lse.data_ptr() if return_lse else None, tp, query_start.data_ptr(),
        kv_len.data_ptr(), _status_buffer(dev).data_ptr(), q.stride(0), q.stride(1), o.stride(0), o.stride(1),
        kc.stride(0), kc.stride(1), kc.stride(2), vc.stride(0), vc.stride(1), vc.stride(2), page_table.stride(0),
        page_table.shape[1], batch, T, Hq, kc.shape[1], D, kc.shape[0], kc.shape[2], _DTYPES[dtype], bool(causal), window, scale)
    lib = _lib.load()
    with _on_device(dev):
        need = lib.dtb_paged_attn_workspace_bytes(ctypes.byref(p))
        # a workspace of its own for each call: calls on other streams and replays of captured ones may overlap
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        st = lib.dtb_paged_attn(ctypes.byref(p), ws.data_ptr() if need else None, need, _stream_ptr(dev))
    _lib.check(st, "dtb_paged_attn")
    if o is not out:
        out.copy_(o)
    return (out, lse) if return_lse else out


def paged_key_weights(query: torch.Tensor, key_cache: torch.Tensor, lse: torch.Tensor, *, page_table: torch.Tensor,
                      query_start: torch.Tensor, kv_len: torch.Tensor, scale: Optional[float] = None, causal: bool = True,
                      window: Optional[int] = None, prior: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """What each key got of the new tokens' attention: f32 ``[B, heads_kv, slots]``, ``slots`` being the page table's.

    Entry ``s`` of a head is ``prior``'s (zero without) plus the softmax weights of slot ``s`` summed over the sequence's new
    tokens and the query heads of the group; zero at and past ``kv_len``.  ``lse`` is what :func:`paged_attention` returned
    for the same call, whose ``scale``, ``causal`` and ``window`` are given again.  ``out`` may be ``prior``: a running sum.
    """
    _check_heads(query, key_cache)
    dev, dtype = query.device, query.dtype
    _check_cache("key_cache", key_cache, dev, dtype)
    batch = _check_where(page_table, query_start, kv_len, dev)
    scale, window = _check_scale(scale), _check_window(causal, window)
    T, Hq, D = query.shape
    _need_cuda("lse", lse, dev)
    if lse.dtype != torch.float32 or tuple(lse.shape) != (T, Hq):
        raise ValueError(f"lse must be f32 [{T}, {Hq}], got {lse.dtype} {tuple(lse.shape)}")
    kc = key_cache
    shape = (batch, kc.shape[1], page_table.shape[1] * kc.shape[2])
    for name, t in (("prior", prior), ("out", out)):
        if t is None:
            continue
        _need_cuda(name, t, dev)
        if t.dtype != torch.float32 or tuple(t.shape) != shape:
            raise ValueError(f"{name} must be f32 {list(shape)}, got {t.dtype} {list(t.shape)}")
        if (shape[2] > 1 and t.stride(2) != 1) or (name == "out" and any(s == 0 and n > 1 for s, n in zip(t.stride(), shape))):
            raise ValueError(f"{name} must be contiguous in its last axis and no broadcast")
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=dev)
    q, lse = _rows16(query), lse.contiguous()
    p = _lib.PagedKeyWeightsParams(
        q.data_ptr(), kc.data_ptr() or 4096, lse.data_ptr(), prior.data_ptr() if prior is not None else None, out.data_ptr(),
        page_table.data_ptr(), query_start.data_ptr(), kv_len.data_ptr(), _status_buffer(dev).data_ptr(), q.stride(0), q.stride(1),
        kc.stride(0), kc.stride(1), kc.stride(2), page_table.stride(0),
        prior.stride(0) if prior is not None else 0, prior.stride(1) if prior is not None else 0, out.stride(0), out.stride(1),
        page_table.shape[1], batch, T, Hq, kc.shape[1], D, kc.shape[0], kc.shape[2], _DTYPES[dtype], bool(causal), window, scale)
    with _on_device(dev):
        st = _lib.load().dtb_paged_key_weights(ctypes.byref(p), _stream_ptr(dev))
    _lib.check(st, "dtb_paged_key_weights")
    return out


def paged_evict(key_cache: torch.Tensor, value_cache: torch.Tensor, weights: torch.Tensor, *, page_table: torch.Tensor,
                out_table: torch.Tensor, kv_len: torch.Tensor, keep: int,
                recent: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Cuts sequences to ``keep`` tokens by the weights that their keys have gathered (:func:`paged_key_weights`).

    Each key/value head keeps the last ``recent`` tokens and, of those before, the ones of the largest weights - the earlier
    where weights are equal, NaN above all - in their order.  Their rows of both caches are copied to the pages that
    ``out_table`` names, which may hold nothing that is still needed: no page of it may be in ``page_table`` too, or twice.
    Sequences of at most ``keep`` tokens are copied whole.

    Returns ``(kept, weights, kv_len)``: the slot that each kept one came from, int32 ``[B, heads_kv, keep]`` (-1 past a shorter
    sequence's end); the kept weights in their new places, f32 ``[B, heads_kv, slots of out_table]``, zeros behind; and the new
    lengths, int32 ``[B]``.  The next step goes on with ``page_table=out_table`` and the lengths plus its new tokens.
    """
    _need_cuda("key_cache", key_cache)
    dev = key_cache.device
    _check_cache("key_cache", key_cache, dev)
    _check_cache("value_cache", value_cache, dev, key_cache.dtype)
    if key_cache.shape != value_cache.shape:
        raise ValueError("the caches must have the same shape")
    pages, Hkv, page_size, D = key_cache.shape
    if D % 8:
        raise NotImplementedError(f"heads must have a multiple of 8 channels, got {D}")
    batch = _check_where(page_table, None, kv_len, dev)
    _need_cuda("out_table", out_table, dev)
    if out_table.dtype != torch.int32 or out_table.dim() != 2 or out_table.shape[0] != batch or (out_table.shape[1] > 1 and out_table.stride(1) != 1):
        raise ValueError(f"out_table must be int32 [{batch}, pages of a sequence], contiguous in its last axis")
    slots, out_slots = page_table.shape[1] * page_size, out_table.shape[1] * page_size
    _need_cuda("weights", weights, dev)
    if weights.dtype != torch.float32 or tuple(weights.shape) != (batch, Hkv, slots) or (slots > 1 and weights.stride(2) != 1):
        raise ValueError(f"weights must be f32 [{batch}, {Hkv}, {slots}], contiguous in the last axis, got {weights.dtype} {tuple(weights.shape)}")
    keep, recent = int(keep), int(recent)
    if not 1 <= keep <= out_slots or not 0 <= recent <= keep:
        raise ValueError(f"needs 1 <= keep <= {out_slots} (the slots of out_table) and 0 <= recent <= keep, got {keep} and {recent}")
    kept = torch.empty(batch, Hkv, keep, dtype=torch.int32, device=dev)
    weights_out = torch.empty(batch, Hkv, out_slots, dtype=torch.float32, device=dev)
    kv_len_out = torch.empty(batch, dtype=torch.int32, device=dev)
    if not batch or not Hkv:
        return kept, weights_out, kv_len_out
    kc, vc = key_cache, value_cache
    p = _lib.PagedEvictParams(
        kc.data_ptr() or 4096, vc.data_ptr() or 4096, weights.data_ptr() or 4096, page_table.data_ptr() or 4096, out_table.data_ptr(),
        kv_len.data_ptr(), kept.data_ptr(), weights_out.data_ptr(), kv_len_out.data_ptr(),
        _stride(kc, 0), _stride(kc, 1), _stride(kc, 2), _stride(vc, 0), _stride(vc, 1), _stride(vc, 2),
        weights.stride(0), weights.stride(1), page_table.stride(0), out_table.stride(0),
        page_table.shape[1], out_table.shape[1], batch, Hkv, D, pages, page_size, keep, recent)
    with _on_device(dev):
        st = _lib.load().dtb_paged_evict(ctypes.byref(p), _stream_ptr(dev))
    _lib.check(st, "dtb_paged_evict")
    return kept, weights_out, kv_len_out
