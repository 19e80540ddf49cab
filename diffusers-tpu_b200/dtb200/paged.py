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

A length past what the page table can name ends at it: :func:`paged_append_` drops tokens that have no slot, and the others
attend to what the table holds, each new token from the slot that it was appended to, those without one from behind the end.
(Where none of a sequence's new tokens has a slot, they attend as if they were the last ones of the table.)

The reference has no paged cache (one of its models keeps a block's keys and values from step to step, whole:
``diffusers_tpu/backends/qwen21_core_tt.py``); its rotary embedding takes precomputed tables
(``diffusers_tpu/models/minimax_h3/jax_dit.py:251-262``).
All compute goes through the C ABI in ``libdtb200_attn.so``; nothing here falls back to PyTorch.  Gradients pass through
:func:`rotary`; the calls on a cache form none.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .ops import _status_buffer, _status_bufs, _workspace_lock

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_I32 = torch.int32
_POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


class RotaryTable:
    """What :func:`make_rotary_table` builds and :func:`rotary` and :func:`paged_append_` take: how far each pair of channels
    turns per position, on the device in 64 bits, which row of the positions turns it, and the factor on the result."""

    def __init__(self, turns: torch.Tensor, axis: Optional[torch.Tensor], n_axes: int, interleaved: bool, amplitude: float):
        self.turns, self.axis, self.n_axes, self.interleaved, self.amplitude = turns, axis, n_axes, interleaved, amplitude
        self.rotary = 2 * turns.numel()
        self.device = turns.device
        self._ptrs = (turns.data_ptr(), axis.data_ptr() if axis is not None else 0)


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

            # where the slowest pair makes more than slow_turns turns, the ramp ends behind it
            low, high = max(math.floor(pair_of(fast_turns)), 0), math.ceil(pair_of(slow_turns))
            for j in range(n):
                ramp = min(max((j - low) / max(high - low, 1e-3), 0.0), 1.0) if high > 0 else 1.0
                ladder[j] = ladder[j] / factor * ramp + ladder[j] * (1.0 - ramp)
            amplitude = 0.1 * math.log(factor) + 1.0
        turns += [f / (2 * math.pi) for f in ladder]
        axis += [a] * n
    device = torch.device(device)
    return RotaryTable(torch.tensor(turns, dtype=torch.float64, device=device),
                       torch.tensor(axis, dtype=torch.int32, device=device) if len(counts) > 1 else None,
                       len(counts), layout == "interleaved", amplitude)


_pack_rotary, _pack_append, _pack_attn = (_lib.packer(c) for c in (_lib.RotaryParams, _lib.PagedAppendParams, _lib.PagedAttnParams))
_pack_weights, _pack_evict = (_lib.packer(c) for c in (_lib.PagedKeyWeightsParams, _lib.PagedEvictParams))
_status_ptrs: dict = {}
_workspaces: dict = {}


def _need_cuda(name: str, t: torch.Tensor, index: int = -1) -> int:
    """Index of the device that ``t`` is on, which must be ``index`` where that is one."""
    at = t.get_device()
    if at < 0:
        raise RuntimeError(f"{name} must be a CUDA tensor: dtb200 has no CPU path")
    if index >= 0 and at != index:
        raise ValueError(f"{name} is on cuda:{at}, not on cuda:{index}")
    return at


def _status_ptr(device: torch.device) -> int:
    ptr = _status_ptrs.get(device.index)
    if ptr is None:
        if torch.cuda.is_current_stream_capturing() and (device.type, device.index) not in _status_bufs:
            return 0     # a buffer made now would belong to the graph, and be zeroed by its replays only: none is passed
        ptr = _status_ptrs[device.index] = _status_buffer(device).data_ptr()
    return ptr


def _launch(name: str, params: bytes, device: torch.device, index: int) -> None:
    fn = getattr(_lib._lib or _lib.load(), name)
    if torch._C._cuda_getDevice() == index:
        st = fn(params, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            st = fn(params, torch._C._cuda_getCurrentRawStream(index))
    if st:
        _lib.check(st, name)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` where the kernels can address it (contiguous channels, no broadcast axis), else a copy."""
    if t.is_contiguous():
        return t
    st, sh = t.stride(), t.shape
    if st[-1] == 1 or sh[-1] == 1:
        for i in range(len(sh) - 1):
            if st[i] <= 0 and sh[i] > 1:
                return t.contiguous()
        return t
    return t.contiguous()


def _rows16(t: torch.Tensor) -> torch.Tensor:
    """As :func:`_rows`, for 16-bit rows of 64 or 128 channels, with pointer and strides multiples of 16 bytes."""
    if t.is_contiguous() and not t.data_ptr() % 16:
        return t
    st, sh = t.stride(), t.shape
    if st[-1] == 1 and not t.data_ptr() % 16 and all(n == 1 or (s > 0 and not s % 8) for s, n in zip(st[:-1], sh[:-1])):
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def _strides(t: torch.Tensor) -> Tuple[int, int]:
    """(token, head) strides; of an axis with a single entry, which torch may give any stride, one that is harmless."""
    st, sh = t.stride(), t.shape
    return (st[0] if sh[0] != 1 else 0, st[1] if sh[1] != 1 else 0)


def _need_out(name: str, out: torch.Tensor, like: torch.Tensor) -> None:
    if out.shape != like.shape or out.dtype != like.dtype or out.get_device() != like.get_device():
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    if out.shape[-1] > 1 and out.stride(-1) != 1 or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{name} must have contiguous channels and no broadcast axis")


def _positions(positions: torch.Tensor, table: RotaryTable, batch: int, tokens: int, device: torch.device):
    """Checked positions and their (axis, batch, token) strides."""
    if not isinstance(positions, torch.Tensor):
        raise TypeError("positions must be a tensor")
    _need_cuda("positions", positions, device.index)
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
    where the table does not scale).  Inputs that require their gradient get it so; with ``out`` or ``key_out``, which may be the
    inputs, that is refused.  Returns the turned query, or (query, key).
    """
    index = _need_cuda("query", query)
    dev = query.device
    if torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad)):
        if out is not None or key_out is not None:
            raise RuntimeError("rotary into out or key_out forms no gradient, and an input requires one")
        return _Turn.apply(query, key, table, positions, transpose)
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
        _need_cuda("key", key, index)
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
        q, k = _rows(query), (_rows(key) if key is not None else None)
        qo, ko = out, key_out
        if not query.shape[-2]:
            q, qo, k, ko = k, ko, None, None
        elif k is not None and not key.shape[-2]:
            k = ko = None
        plain = q.is_contiguous() and qo.is_contiguous() and (k is None or (k.is_contiguous() and ko.is_contiguous()))
        # empty_like of a view may not keep its channels contiguous
        fix = (qo, ko) if plain else [t if t is None or t.stride(-1) == 1 or D == 1 else torch.empty(t.shape, dtype=t.dtype, device=dev)
                                      for t in (qo, ko)]

        def strides(t):
            if t is None:
                return (0, 0, 0)
            if plain:
                h = t.shape[-2] * D
                return (h * tokens, h, D)
            st, sh = t.stride(), t.shape     # an axis of one entry may come with any stride: a harmless one
            return (st[0] if four and batch > 1 else 0, st[-3] if tokens > 1 else 0, st[-2] if sh[-2] > 1 else 0)

        p = _pack_rotary(q.data_ptr(), fix[0].data_ptr(), k.data_ptr() if k is not None else 0,
                         fix[1].data_ptr() if fix[1] is not None else 0, *table._ptrs, positions.data_ptr(),
                         *strides(q), *strides(fix[0]), *strides(k), *strides(fix[1]), pa, pb, ps,
                         _POSITION_TYPES[positions.dtype], batch, tokens, q.shape[-2], k.shape[-2] if k is not None else 0, D,
                         table.rotary, table.n_axes, table.interleaved, bool(transpose), _DTYPES[query.dtype], table.amplitude)
        _launch("dtb_rotary", p, dev, index)
        if fix[0] is not qo:
            qo.copy_(fix[0])
        if fix[1] is not ko:
            ko.copy_(fix[1])
    return out if key is None else (out, key_out)


class _Turn(torch.autograd.Function):
    """:func:`rotary` of inputs that require their gradient, which is the transposed map of the results'."""

    @staticmethod
    def forward(ctx, query, key, table, positions, transpose):
        turned = rotary(query, key, table=table, positions=positions, transpose=transpose)
        ctx.save_for_backward(positions)
        ctx.table, ctx.transpose = table, transpose
        return turned

    @staticmethod
    def backward(ctx, *up):
        need = [i for i in range(len(up)) if ctx.needs_input_grad[i]]
        back = rotary(*(up[i] for i in need), table=ctx.table, positions=ctx.saved_tensors[0], transpose=not ctx.transpose)
        grads = dict(zip(need, back if len(need) > 1 else (back,)))
        return grads.get(0), grads.get(1), None, None, None


def _check_cache(name: str, cache: torch.Tensor, index: int, dtype: Optional[torch.dtype] = None):
    """Checks a cache; returns its shape and (page, head, row) strides."""
    _need_cuda(name, cache, index)
    if cache.dtype != torch.bfloat16 and cache.dtype != torch.float16:
        raise NotImplementedError(f"{name} must be bf16 or fp16, got {cache.dtype}")
    if dtype is not None and cache.dtype != dtype:
        raise ValueError(f"{name} is {cache.dtype}, not {dtype}")
    sh = cache.shape
    if len(sh) != 4:
        raise ValueError(f"{name} must be [pages, heads_kv, page_size, dim], got {tuple(sh)}")
    if not sh[1]:
        raise ValueError(f"{name} has no key/value heads")
    sp, shd, sr, sc = cache.stride()
    # a cache is never copied to make it fit
    if sc != 1 or cache.data_ptr() % 16 or (sp | shd | sr) % 8 or sp <= 0 or shd <= 0 or sr <= 0:
        # an axis of one entry may come with any stride: a harmless one
        sp, shd, sr = (s if n > 1 else 128 for s, n in zip((sp, shd, sr), sh))
        if (sc != 1 and sh[3] != 1) or cache.data_ptr() % 16 or any(s <= 0 or s % 8 for s in (sp, shd, sr)):
            raise ValueError(f"{name} needs contiguous channels, positive strides and rows on 16-byte boundaries, got strides {cache.stride()}")
    return sh, (sp, shd, sr)


def _check_values(cache: torch.Tensor, keys: torch.Tensor, strides: Tuple[int, int, int], index: int) -> Tuple[int, int, int]:
    """Checks the value cache beside a checked key cache, whose shape it must have; returns its strides."""
    if cache.shape != keys.shape:
        raise ValueError(f"the caches must have the same shape, got {tuple(keys.shape)} and {tuple(cache.shape)}")
    if cache.stride() == keys.stride() and cache.dtype is keys.dtype and cache.get_device() == index and not cache.data_ptr() % 16:
        return strides
    return _check_cache("value_cache", cache, index, keys.dtype)[1]


def _check_where(page_table: torch.Tensor, query_start: Optional[torch.Tensor], kv_len: torch.Tensor, index: int) -> int:
    """Checks what says where new tokens and pages lie; returns the number of sequences."""
    sk, sp = kv_len.shape, page_table.shape
    if (kv_len.dtype is _I32 and page_table.dtype is _I32 and len(sk) == 1 and len(sp) == 2 and sp[0] == sk[0] and
            kv_len.get_device() == index and page_table.get_device() == index and kv_len.is_contiguous() and page_table.is_contiguous() and
            (query_start is None or (query_start.dtype is _I32 and query_start.shape == (sk[0] + 1,) and query_start.get_device() == index and
                                     query_start.is_contiguous()))):
        return sk[0]
    # something is unusual, or wrong
    batch = kv_len.shape[0] if kv_len.dim() == 1 else -1
    for name, t, dims, n in (("kv_len", kv_len, 1, batch), ("page_table", page_table, 2, batch), ("query_start", query_start, 1, batch + 1)):
        if t is None:
            continue
        if t.get_device() != index:
            _need_cuda(name, t, index)
        if t.dtype != torch.int32:
            raise NotImplementedError(f"{name} must be int32, got {t.dtype}")
        if t.dim() != dims or batch < 0 or t.shape[0] != n:
            raise ValueError(f"{name} has shape {tuple(t.shape)}: kv_len is [B], query_start [B + 1], page_table [B, pages of a sequence]")
        if not t.is_contiguous() and t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"{name} must be contiguous in its last axis")
    return batch


def _check_heads(query: torch.Tensor, cache: torch.Tensor) -> int:
    index = _need_cuda("query", query)
    sq, sc = query.shape, cache.shape
    if len(sq) != 3:
        raise ValueError(f"query must be [tokens, heads, dim], got {tuple(sq)}")
    if len(sc) == 4:
        if sq[2] != sc[3]:
            raise ValueError(f"query heads have {sq[2]} channels, the cache's {sc[3]}")
        if not sc[1] or not sq[1] or sq[1] % sc[1]:
            raise ValueError("query heads must be a multiple of key/value heads")
    return index


def _workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Scratch of a call, for a caller that holds the lock until it has launched.  Calls of a stream run one after the other and
    share one; a captured call, whose replays may overlap with those of other graphs, takes its own from its graph's memory."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, torch._C._cuda_getCurrentRawStream(device.index))
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = _workspaces[key] = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws


def _launch_attention(p: bytes, device: torch.device) -> int:
    lib = _lib._lib or _lib.load()
    with _workspace_lock:
        need = lib.dtb_paged_attn_workspace_bytes(p)
        ws = _workspace(device, need) if need else None
        return lib.dtb_paged_attn(p, ws.data_ptr() if need else 0, need, torch._C._cuda_getCurrentRawStream(device.index))


def _check_scale(scale: Optional[float]) -> float:
    if scale is None:
        return 0.0
    scale = float(scale)
    # the kernels hold it, and its product with log2(e), in 32 bits
    if not 2.0 ** -126 <= scale <= 2.0 ** 126:
        raise ValueError(f"scale must be positive and finite, from 2^-126 to 2^126, got {scale}")
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
    index = _need_cuda("key", key)
    dev, dtype = key.device, key.dtype
    shape, kc_strides = _check_cache("key_cache", key_cache, index, dtype)
    vc_strides = _check_values(value_cache, key_cache, kc_strides, index)
    if key.dim() != 3 or value.shape != key.shape or value.dtype != dtype or value.get_device() != index:
        raise ValueError(f"key and value must both be [tokens, heads_kv, dim], got {tuple(key.shape)} and {tuple(value.shape)} {value.dtype}")
    if key.shape[1] != shape[1] or key.shape[2] != shape[3]:
        raise ValueError(f"key {tuple(key.shape)} does not go with caches {tuple(key_cache.shape)} and {tuple(value_cache.shape)}")
    batch = _check_where(page_table, query_start, kv_len, index)
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
        _need_cuda("query", query, index)
        if query.dim() != 3 or query.shape[0] != T or query.shape[2] != D or query.dtype != dtype:
            raise ValueError(f"query {tuple(query.shape)} {query.dtype} does not go with key {tuple(key.shape)} {dtype}")
        if query_out is None:
            query_out = torch.empty_like(query, memory_format=torch.contiguous_format)
        else:
            _need_out("query_out", query_out, query)
    elif query_out is not None:
        raise ValueError("query_out without query")
    if not T or not batch:
        return query_out
    k, v = _rows(key), _rows(value)
    q = _rows(query) if query is not None and query.shape[1] else None
    table_width, table_stride = page_table.shape[1], page_table.stride(0)
    if not shape[0] or not table_width:
        if q is None:
            return query_out
        key_cache = value_cache = page_table = q      # no page to write to, and no entry to look at; the queries are still turned
        shape, table_width, table_stride = (0, Hkv, shape[2] or 1, D), 0, 0
    ks, vs = k.stride(), v.stride()
    qs, os = (q.stride(), query_out.stride()) if q is not None else ((0, 0), (0, 0))
    # an axis of one entry may come with any stride: a harmless one
    if T == 1:
        ks, vs, qs, os = ((0, x[1]) for x in (ks, vs, qs, os))
    if Hkv == 1:
        ks, vs = (ks[0], 0), (vs[0], 0)
    if q is not None and q.shape[1] == 1:
        qs, os = (qs[0], 0), (os[0], 0)
    p = _pack_append(
        k.data_ptr(), v.data_ptr(), q.data_ptr() if q is not None else 0, query_out.data_ptr() if q is not None else 0,
        key_cache.data_ptr(), value_cache.data_ptr(), page_table.data_ptr(), query_start.data_ptr(), kv_len.data_ptr(),
        *(table._ptrs if table is not None else (0, 0)), positions.data_ptr() if positions is not None else 0,
        ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], os[0], os[1], *kc_strides, *vc_strides, table_stride, pa, ps,
        table_width, batch, T, q.shape[1] if q is not None else 0, Hkv, D, shape[0], shape[2], _DTYPES[dtype],
        _POSITION_TYPES[positions.dtype] if positions is not None else 0, *((table.rotary, table.n_axes, table.interleaved, table.amplitude)
                                                                            if table is not None else (0, 1, 0, 1.0)))
    _launch("dtb_paged_append", p, dev, index)
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
    NaN or not, and a call takes at most 8192 sequences.  (A NaN or an infinity among the values of a token that counts reaches,
    besides the rows that see it, those of their query block that do not - up to 255 rows of (token, head of the group) in front of
    it, and with a window as many behind those that see it - as it does through a masked softmax and a matrix product.)

    Rows that see nothing come out as zeros; rows of no sequence are not written.  With ``return_lse`` also returns f32
    ``[tokens, heads]``, the base-2 logarithm of the sum of exponentials of the scaled logits (``m + log2(l)`` of
    :class:`ResidualState`), -inf for rows that see nothing.
    """
    index = _check_heads(query, key_cache)
    dev, dtype = query.device, query.dtype
    shape, kc_strides = _check_cache("key_cache", key_cache, index, dtype)
    vc_strides = _check_values(value_cache, key_cache, kc_strides, index)
    batch = _check_where(page_table, query_start, kv_len, index)
    scale, window = _check_scale(scale), _check_window(causal, window)
    T, Hq, D = query.shape
    if out is None:
        out = o = torch.empty_like(query, memory_format=torch.contiguous_format)
    else:
        _need_out("out", out, query)
        o = _rows16(out)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    q = _rows16(query)
    qs, os = _strides(q), _strides(o)
    p = _pack_attn(
        q.data_ptr(), key_cache.data_ptr() or q.data_ptr(), value_cache.data_ptr() or q.data_ptr(), o.data_ptr(),
        lse.data_ptr() if return_lse else 0, page_table.data_ptr() or kv_len.data_ptr(), query_start.data_ptr(), kv_len.data_ptr(),
        _status_ptr(dev), qs[0], qs[1], os[0], os[1], *kc_strides, *vc_strides, page_table.stride(0),
        page_table.shape[1], batch, T, Hq, shape[1], D, shape[0], shape[2], _DTYPES[dtype], bool(causal), window, scale)
    if torch._C._cuda_getDevice() == index:
        st = _launch_attention(p, dev)
    else:
        with torch.cuda.device(dev):
            st = _launch_attention(p, dev)
    if st:
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
    for the same call, whose ``scale``, ``causal`` and ``window`` are given again.  ``out`` may be ``prior``: a running sum.  A call
    takes at most 8192 sequences.
    """
    index = _check_heads(query, key_cache)
    dev, dtype = query.device, query.dtype
    c_shape, kc_strides = _check_cache("key_cache", key_cache, index, dtype)
    batch = _check_where(page_table, query_start, kv_len, index)
    scale, window = _check_scale(scale), _check_window(causal, window)
    T, Hq, D = query.shape
    _need_cuda("lse", lse, index)
    if lse.dtype != torch.float32 or lse.shape != (T, Hq):
        raise ValueError(f"lse must be f32 [{T}, {Hq}], got {lse.dtype} {tuple(lse.shape)}")
    shape = (batch, c_shape[1], page_table.shape[1] * c_shape[2])
    for name, t in (("prior", prior), ("out", out)):
        if t is None:
            continue
        _need_cuda(name, t, index)
        if t.dtype != torch.float32 or t.shape != shape:
            raise ValueError(f"{name} must be f32 {list(shape)}, got {t.dtype} {list(t.shape)}")
        if t.is_contiguous():
            continue
        if (shape[2] > 1 and t.stride(2) != 1) or (name == "out" and any(s == 0 and n > 1 for s, n in zip(t.stride(), shape))):
            raise ValueError(f"{name} must be contiguous in its last axis and no broadcast")
    if out is None:
        out = lse.new_empty(shape)
    q, lse = _rows16(query), lse.contiguous()
    qs, os = _strides(q), out.stride()
    pr = prior.stride() if prior is not None else (0, 0)
    p = _pack_weights(
        q.data_ptr(), key_cache.data_ptr() or out.data_ptr(), lse.data_ptr(), prior.data_ptr() if prior is not None else 0, out.data_ptr(),
        page_table.data_ptr(), query_start.data_ptr(), kv_len.data_ptr(), _status_ptr(dev), qs[0], qs[1], *kc_strides, page_table.stride(0),
        pr[0], pr[1], os[0], os[1], page_table.shape[1], batch, T, Hq, c_shape[1], D, c_shape[0], c_shape[2], _DTYPES[dtype], bool(causal),
        window, scale)
    _launch("dtb_paged_key_weights", p, dev, index)
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
    lengths, int32 ``[B]``.  The next step goes on with ``page_table=out_table`` and the lengths plus its new tokens.  A token's slot
    is its position no longer: :func:`paged_append_` has to be given the ``positions`` of new tokens from then on, and a ``window`` of
    :func:`paged_attention` counts the tokens that were kept.
    """
    index = _need_cuda("key_cache", key_cache)
    dev = key_cache.device
    shape, kc_strides = _check_cache("key_cache", key_cache, index)
    vc_strides = _check_values(value_cache, key_cache, kc_strides, index)
    pages, Hkv, page_size, D = shape
    if D % 8:
        raise NotImplementedError(f"heads must have a multiple of 8 channels, got {D}")
    batch = _check_where(page_table, None, kv_len, index)
    _need_cuda("out_table", out_table, index)
    if out_table.dtype != torch.int32 or out_table.dim() != 2 or out_table.shape[0] != batch or (out_table.shape[1] > 1 and out_table.stride(1) != 1):
        raise ValueError(f"out_table must be int32 [{batch}, pages of a sequence], contiguous in its last axis")
    slots, out_slots = page_table.shape[1] * page_size, out_table.shape[1] * page_size
    _need_cuda("weights", weights, index)
    if weights.dtype != torch.float32 or weights.shape != (batch, Hkv, slots) or (slots > 1 and weights.stride(2) != 1):
        raise ValueError(f"weights must be f32 [{batch}, {Hkv}, {slots}], contiguous in the last axis, got {weights.dtype} {tuple(weights.shape)}")
    keep, recent = int(keep), int(recent)
    if not 1 <= keep <= out_slots or not 0 <= recent <= keep:
        raise ValueError(f"needs 1 <= keep <= {out_slots} (the slots of out_table) and 0 <= recent <= keep, got {keep} and {recent}")
    kept = page_table.new_empty((batch, Hkv, keep))
    weights_out = weights.new_empty((batch, Hkv, out_slots))
    kv_len_out = torch.empty_like(kv_len, memory_format=torch.contiguous_format)
    if not batch:
        return kept, weights_out, kv_len_out
    kept_ptr = kept.data_ptr()
    p = _pack_evict(
        key_cache.data_ptr() or kept_ptr, value_cache.data_ptr() or kept_ptr, weights.data_ptr() or kept_ptr, page_table.data_ptr() or kept_ptr,
        out_table.data_ptr(), kv_len.data_ptr(), kept_ptr, weights_out.data_ptr(), kv_len_out.data_ptr(), *kc_strides, *vc_strides,
        weights.stride(0), weights.stride(1), page_table.stride(0), out_table.stride(0),
        page_table.shape[1], out_table.shape[1], batch, Hkv, D, pages, page_size, keep, recent)
    _launch("dtb_paged_evict", p, dev, index)
    return kept, weights_out, kv_len_out
