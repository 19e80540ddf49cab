"""What the paged-cache operators refuse, before any launch: through the C ABI without a device, and in Python."""
import ctypes

import pytest
import torch

import dtb200
from dtb200 import _lib

NULL, DTYPE, SHAPE, ALIGN = 1, 2, 3, 4


def _fill(cls, **kw):
    p = cls()
    for name, kind in cls._fields_:
        if kind is ctypes.c_void_p:
            setattr(p, name, 4096)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


CACHE = {"kc_stride_p": 4 * 16 * 128, "kc_stride_h": 16 * 128, "kc_stride_r": 128}
VALUES = {"vc_stride_p": 4 * 16 * 128, "vc_stride_h": 16 * 128, "vc_stride_r": 128}
BATCH = {"table_width": 4, "B": 2, "T": 3, "Hq": 8, "Hkv": 4, "D": 128, "pages": 8, "page_size": 16, "q_stride_t": 1024, "q_stride_h": 128}


@pytest.mark.parametrize("kw,code", [
    ({"q": None}, NULL), ({"value_cache": None}, NULL), ({"query_start": None}, NULL), ({"o": None}, NULL),
    ({"dtype": 2}, DTYPE), ({"D": 96}, SHAPE), ({"Hkv": 3}, SHAPE), ({"Hkv": 0}, SHAPE), ({"Hq": 4 * 129}, SHAPE),
    ({"page_size": 24}, SHAPE), ({"page_size": 0}, SHAPE), ({"page_size": 192}, SHAPE), ({"window": 5}, SHAPE), ({"window": -1, "causal": 1}, SHAPE),
    ({"T": -1}, SHAPE), ({"B": -1}, SHAPE), ({"table_width": 2 ** 30}, SHAPE), ({"kc_stride_r": 0}, SHAPE), ({"vc_stride_p": -128}, SHAPE),
    ({"q_stride_t": 0}, SHAPE), ({"q": 4100}, ALIGN), ({"key_cache": 4104}, ALIGN), ({"vc_stride_h": 1027}, ALIGN), ({"o_stride_h": 4}, ALIGN),
])
def test_paged_attention_validation(kw, code):
    p = _fill(_lib.PagedAttnParams, **{**CACHE, **VALUES, **BATCH, "o_stride_t": 1024, "o_stride_h": 128, **kw})
    assert _lib.load().dtb_paged_attn(ctypes.byref(p), None, 0, None) == code


@pytest.mark.parametrize("kw,code", [
    ({"q": None}, NULL), ({"lse": None}, NULL), ({"out": None}, NULL), ({"key_cache": None}, NULL), ({"dtype": 7}, DTYPE), ({"D": 32}, SHAPE),
    ({"page_size": 12}, SHAPE), ({"Hq": 7}, SHAPE), ({"kc_stride_p": 4}, ALIGN), ({"window": 5}, SHAPE),
])
def test_key_weights_validation(kw, code):
    p = _fill(_lib.PagedKeyWeightsParams, **{**CACHE, **BATCH, "out_stride_b": 256, "out_stride_h": 64, **kw})
    assert _lib.load().dtb_paged_key_weights(ctypes.byref(p), None) == code


ROTARY = {"B": 1, "S": 5, "Hq": 2, "Hk": 1, "D": 128, "rotary": 64, "n_axes": 1}


@pytest.mark.parametrize("kw,code", [
    ({"q": None}, NULL), ({"q_out": None}, NULL), ({"k": None}, NULL), ({"turns": None}, NULL), ({"positions": None}, NULL), ({"dtype": 3}, DTYPE),
    ({"pos_type": 3}, DTYPE), ({"rotary": 130}, SHAPE), ({"rotary": 63}, SHAPE), ({"rotary": 0}, SHAPE), ({"D": 513}, SHAPE), ({"n_axes": 0}, SHAPE),
    ({"n_axes": 2, "axis": None}, SHAPE), ({"Hq": 0}, SHAPE), ({"Hk": 0}, SHAPE), ({"S": -1}, SHAPE),
])
def test_rotary_validation(kw, code):
    p = _fill(_lib.RotaryParams, **{**ROTARY, **kw})
    assert _lib.load().dtb_rotary(ctypes.byref(p), None) == code


@pytest.mark.parametrize("kw,code", [
    ({"k": None}, NULL), ({"v": None}, NULL), ({"q_out": None}, NULL), ({"kv_len": None}, NULL), ({"positions": None, "n_axes": 2}, NULL),
    ({"dtype": 2}, DTYPE), ({"rotary": 0}, SHAPE), ({"rotary": 200}, SHAPE), ({"page_size": 0}, SHAPE), ({"Hkv": 0}, SHAPE), ({"pages": -1}, SHAPE),
])
def test_append_validation(kw, code):
    p = _fill(_lib.PagedAppendParams, **{**CACHE, **VALUES, **BATCH, "rotary": 64, "n_axes": 1, **kw})
    assert _lib.load().dtb_paged_append(ctypes.byref(p), None) == code


EVICT = {"table_width": 8, "out_width": 4, "B": 2, "Hkv": 4, "D": 128, "pages": 20, "page_size": 16, "keep": 64, "recent": 8}


@pytest.mark.parametrize("kw,code", [
    ({"weights": None}, NULL), ({"kept": None}, NULL), ({"out_table": None}, NULL), ({"keep": 0}, SHAPE), ({"keep": 65}, SHAPE), ({"recent": 65}, SHAPE),
    ({"recent": -1}, SHAPE), ({"D": 100}, SHAPE), ({"page_size": 0}, SHAPE), ({"out_width": 0}, SHAPE), ({"Hkv": 0}, SHAPE), ({"key_cache": 4100}, ALIGN),
    ({"kc_stride_r": 132}, ALIGN), ({"table_width": 2 ** 30}, SHAPE),
])
def test_evict_validation(kw, code):
    p = _fill(_lib.PagedEvictParams, **{**CACHE, **VALUES, **EVICT, **kw})
    assert _lib.load().dtb_paged_evict(ctypes.byref(p), None) == code


def test_no_cpu_path():
    q, cache = torch.zeros(3, 4, 128, dtype=torch.bfloat16), torch.zeros(2, 4, 16, 128, dtype=torch.bfloat16)
    one = torch.zeros(1, dtype=torch.int32)
    where = {"page_table": torch.zeros(1, 2, dtype=torch.int32), "query_start": torch.zeros(2, dtype=torch.int32), "kv_len": one}
    table = dtb200.make_rotary_table(64, device="cpu")
    for call in (lambda: dtb200.paged_attention(q, cache, cache, **where),
                 lambda: dtb200.paged_key_weights(q, cache, torch.zeros(3, 4), **where),
                 lambda: dtb200.paged_append_(cache, cache, q, q, **where),
                 lambda: dtb200.rotary(q, table=table, positions=torch.zeros(3)),
                 lambda: dtb200.paged_evict(cache, cache, torch.zeros(1, 4, 32), page_table=where["page_table"], out_table=where["page_table"],
                                            kv_len=one, keep=4)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


@pytest.mark.parametrize("args,kw", [((0,), {}), ((7,), {}), ((64,), {"layout": "pairs"}), ((64,), {"scaling": "cubic"}), ((64,), {"axes": [16, 15]}),
                                     ((64,), {"axes": [32, 0]}), ((64,), {"base": 1.0}), ((64,), {"factor": 0.0})])
def test_rotary_tables_are_checked(args, kw):
    with pytest.raises(ValueError):
        dtb200.make_rotary_table(*args, device="cpu", **kw)


def test_rotary_table_has_a_ladder_for_each_axis():
    t = dtb200.make_rotary_table(64, axes=[8, 12, 12], device="cpu")
    assert t.rotary == 64 and t.n_axes == 3 and t.axis.tolist() == [0] * 8 + [1] * 12 + [2] * 12
    two_pi = 6.283185307179586
    assert abs(t.turns[0].item() * two_pi - 1) < 1e-15 and abs(t.turns[8].item() * two_pi - 1) < 1e-15
    assert abs(t.turns[13].item() * two_pi - 10000.0 ** (-5 / 12)) < 1e-15
    assert dtb200.make_rotary_table(64, device="cpu").axis is None
