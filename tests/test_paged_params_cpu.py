"""What the paged calls hand to the library, looked at on the CPU: launches are caught, and no tensor has to be on a device."""
import pytest
import torch

import dtb200
from dtb200 import _lib, paged

BF = torch.bfloat16


@pytest.fixture
def caught(monkeypatch):
    """Parameters of the launches, in order, with tensors of the CPU taken for a device's."""
    calls = []

    def launch(name, params, device, index):
        cls = {"dtb_rotary": _lib.RotaryParams, "dtb_paged_append": _lib.PagedAppendParams, "dtb_paged_key_weights": _lib.PagedKeyWeightsParams,
               "dtb_paged_evict": _lib.PagedEvictParams}[name]
        calls.append(cls.from_buffer_copy(params))

    monkeypatch.setattr(paged, "_need_cuda", lambda name, t, index=-1: t.get_device())
    monkeypatch.setattr(paged, "_launch", launch)
    monkeypatch.setattr(paged, "_status_ptr", lambda device: 0)
    return calls


def _where(new, kv, width):
    return {"page_table": torch.zeros(len(new), width, dtype=torch.int32), "kv_len": torch.tensor(kv, dtype=torch.int32),
            "query_start": torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)}


@pytest.mark.parametrize("pages, width", [(0, 4), (5, 0), (0, 0)])
def test_append_without_pages_names_no_entry_of_a_table(caught, pages, width):
    B, Hq, D = 6, 8, 128                                # single tokens: an entry of sequence 3 in a table of Hq columns lies past the queries
    q, k = torch.zeros(B, Hq, D, dtype=BF), torch.zeros(B, 2, D, dtype=BF)
    cache = torch.zeros(pages, 2, 16, D, dtype=BF)
    dtb200.paged_append_(cache, cache, k, k, query=q, **_where([1] * B, [20] * B, width))
    p, = caught
    assert p.table_width == 0 and p.table_stride == 0
    assert p.q == q.data_ptr() and (p.T, p.Hq, p.Hkv) == (B, Hq, 2)
    dtb200.paged_append_(cache, cache, k, k, **_where([1] * B, [20] * B, width))
    assert len(caught) == 1                             # nothing to write and nothing to turn


@pytest.fixture
def attention_caught(caught, monkeypatch):
    monkeypatch.setattr(paged, "_launch_attention", lambda p, device: caught.append(_lib.PagedAttnParams.from_buffer_copy(p)) or 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1, raising=False)
    return caught


@pytest.mark.parametrize("T, H, strides", [(1, 8, (8 * 128 + 4, 128)), (5, 1, (128, 3)), (1, 1, (7, 13)), (1, 8, (0, 128)), (1, 4, (-3, 256)), (4, 2, (264, 128))])
def test_axes_of_one_entry_may_have_any_stride(attention_caught, T, H, strides):
    """A single token cut out of a wider row, say: torch keeps whatever stride the axis had, and calls such a tensor contiguous."""
    q = torch.zeros(4096, dtype=BF)
    out = torch.zeros(4096, dtype=BF)
    q, out = (torch.as_strided(x, (T, H, 128), (*(max(s, 0) for s in strides), 1)) for x in (q, out))
    cache = torch.zeros(4, H, 16, 128, dtype=BF)
    dtb200.paged_attention(q, cache, cache, out=out, **_where([T], [40], 3))
    dtb200.paged_key_weights(q, cache, torch.zeros(T, H), **_where([T], [40], 3))
    a, w = attention_caught
    assert a.q == w.q == q.data_ptr() and a.o == out.data_ptr()          # taken in place
    for st, n in ((a.q_stride_t, T), (a.q_stride_h, H), (a.o_stride_t, T), (a.o_stride_h, H), (w.q_stride_t, T), (w.q_stride_h, H)):
        assert st % 8 == 0 and (n == 1 or st > 0)
    if T > 1 and H > 1:
        assert (a.q_stride_t, a.q_stride_h) == strides


def test_caches_without_heads_are_refused(attention_caught):
    """Rather than queries that are not turned, and lengths that nobody wrote."""
    cache, k, q = torch.zeros(4, 0, 16, 128, dtype=BF), torch.zeros(2, 0, 128, dtype=BF), torch.zeros(2, 8, 128, dtype=BF)
    where = _where([1, 1], [20, 20], 2)
    for call in (lambda: dtb200.paged_append_(cache, cache, k, k, query=q, **where), lambda: dtb200.paged_attention(q, cache, cache, **where),
                 lambda: dtb200.paged_evict(cache, cache, torch.zeros(2, 0, 32), page_table=where["page_table"], kv_len=where["kv_len"],
                                            out_table=where["page_table"] + 2, keep=10)):
        with pytest.raises(ValueError, match="heads"):
            call()
    assert not attention_caught


def test_rotary_hands_its_gradient_on(caught):
    table = dtb200.make_rotary_table(64, device="cpu")
    q, k = (torch.zeros(5, h, 128, dtype=BF) for h in (4, 2))
    positions = torch.arange(5)
    for which in ("qk", "q", "k"):
        del caught[:]
        q.requires_grad_("q" in which), k.requires_grad_("k" in which)
        q.grad = k.grad = None
        a, b = dtb200.rotary(q, k, table=table, positions=positions)
        (a.float().sum() + b.float().sum()).backward()
        forward, back = caught
        assert (forward.transpose, back.transpose) == (0, 1) and forward.q == q.data_ptr() and back.amplitude == forward.amplitude
        assert back.positions == positions.data_ptr() and (back.Hq, back.Hk) == {"qk": (4, 2), "q": (4, 0), "k": (2, 0)}[which]
        assert all((x.grad is None) == (not x.requires_grad) and (x.grad is None or x.grad.shape == x.shape) for x in (q, k))
    del caught[:]
    x = torch.zeros(5, 4, 128, dtype=BF, requires_grad=True)
    y = dtb200.rotary(x, table=table, positions=positions, transpose=True)
    g, = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    assert [p.transpose for p in caught] == [1, 0] and g.shape == x.shape
    with pytest.raises(RuntimeError, match="out"):
        dtb200.rotary(x, table=table, positions=positions, out=torch.zeros_like(x))
    with torch.no_grad():
        assert not dtb200.rotary(x, table=table, positions=positions, out=torch.zeros(5, 4, 128, dtype=BF)).requires_grad
    assert not dtb200.rotary(x.detach(), table=table, positions=positions).requires_grad


@pytest.mark.parametrize("kw, code", [({"table_width": 2 ** 31 - 5000, "out_width": 64, "page_size": 1}, 2), ({"out_width": 2 ** 31 - 5000, "page_size": 1}, 2),
                                      ({"table_width": 2 ** 31 - 8200, "out_width": 2 ** 31 - 8200, "page_size": 1, "kc_stride_r": 4}, 4)])
def test_eviction_refuses_tables_whose_places_pass_an_int(kw, code):
    """Runs of slots and of copied rows are rounded up to whole ones of some thousand."""
    import ctypes

    from test_paged_cpu import ALIGN, CACHE, EVICT, SHAPE, VALUES, _fill

    p = _fill(_lib.PagedEvictParams, **{**CACHE, **VALUES, **EVICT, "keep": 10, "recent": 0, **kw})
    assert _lib.load().dtb_paged_evict(ctypes.byref(p), None) == {2: SHAPE, 4: ALIGN}[code]


@pytest.mark.parametrize("scale", [1e-50, 1e-40, 1e39, 2.0 ** 127])
def test_scales_that_32_bits_cannot_hold_are_refused(attention_caught, scale):
    """1e-50 came to the kernel as 0, which stands for the usual scale there."""
    q, cache = torch.zeros(2, 4, 128, dtype=BF), torch.zeros(4, 2, 16, 128, dtype=BF)
    for call in (lambda: dtb200.paged_attention(q, cache, cache, scale=scale, **_where([1, 1], [9, 9], 2)),
                 lambda: dtb200.paged_key_weights(q, cache, torch.zeros(2, 4), scale=scale, **_where([1, 1], [9, 9], 2))):
        with pytest.raises(ValueError, match="scale"):
            call()
    assert not attention_caught


@pytest.mark.parametrize("width, cut", [(63, False), (64, True), (1000, True)])
def test_workspace_of_calls_whose_units_cannot_be_cut(width, cut):
    """Pieces leave at least 512 keys on both sides of a cut: tables of fewer than 1024 slots need no room for their states."""
    import ctypes

    from test_paged_cpu import BATCH, CACHE, VALUES, _fill

    p = _fill(_lib.PagedAttnParams, **{**CACHE, **VALUES, **BATCH, "o_stride_t": 1024, "o_stride_h": 128, "table_width": width})
    need = _lib.load().dtb_paged_attn_workspace_bytes(ctypes.byref(p))
    assert need > 2 ** 24 if cut else 0 < need <= 2 ** 14
