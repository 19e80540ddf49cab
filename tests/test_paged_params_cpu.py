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
