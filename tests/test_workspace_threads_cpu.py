"""Calls that go through a workspace, from several host threads: the lookup and the launches of one call come one after the other."""
import threading
import time
import types

import pytest
import torch

from dtb200 import _lib, ops, paged

CPU = torch.device("cpu")


@pytest.fixture
def library(monkeypatch):
    """A library whose calls take a while, as those that let go of the interpreter's lock do; what they were given, and overlaps."""
    lib = types.SimpleNamespace(inside=0, most=0, seen=[])

    def launches(workspace, nbytes):
        lib.inside += 1
        lib.most = max(lib.most, lib.inside)
        time.sleep(0.02)
        alive = [ws for ws in (*paged._workspaces.values(), *ops._workspaces.values()) if ws.data_ptr() == workspace]
        lib.seen.append((nbytes, alive[0].numel() if alive else -1))
        lib.inside -= 1
        return 0

    sizes = iter([1000, 5000, 200, 9000] * 3)
    lib.dtb_paged_attn_workspace_bytes = lambda p: next(sizes)
    lib.dtb_attn_workspace_bytes = lambda p: next(sizes)
    lib.dtb_paged_attn = lambda p, ws, n, stream: launches(ws, n)
    lib.dtb_attn_fwd = lambda p, ws, n, stream: launches(ws, n)
    monkeypatch.setattr(_lib, "_lib", lib)
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(paged, "_workspaces", {})
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 7, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: types.SimpleNamespace(cuda_stream=7))
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(ops, "_on_device", lambda device: ops.contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream_ptr", lambda device: 7)
    return lib


def _together(calls):
    errors = []

    def run(f):
        try:
            f()
        except Exception as e:           # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(f,)) for f in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_paged_attention(library):
    _together([lambda: paged._launch_attention(b"", CPU)] * 4)
    assert library.most == 1, "two calls in the library at a time, on one workspace"
    assert len(library.seen) == 4 and all(0 < need <= have for need, have in library.seen), library.seen


def test_attention(library, monkeypatch):
    monkeypatch.setattr(ops, "_check_inputs", lambda *a: None)
    monkeypatch.setattr(ops, "_status_buffer", lambda device: torch.zeros(4, dtype=torch.int32))
    x = torch.zeros(1, 2, 128, 128, dtype=torch.bfloat16)
    _together([lambda: ops.attention(x, x, x)] * 4)
    assert library.most == 1, "two calls in the library at a time, on one workspace"
    assert len(library.seen) == 4 and all(0 < need <= have for need, have in library.seen), library.seen


@pytest.mark.parametrize("module", [ops, paged])
def test_captured_calls_share_no_workspace(library, monkeypatch, module):
    """Replays of two graphs may overlap; and what a capture allocates belongs to its graph, not to the calls behind it."""
    plain = module._workspace(CPU, 100)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    first, second = module._workspace(CPU, 200), module._workspace(CPU, 200)
    assert len({t.data_ptr() for t in (plain, first, second)}) == 3
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    assert module._workspace(CPU, 100) is plain
