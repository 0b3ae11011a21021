"""CPU: whose workspace a call without one of its own gets, and which explicit
workspaces are refused (the device side is replaced by fakes)."""
from __future__ import annotations

import pytest
import torch

from ps_attn import ops


class Fakes:
    stream, capture = 7, 0

    class Lib:
        @staticmethod
        def ps_stream_capture_id(stream):
            return Fakes.capture if stream == Fakes.stream else 0


@pytest.fixture
def fakes(monkeypatch):
    Fakes.stream, Fakes.capture = 7, 0

    class Workspace:
        def __init__(self, max_num_seqs, *shape, cascade=False):
            self.max_num_seqs, self.shape, self.cascade = max_num_seqs, shape, cascade

    monkeypatch.setattr(ops, "DecodeWorkspace", Workspace)
    monkeypatch.setattr(ops, "_stream_ptr", lambda device: Fakes.stream)
    monkeypatch.setattr(ops._lib, "load", lambda: Fakes.Lib)
    monkeypatch.setattr(ops, "_WS_CACHE", {})
    if hasattr(ops, "_WS_CAPTURES"):
        monkeypatch.setattr(ops, "_WS_CAPTURES", {})
    return Fakes


def get(n=4, hq=8, hkv=2, **kw):
    return ops.get_workspace(n, hq, hkv, 128, torch.device("cuda", 0), **kw)


def test_a_stream_keeps_its_workspace_and_grows_it(fakes):
    a = get()
    assert get(200) is a and a.max_num_seqs == 256
    b = get(300)
    assert b is not a and b.max_num_seqs == 512 and get(4) is b
    assert get(cascade=True) is not b and get(hkv=4) is not b


def test_streams_do_not_share(fakes):
    a = get()
    fakes.stream = 9
    b = get()
    assert b is not a
    fakes.stream = 7
    assert get() is a


def test_a_captured_graph_has_its_own(fakes):
    eager = get()
    fakes.capture = 41
    first = get()
    assert first is not eager and get(100) is first
    bigger = get(1000)
    assert bigger is not first
    fakes.capture = 42
    second = get()
    assert second is not eager and second is not first and second is not bigger
    fakes.capture = 0
    assert get() is eager  # never a buffer that only a graph's replay zeroes
    fakes.capture = 42     # (the same capture, asked again)
    assert get() is second


def test_a_first_call_inside_a_capture_leaves_nothing_behind(fakes):
    fakes.capture = 43
    captured = get()
    fakes.capture = 0
    assert get() is not captured


@pytest.mark.parametrize("cache", ["16bit", "nvfp4"])
def test_a_workspace_of_another_head_count_is_refused(cache):
    """Its counters lie where calls with this many heads put partial rows."""
    class Workspace:
        max_num_seqs, num_q_heads, num_kv_heads = 8, 16, 8

    q = torch.zeros(2, 16, 128, dtype=torch.bfloat16)
    kc = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    if cache == "nvfp4":
        kc = torch.zeros(ops.nvfp4_cache_shape(4, 16, 2), dtype=torch.uint8)
    table, lens = torch.zeros(2, 4, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="8 kv heads, the call has 2"):
        ops.paged_decode(q, kc, kc, table, lens, 0.1, q, workspace=Workspace())
    Workspace.num_kv_heads = 2
    with pytest.raises(ValueError, match="CUDA"):  # past the workspace's checks
        ops.paged_decode(q, kc, kc, table, lens, 0.1, q, workspace=Workspace())
