"""CPU: every call launches with its tensors' device current, not whichever is
(the C library launches on the current device); devices and library are fakes."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from ps_attn import ops


@pytest.fixture
def trace(monkeypatch):
    """Launches as (entry point, the device that was current), with tensors of "cuda:3" while device 0 is."""
    seen = SimpleNamespace(calls=[], current=0)

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.back, seen.current = seen.current, self.index

        def __exit__(self, *a):
            seen.current = self.back

    class Lib:
        def __getattr__(self, name):
            return lambda *a: seen.calls.append((name, seen.current)) or 0

    monkeypatch.setattr(ops._lib, "load", lambda: Lib())
    monkeypatch.setattr(ops.torch._C, "_cuda_getDevice", lambda: seen.current, raising=False)
    monkeypatch.setattr(ops.torch.cuda, "device", Device)
    monkeypatch.setattr(ops, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "_stream_ptr", lambda device: 1)
    return seen


class On3(torch.Tensor):
    """A CPU tensor that says it lives on cuda:3."""

    device = property(lambda self: torch.device("cuda", 3))
    is_cuda = property(lambda self: True)
    dtype = property(lambda self: torch.Tensor.dtype.__get__(self))


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(On3)


def test_every_call_makes_its_device_current(trace):
    q, kc, bt, n = t(2, 4, 128), t(3, 16, 2, 128), t(2, 2, dtype=torch.int32), t(2, dtype=torch.int32)
    k, slots, qsl = t(2, 2, 128), t(2, dtype=torch.int64), t(3, dtype=torch.int32)
    four, eight = t(3, 2, 16, 72, dtype=torch.uint8), t(3, 16, 2, 128, dtype=torch.uint8)
    ws = SimpleNamespace(max_num_seqs=8, num_kv_heads=2, nbytes=256, buffer=t(256, dtype=torch.uint8))
    for cache in (kc, four, eight):
        ops.kv_append(k, k, cache, cache, slots)
        ops.paged_decode(q, cache, cache, bt, n, 0.1, q, workspace=ws)
        ops.paged_decode(q, cache, cache, bt, n, 0.1, q, workspace=ws, score_mod=ops.ScoreMod())
    for cache in (four, eight):
        ops.dequant_gather(cache, cache, bt, n, 2, torch.bfloat16, out=(t(4, 16, 2, 128), t(4, 16, 2, 128)))
    ops.chunked_prefill(q, kc, kc, bt, n, qsl, 0.1, q)
    ops.chunked_prefill(q, kc, kc, bt, n, qsl, 0.1, q, workspace=ws)
    ops.chunked_prefill(q, kc, kc, bt, n, qsl, 0.1, q, score_mod=ops.ScoreMod())
    plan = SimpleNamespace(max_num_seqs=8, num_seqs=0, nbytes=256, buffer=t(64, dtype=torch.int32))
    ops.cascade_plan(bt, n, 4, 2, 16, plan=plan)
    ops.paged_decode(q, kc, kc, bt, n, 0.1, q, workspace=ws, cascade=plan)
    ops.paged_decode(q, kc, kc, bt, n, 0.1, q, workspace=ws, head_gather=ops._lib.HeadGatherProblem())
    lse = t(4, 2, dtype=torch.float32)
    ops.merge_attn_states(q, q, lse, q, lse)
    ops.rope_kv_append(q, k, k, slots, t(16, 128), True, kc, kc, slots)
    assert len(trace.calls) == 19
    assert [c for c in trace.calls if c[1] != 3] == [] and trace.current == 0
