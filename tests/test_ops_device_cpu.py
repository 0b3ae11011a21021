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


SHORT = {
    "table rows": (dict(bt=lambda x: x[:1]), "block_table has 1 rows"),
    "query rows": (dict(q=lambda x: x[:1], out=lambda x: x[:1]), "q has 1 rows"),
    "query offsets": (dict(qsl=lambda x: x[:2]), "3 entries"),
    "strided query offsets": (dict(qsl=lambda x: t(6, dtype=torch.int32)[::2]), "3 entries"),
    "head size": (dict(q=lambda x: t(2, 4, 64), out=lambda x: t(2, 4, 64)), "head size"),
    "output heads": (dict(out=lambda x: t(2, 2, 128)), "out must have"),
    "output head size": (dict(out=lambda x: t(2, 4, 64)), "out must have"),
    "LSE heads": (dict(lse=lambda x: t(3, 2, dtype=torch.float32)), "lse"),
    "LSE rows": (dict(lse=lambda x: t(4, 1, dtype=torch.float32)), "lse"),
    "new values": (dict(nv=lambda x: x[:1]), "per query row"),
}


@pytest.mark.parametrize("what", SHORT)
@pytest.mark.parametrize("kind", ["16bit", "nvfp4"])
def test_arrays_shorter_than_the_kernels_read_are_refused(trace, what, kind):
    if kind == "nvfp4" and what == "head size":
        pytest.skip("a cache of its shape is not a 4-bit one for this head size")
    a = dict(q=t(2, 4, 128), bt=t(2, 2, dtype=torch.int32), n=t(2, dtype=torch.int32), out=t(2, 4, 128), qsl=None,
             lse=t(4, 2, dtype=torch.float32), nk=t(2, 2, 128), nv=t(2, 2, 128), slots=t(2, dtype=torch.int64))
    if "offsets" in what:
        a["qsl"] = t(3, dtype=torch.int32)
    cache = t(3, 16, 2, 128) if kind == "16bit" else t(3, 2, 16, 72, dtype=torch.uint8)
    ws = SimpleNamespace(max_num_seqs=8, num_kv_heads=2, nbytes=256, buffer=t(256, dtype=torch.uint8))

    def go(a):
        ops.paged_decode(a["q"], cache, cache, a["bt"], a["n"], 0.1, a["out"], lse=a["lse"], query_start_loc=a["qsl"],
                         workspace=ws, new_key=a["nk"], new_value=a["nv"], slot_mapping=a["slots"])

    go(a)
    changes, match = SHORT[what]
    with pytest.raises(ValueError, match=match):
        go({k: changes[k](v) if k in changes else v for k, v in a.items()})
    assert len(trace.calls) == 1
    if what == "table rows" and kind == "nvfp4":
        with pytest.raises(ValueError, match=match):
            ops.dequant_gather(cache, cache, a["bt"][:1], a["n"], 2, torch.bfloat16,
                               out=(t(4, 16, 2, 128), t(4, 16, 2, 128)))


@pytest.mark.parametrize("rows", [1, 3])
def test_paged_attention_passes_the_scales_on(trace, monkeypatch, rows):
    got = []
    for name in ("paged_decode", "chunked_prefill"):
        monkeypatch.setattr(ops, name, lambda *a, _n=name, **k: got.append((_n, k["k_scale"], k["v_scale"])))
    ops.paged_attention("q", "k", "v", "o", None, rows, "n", 0.1, "bt", k_scale=2, v_scale=3)
    assert got == [("paged_decode" if rows == 1 else "chunked_prefill", 2, 3)]
