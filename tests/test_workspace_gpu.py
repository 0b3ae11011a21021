"""GPU: decodes without a workspace of their own, captured, grown past and run side by side."""
from __future__ import annotations

import pytest
import torch

import mod_ref
from ps_attn import ops

pytestmark = pytest.mark.gpu


def decode(b, mod, out, lse):
    ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, b.scale, out, lse=lse, score_mod=mod, **b.scales)


def capture(b, mod):
    out, lse = torch.empty_like(b.q), torch.empty(b.hq, b.q.shape[0], device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        decode(b, mod, out, lse)
    return g, out, lse


@pytest.mark.parametrize("kind", ["16bit", "nvfp4"])
def test_a_graph_outlives_a_larger_batch(kind):
    """The first call of its heads is captured; then larger batches come and go and what they freed is overwritten."""
    hq, hkv = (6, 3) if kind == "16bit" else (10, 5)
    b = mod_ref.Batch([9000, 33, 1200], [1] * 3, hq, hkv, kind=kind, seed=81)
    ref = b.reference(dict(softcap=20.0))
    g, out, lse = capture(b, ops.ScoreMod(softcap=20.0))
    many = mod_ref.Batch([17 + i % 40 for i in range(700)], [1] * 700, hq, hkv, kind=kind, seed=82)
    o, l = torch.empty_like(many.q), torch.empty(hq, 700, device="cuda")
    for _ in range(3):
        decode(many, ops.ScoreMod(softcap=20.0), o, l)
        junk = [torch.full((1 << 20,), 0x5A5A5A5A, dtype=torch.int32, device="cuda") for _ in range(8)]
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        mod_ref.check(out, lse, ref)
        assert all(bool((j == 0x5A5A5A5A).all()) for j in junk)
    mod_ref.check(o, l, many.reference(dict(softcap=20.0)))


def test_graphs_and_calls_on_their_own_streams():
    """Two graphs and plain calls on a third stream, none with a workspace of its own, run at the same time."""
    bs = [mod_ref.Batch([5000 + 311 * i, 700, 2000], [1] * 3, 8, 2, kind="nvfp4", seed=83 + i) for i in range(3)]
    refs = [b.reference(dict(softcap=15.0)) for b in bs]
    mod = ops.ScoreMod(softcap=15.0)
    graphs = [capture(b, mod) for b in bs[:2]]
    out, lse = torch.empty_like(bs[2].q), torch.empty(8, 3, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(30):
        for s, (g, _, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            decode(bs[2], mod, out, lse)
    torch.cuda.synchronize()
    for (o, l), r in zip([g[1:] for g in graphs] + [(out, lse)], refs):
        mod_ref.check(o, l, r)
