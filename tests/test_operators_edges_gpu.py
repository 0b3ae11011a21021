"""GPU: the score modifiers and the 4-bit cache at the ends of their ranges: the most sequences of a launch, offsets
past 32 bits, merges in two levels, inconsistent lengths and slots, saturated caps, NaN rows, other streams, graphs."""
from __future__ import annotations

import ctypes

import pytest
import torch

import mod_ref
from ps_attn import _lib, ops
from test_score_mod_gpu import run_decode, run_prefill, slopes, to_mod

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["16bit", "nvfp4"])
def test_most_sequences_of_one_launch(kind):
    lens = [(i * 37) % 41 for i in range(4096)]  # some empty
    b = mod_ref.Batch(lens, [1] * 4096, 1, 1, kind=kind, seed=41)
    m = dict(window_left=20, softcap=11.0)
    mod_ref.check(*run_decode(b, m), b.reference(m))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
@pytest.mark.parametrize("hq", [1, 2, 3, 8, 13])
def test_merges_in_two_levels(kind, hq):
    """One kv head, one or two sequences: hundreds of splits, chunks of 16 and of 32 and a ragged last one."""
    for lens in ([5000], [33001, 700], [9000, 8999]):
        b = mod_ref.Batch(lens, [1] * len(lens), hq, 1, kind=kind, seed=42)
        m = dict(softcap=25.0)
        for _ in range(2):  # the counters are back at zero
            mod_ref.check(*run_decode(b, m), b.reference(m))


def test_one_workspace_for_calls_of_every_kind():
    ws = ops.DecodeWorkspace(4, 8, 1, 128)
    for kind, lens, m in (("nvfp4", [20000], None), ("16bit", [20000], dict(softcap=9.0)), ("fp8", [40, 3000], {}),
                          ("nvfp4", [700, 1, 1500, 64], dict(window_left=300)), ("16bit", [900, 5], None)):
        b = mod_ref.Batch(lens, [1] * len(lens), 8, 1, kind=kind, seed=43)
        out, lse = torch.empty_like(b.q), torch.empty(8, len(lens), device="cuda")
        ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, b.scale, out, lse=lse, workspace=ws,
                         score_mod=None if m is None else to_mod(m), **b.scales)
        mod_ref.check(out, lse, b.reference(m))
    assert ws.status() == 0


def test_cache_offsets_past_32_bits():
    """Blocks beyond 4 GiB of each cache half: append, read back, decode (4-bit); decode and prefill (16-bit)."""
    hq, hkv, lens = 16, 8, [100, 333]
    src = mod_ref.Batch(lens, [1, 1], hq, hkv, kind="nvfp4", seed=44)
    nb = 480_000  # of 9,216 bytes
    kc = torch.zeros(ops.nvfp4_cache_shape(nb, 16, hkv), dtype=torch.uint8, device="cuda")
    vc = torch.zeros_like(kc)
    shift = nb - 40
    slots = src.slots.cuda() + shift * 16
    table = torch.where(src.table >= 0, src.table + shift, src.table)
    ops.kv_append(src.rows_k.cuda(), src.rows_v.cuda(), kc, vc, slots, **src.scales)
    out, lse = torch.empty_like(src.q), torch.empty(hq, 2, device="cuda")
    ops.paged_decode(src.q, kc, vc, table, src.lens, src.scale, out, lse=lse, **src.scales)
    mod_ref.check(out, lse, src.reference())
    k16, v16, bt = ops.dequant_gather(kc, vc, table, src.lens, table.shape[1], src.dtype)
    ops.paged_decode(src.q, k16, v16, bt, src.lens, src.scale, out, lse=lse, **src.scales)
    mod_ref.check(out, lse, mod_ref.attention(src.q, src.ks, src.vs, src.starts, src.scale, None, src.dtype))
    del kc, vc
    b = mod_ref.Batch(lens, [20, 50], hq, hkv, seed=45)
    nb = 140_000  # of 32,768 bytes
    kc = torch.zeros(nb, 16, hkv, 128, dtype=b.dtype, device="cuda")
    vc = torch.zeros_like(kc)
    shift = nb - b.kc.shape[0]
    kc[shift:], vc[shift:] = b.kc, b.vc
    b.kc, b.vc, b.table = kc, vc, torch.where(b.table >= 0, b.table + shift, b.table)
    m = dict(window_left=77, alibi_slopes=slopes(hq))
    mod_ref.check(*run_prefill(b, m), b.reference(m, prefill=True))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
def test_inconsistent_lengths_and_slots_are_reported(kind):
    lens = [50, 64, 90]
    b = mod_ref.Batch(lens, [1] * 3, 8, 2, kind=kind, seed=46)
    m = dict(window_left=1000)
    ref = b.reference(m)
    kc, vc = b.kc.clone(), b.vc.clone()
    as_bytes = (lambda t: t.view(torch.uint8) if t.dtype == torch.uint8 else t.view(torch.int16))
    ws = ops.DecodeWorkspace(3, 8, 2, 128)
    out, lse = torch.empty_like(b.q), torch.empty(8, 3, device="cuda")
    # a length past the block table, with a fused append
    bad = b.lens.clone()
    bad[0] = 10_000
    row = torch.randn(3, 2, 128, device="cuda").to(b.dtype)
    slot = torch.tensor([7 * 16, -1, -1], device="cuda")
    for mod in (to_mod(m), None):
        ws.clear_status()
        ops.paged_decode(b.q, b.kc, b.vc, b.table, bad, b.scale, out, lse=lse, workspace=ws, score_mod=mod,
                         new_key=row, new_value=row, slot_mapping=slot, **b.scales)
        assert ws.status() & 8
        assert torch.equal(as_bytes(b.kc), as_bytes(kc)) and torch.equal(as_bytes(b.vc), as_bytes(vc))
        mod_ref.check(out[1:], lse[:, 1:], tuple(x[1:] if x.dim() == 3 else x[:, 1:] for x in ref))
        # a table entry past the pool and the slot that goes with it
        ws.clear_status()
        nb = b.kc.shape[0]
        table = b.table.clone()
        table[0, (lens[0] - 1) // 16] = nb + 5
        past = torch.tensor([(nb + 5) * 16 + (lens[0] - 1) % 16, -1, -1], device="cuda")
        ops.paged_decode(b.q, b.kc, b.vc, table, b.lens, b.scale, out, lse=lse, workspace=ws, score_mod=mod,
                         new_key=row, new_value=row, slot_mapping=past, **b.scales)
        assert ws.status() == 2 | 8
        assert torch.equal(as_bytes(b.kc), as_bytes(kc)) and torch.equal(as_bytes(b.vc), as_bytes(vc))


def test_prefill_rows_before_the_sequence_see_nothing():
    """More query rows than tokens: the first rows lie before the sequence."""
    b = mod_ref.Batch([5, 40], [9, 40], 4, 1, seed=47)
    out, lse = run_prefill(b, dict(window_left=2 ** 31 - 1))
    assert torch.all(out[:4] == 0) and torch.all(torch.isneginf(lse[:, :4]))
    ref = mod_ref.attention(b.q[4:], b.ks, b.vs, [0, 5, 45], b.scale, {}, b.dtype, True)
    mod_ref.check(out[4:], lse[:, 4:], ref)


@pytest.mark.parametrize("cap", [0.05, 1.0, 1e4])
def test_caps_from_saturated_to_idle(cap):
    """Scores far past a small cap (the exponential form) and far inside a large one (the polynomial)."""
    b = mod_ref.Batch([300, 77], [300, 30], 8, 2, seed=48, spread=6.0)
    m = dict(softcap=cap)
    mod_ref.check(*run_prefill(b, m), b.reference(m, prefill=True))
    d = mod_ref.Batch([300, 77], [1, 1], 8, 2, kind="nvfp4", seed=49, spread=6.0)
    mod_ref.check(*run_decode(d, m), d.reference(m))


def test_a_nan_row_stays_with_its_sequence_and_heads():
    b = mod_ref.Batch([200, 200, 60], [1] * 3, 8, 2, kind="nvfp4", seed=50)
    ref = b.reference()
    k = torch.zeros(1, 2, 128, dtype=b.dtype, device="cuda")
    k[0, 1, 7] = float("nan")
    # position 70 of sequence 1, both heads rewritten; head 0's new row is what a reference needs, so keep it masked
    slot = b.slots[200 + 70:200 + 71].cuda()
    keep_k = b.kc.clone()
    ops.kv_append(k, k, b.kc, b.vc, slot, **b.scales)
    out, lse = torch.empty_like(b.q), torch.empty(8, 3, device="cuda")
    ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, b.scale, out, lse=lse, **b.scales)
    assert torch.isnan(out[1, 4:]).any(-1).all()          # kv head 1 of sequence 1
    assert torch.isfinite(out[1, :4]).all()
    for row in (0, 2):
        r = tuple(x[row:row + 1] if x.dim() == 3 else x[:, row:row + 1] for x in ref)
        mod_ref.check(out[row:row + 1], lse[:, row:row + 1], r)
    # a window past it does not see it
    m = dict(window_left=100)
    got, gl = run_decode(b, m)
    r = mod_ref.attention(b.q, b.ks, b.vs, b.starts, b.scale, m, torch.float16)
    mod_ref.check(got, gl, r)
    assert not torch.equal(keep_k, b.kc)


def test_two_streams_with_their_own_workspaces():
    bs = [mod_ref.Batch([3000 + 17 * i, 900], [1, 1], 8, 2, kind="nvfp4", seed=51 + i) for i in range(2)]
    refs = [b.reference(dict(softcap=20.0)) for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    outs = [(torch.empty_like(b.q), torch.empty(8, 2, device="cuda")) for b in bs]
    ws = [ops.DecodeWorkspace(2, 8, 2, 128) for _ in bs]
    mod = ops.ScoreMod(softcap=20.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for b, s, (o, l), w in zip(bs, streams, outs, ws):
            with torch.cuda.stream(s):
                ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, b.scale, o, lse=l, workspace=w, score_mod=mod,
                                 **b.scales)
    torch.cuda.synchronize()
    for (o, l), r, w in zip(outs, refs, ws):
        mod_ref.check(o, l, r)
        assert w.status() == 0


def test_captured_store_and_prefill_follow_their_inputs():
    """Append, gather and prefill over the 4-bit cache as one graph, replayed on other rows."""
    b = mod_ref.Batch([40, 130], [40, 30], 8, 2, kind="nvfp4", seed=53)
    rows = [torch.empty(170, 2, 128, dtype=b.dtype, device="cuda") for _ in range(2)]
    slots = b.slots.cuda()
    starts = b.starts.cuda()
    out, lse = torch.empty_like(b.q), torch.empty(8, 70, device="cuda")
    ws = ops.DecodeWorkspace(2, 8, 2, 128)
    scratch = ops.dequant_gather(b.kc, b.vc, b.table, b.lens, 9, b.dtype)
    mod = ops.ScoreMod(softcap=30.0)

    def step():
        ops.kv_append(rows[0], rows[1], b.kc, b.vc, slots, **b.scales)
        k, v, bt = ops.dequant_gather(b.kc, b.vc, b.table, b.lens, 9, b.dtype, out=scratch)
        ops.chunked_prefill(b.q, k, v, bt, b.lens, starts, b.scale, out, lse=lse, workspace=ws, score_mod=mod, **b.scales)

    for r in rows:
        r.zero_()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator().manual_seed(54)
    for _ in range(3):
        k, v = (torch.randn(170, 2, 128, generator=g).to(b.dtype) for _ in range(2))
        rows[0].copy_(k)
        rows[1].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        ks = [mod_ref.nvfp4_values(x, b.gk) for x in (k[:40], k[40:])]
        vs = [mod_ref.nvfp4_values(x, b.gv) for x in (v[:40], v[40:])]
        mod_ref.check(out, lse, mod_ref.attention(b.q, ks, vs, b.starts, b.scale, dict(softcap=30.0), b.dtype, True))
    assert ws.status() == 0


def test_static_scratch_takes_a_4bit_cache():
    lib = _lib.load()
    b = mod_ref.Batch([20000, 70], [1, 1], 8, 1, kind="nvfp4", seed=55)
    status = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    for _ in range(2):
        out, lse = torch.empty_like(b.q), torch.empty(8, 2, device="cuda")
        pr = ops._problem(b.q, b.kc, b.vc, b.table, b.lens, None, b.scale, out, lse, status=status, **b.scales)
        _lib.check(lib.ps_paged_decode_static_scratch(ctypes.byref(pr), torch.cuda.current_stream().cuda_stream))
        mod_ref.check(out, lse, b.reference())
        assert int(status) == 0


@pytest.mark.parametrize("m", [None, dict(softcap=30.0, window_left=40)], ids=["plain", "mod"])
@pytest.mark.parametrize("B,hkv", [(24, 8), (60, 8), (128, 2), (129, 2)])
def test_prefill_of_many_unequal_sequences(B, hkv, m):
    """Around the rules that list a batch's sequences by falling length: some without rows, equal lengths, one long."""
    q_lens = [(i * 5) % 13 for i in range(B)]
    lens = [q + (i * i * 7) % 90 for i, q in enumerate(q_lens)]
    lens[B // 2] += 700
    b = mod_ref.Batch(lens, q_lens, 2 * hkv, hkv, seed=56)
    mod_ref.check(*run_prefill(b, m), b.reference(m, prefill=True))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
def test_a_bad_query_stays_with_its_row_and_head(kind):
    """A NaN or infinite query in one head of one row: every other (row, head) as without it."""
    b = mod_ref.Batch([90, 300, 33], [1] * 3, 8, 2, kind=kind, seed=57)
    m = dict(softcap=12.0, window_left=120)
    ref = b.reference(m)
    keep = torch.ones(3, 8, dtype=torch.bool, device="cuda")
    b.q = b.q.clone()
    b.q[1, 2, 5], keep[1, 2] = float("nan"), False
    b.q[2, 7, 100], keep[2, 7] = float("inf"), False
    out, lse = run_decode(b, m)
    for t in range(3):
        for h in torch.nonzero(keep[t]).flatten().tolist():
            r = tuple(x[t:t + 1, h:h + 1] if x.dim() == 3 else x[h:h + 1, t:t + 1] for x in ref)
            mod_ref.check(out[t:t + 1, h:h + 1], lse[h:h + 1, t:t + 1], r)


def test_a_bad_query_row_of_a_prompt_stays_with_its_row():
    b = mod_ref.Batch([300], [300], 8, 2, seed=58)
    m = dict(softcap=12.0, window_left=120)
    ref = b.reference(m, prefill=True)
    b.q = b.q.clone()
    b.q[140, 3, 9] = float("nan")
    out, lse = run_prefill(b, m)
    out[140, 3], lse[3, 140] = ref[0][140, 3].to(out.dtype), ref[1][3, 140].float()
    mod_ref.check(out, lse, ref)
