"""GPU: attention with score modifiers (tanh cap, distance bias, sliding window,
document and prefix masks) against plain 64-bit attention, over 16-bit, fp8 and
4-bit caches whose unused slots hold NaN."""
from __future__ import annotations

import pytest
import torch

import mod_ref
from ps_attn import ops

pytestmark = pytest.mark.gpu


def slopes(hq):
    return torch.exp2(-8.0 * torch.arange(1, hq + 1, dtype=torch.float32) / hq)


def to_mod(mod, dev="cuda"):
    kw = {k: (v.to(dev) if isinstance(v, torch.Tensor) else v) for k, v in mod.items()}
    return ops.ScoreMod(**kw)


def run_decode(b, mod, **kw):
    out = torch.full_like(b.q, float("nan"))
    lse = torch.full((b.hq, b.q.shape[0]), float("nan"), device="cuda")
    ws = ops.DecodeWorkspace(max(len(b.lens_list), 1), b.hq, b.hkv, 128)
    ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, b.scale, out, lse=lse, query_start_loc=b.starts.cuda(),
                     workspace=ws, score_mod=to_mod(mod) if mod is not None else None, **b.scales, **kw)
    torch.cuda.synchronize()
    assert ws.status() == 0
    return out, lse


def run_prefill(b, mod, workspace=True):
    out = torch.full_like(b.q, float("nan"))
    lse = torch.full((b.hq, b.q.shape[0]), float("nan"), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = ops.DecodeWorkspace(len(b.lens_list), b.hq, b.hkv, 128) if workspace else None
    ops.chunked_prefill(b.q, b.kc, b.vc, b.table, b.lens, b.starts.cuda(), b.scale, out, lse=lse, status=status,
                        workspace=ws, score_mod=to_mod(mod) if mod is not None else None)
    torch.cuda.synchronize()
    assert int(status) == 0
    return out, lse


LENS = [1, 15, 16, 17, 63, 64, 65, 130, 257, 1000, 2049]
MODS = {
    "cap": lambda hq: dict(softcap=7.5),
    "bias": lambda hq: dict(alibi_slopes=slopes(hq)),
    "window0": lambda hq: dict(window_left=0),
    "window15": lambda hq: dict(window_left=15),
    "window16": lambda hq: dict(window_left=16),
    "window100": lambda hq: dict(window_left=100),
    "all": lambda hq: dict(softcap=30.0, alibi_slopes=slopes(hq), window_left=333),
    "none": lambda hq: dict(),
}


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
@pytest.mark.parametrize("mod", MODS)
def test_decode_matches_plain(kind, mod):
    b = mod_ref.Batch(LENS, [1] * len(LENS), 8, 2, kind=kind, seed=3)
    m = MODS[mod](8)
    mod_ref.check(*run_decode(b, m), b.reference(m))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
@pytest.mark.parametrize("hq,hkv,dtype,bs", [(1, 1, torch.float16, 16), (5, 1, torch.bfloat16, 32),
                                             (16, 2, torch.float16, 64), (24, 2, torch.bfloat16, 16),
                                             (16, 1, torch.float16, 256)])
def test_decode_heads_types_blocks(kind, hq, hkv, dtype, bs):
    lens = [700, 3, 4097, 96, 31]
    b = mod_ref.Batch(lens, [1] * 5, hq, hkv, dtype=dtype, bs=bs, kind=kind, seed=4)
    m = dict(softcap=12.0, alibi_slopes=slopes(hq), window_left=600)
    mod_ref.check(*run_decode(b, m), b.reference(m))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
def test_decode_documents_and_empty_rows(kind):
    lens = [40, 40, 40, 40, 500, 500, 0, 1, 1]
    b = mod_ref.Batch(lens, [1] * 9, 8, 2, kind=kind, seed=5)
    # first key: 0, inside, the last key, past the row (nothing left), far past, a page's first
    start = torch.tensor([0, 17, 39, 40, 10 ** 6, 496, 0, 0, 1], dtype=torch.int32)
    m = dict(key_start=start, softcap=20.0, prefix_lens=torch.full((9,), 30, dtype=torch.int32))
    out, lse = run_decode(b, m)
    ref = b.reference(dict(key_start=start, softcap=20.0))
    mod_ref.check(out, lse, ref)
    for row in (3, 4, 6, 8):
        assert torch.all(out[row] == 0) and torch.all(torch.isneginf(lse[:, row]))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
def test_decode_window_never_looks_below(kind):
    """Pages below the window have been given away: their entries are invalid."""
    lens = [1000, 777, 300]
    b = mod_ref.Batch(lens, [1] * 3, 8, 2, kind=kind, seed=6)
    m = dict(window_left=200)
    ref = b.reference(m)
    for i, n in enumerate(lens):
        b.table[i, :max(0, n - 1 - 200) // 16] = -1
    mod_ref.check(*run_decode(b, m), ref)


@pytest.mark.parametrize("kind", ["16bit", "nvfp4"])
def test_decode_one_long_sequence_over_many_splits(kind):
    b = mod_ref.Batch([40003], [1], 8, 1, kind=kind, seed=7)
    for m in (dict(softcap=50.0), dict(alibi_slopes=slopes(8)), dict(window_left=20001)):
        mod_ref.check(*run_decode(b, m), b.reference(m))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
def test_decode_fused_append(kind):
    """The appended token is attended and stored, also where the masks hide it."""
    lens = [1, 16, 17, 100, 1025, 50]
    b = mod_ref.Batch(lens, [1] * 6, 8, 2, kind=kind, seed=8)
    want_k, want_v = b.kc.clone(), b.vc.clone()
    ends = torch.tensor(lens).cumsum(0) - 1
    slot = b.slots[ends].cuda()
    # take the last tokens out of the cache again
    if kind == "nvfp4":
        nan = torch.full((6, 2, 128), float("nan"), dtype=b.dtype, device="cuda")
        ops.kv_append(nan, nan, b.kc, b.vc, slot, **b.scales)
    else:
        flat = (lambda c: c.view(-1, 2, 128))
        fill = 0x7F if kind == "fp8" else float("nan")
        flat(b.kc)[slot] = fill
        flat(b.vc)[slot] = fill
    start = torch.tensor([0, 0, 0, 0, 0, 50], dtype=torch.int32)
    m = dict(window_left=64, key_start=start)
    out, lse = run_decode(b, m, new_key=b.rows_k[ends].cuda(), new_value=b.rows_v[ends].cuda(), slot_mapping=slot)
    mod_ref.check(out, lse, b.reference(m))
    as_bytes = (lambda t: t.view(torch.uint8) if t.dtype == torch.uint8 else t.view(torch.int16))
    assert torch.equal(as_bytes(b.kc), as_bytes(want_k)) and torch.equal(as_bytes(b.vc), as_bytes(want_v))


def test_decode_strided_rows_and_skipped_sequences():
    lens, qlens = [33, 500, 64, 129], [1, 0, 1, 1]
    b = mod_ref.Batch(lens, qlens, 8, 2, seed=9)
    m = dict(window_left=50, softcap=9.0)
    ref = b.reference(m)
    wide = torch.zeros(b.q.shape[0], 8, 384, dtype=b.dtype, device="cuda")
    wide[..., 128:256] = b.q
    out = torch.full((b.q.shape[0] + 2, 8, 256), 7.0, dtype=b.dtype, device="cuda")
    lse = torch.full((8, b.q.shape[0]), float("nan"), device="cuda")
    ops.paged_decode(wide[..., 128:256], b.kc, b.vc, b.table, b.lens, b.scale, out[..., :128], lse=lse,
                     query_start_loc=b.starts.cuda(), score_mod=to_mod(m))
    mod_ref.check(out[:3, :, :128], lse, ref)
    assert torch.all(out[..., 128:] == 7.0) and torch.all(out[3:] == 7.0)


# ---------------------------------------------------------------- prefill

PREFILL = {
    "cap": lambda hq, T, B: dict(softcap=7.5),
    "bias": lambda hq, T, B: dict(alibi_slopes=slopes(hq)),
    "window0": lambda hq, T, B: dict(window_left=0),
    "window17": lambda hq, T, B: dict(window_left=17),
    "window300": lambda hq, T, B: dict(window_left=300, softcap=25.0),
    "prefix": lambda hq, T, B: dict(prefix_lens=(torch.arange(B) * 97 % 421).int()),
    "prefix_bias": lambda hq, T, B: dict(prefix_lens=(torch.arange(B) * 97 % 421).int(), alibi_slopes=slopes(hq)),
    "all": lambda hq, T, B: dict(prefix_lens=(torch.arange(B) * 97 % 421).int(), alibi_slopes=slopes(hq),
                                 softcap=30.0, window_left=200),
    "none": lambda hq, T, B: dict(),
}


@pytest.mark.parametrize("mod", PREFILL)
def test_prefill_matches_plain(mod):
    lens = [1, 5, 16, 129, 300, 777, 600]
    qlens = [1, 5, 7, 129, 111, 777, 1]
    b = mod_ref.Batch(lens, qlens, 8, 2, seed=11)
    m = PREFILL[mod](8, sum(qlens), len(lens))
    mod_ref.check(*run_prefill(b, m), b.reference(m, prefill=True))


@pytest.mark.parametrize("hq,hkv,dtype,bs", [(1, 1, torch.float16, 16), (5, 1, torch.bfloat16, 32),
                                             (16, 1, torch.float16, 64), (12, 2, torch.bfloat16, 256)])
def test_prefill_heads_types_blocks(hq, hkv, dtype, bs):
    lens, qlens = [400, 90, 1200], [257, 90, 300]
    b = mod_ref.Batch(lens, qlens, hq, hkv, dtype=dtype, bs=bs, seed=12)
    m = dict(softcap=15.0, alibi_slopes=slopes(hq), window_left=250,
             prefix_lens=torch.tensor([0, 40, 950], dtype=torch.int32))
    mod_ref.check(*run_prefill(b, m), b.reference(m, prefill=True))
    m = dict(window_left=140)
    mod_ref.check(*run_prefill(b, m, workspace=False), b.reference(m, prefill=True))


def test_prefill_documents_any_order_and_empty_rows():
    lens, qlens = [700, 64, 300], [700, 64, 40]
    b = mod_ref.Batch(lens, qlens, 4, 2, seed=13)
    g = torch.Generator().manual_seed(1)
    # packed documents in the first sequence, arbitrary starts in the second, none visible in parts of the third
    start = torch.zeros(804, dtype=torch.int32)
    pos = torch.arange(700)
    for cut in (100, 333, 334, 600):
        start[:700] = torch.where(pos >= cut, torch.tensor(cut), start[:700]).int()
    start[700:764] = torch.randint(0, 64, (64,), generator=g).int()
    start[764:784] = 10 ** 6
    start[784:804] = 290
    m = dict(key_start=start)
    out, lse = run_prefill(b, m)
    mod_ref.check(out, lse, b.reference(m, prefill=True))
    assert torch.all(out[764:784] == 0) and torch.all(torch.isneginf(lse[:, 764:784]))
    # no row of the batch sees anything
    m = dict(key_start=torch.full((804,), 10 ** 6, dtype=torch.int32))
    out, lse = run_prefill(b, m)
    assert torch.all(out == 0) and torch.all(torch.isneginf(lse))


def test_prefill_window_never_looks_below():
    lens, qlens = [2000, 1500], [64, 40]
    b = mod_ref.Batch(lens, qlens, 4, 1, seed=14)
    m = dict(window_left=100, softcap=10.0)
    ref = b.reference(m, prefill=True)
    for i, (n, k) in enumerate(zip(lens, qlens)):
        b.table[i, :(n - k - 100) // 16] = -1
    mod_ref.check(*run_prefill(b, m), ref)


def test_decode_and_prefill_agree_on_one_row():
    lens = [1, 77, 512, 1300]
    b = mod_ref.Batch(lens, [1] * 4, 8, 2, seed=15)
    m = dict(softcap=20.0, alibi_slopes=slopes(8), window_left=400)
    ref = b.reference(m, prefill=True)
    mod_ref.check(*run_decode(b, m), ref)
    mod_ref.check(*run_prefill(b, m), ref)


def test_an_empty_modifier_is_plain_attention():
    """The same scores and weights; only the merge of a sequence's splits sums in another order.  Up to 24
    positive terms: each sum is off by 24 * 2^-24 at most, the logarithm by 2^-22 and the LSE (below 16) by its
    own rounding, 2^-21; outputs differ by the rounding to bf16 of values that agree to 2^-19."""
    b = mod_ref.Batch(LENS, [1] * len(LENS), 8, 2, seed=16)
    a, la = run_decode(b, None)
    c, lc = run_decode(b, {})
    assert float((la - lc).abs().max()) <= 2 * (24 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -21)
    a, c = a.double(), c.double()
    # one bf16 step apart at most: a step is 2^-7 of the value's power of two
    assert bool(((a - c).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), c.abs())).all())


def test_captured_and_replayed():
    """A step captured in a CUDA graph follows its inputs: lengths, documents, slopes and the query rows."""
    lens = [100, 900, 33]
    b = mod_ref.Batch(lens, [1] * 3, 8, 2, kind="nvfp4", seed=17)
    start = torch.zeros(3, dtype=torch.int32, device="cuda")
    sl = slopes(8).cuda()
    out, lse = torch.empty_like(b.q), torch.empty(8, 3, device="cuda")
    ws = ops.DecodeWorkspace(3, 8, 2, 128)
    mod = ops.ScoreMod(softcap=20.0, alibi_slopes=sl, window_left=500, key_start=start)

    def step():
        ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, b.scale, out, lse=lse, workspace=ws, score_mod=mod,
                         **b.scales)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(3):
        start.copy_(torch.tensor([i * 7, 450 + i, 0], dtype=torch.int32))
        sl.mul_(0.5)
        b.q.mul_(1.0 if i == 0 else -0.5)
        b.lens.copy_(torch.tensor([100 - i, 900 - 16 * i, 33], dtype=torch.int32))
        cur = [int(x) for x in b.lens]
        graph.replay()
        torch.cuda.synchronize()
        m = dict(softcap=20.0, alibi_slopes=sl.cpu(), window_left=500, key_start=start.cpu())
        ref = mod_ref.attention(b.q, [k[:n] for k, n in zip(b.ks, cur)], [v[:n] for v, n in zip(b.vs, cur)],
                                b.starts, b.scale, m, torch.float16)
        mod_ref.check(out, lse, ref)
    assert ws.status() == 0
