"""GPU: the backend's forward over a 4-bit cache and with score modifiers on a
mixed decode + prefill batch, step after step, against plain 64-bit attention;
and the ``torch.ops.ps_attn`` operators of both."""
from __future__ import annotations

import pytest
import torch

import mod_ref
from ps_attn import ops, torch_ops

pytestmark = pytest.mark.gpu

HQ, HKV = 16, 4
SLOPES = [2.0 ** (-0.5 * (i + 1)) for i in range(HQ)]


@pytest.mark.parametrize("kv_dtype,kw", [
    ("nvfp4", {}),
    ("nvfp4", dict(sliding_window=50, logits_soft_cap=20.0)),
    ("auto", dict(sliding_window=100, logits_soft_cap=15.0)),
    ("auto", dict(alibi_slopes=SLOPES)),
    ("fp8", dict(sliding_window=70, alibi_slopes=SLOPES)),
])
def test_forward_over_steps(cuda_device, kv_dtype, kw):
    psb = pytest.importorskip("ps_attn.backend")
    bs, dtype = 32, torch.bfloat16
    gen = torch.Generator().manual_seed(31)
    args = dict(alibi_slopes=None, sliding_window=None, kv_cache_dtype=kv_dtype)
    args.update(kw)
    cls = psb.PSScoreModAttentionImpl if kw else psb.PSAttentionImpl
    impl = cls(HQ, 128, 128 ** -0.5, HKV, **args)
    gk, gv = (0.043, 0.037) if kv_dtype != "auto" else (1.0, 1.0)

    class Layer:
        _k_scale = torch.tensor(gk, device=cuda_device)
        _v_scale = torch.tensor(gv, device=cuda_device)

    nb, width = 30, 7
    shape = psb.PSAttentionBackend.get_kv_cache_shape(nb, bs, HKV, 128, kv_dtype)
    quant = kv_dtype != "auto"
    cache = torch.zeros(shape, dtype=torch.uint8 if quant else dtype, device=cuda_device)
    cache.fill_(0x7F if quant else float("nan"))
    table = torch.randperm(nb, generator=gen)[:4 * width].view(4, width).int()
    held = [[torch.zeros(0, HKV, 128, dtype=torch.float64)] * 2 for _ in range(4)]

    def as_held(x, g):
        if kv_dtype == "nvfp4":
            return mod_ref.nvfp4_values(x, g)
        if kv_dtype == "fp8":
            g32 = torch.tensor(g, dtype=torch.float32)
            return (x.float() / g32).clamp(-448, 448).to(torch.float8_e4m3fn).double() * float(g32)
        return x.double()

    ws = ops.DecodeWorkspace(4, HQ, HKV, 128, cuda_device)
    mod = dict(softcap=kw.get("logits_soft_cap", 0.0), window_left=kw["sliding_window"] - 1 if "sliding_window" in kw else -1)
    if "alibi_slopes" in kw:
        mod["alibi_slopes"] = torch.tensor(SLOPES)
    # decode rows first: (sequence, new tokens) of each step
    for step in ([(0, 80), (1, 33), (2, 1)], [(2, 1), (0, 1), (1, 40), (3, 90)], [(0, 1), (1, 1), (2, 1), (3, 1)]):
        seqs, new = [s for s, _ in step], [n for _, n in step]
        nd = sum(1 for i, n in enumerate(new) if n == 1 and all(m == 1 for m in new[:i]))
        T = sum(new)
        k = torch.randn(T, HKV, 128, generator=gen).to(dtype)
        v = torch.randn(T, HKV, 128, generator=gen).to(dtype)
        q = torch.randn(T, HQ, 128, generator=gen).to(dtype)
        starts = torch.tensor([0] + new).cumsum(0).int()
        slots = []
        for i, (s, n) in enumerate(step):
            pos = torch.arange(held[s][0].shape[0], held[s][0].shape[0] + n)
            slots.append(table[s][pos // bs].long() * bs + pos % bs)
            rows = slice(int(starts[i]), int(starts[i + 1]))
            held[s] = [torch.cat([held[s][0], as_held(k[rows], gk)]), torch.cat([held[s][1], as_held(v[rows], gv)])]
        lens = [held[s][0].shape[0] for s in seqs]
        md = psb.PSAttentionMetadata(
            num_actual_tokens=T, max_query_len=max(new), query_start_loc=starts.to(cuda_device), max_seq_len=max(lens),
            seq_lens=torch.tensor(lens, dtype=torch.int32, device=cuda_device),
            block_table=table[seqs].to(cuda_device), slot_mapping=torch.cat(slots).to(cuda_device), num_decodes=nd,
            num_decode_tokens=nd, num_prefills=len(step) - nd, workspace=ws)
        out = torch.full((T + 3, HQ, 128), 9.0, dtype=dtype, device=cuda_device)
        pad = torch.zeros(3, HQ, 128, dtype=dtype)  # vLLM pads its buffers
        impl.forward(Layer(), torch.cat([q, pad]).to(cuda_device), k.to(cuda_device), v.to(cuda_device), cache, md, out)
        ref = mod_ref.attention(q, [held[s][0] for s in seqs], [held[s][1] for s in seqs], starts, impl.scale, mod,
                                dtype, prefill=True)
        torch.cuda.synchronize()
        ro, _, otol, _ = ref
        assert bool(((out[:T].cpu().double() - ro).abs() <= otol).all())
        assert torch.all(out[T:] == 9.0)
    assert ws.status() == 0


def test_torch_operators(cuda_device):
    b = mod_ref.Batch([100, 33, 700], [1, 1, 1], HQ, HKV, kind="nvfp4", seed=32)
    ws = torch_ops.workspace_tensor(3, HQ, HKV, device=cuda_device)
    out, lse = torch.empty_like(b.q), torch.empty(HQ, 3, device=cuda_device)
    sl = torch.tensor(SLOPES, device=cuda_device)
    args = (b.q, b.kc, b.vc, b.table, b.lens, None, b.scale, out, lse, ws, 20.0, sl, 300, None, b.scales["k_scale"],
            b.scales["v_scale"])
    torch.ops.ps_attn.paged_decode_mod(*args)
    m = dict(softcap=20.0, alibi_slopes=sl.cpu(), window_left=300)
    mod_ref.check(out, lse, b.reference(m))
    torch.library.opcheck(torch.ops.ps_attn.paged_decode_mod.default, args,
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
    p = mod_ref.Batch([100, 333], [100, 50], HQ, HKV, seed=33)
    out, lse = torch.empty_like(p.q), torch.empty(HQ, 150, device=cuda_device)
    args = (p.q, p.kc, p.vc, p.table, p.lens, p.starts.cuda(), p.scale, out, lse, ws, 20.0, sl, 60)
    torch.ops.ps_attn.chunked_prefill_mod(*args)
    m["window_left"] = 60
    mod_ref.check(out, lse, p.reference(m, prefill=True))
    kc, vc = torch.zeros_like(b.kc), torch.zeros_like(b.vc)
    args = (b.rows_k.cuda(), b.rows_v.cuda(), kc, vc, b.slots.cuda(), b.scales["k_scale"], b.scales["v_scale"])
    torch.ops.ps_attn.kv_append_scaled(*args)
    want = torch.full_like(b.kc, 0)
    ops.kv_append(b.rows_k.cuda(), b.rows_v.cuda(), want, torch.zeros_like(b.vc), b.slots.cuda(), **b.scales)
    assert torch.equal(kc, want)
    torch.library.opcheck(torch.ops.ps_attn.kv_append_scaled.default, args,
                          test_utils=("test_schema", "test_faketensor", "test_autograd_registration"))
