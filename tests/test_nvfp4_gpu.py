"""GPU: the 4-bit (nvfp4) KV cache -- append, read-back, decode and prefill --
against the format's definition and plain 64-bit attention."""
from __future__ import annotations

import math

import pytest
import torch

import mod_ref
from ps_attn import ops

pytestmark = pytest.mark.gpu


def appended(rows_k, rows_v, nb, bs, hkv, slots, gk, gv, fill=0):
    kc = torch.full(ops.nvfp4_cache_shape(nb, bs, hkv), fill, dtype=torch.uint8, device="cuda")
    vc = torch.full_like(kc, fill)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv_append(rows_k.cuda(), rows_v.cuda(), kc, vc, slots.cuda(), status=status,
                  k_scale=torch.tensor([gk], device="cuda"), v_scale=torch.tensor([gv], device="cuda"))
    torch.cuda.synchronize()
    return kc, vc, int(status)


def same(a, b):
    return torch.equal(a.nan_to_num(nan=1e9), b.nan_to_num(nan=1e9))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,hkv,bs,g", [(1, 1, 16, 1.0), (7, 3, 16, 0.5), (100, 8, 32, 0.0037), (333, 2, 64, 0.11)])
def test_append_stores_the_definition(dtype, T, hkv, bs, g):
    gen = torch.Generator().manual_seed(T)
    nb = T // bs + 4
    slots = torch.randperm(nb * bs, generator=gen)[:T]
    k = (torch.randn(T, hkv, 128, generator=gen) * torch.exp2(torch.randn(T, hkv, 1, generator=gen) * 3)).to(dtype)
    v = torch.randn(T, hkv, 128, generator=gen).to(dtype)
    kc, vc, status = appended(k, v, nb, bs, hkv, slots, g, g / 2)
    assert status == 0
    for cache, x, s, value in ((kc, k, g, False), (vc, v, g / 2, True)):
        held, sc = mod_ref.quantize_nvfp4(x, s)
        want = torch.zeros(nb * bs, hkv, 128, dtype=torch.float64)
        want[slots] = (held.unflatten(-1, (8, 16)) * sc[..., None]).flatten(-2)
        assert torch.equal(mod_ref.decode_tiles(cache.cpu(), value).view(nb * bs, hkv, 128), want)


def test_append_special_values():
    """Ties of both roundings, zeros, infinities, NaN, blocks below the smallest scale."""
    x = torch.zeros(10, 1, 128, dtype=torch.bfloat16)
    x[0, 0, :16] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6])
    x[1, 0, 0] = 6 * 1.0625   # the scale lies between two e4m3 values
    x[2, 0, 0] = 6 * 1.1875
    x[3, 0, :4] = torch.tensor([math.inf, -math.inf, 1.0, -1.0])
    x[4, 0, 5] = math.nan
    x[4, 0, 6] = 3.0
    x[5, 0, :2] = torch.tensor([6 * 2.0 ** -10, 1e-30])  # a tie between no scale and the smallest
    x[6, 0, :2] = torch.tensor([1e-4, -1e-4])
    x[7] = 3.38e38
    x[8] = torch.randn(1, 128)
    kc, vc, _ = appended(x, x, 1, 16, 1, torch.arange(10), 1.0, 1.0)
    held, s = mod_ref.quantize_nvfp4(x, 1.0)
    want = (held.unflatten(-1, (8, 16)) * s[..., None]).flatten(-2)
    for cache, value in ((kc, False), (vc, True)):
        got = mod_ref.decode_tiles(cache.cpu(), value).view(16, 1, 128)[:10]
        assert same(got, want)
    assert torch.isnan(got[4, 0, :16]).all() and got[3, 0, 0] == 2688 and got[3, 0, 1] == -2688
    assert torch.all(got[6] == 0)


def test_append_padding_bounds_and_strided_rows():
    gen = torch.Generator().manual_seed(2)
    wide = torch.randn(9, 2, 3, 128, generator=gen).to(torch.bfloat16).cuda()
    k, v = wide[:, :, 1], wide[:, :, 2]
    slots = torch.tensor([3, -1, 40, 47, 48, 5, 10 ** 12, 0], dtype=torch.int64)  # 48 and more: past the pool
    kc, vc, status = appended(k, v, 3, 16, 2, slots, 0.1, 0.1, fill=0x11)
    assert status == 1
    good = [0, 2, 3, 5, 7]
    for cache, x, value in ((kc, k, False), (vc, v, True)):
        got = mod_ref.decode_tiles(cache.cpu(), value).view(48, 2, 128)
        held, s = mod_ref.quantize_nvfp4(x.cpu(), 0.1)
        want = (held.unflatten(-1, (8, 16)) * s[..., None]).flatten(-2)
        assert torch.equal(got[slots[good]], want[good])
        rest = torch.ones(48, dtype=torch.bool)
        rest[slots[good]] = False
        untouched = mod_ref.decode_tiles(torch.full_like(cache, 0x11).cpu(), value).view(48, 2, 128)
        assert torch.equal(got[rest], untouched[rest])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bs,hkv", [(16, 1), (32, 3), (256, 8)])
def test_gather_reads_back(dtype, bs, hkv):
    lens = [1, 15, 16, 17, 300, 0]
    b = mod_ref.Batch(lens, [1] * 6, hkv, hkv, dtype=dtype, bs=bs, kind="nvfp4", seed=21)
    width = b.table.shape[1]
    plain = ops.dequant_gather(b.kc, b.vc, b.table, b.lens, width, dtype)
    out = tuple(torch.full((6 * width, bs, hkv, 128), 5.0, dtype=dtype, device="cuda") for _ in range(2))
    scaled = ops.dequant_gather(b.kc, b.vc, b.table, b.lens, width, dtype, out=out, **b.scales)
    assert scaled[0].data_ptr() == out[0].data_ptr()
    at = 0
    for i, n in enumerate(lens):
        for x, y, rows, g in ((plain[0], scaled[0], b.rows_k, b.gk), (plain[1], scaled[1], b.rows_v, b.gv)):
            held, s = mod_ref.quantize_nvfp4(rows[at:at + n], g)
            v = (held.unflatten(-1, (8, 16)) * s[..., None]).flatten(-2)
            got = x.view(6, width * bs, hkv, 128)[i, :n].cpu()
            assert torch.equal(got.double(), v)  # exact in either type
            g32 = torch.tensor(g, dtype=torch.float32)
            got = y.view(6, width * bs, hkv, 128)[i, :n].cpu()
            assert torch.equal(got, (v.float() * g32).to(dtype))
            used = (n + bs - 1) // bs
            assert torch.all(y.view(6, width, bs, hkv, 128)[i, used:] == 5.0)  # pages past the length: as they were
        at += n


@pytest.mark.parametrize("hq,hkv,dtype,bs", [(1, 1, torch.float16, 16), (16, 8, torch.bfloat16, 16),
                                             (10, 2, torch.float16, 32), (24, 2, torch.bfloat16, 64),
                                             (32, 2, torch.bfloat16, 256)])
def test_decode_matches_plain(hq, hkv, dtype, bs):
    lens = [1, 15, 16, 17, 63, 64, 65, 128, 999, 0, 3001]
    b = mod_ref.Batch(lens, [1] * len(lens), hq, hkv, dtype=dtype, bs=bs, kind="nvfp4", seed=22)
    out = torch.full_like(b.q, float("nan"))
    lse = torch.full((hq, len(lens)), float("nan"), device="cuda")
    ws = ops.DecodeWorkspace(len(lens), hq, hkv, 128)
    for _ in range(2):  # the workspace serves call after call
        ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, b.scale, out, lse=lse, workspace=ws, **b.scales)
        mod_ref.check(out, lse, b.reference())
    assert ws.status() == 0


def test_decode_without_scales_and_large_queries():
    """No tensor scales (1.0); query rows beyond f16's range, tiny and zero ones."""
    b = mod_ref.Batch([300] * 4, [1] * 4, 8, 2, kind="nvfp4", seed=23)
    b.q[1] *= 1e-30
    b.q[2] = 0
    b.q[3] *= 3e5
    k = [x / b.gk for x in b.ks]
    v = [x / b.gv for x in b.vs]
    scale = b.scale * b.gk
    ref = mod_ref.attention(b.q, k, v, b.starts, scale, None, torch.float16)
    out, lse = torch.empty_like(b.q), torch.empty(8, 4, device="cuda")
    ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, scale, out, lse=lse)
    # scores of the last row reach 1e6: fp32 holds them to 2^-23 of that
    mod_ref.check(out[:3], lse[:, :3], tuple(x[:3] if x.dim() == 3 else x[:, :3] for x in ref))
    assert torch.isfinite(out).all()
    big = torch.softmax((b.q[3].double().cpu().view(2, 4, 128) @ k[3].permute(1, 2, 0)) * scale, -1)
    top = big.amax(-1) > 0.999  # rows decided by one key
    want = (big @ v[3].transpose(0, 1)).view(8, 128)
    got = out[3].double().cpu()
    for h in range(8):
        if top.view(8)[h]:
            assert (got[h] - want[h]).abs().max() <= 2.0 ** -7 * want[h].abs().max()


def test_decode_reports_blocks_outside_the_pool():
    b = mod_ref.Batch([100, 50], [1, 1], 8, 2, kind="nvfp4", seed=24)
    b.table[1, 2] = 10 ** 6
    ws = ops.DecodeWorkspace(2, 8, 2, 128)
    out = torch.empty_like(b.q)
    ops.paged_decode(b.q, b.kc, b.vc, b.table, b.lens, b.scale, out, workspace=ws, **b.scales)
    assert ws.status() == 2
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.dequant_gather(b.kc, b.vc, b.table, b.lens, b.table.shape[1], b.dtype, status=status)
    assert int(status) == 2


def test_decode_cache_inside_a_wider_allocation():
    """Block and head strides that are not the packed ones."""
    b = mod_ref.Batch([200, 70], [1, 1], 8, 2, kind="nvfp4", seed=25)
    nb = b.kc.shape[0]
    wide = torch.full((nb, 5, 2, 16, 72), 0x7F, dtype=torch.uint8, device="cuda")
    kc, vc = wide[:, 1], wide[:, 3]
    kc.copy_(b.kc)
    vc.copy_(b.vc)
    out, lse = torch.empty_like(b.q), torch.empty(8, 2, device="cuda")
    ops.paged_decode(b.q, kc, vc, b.table, b.lens, b.scale, out, lse=lse, **b.scales)
    mod_ref.check(out, lse, b.reference())
    k16, v16, bt = ops.dequant_gather(kc, vc, b.table, b.lens, b.table.shape[1], b.dtype)
    k2, v2, _ = ops.dequant_gather(b.kc, b.vc, b.table, b.lens, b.table.shape[1], b.dtype)
    used = [i * b.table.shape[1] + j for i, n in enumerate((200, 70)) for j in range((n + 15) // 16)]
    assert torch.equal(k16[used].view(torch.int16), k2[used].view(torch.int16))
    assert torch.equal(v16[used].view(torch.int16), v2[used].view(torch.int16))


@pytest.mark.parametrize("dtype,bs", [(torch.bfloat16, 16), (torch.float16, 64)])
def test_a_sequence_served_from_a_4bit_cache(dtype, bs):
    """Prompt, follow-up chunk and decode steps as a server runs them: rows appended, pages gathered for the
    prefill, the decode's append fused; every step against plain attention over what the cache holds."""
    gen = torch.Generator().manual_seed(26)
    hq, hkv, B = 8, 2, 3
    gk, gv = torch.tensor([0.043], device="cuda"), torch.tensor([0.037], device="cuda")
    sc = dict(k_scale=gk, v_scale=gv)
    nb, width = 40, 12 * 16 // bs
    kc = torch.full(ops.nvfp4_cache_shape(nb, bs, hkv), 0x7F, dtype=torch.uint8, device="cuda")
    vc = torch.full_like(kc, 0x7F)
    table = torch.randperm(nb, generator=gen)[:B * width].view(B, width).int().cuda()
    held = [[torch.zeros(0, hkv, 128, dtype=torch.float64)] * 2 for _ in range(B)]
    ws = ops.DecodeWorkspace(B, hq, hkv, 128)
    lens = [0] * B
    scale = 128 ** -0.5
    for step, new in enumerate(([37, 16, 90], [20, 1, 33], [1, 1, 1], [1, 1, 1], [1, 1, 1])):
        starts = torch.tensor([0] + new).cumsum(0).int()
        T = sum(new)
        k = torch.randn(T, hkv, 128, generator=gen).to(dtype)
        v = torch.randn(T, hkv, 128, generator=gen).to(dtype)
        q = torch.randn(T, hq, 128, generator=gen).to(dtype)
        slots = []
        for b, n in enumerate(new):
            pos = torch.arange(lens[b], lens[b] + n)
            slots.append(table[b].cpu()[pos // bs].long() * bs + pos % bs)
            rows = slice(int(starts[b]), int(starts[b + 1]))
            held[b] = [torch.cat([held[b][0], mod_ref.nvfp4_values(k[rows], 0.043)]),
                       torch.cat([held[b][1], mod_ref.nvfp4_values(v[rows], 0.037)])]
            lens[b] += n
        slots = torch.cat(slots).cuda()
        L = torch.tensor(lens, dtype=torch.int32, device="cuda")
        qc, out = q.cuda(), torch.empty(T, hq, 128, dtype=dtype, device="cuda")
        lse = torch.empty(hq, T, device="cuda")
        if max(new) > 1:
            ops.kv_append(k.cuda(), v.cuda(), kc, vc, slots, **sc)
            k16, v16, bt = ops.dequant_gather(kc, vc, table, L, (max(lens) + bs - 1) // bs, dtype)
            ops.chunked_prefill(qc, k16, v16, bt, L, starts.cuda(), scale, out, lse=lse, workspace=ws, **sc)
        else:
            ops.paged_decode(qc, kc, vc, table, L, scale, out, lse=lse, workspace=ws, new_key=k.cuda(),
                             new_value=v.cuda(), slot_mapping=slots, **sc)
        ref = mod_ref.attention(q, [h[0] for h in held], [h[1] for h in held], starts, scale, None,
                                dtype if max(new) > 1 else torch.float16, prefill=max(new) > 1)
        mod_ref.check(out, lse, ref)
    assert ws.status() == 0
