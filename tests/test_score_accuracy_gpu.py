"""GPU: score modifiers held to what their arithmetic allows, 30 times and more
below a plain prefill's cubic exponential: LSEs of prompts and of single rows
under a bias, a window, documents, a prefix and all together."""
from __future__ import annotations

import math

import pytest
import torch

import mod_ref
from ps_attn import ops
from test_score_mod_gpu import run_decode, run_prefill, slopes

pytestmark = pytest.mark.gpu


def reference(b, mod, prefill):
    """(LSE, its tolerance) in float64.

    A score is off by 2^-18 of sum |q| |k| scale (its 128 products are summed in
    fp32 over at most 9 steps of 2^-22), 2^-20 of max(|z|, 1) (scale, cap and the
    exponent's argument) and 2^-21 of its bias (at most four roundings of it, and
    two of the sum); its exponential by 2^-21, in the prefill by 2.6e-6.  The LSE
    is off by the mean of that under the weights, and by its own roundings."""
    f = torch.float64
    T, hq, _ = b.q.shape
    lse, tol = torch.full((hq, T), -math.inf, dtype=f), torch.zeros(hq, T, dtype=f)
    for i, k in enumerate(b.ks):
        r0, r1, L = int(b.starts[i]), int(b.starts[i + 1]), k.shape[0]
        prefix = int(mod["prefix_lens"][i]) if "prefix_lens" in mod else 0
        low, last = mod_ref.visible_range(L, r1 - r0, r0, mod.get("window_left", -1), mod.get("key_start"), prefix)
        key, pos = torch.arange(L), torch.arange(L - (r1 - r0), L)
        seen = (key[None] >= low[:, None]) & (key[None] <= last[:, None])
        for h in range(hq):
            q, kk = b.q[r0:r1, h].cpu().to(f), k[:, h // (hq // b.hkv)].cpu()
            z = q @ kk.T * b.scale
            e = q.abs() @ kk.abs().T * b.scale * 2.0 ** -18
            if mod.get("softcap"):
                z = mod["softcap"] * torch.tanh(z / mod["softcap"])
            e = e + z.abs().clamp(min=1.0) * 2.0 ** -20
            if "alibi_slopes" in mod:
                bias = float(mod["alibi_slopes"][h]) * (pos[:, None] - key[None]).abs().to(f)
                z, e = z - bias, e + bias * 2.0 ** -21
            e = e + 2.0 ** -21 + (2.6e-6 if prefill else 0.0)
            z, e = torch.where(seen, z, -math.inf), torch.where(seen, e, 0.0)
            ll = torch.logsumexp(z, -1)
            w = torch.exp(z - torch.where(ll == -math.inf, 0.0, ll)[:, None])
            lse[h, r0:r1] = ll
            tol[h, r0:r1] = ((w * e).sum(-1) + 2.0 ** -20 + ll.abs().nan_to_num(posinf=0.0) * 2.0 ** -21) * 1.01
    return lse, tol


def check(lse, ref):
    want, tol = ref
    lse = lse.cpu().double()
    assert torch.equal(torch.isneginf(lse), torch.isneginf(want))
    fine = ~torch.isneginf(want)
    worst = ((lse - want).abs() - tol)[fine].max()
    assert worst <= 0, f"off by {float((lse - want)[fine].abs().max()):.3e}, {float(worst):.3e} past its bound"


def mods(hq, rows, lens):
    g = torch.Generator().manual_seed(5)
    docs = torch.cat([(torch.arange(n - q, n) // 37 * 37).int() for n, q in zip(lens, rows)])
    return {
        "none": {},
        "cap": dict(softcap=20.0),
        "bias": dict(alibi_slopes=slopes(hq)),
        "window": dict(window_left=50),
        "documents": dict(key_start=docs),
        "prefix": dict(prefix_lens=torch.tensor([n // 3 for n in lens], dtype=torch.int32)),
        "all": dict(softcap=20.0, alibi_slopes=slopes(hq) * 0.3, window_left=150, key_start=(docs - 20).clamp(min=0),
                    prefix_lens=torch.randint(0, 60, (len(lens),), generator=g).int()),
    }


NAMES = ["none", "cap", "bias", "window", "documents", "prefix", "all"]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", NAMES)
def test_prefill_lse(name, dtype):
    rows, lens = [200, 1, 333, 64], [200, 90, 500, 700]
    b = mod_ref.Batch(lens, rows, 8, 2, dtype=dtype, seed=61)
    m = mods(8, rows, lens)[name]
    check(run_prefill(b, m)[1], reference(b, m, True))


@pytest.mark.parametrize("kind", ["16bit", "fp8", "nvfp4"])
@pytest.mark.parametrize("name", NAMES)
def test_decode_lse(name, kind):
    lens = [1, 17, 300, 1025, 4000]
    b = mod_ref.Batch(lens, [1] * 5, 8, 2, kind=kind, seed=62)
    m = mods(8, [1] * 5, lens)[name]
    check(run_decode(b, m)[1], reference(b, m, False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["fp8", "nvfp4"])
def test_prefill_lse_over_a_quantized_cache(kind, dtype):
    """Rows of few keys among them, whose sums a coarse exponential of one key in eight would show in."""
    rows, lens = [25, 1, 60, 3, 90], [25, 31, 200, 400, 90]
    b = mod_ref.Batch(lens, rows, 4, 2, dtype=dtype, kind=kind, seed=63)
    k, v, table = ops.dequant_gather(b.kc, b.vc, b.table, b.lens, b.table.shape[1], b.dtype)
    out, lse = torch.empty_like(b.q), torch.empty(4, sum(rows), device="cuda")
    ops.chunked_prefill(b.q, k, v, table, b.lens, b.starts.cuda(), b.scale, out, lse=lse, **b.scales)
    check(lse, reference(b, {}, True))
