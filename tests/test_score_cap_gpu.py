"""GPU: the tanh cap over its whole accepted range.  A capped score has to be as
accurate as the plain one whatever the cap is, so the tolerances here grow with
the scores and not with the cap."""
from __future__ import annotations

import math

import pytest
import torch

import mod_ref
from test_score_mod_gpu import run_decode, run_prefill, to_mod  # noqa: F401  (to_mod: for callers of this module)

pytestmark = pytest.mark.gpu

CAPS = [1e-30, 1e-9, 1e-6, 0.05, 50.0, 1e4, 1e6, 1e30, 1e38]


def capped(b, cap, prefill, window=None):
    """(out, lse, tolerance of out, tolerance of lse) of a batch under a cap, float64.

    Errors of one score z with key k: the product of 128 elements is summed in
    fp32 over at most 9 steps that each lose at most 2^-22 of sum |q| |k|, below
    2^-18 of it; the cap, the scale and the exponent's argument are each a few
    fp32 roundings of a number no larger than max(|z|, 1): 2^-20 of it (the
    exponential form's 2^-22 c is used where |z| >= c tanh(1/2) = 0.46 c).  A
    weight then has that error, 2^-21 of an exponential of 2^-22, and in the
    prefill one of 2.6e-6.  The LSE is off by the weights' mean error, an output
    by that and the errors of its own terms, a weight's rounding to its type
    (half a step, below 2^-14 in f16 an absolute 2^-25 of the largest) and the
    output's."""
    f = torch.float64
    T, hq, _ = b.q.shape
    out, otol = torch.zeros(T, hq, 128, dtype=f), torch.zeros(T, hq, 128, dtype=f)
    lse, ltol = torch.full((hq, T), -math.inf, dtype=f), torch.zeros(hq, T, dtype=f)
    p_dtype = b.dtype if prefill else b.p_dtype
    hp, tiny = mod_ref.half_step(p_dtype), 2.0 ** -25 if p_dtype == torch.float16 else 0.0
    g = hq // b.hkv
    for i, (k, v) in enumerate(zip(b.ks, b.vs)):
        r0, r1, L = int(b.starts[i]), int(b.starts[i + 1]), k.shape[0]
        if r1 == r0 or L == 0:
            continue
        pos, key = torch.arange(L - (r1 - r0), L), torch.arange(L)
        seen = key[None] <= pos[:, None]
        if window is not None:
            seen &= key[None] >= pos[:, None] - window
        for h in range(hq):
            q, kk, vv = b.q[r0:r1, h].cpu().to(f), k[:, h // g].cpu(), v[:, h // g].cpu()
            z = cap * torch.tanh(q @ kk.T * (b.scale / cap))
            e = q.abs() @ kk.abs().T * b.scale * 2.0 ** -18 + z.abs().clamp(min=1.0) * 2.0 ** -20
            e = e + 2.0 ** -21 + (2.6e-6 if prefill else 0.0)
            z = torch.where(seen, z, -math.inf)
            ll = torch.logsumexp(z, -1)
            w = torch.exp(z - ll[:, None])
            e = torch.where(seen, e, 0.0)
            mean = (w * e).sum(-1, keepdim=True)
            o = w @ vv
            top = w.amax(-1, keepdim=True)
            out[r0:r1, h], lse[h, r0:r1] = o, ll
            spread = (w * (e + mean + hp) + torch.where(seen, tiny * top, 0.0)) @ vv.abs()
            otol[r0:r1, h] = (mod_ref.half_step(b.dtype) * o.abs() + spread) * 1.01 + 1e-7
            ltol[h, r0:r1] = (mean[:, 0] + 2.0 ** -20 + ll.abs() * 2.0 ** -21) * 1.01
    return out, lse, otol, ltol


@pytest.mark.parametrize("kind,dtype", [("16bit", torch.bfloat16), ("16bit", torch.float16), ("fp8", torch.bfloat16),
                                        ("nvfp4", torch.float16), ("nvfp4", torch.bfloat16)])
@pytest.mark.parametrize("cap", CAPS)
def test_decode_caps_of_every_size(kind, dtype, cap):
    b = mod_ref.Batch([1, 2, 16, 65, 300, 1000], [1] * 6, 8, 2, dtype=dtype, kind=kind, seed=71, spread=2.0)
    b.q[2] = 0  # scores of exactly zero: the mean of the values
    mod_ref.check(*run_decode(b, dict(softcap=cap)), capped(b, cap, False))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cap", CAPS)
def test_prefill_caps_of_every_size(dtype, cap):
    b = mod_ref.Batch([1, 2, 65, 300], [1, 2, 30, 300], 8, 2, dtype=dtype, seed=73, spread=2.0)
    b.q[1] = 0  # scores of exactly zero, in a warp with others and in warps of their own
    b.q[-150:] = 0
    mod_ref.check(*run_prefill(b, dict(softcap=cap)), capped(b, cap, True))


def one_far_key(kind, cap, qlens, lens):
    """Every sequence's key 5 is far below or above the others for every head of kv head 0 and 1: z of about -0.8
    and 0.8 cap, in the reach of the exponential form, beside ordinary scores."""
    b = mod_ref.Batch(lens, qlens, 2, 2, kind=kind, seed=72)
    b.q[:] = b.q[:1]  # one query for all rows, so that the key is far for each
    q = b.q[0].cpu().double()
    from ps_attn import ops

    for i, n in enumerate(lens):
        sign = -1.0 if i % 2 == 0 else 1.0
        size = (q * q).sum(-1, keepdim=True) * b.scale
        row = (sign * 0.8 * cap * q / size).to(b.dtype)[None]
        at = sum(lens[:i]) + 5
        dev = b.kc.device
        ops.kv_append(row.to(dev), b.rows_v[at:at + 1].to(dev), b.kc, b.vc, b.slots[at:at + 1].to(dev), **b.scales)
        b.ks[i][5] = b._held(row, b.gk)[0]
    return b


@pytest.mark.parametrize("kind", ["16bit", "nvfp4"])
@pytest.mark.parametrize("cap", [1e3, 1e4])
def test_decode_one_far_key(kind, cap):
    """A score far beyond c / 2 leaves the accuracy of the others in its tile alone."""
    b = one_far_key(kind, cap, [1, 1, 1], [40, 50, 300])
    mod_ref.check(*run_decode(b, dict(softcap=cap)), capped(b, cap, False))


@pytest.mark.parametrize("cap", [1e3, 1e4])
def test_prefill_one_far_key(cap):
    b = one_far_key("16bit", cap, [40, 40, 40], [40, 50, 300])
    mod_ref.check(*run_prefill(b, dict(softcap=cap)), capped(b, cap, True))


@pytest.mark.parametrize("window", [None, 40])
def test_prefill_bits_do_not_depend_on_keys_nobody_sees(window):
    """Slots past a sequence, keys below its window and unused blocks hold NaN, then small, then huge values; more
    units than CTAs, handed out dynamically or in turn: the same bits each time."""
    lens = [5 + (i * 29) % 150 for i in range(40)]
    b = mod_ref.Batch(lens, [min(n, 3 + i % 50) for i, n in enumerate(lens)], 16, 8, seed=74, spread=2.0)
    m = dict(softcap=9.0) if window is None else dict(softcap=9.0, window_left=window)
    unused = torch.isnan(b.kc)
    if window is not None:  # keys that no row of their sequence sees
        row = 0
        for i, n in enumerate(lens):
            for slot in b.slots[row:row + max(0, n - b.qlens[i] - window)].tolist():
                unused[slot // b.bs, slot % b.bs] = True
            row += n
    first = run_prefill(b, m)
    for value in (0.01, 3e38, -3e38):
        b.kc, b.vc = b.kc.masked_fill(unused, value), b.vc.masked_fill(unused, value)
        for ws in (True, False, True):
            again = run_prefill(b, m, workspace=ws)
            assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])
    mod_ref.check(*first, capped(b, 9.0, True, window))
