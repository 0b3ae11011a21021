"""Plain 64-bit attention with score modifiers, the 4-bit cache format spelled
out element by element, and the error bounds that tests hold the kernels to."""
from __future__ import annotations

import math

import torch

D = 128
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def half_step(dtype) -> float:
    """Largest relative error of rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------- 4-bit cache

def quantize_nvfp4(x: torch.Tensor, g: float):
    """x [..., 128] (16-bit) -> (values [..., 128] without the tensor's scale g, block scales [..., 8]), float64.

    The definition with the roundings it names: 6 g, the block's quotient,
    scale * g and each element's quotient rounded to fp32; e4m3 and e2m1 to the
    nearest code, ties to even, saturating."""
    f32 = torch.float32
    b = x.to(f32).unflatten(-1, (8, 16))
    g32 = torch.tensor(g, dtype=f32, device=x.device)
    nan = b.isnan().any(-1)
    amax = b.abs().nan_to_num(nan=0.0, posinf=math.inf).amax(-1)
    s = (amax / (6.0 * g32)).clamp(max=448.0).to(torch.float8_e4m3fn).to(f32)
    d = s * g32
    ok = (d > 0) & ~nan
    r = torch.where(ok[..., None], b / torch.where(ok, d, torch.ones_like(d))[..., None], torch.zeros_like(b)).double()
    # nearest e2m1 by distance, ties to the even code
    a = r.abs().clamp(max=6.0)
    lv = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    dist = (a[..., None] - lv).abs()
    best = dist.amin(-1, keepdim=True)
    even = torch.tensor([0, 1] * 4, device=x.device)
    code = torch.where(dist == best, even, 9).argmin(-1)
    v = torch.where(r < 0, -lv[code], lv[code])
    s = torch.where(nan, torch.full_like(s, math.nan), s).double()
    return v.flatten(-2), s


def nvfp4_values(x: torch.Tensor, g: float) -> torch.Tensor:
    """What a 4-bit cache holds for rows x under the tensor's scale g, float64."""
    v, s = quantize_nvfp4(x, g)
    return (v.unflatten(-1, (8, 16)) * s[..., None]).flatten(-2) * float(torch.tensor(g, dtype=torch.float32))


def decode_tiles(cache: torch.Tensor, value: bool) -> torch.Tensor:
    """Values [num_blocks, bs, H, 128] of a cache half [num_blocks, H, bs, 72], without the tensor's scale."""
    nb, H, bs, _ = cache.shape
    tile = cache.reshape(nb, H, bs // 16, 1152)
    out = torch.empty(nb, H, bs // 16, 16, D, dtype=torch.float64, device=cache.device)
    lv = torch.tensor(LEVELS + tuple(-x for x in LEVELS), dtype=torch.float64, device=cache.device)
    for r in range(16):
        for d in range(0, D, 2):
            if value:
                m, g, i = d // 64, (d % 64) // 8, d % 8
                byte = m * 512 + (4 * g + (r % 8) // 2) * 16 + (r // 8) * 8 + (r % 2) * 4 + i // 2
                k = d // 16
                so = 1024 + (k % 4) * 32 + ((r % 8) // 2) * 8 + (k // 4) * 4 + (r // 8) * 2 + r % 2
            else:
                byte, so = r * 64 + d // 2, 1024 + r * 8 + d // 16
            s = tile[..., so].contiguous().view(torch.float8_e4m3fn).double()
            b = tile[..., byte].long()
            out[..., r, d] = lv[b & 15] * s
            out[..., r, d + 1] = lv[b >> 4] * s
    return out.permute(0, 2, 3, 1, 4).reshape(nb, bs, H, D).contiguous()


# ---------------------------------------------------------------- attention

def visible_range(L, qlen, start_row, window_left=-1, key_start=None, prefix=0):
    """(low, last) of each row, int64 tensors [qlen] (last inclusive)."""
    pos = torch.arange(L - qlen, L)
    low = torch.zeros_like(pos)
    if window_left >= 0:
        low = torch.maximum(low, pos - window_left)
    if key_start is not None:
        low = torch.maximum(low, key_start[start_row:start_row + qlen].cpu().long())
    last = torch.maximum(pos, torch.full_like(pos, min(prefix, L) - 1))
    return low, last


def attention(q, ks, vs, starts, scale, mod=None, p_dtype=None, prefill=False):
    """q [T, Hq, 128]; ks, vs: each sequence's [L, Hkv, 128] (float64, any device); starts [B + 1].

    Returns (out, lse, tolerance of out, tolerance of lse), all float64 on the
    CPU.  The tolerance of out is h |out| + (h_p + 2 e) sum_j p_j |v_j| with h
    the output's half step, h_p that of the type the weights are rounded to,
    and e the error of a score (fp32 products and sums, exp and reciprocal
    approximations of 2^-22, cubic exponentials of 7.5e-5 in the prefill);
    the weights' sum has no rounding, so h_p counts once."""
    mod = mod or {}
    T, hq, _ = q.shape
    f = torch.float64
    out = torch.zeros(T, hq, D, dtype=f)
    lse = torch.full((hq, T), -math.inf, dtype=f)
    otol = torch.zeros(T, hq, D, dtype=f)
    ltol = torch.zeros(hq, T, dtype=f)
    h, hp = half_step(q.dtype), half_step(p_dtype or q.dtype)
    starts = [int(x) for x in starts]
    cap = mod.get("softcap", 0.0)
    for b, (k, v) in enumerate(zip(ks, vs)):
        r0, r1 = starts[b], starts[b + 1]
        n = r1 - r0
        if n == 0 or k.shape[0] == 0:
            continue
        L, hkv = k.shape[0], k.shape[1]
        prefix = int(mod["prefix_lens"][b]) if mod.get("prefix_lens") is not None else 0
        low, last = visible_range(L, n, r0, mod.get("window_left", -1), mod.get("key_start"), prefix)
        key = torch.arange(L)
        seen = (key[None] >= low[:, None]) & (key[None] <= last[:, None])
        for hh in range(hq):
            kk, vv = k[:, hh // (hq // hkv)].cpu().to(f), v[:, hh // (hq // hkv)].cpu().to(f)
            qq = q[r0:r1, hh].cpu().to(f)
            z = qq @ kk.T * scale
            # 128 products summed in fp32: each partial sum is off by 2^-23 at most
            e = torch.where(seen, qq.abs() @ kk.abs().T * scale * 2.0 ** -17, 0.0).nan_to_num(0.0).amax(-1, keepdim=True)
            if cap > 0:
                z = cap * torch.tanh(z / cap)
                e = e + cap * 2.0 ** -20
            if mod.get("alibi_slopes") is not None:
                pos = torch.arange(L - n, L)
                bias = float(mod["alibi_slopes"][hh]) * (pos[:, None] - key[None]).abs().to(f)
                z = z - bias
                # only scores near the row's maximum count: their bias is below 2^7
                e = e + 2.0 ** -16
            z = torch.where(seen, z, -math.inf)
            e = e + 2.0 ** -19 * (1 + torch.where(seen, z.abs(), 0.0).clamp(max=64.0).amax(-1, keepdim=True))
            if prefill:
                e = e + 7.5e-5
            ll = torch.logsumexp(z, -1)
            w = torch.where(seen, torch.exp(z - torch.where(ll == -math.inf, 0.0, ll)[:, None]), 0.0)
            vz = torch.where(seen.any(0)[:, None], vv, 0.0)
            o = w @ vz
            out[r0:r1, hh] = o
            lse[hh, r0:r1] = ll
            otol[r0:r1, hh] = (h * o.abs() + (hp + 2 * e) * (w @ vz.abs())) * 1.01 + 1e-7
            ltol[hh, r0:r1] = (e[:, 0] + 2.0 ** -20) * 1.01 + 1e-6
    return out, lse, otol, ltol


def check(out, lse, ref):
    ro, rl, otol, ltol = ref
    out, lse = out.detach().cpu().double(), lse.detach().cpu().double()
    assert torch.isfinite(out).all(), "non-finite output"
    bad = (out - ro).abs() - otol
    assert bad.max() <= 0, f"output off by {float((out - ro).abs().flatten()[bad.argmax()]):.3e}, " \
                           f"tolerance {float(otol.flatten()[bad.argmax()]):.3e}"
    assert torch.equal(torch.isneginf(lse), torch.isneginf(rl)), "LSE -inf pattern differs"
    fine = ~torch.isneginf(rl)
    d = (lse - rl)[fine].abs() - ltol[fine]
    assert d.numel() == 0 or d.max() <= 0, f"LSE off by {float((lse - rl)[fine].abs().max()):.3e}"


# ---------------------------------------------------------------- batches

class Batch:
    """Random rows in a paged pool whose unused slots and blocks hold NaN.

    kind: "16bit", "fp8" or "nvfp4".  ks / vs: what the cache holds for each
    sequence, float64, the tensors' scales included."""

    def __init__(self, lens, qlens, hq, hkv, dtype=torch.bfloat16, bs=16, kind="16bit", seed=0, device="cuda",
                 spread=1.0):
        from ps_attn import ops

        g = torch.Generator().manual_seed(seed)
        self.lens_list, self.qlens = list(lens), list(qlens)
        B, T = len(lens), sum(qlens)
        pages = [(n + bs - 1) // bs for n in lens]
        nb = sum(pages) + 3
        perm = torch.randperm(nb, generator=g)
        width = max(max(pages), 1)
        table = torch.full((B, width), -1, dtype=torch.int32)  # entries past a sequence are invalid
        k16 = torch.full((nb, bs, hkv, D), math.nan).to(dtype)
        v16 = torch.full((nb, bs, hkv, D), math.nan).to(dtype)
        self.kind, self.dtype, self.bs, self.hq, self.hkv = kind, dtype, bs, hq, hkv
        self.gk, self.gv = (1.0, 1.0) if kind == "16bit" else (0.043, 0.037)
        slots, rows_k, rows_v, c = [], [], [], 0
        self.ks, self.vs = [], []
        for b, n in enumerate(lens):
            ids = perm[c:c + pages[b]]
            c += pages[b]
            table[b, :pages[b]] = ids.int()
            k = (torch.randn(n, hkv, D, generator=g) * spread).to(dtype)
            v = torch.randn(n, hkv, D, generator=g).to(dtype)
            at = torch.arange(n)
            slot = ids[at // bs] * bs + at % bs
            slots.append(slot)
            rows_k.append(k)
            rows_v.append(v)
            k16.view(nb * bs, hkv, D)[slot] = k
            v16.view(nb * bs, hkv, D)[slot] = v
            self.ks.append(self._held(k, self.gk))
            self.vs.append(self._held(v, self.gv))
        dev = torch.device(device)
        self.slots = torch.cat(slots) if slots else torch.zeros(0, dtype=torch.int64)
        self.rows_k, self.rows_v = torch.cat(rows_k), torch.cat(rows_v)
        self.table = table.to(dev)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=dev)
        self.starts = torch.tensor([0] + list(qlens)).cumsum(0).int()
        self.q = torch.randn(T, hq, D, generator=g).to(dtype).to(dev)
        self.scale = 1.0 / math.sqrt(D)
        self.scales = {}
        if kind != "16bit":
            self.scales = dict(k_scale=torch.tensor([self.gk], device=dev), v_scale=torch.tensor([self.gv], device=dev))
        if kind == "nvfp4":
            shape = ops.nvfp4_cache_shape(nb, bs, hkv)
            # 0x7f: a NaN block scale in every slot nothing was written to
            self.kc = torch.full(shape, 0x7F, dtype=torch.uint8, device=dev)
            self.vc = torch.full(shape, 0x7F, dtype=torch.uint8, device=dev)
        elif kind == "fp8":
            self.kc = torch.full((nb, bs, hkv, D), 0x7F, dtype=torch.uint8, device=dev)
            self.vc = torch.full((nb, bs, hkv, D), 0x7F, dtype=torch.uint8, device=dev)
        else:
            self.kc, self.vc = k16.to(dev), v16.to(dev)
        if kind != "16bit" and len(self.slots):
            ops.kv_append(self.rows_k.to(dev), self.rows_v.to(dev), self.kc, self.vc, self.slots.to(dev),
                          **self.scales)

    def _held(self, x, g):
        if self.kind == "16bit":
            return x.double()
        if self.kind == "nvfp4":
            return nvfp4_values(x, g)
        g32 = torch.tensor(g, dtype=torch.float32)
        q = (x.float() / g32).clamp(-448, 448).to(torch.float8_e4m3fn).double()
        return q * float(g32)

    @property
    def p_dtype(self):
        return self.dtype if self.kind == "16bit" else torch.float16

    def reference(self, mod=None, prefill=False):
        return attention(self.q, self.ks, self.vs, self.starts, self.scale, mod, self.p_dtype, prefill)
