"""What the measured operators compute, on what inputs, and how a user calls them.

Two families that an inference server needs beside plain paged attention:

* a KV cache held in 4 bits ("nvfp4": e2m1 codes, one e4m3 scale per 16
  elements, one fp32 scale per tensor): appending rows and reading them back
  (``store``), decode attention over it (``fp4_decode``) and chunked prefill
  over it (``fp4_prefill``);
* attention whose scores are capped by a tanh, get a bias that falls with the
  distance, or are masked by a sliding window, a document start or a
  bidirectional prefix: decode (``mod_decode``) and chunked prefill
  (``mod_prefill``) over a 16-bit paged cache.

``own = False`` computes each operator from elementary torch operations in
32 bits; ``own = True`` calls the framework.
"""
import math

import torch

own = False

D = 128        # head size
PAGE = 16      # tokens of a cache page
ROW = 72       # bytes of a token's 4-bit row of one head: 64 of codes, 8 of scales
TILE = PAGE * ROW
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # magnitudes of an e2m1 code


# ---------------------------------------------------------------- cases

def _lengths(case):
    """Tokens cached for each sequence, new ones included: spread over the logarithm."""
    g = torch.Generator().manual_seed(case["lens_seed"])
    u = torch.rand(case["seqs"], generator=g, dtype=torch.float64)
    lo, hi = math.log(case["len_min"]), math.log(case["len_max"] + 1)
    return [min(case["len_max"], int(math.exp(lo + x * (hi - lo)))) for x in u.tolist()]


def _queries(case):
    """New tokens of each sequence."""
    lens = _lengths(case)
    return [min(case.get("new", 1), n) for n in lens]


def listed():
    # sizes: the framework's own configurations (16/8, 32/8 and 64/8 heads, 16-token
    # blocks, contexts of 1k to 32k, chunks of 2048), and odd ones beside them
    c = []

    def add(name, op, **kw):
        d = dict(name=name, op=op, dtype="bf16", block=16, lens_seed=len(c) + 1)
        d.update(kw)
        c.append(d)

    # a decode step's new tokens, one per sequence: latency
    add("store_step_256", "store", seqs=256, len_min=16, len_max=16, new=1, hkv=8)
    # eight prompts of one prefill step, odd lengths
    add("store_prompts_16k", "store", seqs=8, len_min=1801, len_max=2311, new=2311, hkv=8, dtype="fp16")
    # one chat turn answered alone: latency of a single short sequence
    add("fp4_decode_one", "fp4_decode", seqs=1, len_min=1531, len_max=1531, hq=16, hkv=8)
    # a batch of ordinary chats
    add("fp4_decode_64", "fp4_decode", seqs=64, len_min=1024, len_max=4096, hq=16, hkv=8)
    # long reasoning rollouts of a large model
    add("fp4_decode_long", "fp4_decode", seqs=40, len_min=2048, len_max=32768, hq=64, hkv=8)
    # chunks of prompts that continue a cached context
    add("fp4_prefill_chunks", "fp4_prefill", seqs=4, len_min=3001, len_max=6001, new=1024, hq=32, hkv=8)
    # many short follow-up turns, odd lengths, wide cache blocks
    add("fp4_prefill_turns", "fp4_prefill", seqs=24, len_min=129, len_max=1999, new=77, hq=16, hkv=8,
        dtype="fp16", block=32)
    # a sliding-window layer with capped scores over long contexts: only the window is read
    add("window_cap_decode", "mod_decode", seqs=64, len_min=1024, len_max=16384, hq=32, hkv=8,
        window=1023, cap=50.0)
    # a distance-biased model without shared heads, long contexts
    add("bias_decode_long", "mod_decode", seqs=16, len_min=2048, len_max=32768, hq=16, hkv=16, bias=True,
        dtype="fp16")
    # capped scores with a sliding window over prompts
    add("window_cap_prefill", "mod_prefill", seqs=4, len_min=2501, len_max=4096, new=4096, hq=32, hkv=8,
        window=1023, cap=50.0)
    # the same kind of prompts under a distance bias
    add("bias_prefill", "mod_prefill", seqs=2, len_min=4001, len_max=4096, new=2048, hq=16, hkv=16, bias=True,
        dtype="fp16")
    # packed documents behind a bidirectional prefix (an image or an instruction)
    add("prefix_docs_prefill", "mod_prefill", seqs=6, len_min=1501, len_max=3500, new=3500, hq=32, hkv=8,
        docs=3, prefix=301)
    return c


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["store", "fp4_decode", "fp4_prefill", "mod_decode", "mod_prefill"])
    hkv = rng.choice([1, 2, 4, 8])
    c = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), block=rng.choice([16, 32, 64]),
             lens_seed=rng.randrange(1 << 30), hkv=hkv, hq=hkv * rng.choice([1, 2, 4, 5, 8, 16]))
    if op == "store":
        c.update(seqs=log(1, 256))
        hi = log(1, max(1, 16384 // c["seqs"]))
        c.update(len_min=max(1, hi // 3), len_max=hi, new=log(1, hi))
    elif op in ("fp4_decode", "mod_decode"):
        c.update(seqs=log(1, 64))
        hi = log(16, min(32768, 196608 // c["seqs"]))
        c.update(len_min=log(1, hi), len_max=hi)
    else:
        c.update(seqs=log(1, 8), hq=hkv * rng.choice([1, 2, 4]))
        hi = log(16, 4096)
        most = int(1.2e10 / (c["seqs"] * c["hq"] * hi * 8))  # the largest listed case's pairs of rows and keys
        c.update(len_min=max(1, hi // 2), len_max=hi, new=log(2, max(2, min(hi, 2048, most))))
    if op.startswith("mod"):
        kind = rng.choice(["cap", "bias", "window", "docs"])
        if kind == "cap" or rng.random() < 0.3:
            c["cap"] = float(rng.choice([5, 15, 30, 50]))
        if kind == "bias":
            c["bias"] = True
        if kind == "window" or rng.random() < 0.3:
            c["window"] = log(1, 4096)
        if kind == "docs":
            c["docs"] = rng.choice([1, 2, 5])
        if op == "mod_prefill" and rng.random() < 0.3:
            c["prefix"] = log(1, hi)
    return c


# ---------------------------------------------------------------- inputs

def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _quantize(x, g):
    """x [..., 128] -> (codes 0..15 [..., 128] uint8, block scales [..., 8] e4m3) under the tensor's scale g:
    scale = e4m3(max|x| / (6 g)), code = e2m1(x / (scale * g)), both to nearest, ties to even."""
    b = x.float().unflatten(-1, (8, 16))
    s = (b.abs().amax(-1) / (6.0 * g)).clamp(max=448.0).to(torch.float8_e4m3fn)
    d = s.float() * g
    r = torch.where(d[..., None] > 0, b / d[..., None], torch.zeros_like(b))
    a = r.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5)
            + (a > 5.0)).to(torch.uint8)
    code |= (torch.signbit(r).to(torch.uint8) << 3)
    return code.flatten(-2), s


def _pack(codes, scales, value):
    """codes [NB, bs, H, 128], scales [NB, bs, H, 8] -> cache [NB, H, bs, 72] of one 1152-byte tile per 16 tokens."""
    NB, bs, H, _ = codes.shape
    c = codes.view(NB, bs // PAGE, PAGE, H, D).permute(0, 3, 1, 2, 4)      # [NB, H, P, 16, 128]
    s = scales.view(torch.uint8).view(NB, bs // PAGE, PAGE, H, 8).permute(0, 3, 1, 2, 4)
    if value:
        # token = 8a + 2t + e, dim = 64m + 8g + i: 4-byte words in the order [m][g][t][a][e], the nibbles of
        # i in order; scale block = 4m + k in the order [k][t][m][a][e]
        c = c.reshape(NB, H, bs // PAGE, 2, 4, 2, 2, 8, 8).permute(0, 1, 2, 6, 7, 4, 3, 5, 8)
        s = s.reshape(NB, H, bs // PAGE, 2, 4, 2, 2, 4).permute(0, 1, 2, 7, 4, 6, 3, 5)
    c = c.reshape(NB, H, bs // PAGE, PAGE * D // 2, 2)
    c = c[..., 0] | (c[..., 1] << 4)
    s = s.reshape(NB, H, bs // PAGE, PAGE * 8)
    return torch.cat([c, s], -1).reshape(NB, H, bs, ROW).contiguous()


def _unpack(tiles, value):
    """tiles uint8 [..., 1152] -> (values of the codes [..., 16, 128], block scales [..., 16, 8]), fp32."""
    lead = tiles.shape[:-1]
    c, s = tiles[..., :PAGE * D // 2], tiles[..., PAGE * D // 2:]
    level = torch.tensor(LEVELS + tuple(-x for x in LEVELS), device=tiles.device)
    c = torch.stack([c & 15, c >> 4], -1)
    s = s.contiguous().view(torch.float8_e4m3fn).float()
    if value:
        n = len(lead)
        ax = list(range(n))
        c = c.reshape(*lead, 2, 8, 4, 2, 2, 8).permute(*ax, n + 3, n + 2, n + 4, n, n + 1, n + 5)
        s = s.reshape(*lead, 4, 4, 2, 2, 2).permute(*ax, n + 3, n + 1, n + 4, n + 2, n)
    return level[c.reshape(*lead, PAGE, D).int()], s.reshape(*lead, PAGE, 8)


def _slopes(hq, device):
    """The bias' slope for each head: 2^(-8 (h + 1) / hq)."""
    return torch.exp2(-8.0 * torch.arange(1, hq + 1, device=device, dtype=torch.float32) / hq)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, bs, hkv = _dtype(case), case["block"], case["hkv"]
    lens, new = _lengths(case), _queries(case)
    B, T = len(lens), sum(new)
    blocks = [(n + bs - 1) // bs for n in lens]
    nb, width = sum(blocks) + 8, max(blocks)
    order = torch.randperm(nb, generator=g, device=dev).int()
    first = torch.tensor([0] + blocks).cumsum(0)[:-1].to(dev)
    count = torch.tensor(blocks, device=dev)
    col = torch.arange(width, device=dev)
    table = torch.where(col[None] < count[:, None], order[(first[:, None] + col[None]).clamp(max=nb - 1)], 0).int()
    st = dict(case=case, table=table.contiguous(), lens=torch.tensor(lens, dtype=torch.int32, device=dev),
              starts=torch.tensor([0] + new).cumsum(0).int().to(dev), width=width, longest=max(lens),
              rows=max(new), scale=1.0 / math.sqrt(D))
    four = case["op"] in ("store", "fp4_decode", "fp4_prefill")
    if four:
        # a channel-wise spread as keys have it, and a per-tensor scale that uses the whole e4m3 range
        spread = torch.exp2(torch.randn(2, 1, 1, hkv, D, generator=g, device=dev) * 0.5)
        st["k_scale"] = torch.tensor([0.0037], device=dev)
        st["v_scale"] = torch.tensor([0.0041], device=dev)
        cache = []
        for i, s in enumerate((st["k_scale"], st["v_scale"])):
            parts = []
            for n in torch.split(torch.arange(nb), max(1, (1 << 26) // (bs * hkv * D))):
                x = torch.randn(len(n), bs, hkv, D, generator=g, device=dev) * spread[i]
                parts.append(_pack(*_quantize(x.to(dt), s), value=i == 1))
            cache.append(torch.cat(parts))
        st["kc"], st["vc"] = cache
    else:
        st["kc"] = torch.randn(nb, bs, hkv, D, generator=g, device=dev, dtype=dt)
        st["vc"] = torch.randn(nb, bs, hkv, D, generator=g, device=dev, dtype=dt)
    # the new tokens, flat: the sequence and the position of each
    seq = torch.repeat_interleave(torch.arange(B), torch.tensor(new))
    pos = torch.tensor(lens)[seq] - torch.tensor(new)[seq] + torch.arange(T) - torch.tensor([0] + new).cumsum(0)[seq]
    st["seq"], st["pos"] = seq.to(dev), pos.to(dev)
    if case["op"] == "store":
        st["key"] = (torch.randn(T, hkv, D, generator=g, device=dev) * spread[0, 0]).to(dt)
        st["value"] = (torch.randn(T, hkv, D, generator=g, device=dev) * spread[1, 0]).to(dt)
        st["slots"] = table[st["seq"], st["pos"] // bs].long() * bs + st["pos"] % bs
        st["scratch"] = [torch.zeros(B * width, bs, hkv, D, dtype=dt, device=dev) for _ in range(2)]
        return st
    hq = case["hq"]
    st["q"] = torch.randn(T, hq, D, generator=g, device=dev, dtype=dt)
    st["out"] = torch.empty_like(st["q"])
    st["lse"] = torch.empty(hq, T, dtype=torch.float32, device=dev)
    if case.get("bias"):
        st["slopes"] = _slopes(hq, dev)
    if case.get("docs"):
        # the first key of each row's document: the sequence cut at drawn places
        cuts = (torch.rand(B, case["docs"], generator=g, device=dev) * st["lens"][:, None]).int()
        at = torch.where(cuts[st["seq"]] <= st["pos"][:, None], cuts[st["seq"]], 0).amax(-1)
        if case.get("prefix"):
            at = torch.where(st["pos"] < case["prefix"], 0, at)
        st["key_start"] = at.int().contiguous()
    if case.get("prefix"):
        st["prefix"] = torch.full((B,), case["prefix"], dtype=torch.int32, device=dev)
    return st


# ---------------------------------------------------------------- one pass

def run(st):
    if own:
        return _own(st)
    case = st["case"]
    if case["op"] == "store":
        return _plain_store(st)
    tables = st["table"].long()
    if case["op"].startswith("fp4"):
        kv = []
        for cache, scale, value in ((st["kc"], st["k_scale"], False), (st["vc"], st["v_scale"], True)):
            pages = cache.flatten(2).unflatten(2, (-1, TILE)).transpose(1, 2)[tables]  # [B, W, P, H, 1152]
            x, s = _unpack(pages, value)
            x = (x.unflatten(-1, (8, 16)) * s[..., None]).flatten(-2) * scale     # [B, W, P, H, 16, 128]
            kv.append(x.transpose(3, 4).flatten(1, 3))                            # [B, L, H, 128]
        return _plain_attention(st, *kv)
    return _plain_attention(st, st["kc"][tables].flatten(1, 2).float(), st["vc"][tables].flatten(1, 2).float())


def _plain_store(st):
    outs = []
    bs, dt = st["case"]["block"], _dtype(st["case"])
    used = torch.arange(st["width"], device=st["lens"].device)[None] * bs < st["lens"][:, None]
    for cache, rows, scale, value in ((st["kc"], st["key"], st["k_scale"], False),
                                      (st["vc"], st["value"], st["v_scale"], True)):
        tiles = cache.flatten(2).unflatten(2, (-1, TILE))[st["table"].long()]     # [B, W, H, P, 1152]
        x, s = _unpack(tiles, value)
        x = (x.unflatten(-1, (8, 16)) * s[..., None]).flatten(-2) * scale
        x = x.flatten(3, 4).transpose(2, 3).to(dt)                                # [B, W, bs, H, 128]
        codes, s = _quantize(rows, scale)
        level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=rows.device)
        y = ((level[codes.int()].unflatten(-1, (8, 16)) * s.float()[..., None]).flatten(-2) * scale).to(dt)
        x[st["seq"], st["pos"] // bs, st["pos"] % bs] = y
        outs.append(torch.where(used[:, :, None, None, None], x, 0).flatten(0, 1))
    return outs


def _plain_attention(st, k, v):
    """softmax(bias(cap(q k^T scale))) v over the visible keys of each row; k, v [B, L, Hkv, 128] fp32."""
    case, q, B = st["case"], st["q"], st["lens"].shape[0]
    T, hq, _ = q.shape
    hkv, L = k.shape[2], k.shape[1]
    at = torch.arange(T, device=q.device) - st["starts"].long()[st["seq"]]
    qp = q.new_zeros(B, st["rows"], hq, D, dtype=torch.float32)
    qp[st["seq"], at] = q.float()
    qp = qp.unflatten(2, (hkv, hq // hkv)).permute(0, 2, 3, 1, 4).flatten(2, 3)          # [B, Hkv, G*R, 128]
    s = (qp @ k.permute(0, 2, 3, 1)).unflatten(2, (hq // hkv, st["rows"])) * st["scale"]  # [B, Hkv, G, R, L]
    if case.get("cap"):
        s = case["cap"] * torch.tanh(s / case["cap"])
    key = torch.arange(L, device=q.device)
    pos = torch.full((B, st["rows"]), -1, device=q.device)
    pos[st["seq"], at] = st["pos"]
    if case.get("bias"):
        far = (key[None, None] - pos[..., None]).abs().float()                           # [B, R, L]
        s = s - st["slopes"].view(1, hkv, hq // hkv, 1, 1) * far[:, None, None]
    last, low = pos, torch.zeros_like(pos)
    if case.get("prefix"):
        last = torch.maximum(pos, torch.minimum(st["prefix"], st["lens"]).long()[:, None] - 1)
    if case.get("window"):
        low = pos - case["window"]
    if case.get("docs"):
        first = torch.zeros_like(pos)
        first[st["seq"], at] = st["key_start"].long()
        low = torch.maximum(low, first)
    seen = (key >= low[..., None]) & (key <= last[..., None]) & (key < st["lens"][:, None, None])
    s = s.masked_fill(~seen[:, None, None], -torch.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -torch.inf, 0.0, m)
    p = torch.exp(s - m)
    l = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v.transpose(1, 2)).unflatten(2, (hq // hkv, st["rows"]))
    o = torch.where(l > 0, o / l, 0.0)
    lse = (m + torch.log(l))[..., 0]
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[st["seq"], at].to(q.dtype)
    return [o, lse.permute(0, 3, 1, 2).flatten(2, 3)[st["seq"], at].T.contiguous()]


def _own(st):
    import sys
    from pathlib import Path

    here = str(Path(__file__).resolve().parent.parent / "prime-rl_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    from ps_attn import ops

    case = st["case"]
    op = case["op"]
    if op == "store":
        sc = dict(k_scale=st["k_scale"], v_scale=st["v_scale"])
        ops.kv_append(st["key"], st["value"], st["kc"], st["vc"], st["slots"], **sc)
        k, v, _ = ops.dequant_gather(st["kc"], st["vc"], st["table"], st["lens"], st["width"], _dtype(case),
                                     out=tuple(st["scratch"]), **sc)
        return [k, v]
    q, out, lse = st["q"], st["out"], st["lse"]
    ws = ops.get_workspace(st["lens"].shape[0], q.shape[1], case["hkv"], D, q.device)
    args = dict(lse=lse, query_start_loc=st["starts"], workspace=ws)
    mod = None
    if op.startswith("mod"):
        mod = ops.ScoreMod(softcap=case.get("cap", 0.0), alibi_slopes=st.get("slopes"),
                           window_left=case.get("window", -1), key_start=st.get("key_start"),
                           prefix_lens=st.get("prefix"))
        args["score_mod"] = mod
    if op == "fp4_decode":
        args.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    if op in ("fp4_decode", "mod_decode"):
        ops.paged_decode(q, st["kc"], st["vc"], st["table"], st["lens"], st["scale"], out, **args)
        return [out, lse]
    kc, vc, table = st["kc"], st["vc"], st["table"]
    if op == "fp4_prefill":
        # the 16-bit prefill reads the 4-bit pages' values; the tensors' scales go into its scores and outputs
        kc, vc, table = ops.dequant_gather(kc, vc, table, st["lens"], st["width"], q.dtype)
        args.update(k_scale=st["k_scale"], v_scale=st["v_scale"])
    starts = args.pop("query_start_loc")
    ops.chunked_prefill(q, kc, vc, table, st["lens"], starts, st["scale"], out, **args)
    return [out, lse]


# ---------------------------------------------------------------- what it cannot do without

def _visible(case):
    """For each sequence: the pairs of (row, key) that a mask can leave (documents, whose cuts are drawn with the
    inputs, count as if they cut nothing), the distinct keys that some row sees, and its rows."""
    got = []
    for n, new in zip(_lengths(case), _queries(case)):
        w = case.get("window", n)
        pos = torch.arange(n - new, n)
        low = (pos - w).clamp(min=0)
        last = torch.maximum(pos, torch.full_like(pos, min(case.get("prefix", 0), n) - 1))
        got.append((int((last - low + 1).sum()), int(last.max() - low.min()) + 1, new))
    return got


def _docs_share(case):
    """The expected share of pairs that documents leave: a row at x of a sequence cut at d uniform places starts
    (x - its last cut) back, so it keeps (1 - (1 - x)^(d + 1)) / ((d + 1) x) of its keys; averaged over pairs."""
    d = case.get("docs", 0)
    if not d:
        return 1.0
    if case["op"] == "mod_decode":
        return 1.0 / (d + 1)
    x = torch.linspace(0.0005, 0.9995, 1000, dtype=torch.float64)
    kept = (1 - (1 - x) ** (d + 1)) / (d + 1)
    return float(kept.mean() / x.mean())


def work(case):
    hkv, hq, B = case["hkv"], case.get("hq", 0), case["seqs"]
    if case["op"] == "store":
        lens, new = _lengths(case), _queries(case)
        rows = sum(new) * hkv
        held = sum((n + case["block"] - 1) // case["block"] * case["block"] for n in lens) * hkv
        # rows in, their codes out, the pages' codes in, their values out; keys and values
        return {"bytes": 2 * (rows * (2 * D + ROW) + held * (ROW + 2 * D)) + sum(new) * 8, "flops": 2 * rows * D * 4}
    pairs = [sum(x) for x in zip(*_visible(case))]
    share = _docs_share(case)
    row = ROW if case["op"].startswith("fp4") else 2 * D
    keys = pairs[1]
    if case["op"] == "mod_decode":
        keys = int(keys * share)
    T = pairs[2]
    return {"bytes": keys * hkv * 2 * row + T * hq * (4 * D + 4) + B * 12 + keys // case["block"] * 4,
            "flops": 4 * int(pairs[0] * share) * hq * D}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    cost = sum(p for p, _, _ in _visible(case)) * case.get("hq", 1)
    if cost > 4e10:
        return None
    st = prepare(case, seed)
    f = torch.float64
    if case["op"] == "store":
        return _exact_store(case, st, f)
    hq, hkv, bs = case["hq"], case["hkv"], case["block"]
    group = hq // hkv
    lens, new = _lengths(case), _queries(case)
    outs, lses, t0 = [], [], 0
    for b, (n, m) in enumerate(zip(lens, new)):
        blocks = st["table"][b, :(n + bs - 1) // bs].long()
        if case["op"].startswith("fp4"):
            k = _exact_rows(st["kc"][blocks], False, bs, f)[:n] * st["k_scale"].to(f)
            v = _exact_rows(st["vc"][blocks], True, bs, f)[:n] * st["v_scale"].to(f)
        else:
            k = st["kc"][blocks].flatten(0, 1)[:n].to(f)
            v = st["vc"][blocks].flatten(0, 1)[:n].to(f)
        at = torch.arange(n - m, n, device=k.device)
        key = torch.arange(n, device=k.device)
        low = torch.zeros_like(at)
        if case.get("window"):
            low = at - case["window"]
        if case.get("docs"):
            low = torch.maximum(low, st["key_start"][t0:t0 + m].long())
        last = at.clone()
        if case.get("prefix"):
            last = torch.maximum(last, torch.full_like(last, min(case["prefix"], n) - 1))
        seen = (key[None] >= low[:, None]) & (key[None] <= last[:, None])
        ob, lb = [], []
        for h in range(hq):
            z = st["q"][t0:t0 + m, h].to(f) @ k[:, h // group].T / math.sqrt(D)
            if case.get("cap"):
                z = torch.tanh(z / case["cap"]) * case["cap"]
            if case.get("bias"):
                z = z - st["slopes"][h].to(f) * (at[:, None] - key[None]).abs().to(f)
            z = torch.where(seen, z, -torch.inf)
            lb.append(torch.logsumexp(z, 1))
            w = torch.where(seen, torch.exp(z - torch.where(lb[-1] == -torch.inf, 0.0, lb[-1])[:, None]), 0.0)
            ob.append(w @ v[:, h // group])
        outs.append(torch.stack(ob, 1))
        lses.append(torch.stack(lb))
        t0 += m
    return [torch.cat(outs), torch.cat(lses, 1)]


def _exact_rows(cache, value, bs, f):
    """The rows [tokens, Hkv, 128] that the blocks [n, Hkv, bs, 72] of a 4-bit cache hold, without the tensor's
    scale: every element looked up by its place in the tile."""
    n, H = cache.shape[:2]
    tile = cache.reshape(n, H, bs // PAGE, TILE)
    r = torch.arange(PAGE, device=cache.device)[:, None]
    d = torch.arange(D, device=cache.device)[None]
    if value:
        e = (d // 64) * 512 + ((d % 64) // 8) * 64 + ((r % 8) // 2) * 16 + (r // 8) * 8 + (r % 2) * 4 + (d % 8) // 2
        b = d // 16
        sc = 1024 + (b % 4) * 32 + ((r % 8) // 2) * 8 + (b // 4) * 4 + (r // 8) * 2 + r % 2
    else:
        e = r * 64 + d // 2
        sc = 1024 + r * 8 + d // 16
    byte = tile[..., e].long()
    code = torch.where((d % 2) == 1, byte >> 4, byte & 15)
    mag, ex = code & 1, (code >> 1) & 3
    x = torch.where(ex == 0, mag.to(f) / 2, torch.exp2((ex - 1).to(f)) * (1 + mag.to(f) / 2))
    x = torch.where(code >= 8, -x, x) * tile[..., sc].contiguous().view(torch.float8_e4m3fn).to(f)
    return x.permute(0, 2, 3, 1, 4).reshape(n * bs, H, D)


def _exact_store(case, st, f):
    bs = case["block"]
    got = []
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=f, device=st["lens"].device)
    even = torch.tensor([0, 1, 0, 1, 0, 1, 0], dtype=torch.bool, device=mids.device)   # a tie rounds up at these
    level = torch.tensor(LEVELS, dtype=f, device=mids.device)
    for cache, rows, scale, value in ((st["kc"], st["key"], st["k_scale"], False),
                                      (st["vc"], st["value"], st["v_scale"], True)):
        g = scale.to(f)
        B, W = st["table"].shape
        x = _exact_rows(cache[st["table"].flatten().long()], value, bs, f) * g
        x = x.view(B, W * bs, -1, D)
        z = rows.to(f).unflatten(-1, (8, 16))
        # an e4m3 value near t: three mantissa bits, exponents from -6 on
        t = z.abs().amax(-1) / (6 * g)
        step = torch.exp2(torch.floor(torch.log2(t.clamp(min=2.0 ** -6))) - 3)
        s = (torch.round(t / step) * step).clamp(max=448.0)
        ratio = torch.where(s[..., None] > 0, z / (s[..., None] * g).clamp(min=1e-300), 0.0)
        a = ratio.abs()[..., None]
        code = ((a > mids) | ((a == mids) & even)).sum(-1)
        y = torch.where(ratio < 0, -level[code], level[code]) * (s[..., None] * g)
        x[st["seq"], st["pos"]] = y.flatten(-2)
        used = torch.arange(W, device=x.device)[None] * bs < st["lens"][:, None]
        got.append(torch.where(used[..., None, None, None], x.view(B, W, bs, -1, D), 0.0).flatten(0, 1))
    return got
