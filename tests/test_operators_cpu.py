"""CPU: refusals, struct layout, bindings and backend routes of the score
modifiers and the 4-bit (nvfp4) cache, and the test reference's own 4-bit format
against hand-computed codes (no kernel is launched here)."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import mod_ref
from ps_attn import _lib, ops
from ps_attn import backend as psb
from ps_attn import torch_ops
from test_abi import _struct_fields


def problem(**kw):
    """A problem that passes the host's checks (fake, aligned pointers)."""
    pr = _lib.PagedProblem()
    for f in ("q", "key_cache", "value_cache", "block_table", "seq_lens", "out", "query_start_loc"):
        setattr(pr, f, 4096)
    pr.num_seqs, pr.dtype, pr.head_size, pr.block_size = 1, _lib.PS_DTYPE_BF16, 128, 16
    pr.num_q_heads, pr.num_kv_heads, pr.num_blocks, pr.num_tokens = 8, 2, 4, 1
    pr.max_blocks_per_seq, pr.block_table_stride = 4, 4
    pr.q_stride_token, pr.q_stride_head = 1024, 128
    pr.out_stride_token, pr.out_stride_head = 1024, 128
    pr.cache_stride_block, pr.cache_stride_slot, pr.cache_stride_head = 16 * 256, 256, 128
    pr.softmax_scale = 0.088
    for k, v in kw.items():
        setattr(pr, k, v)
    return pr


def fp4_problem(**kw):
    base = dict(kv_cache_dtype=_lib.PS_KV_NVFP4, cache_stride_block=2 * 16 * 72, cache_stride_head=16 * 72,
                cache_stride_slot=72)
    base.update(kw)
    return problem(**base)


def passes_host_checks(rc):
    """Past every check of arguments: without a GPU the next step fails on the device, with one on the workspace."""
    return rc in (_lib.PS_ERR_CUDA, _lib.PS_ERR_WORKSPACE)


def test_struct_layout():
    assert _struct_fields("ps_score_mod") == [f for f, _ in _lib.ScoreMod._fields_]
    pr = _lib.PagedProblem.from_buffer_copy(_lib.PAGED_PROBLEM_STRUCT.pack(*range(1, 27), 0.5, *range(28, 40)))
    assert [int(getattr(pr, f) or 0) for f, _ in _lib.PagedProblem._fields_][:26] == list(range(1, 27))
    assert pr.softmax_scale == 0.5 and pr.num_tokens == 28 and pr.v_scale == 39


def test_score_mod_entry_points_refuse_on_the_host():
    lib = _lib.load()
    m = _lib.ScoreMod()
    m.window_left = -1
    for call in (lib.ps_paged_decode_mod, lib.ps_chunked_prefill_mod):
        def go(pr=None, mod=m):
            return call(ctypes.byref(pr) if pr is not None else None, ctypes.byref(mod) if mod is not None else None,
                        None, 0, None)

        assert go(None) == _lib.PS_ERR_INVALID_ARGUMENT
        assert go(problem(), None) == _lib.PS_ERR_INVALID_ARGUMENT and b"NULL" in lib.ps_last_error()
        assert go(problem(head_size=64)) == _lib.PS_ERR_UNSUPPORTED
        for cap in (-1.0, math.nan, math.inf, 1e-44, 3e38):
            bad = _lib.ScoreMod()
            bad.logits_soft_cap, bad.window_left = cap, -1
            assert go(problem(), bad) == _lib.PS_ERR_INVALID_ARGUMENT, cap
        for field in ("alibi_slopes", "key_start", "prefix_lens"):
            bad = _lib.ScoreMod()
            setattr(bad, field, 4098)
            assert go(problem(), bad) == _lib.PS_ERR_INVALID_ARGUMENT and b"aligned" in lib.ps_last_error()
        assert go(problem(num_seqs=0)) == _lib.PS_OK
    assert passes_host_checks(lib.ps_paged_decode_mod(ctypes.byref(problem()), ctypes.byref(m), None, 0, None))


def test_nvfp4_entry_points_refuse_on_the_host():
    lib = _lib.load()
    m = _lib.ScoreMod()
    assert passes_host_checks(lib.ps_paged_decode(ctypes.byref(fp4_problem()), None, 0, None))
    # tiles of 16 tokens are contiguous, blocks and heads apart and 16-byte aligned
    for bad in (dict(cache_stride_slot=80), dict(cache_stride_head=16 * 72 - 16), dict(cache_stride_head=16 * 72 + 8),
                dict(cache_stride_block=2 * 16 * 72 + 8), dict(key_cache=4104)):
        assert lib.ps_paged_decode(ctypes.byref(fp4_problem(**bad)), None, 0, None) == _lib.PS_ERR_INVALID_ARGUMENT
    # one kv head: its stride does not matter
    assert passes_host_checks(lib.ps_paged_decode(
        ctypes.byref(fp4_problem(num_kv_heads=1, cache_stride_head=0)), None, 0, None))
    # entry points without a 4-bit kernel
    pr = fp4_problem()
    assert lib.ps_chunked_prefill(ctypes.byref(pr), None) == _lib.PS_ERR_UNSUPPORTED
    assert lib.ps_chunked_prefill_mod(ctypes.byref(pr), ctypes.byref(m), None, 0, None) == _lib.PS_ERR_UNSUPPORTED
    assert lib.ps_paged_decode_cascade(ctypes.byref(pr), ctypes.c_void_p(4096), 1 << 20, None, 0,
                                       None) == _lib.PS_ERR_UNSUPPORTED
    hp = _lib.HeadGatherProblem()
    hp.world, hp.rank, hp.num_tokens, hp.hq_local, hp.max_tokens = 2, 1, 4, 8, 8
    hp.dtype = _lib.PS_DTYPE_BF16
    hp.slabs[0], hp.slabs[1] = 256, 512
    hp.out, hp.out_stride_token, hp.out_stride_head, hp.status = 1024, 16 * 128, 128, 4096
    assert lib.ps_paged_decode_head_gather(ctypes.byref(pr), None, 0, ctypes.byref(hp), None) == _lib.PS_ERR_UNSUPPORTED
    assert lib.ps_kv_dequant_gather(ctypes.byref(problem()), 4, None, None, None) == _lib.PS_ERR_INVALID_ARGUMENT
    assert lib.ps_kv_dequant_gather(ctypes.byref(fp4_problem(cache_stride_slot=64)), 4, ctypes.c_void_p(4096),
                                    ctypes.c_void_p(4096), None) == _lib.PS_ERR_INVALID_ARGUMENT


def test_nvfp4_append_refuses_on_the_host():
    lib = _lib.load()
    names = ["key", "k_st", "k_sh", "value", "v_st", "v_sh", "kc", "vc", "s_block", "s_head", "nb", "slots", "T", "hkv",
             "d", "bs", "dtype", "ks", "vs", "status", "stream"]
    good = dict(key=4096, k_st=256, k_sh=128, value=4096, v_st=256, v_sh=128, kc=4096, vc=4096, s_block=2304, s_head=1152,
                nb=4, slots=4096, T=2, hkv=2, d=128, bs=16, dtype=_lib.PS_DTYPE_BF16, ks=None, vs=None, status=None,
                stream=None)

    def go(**kw):
        a = dict(good, **kw)
        return lib.ps_kv_append_nvfp4(*[a[n] for n in names])

    if not torch.cuda.is_available():  # (with a GPU these addresses would be launched on)
        assert go() == _lib.PS_ERR_CUDA
    assert go(T=0) == _lib.PS_OK
    for bad in (dict(T=-1), dict(key=None), dict(slots=None), dict(hkv=0), dict(bs=24), dict(nb=0), dict(key=4104),
                dict(k_st=100), dict(kc=4104), dict(s_block=2312), dict(s_head=1136)):
        assert go(**bad) == _lib.PS_ERR_INVALID_ARGUMENT, bad
    assert go(dtype=_lib.PS_DTYPE_FP32) == _lib.PS_ERR_UNSUPPORTED
    assert go(d=64) == _lib.PS_ERR_UNSUPPORTED


def test_score_mod_argument_checks():
    q = torch.zeros(5, 8, 128)
    ok = ops.ScoreMod(softcap=3.0, alibi_slopes=torch.zeros(8), window_left=2 ** 40,
                      key_start=torch.zeros(7, dtype=torch.int32), prefix_lens=torch.zeros(2, dtype=torch.int32))
    m = ok._struct(q, 2)
    assert m.logits_soft_cap == 3.0 and m.window_left == 2 ** 31 - 1 and m.alibi_slopes and m.key_start
    assert ops.ScoreMod(window_left=-5)._struct(q, 2).window_left == -1
    for bad in (dict(softcap=-1.0), dict(softcap=math.nan), dict(softcap=math.inf),
                dict(alibi_slopes=torch.zeros(7)), dict(alibi_slopes=torch.zeros(8, dtype=torch.float64)),
                dict(alibi_slopes=torch.zeros(16)[::2]), dict(key_start=torch.zeros(4, dtype=torch.int32)),
                dict(key_start=torch.zeros(5)), dict(prefix_lens=torch.zeros(3, dtype=torch.int32)),
                dict(prefix_lens=torch.zeros(1, 2, dtype=torch.int32)),
                dict(key_start=torch.zeros(5, dtype=torch.int32, device="meta"))):
        with pytest.raises(ValueError):
            ops.ScoreMod(**bad)._struct(q, 2)


def test_nvfp4_cache_is_known_by_its_shape():
    assert ops.nvfp4_cache_shape(10, 32, 4) == (10, 4, 32, 72)
    for bad in ((10, 24, 4, 128), (10, 16, 4, 64), (10, 0, 4, 128)):
        with pytest.raises(ValueError):
            ops.nvfp4_cache_shape(*bad)
    c = torch.zeros(ops.nvfp4_cache_shape(2, 16, 4), dtype=torch.uint8)
    assert ops.is_nvfp4_cache(c)
    assert not ops.is_nvfp4_cache(c, 72)  # an fp8 cache of head size 72
    assert not ops.is_nvfp4_cache(torch.zeros(2, 16, 4, 128, dtype=torch.uint8))
    ops._check_nvfp4(c, c.clone())
    for k, v in ((c, c[:1]), (c, c.to(torch.int8)), (torch.zeros(2, 4, 8, 72, dtype=torch.uint8),) * 2,
                 (torch.zeros(2, 16, 4, 72, dtype=torch.uint8).transpose(1, 2),) * 2):
        with pytest.raises(ValueError):
            ops._check_nvfp4(k, v)


def test_calls_refuse_cpu_tensors_and_mixed_features():
    c = torch.zeros(ops.nvfp4_cache_shape(2, 16, 1), dtype=torch.uint8)
    k = torch.zeros(2, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_append(k, k, c, c, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="cascade"):
        ops.paged_decode(k, c, c, None, torch.zeros(2), 1.0, k, cascade=object())
    with pytest.raises(ValueError, match="cascade"):
        ops.paged_decode(k, k, k, None, torch.zeros(2), 1.0, k, cascade=object(), score_mod=ops.ScoreMod())


def test_torch_operators_are_registered():
    op = torch.ops.ps_attn

    def mutated(o):
        return {a.name for a in o.default._schema.arguments if a.alias_info is not None and a.alias_info.is_write}

    assert mutated(op.kv_append_scaled) == {"key_cache", "value_cache"}
    assert mutated(op.paged_decode_mod) == {"key_cache", "value_cache", "out", "lse", "workspace"}
    assert mutated(op.chunked_prefill_mod) == {"out", "lse", "workspace"}
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        q = torch.empty(4, 8, 128, dtype=torch.bfloat16)
        c = torch.empty(ops.nvfp4_cache_shape(8, 16, 2), dtype=torch.uint8)
        i = torch.zeros(4, dtype=torch.int32)
        k = torch.empty(4, 2, 128, dtype=torch.bfloat16)
        ws = torch.empty(1 << 20, dtype=torch.uint8)
        op.kv_append_scaled(k, k, c, c, i.long())
        op.paged_decode_mod(q, c, c, i.view(4, 1), i, None, 0.1, q, None, ws, 30.0, None, 100)
        op.chunked_prefill_mod(q, c, c, i.view(4, 1), i, i, 0.1, q, None, None, prefix_lens=i)
    assert torch_ops.paged_decode_mod is not None


# ---------------------------------------------------------------- backend

def test_backend_variants():
    assert "nvfp4" in psb.PSAttentionBackend.supported_kv_cache_dtypes
    assert psb.PSAttentionBackend.get_kv_cache_shape(10, 32, 8, 128, "nvfp4") == (2, 10, 8, 32, 72)
    with pytest.raises(ValueError):
        psb.PSAttentionBackend.get_kv_cache_shape(10, 32, 8, 64, "nvfp4")
    assert psb.PSScoreModAttentionBackend.get_impl_cls() is psb.PSScoreModAttentionImpl
    from vllm.v1.attention.backends.registry import AttentionBackendEnum

    psb.register(score_mods=True)
    assert AttentionBackendEnum.CUSTOM.get_class() is psb.PSScoreModAttentionBackend
    AttentionBackendEnum.CUSTOM.clear_override()
    with pytest.raises(ValueError):
        psb.register(score_mods=True, rope_fusion=True)
    assert psb.PSRopeAttentionImpl(16, 128, 0.088, 8, None, None, "nvfp4").fused_rope_kvcache_supported() is False


def test_score_mod_impl_options():
    cpu = torch.device("cpu")
    impl = psb.PSScoreModAttentionImpl(16, 128, 0.088, 8, [0.5] * 16, 128, "auto", 30.0)
    m = impl.score_mod(cpu)
    assert m.softcap == 30.0 and m.window_left == 127 and m.alibi_slopes.tolist() == [0.5] * 16
    assert impl.score_mod(cpu) is m
    assert psb.PSScoreModAttentionImpl(16, 128, 0.088, 8, None, None, "auto", None).score_mod(cpu) is None
    assert psb.PSScoreModAttentionImpl(16, 128, 0.088, 8, None, None, "nvfp4", 0.0).score_mod(cpu) is None
    assert psb.PSAttentionImpl(16, 128, 0.088, 8, None, None, "auto").score_mod(cpu) is None
    with pytest.raises(ValueError):
        psb.PSScoreModAttentionImpl(16, 128, 0.088, 8, [0.5] * 8, None, "auto")
    with pytest.raises(ValueError):
        psb.PSScoreModAttentionImpl(16, 128, 0.088, 8, None, 0, "auto")
    with pytest.raises(NotImplementedError):
        psb.PSScoreModAttentionImpl(16, 128, 0.088, 8, None, 64, "fp8_e5m2")
    with pytest.raises(NotImplementedError):
        psb.PSScoreModAttentionImpl(16, 128, 0.088, 8, None, 64, "auto", sinks=torch.zeros(16))


@pytest.mark.parametrize("cls,kw,dtype", [("PSAttentionImpl", {}, "nvfp4"),
                                          ("PSScoreModAttentionImpl", dict(sliding_window=64), "nvfp4"),
                                          ("PSScoreModAttentionImpl", dict(logits_soft_cap=20.0), "auto")])
def test_forward_routes(monkeypatch, cls, kw, dtype):
    """Which calls a mixed batch makes, with which scales, modifiers and caches."""
    calls = []
    for name in ("kv_append", "paged_decode", "chunked_prefill"):
        monkeypatch.setattr(psb.ops, name, lambda *a, _n=name, **k: calls.append((_n, a, k)))
    monkeypatch.setattr(psb.ops, "dequant_gather",
                        lambda *a, **k: calls.append(("gather", a, k)) or ("kd", "vd", "bt"))
    args = dict(alibi_slopes=None, sliding_window=None, kv_cache_dtype=dtype)
    args.update(kw)
    impl = getattr(psb, cls)(16, 128, 0.088, 8, **args)

    class Layer:
        _k_scale = torch.tensor(0.5)
        _v_scale = torch.tensor(0.25)

    lens = torch.tensor([10, 20, 40], dtype=torch.int32)
    md = psb.PSAttentionMetadata(
        num_actual_tokens=7, max_query_len=5, query_start_loc=torch.tensor([0, 1, 2, 7], dtype=torch.int32),
        max_seq_len=40, seq_lens=lens, block_table=torch.zeros(3, 4, dtype=torch.int32),
        slot_mapping=torch.arange(7), num_decodes=2, num_decode_tokens=2, num_prefills=1, workspace="ws",
        cascade_plan="plan")
    q = torch.zeros(7, 16, 128, dtype=torch.bfloat16)
    shape = psb.PSAttentionBackend.get_kv_cache_shape(4, 32, 8, 128, dtype)
    kv = torch.zeros(shape, dtype=torch.uint8 if dtype == "nvfp4" else torch.bfloat16)
    impl.forward(Layer(), q, torch.zeros(7, 8, 128), torch.zeros(7, 8, 128), kv, md, torch.zeros_like(q))
    four = dtype == "nvfp4"
    assert [c[0] for c in calls] == ["kv_append", "paged_decode"] + ["gather"] * four + ["chunked_prefill"]
    mod = impl.score_mod(torch.device("cpu"))
    assert (mod is not None) == bool(kw)
    for name, _, k in calls:
        if name != "gather":
            assert k.get("k_scale") is (Layer._k_scale if four else None)
        if name in ("paged_decode", "chunked_prefill"):
            assert k["score_mod"] is mod
    assert calls[1][2]["cascade"] is None and calls[1][1][1].shape == kv[0].shape
    if four:
        assert calls[2][1][4] == 2  # ceil(40 / 32) blocks of the longest sequence
        assert calls[3][1][1:4] == ("kd", "vd", "bt")


# ---------------------------------------------------------------- the reference's own format

def test_reference_quantizer_by_hand():
    x = torch.zeros(1, 128, dtype=torch.bfloat16)
    x[0, :16] = torch.tensor([6, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, -6])
    v, s = mod_ref.quantize_nvfp4(x, 1.0)
    assert s[0, 0] == 1.0 and s[0, 1:].eq(0).all()
    assert v[0, :16].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, 0, -1, -1, -2, -2, -4, -4, -6]
    # values never differ from the input by more than half a code step plus the scale's own rounding
    g = 0.01
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    err = (mod_ref.nvfp4_values(x, g) - x.double()).abs().unflatten(-1, (8, 16)).amax(-1)
    amax = x.double().abs().unflatten(-1, (8, 16)).amax(-1)
    # half of the largest step (2 of 6) of the scale, which e4m3 rounds by 2^-4 at most
    assert bool((err <= amax * (1 / 6) * (1 + 2.0 ** -4) + amax * 2.0 ** -4).all())
