"""The backend's variants as vLLM's attention layer makes and runs them
(``vllm/model_executor/layers/attention/attention.py``): with the positional
arguments of a layer (CPU), and in a layer over a 4-bit cache or with score
modifiers, eager and captured, against 64-bit attention (GPU)."""
from __future__ import annotations

import inspect
import json

import pytest
import torch

import mod_ref
from ps_attn import backend as psb
from test_score_mod_gpu import slopes

HQ, HKV, D, BS = 16, 8, 128, 16


@pytest.mark.parametrize("cls", [psb.PSAttentionImpl, psb.PSRopeAttentionImpl, psb.PSScoreModAttentionImpl])
def test_impls_take_a_layers_positional_arguments(cls):
    """heads, head size, scale, kv heads, ALiBi, window, cache dtype, soft-cap, attention type, KV sharing target."""
    impl = cls(HQ, D, 0.088, HKV, None, None, "auto", None, "decoder", "model.layers.0.attn")
    assert impl.kv_sharing_target_layer_name == "model.layers.0.attn" and impl.attn_type == "decoder"
    names = list(inspect.signature(psb.PSAttentionImpl.__init__).parameters)
    assert list(inspect.signature(cls.__init__).parameters) == names
    with pytest.raises(NotImplementedError, match="decoder"):
        cls(HQ, D, 0.088, HKV, None, None, "auto", None, "encoder", None)


def common(qlens, lens, bound):
    from vllm.v1.attention.backend import CommonAttentionMetadata

    qsl = torch.tensor([0] + qlens).cumsum(0).int()
    return CommonAttentionMetadata(
        query_start_loc=qsl, query_start_loc_cpu=qsl.clone(), seq_lens=torch.tensor(lens, dtype=torch.int32),
        num_reqs=len(qlens), num_actual_tokens=sum(qlens), max_query_len=max(qlens), max_seq_len=max(lens),
        block_table_tensor=torch.zeros(len(qlens), 2048, dtype=torch.int32),
        slot_mapping=torch.arange(sum(qlens)), seq_lens_cpu_upper_bound=bound)


@pytest.mark.parametrize("dtype", ["nvfp4", "fp8"])
def test_prefill_scratch_holds_the_prefills_not_the_longest_decode(monkeypatch, dtype):
    """Two short prompts beside a decode of 32,000 tokens: scratch for the prompts' pages, where the step's lengths
    are known on the host."""
    calls = []
    for name in ("kv_append", "paged_decode", "chunked_prefill"):
        monkeypatch.setattr(psb.ops, name, lambda *a, **k: None)
    monkeypatch.setattr(psb.ops, "dequant_gather", lambda *a, **k: calls.append(a) or ("k", "v", "bt"))
    impl = psb.PSAttentionImpl(HQ, D, 0.088, HKV, None, None, dtype)
    kv = torch.zeros(psb.PSAttentionBackend.get_kv_cache_shape(4, BS, HKV, D, dtype), dtype=torch.uint8)
    q = torch.zeros(71, HQ, D)
    builder = psb.PSAttentionMetadataBuilder.__new__(psb.PSAttentionMetadataBuilder)
    builder.workspace = object()
    lens = [32_000, 50, 70]
    # (a bound for some of the requests only is none)
    for bound, pages in ((torch.tensor([32_001, 50, 71]), 5), (None, 2000), (torch.tensor([32_001, 50]), 2000)):
        md = builder.build(0, common([1, 50, 20], lens, bound))
        impl.forward(object(), q, q[:, :HKV], q[:, :HKV], kv, md, torch.zeros_like(q))
        assert calls.pop()[4] == pages
    # a decode-only step has no prefill
    assert builder.build(0, common([1, 1], [5, 6], torch.tensor([5, 6]))).max_prefill_len == 0


CASES = {
    "nvfp4": ("nvfp4", {}, {}),
    "nvfp4_window_cap": ("nvfp4", dict(per_layer_sliding_window=100, logits_soft_cap=20.0),
                         dict(window_left=99, softcap=20.0)),
    "bias": ("auto", dict(alibi_slopes=slopes(HQ).tolist()), dict(alibi_slopes=slopes(HQ))),
    "window_cap": ("auto", dict(per_layer_sliding_window=64, logits_soft_cap=30.0), dict(window_left=63, softcap=30.0)),
    "fp8_cap": ("fp8", dict(logits_soft_cap=10.0), dict(softcap=10.0)),
}


@pytest.fixture(scope="module")
def config(tmp_path_factory):
    from vllm.config import CacheConfig, ModelConfig, VllmConfig

    d = tmp_path_factory.mktemp("layer_config")
    (d / "config.json").write_text(json.dumps({
        "architectures": ["Qwen3ForCausalLM"], "model_type": "qwen3", "hidden_size": 1024, "intermediate_size": 2048,
        "num_attention_heads": HQ, "num_key_value_heads": HKV, "head_dim": D, "num_hidden_layers": 2,
        "vocab_size": 32000, "max_position_embeddings": 16384, "rms_norm_eps": 1e-6, "rope_theta": 1000000,
        "torch_dtype": "bfloat16", "tie_word_embeddings": True, "attention_bias": False, "hidden_act": "silu"}))

    def make(cache_dtype):
        mc = ModelConfig(model=str(d), skip_tokenizer_init=True, dtype="bfloat16", max_model_len=8192)
        return VllmConfig(model_config=mc, cache_config=CacheConfig(block_size=BS, cache_dtype=cache_dtype))

    return make


def layer_of(vc, name, kw, cls, device):
    from vllm.config import set_current_vllm_config
    from vllm.model_executor.layers.attention.attention import Attention

    torch.set_default_dtype(torch.bfloat16)
    try:
        with set_current_vllm_config(vc), torch.device(device):
            layer = Attention(HQ, D, D ** -0.5, HKV, cache_config=vc.cache_config, prefix=name, attn_backend=cls, **kw)
            spec = layer.get_kv_cache_spec(vc)
            return layer, spec, cls.get_builder_cls()(spec, [name], vc, device)
    finally:
        torch.set_default_dtype(torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_layer_matches_plain_attention(case, config, cuda_device):
    pytest.importorskip("vllm")
    from vllm.forward_context import set_forward_context
    from vllm.v1.attention.backend import CommonAttentionMetadata

    dtype, kw, mod = CASES[case]
    kind = {"auto": "16bit"}.get(dtype, dtype)
    cls = psb.PSScoreModAttentionBackend if mod else psb.PSAttentionBackend
    vc = config(dtype)
    name = f"model.layers.{list(CASES).index(case)}.{case}.attn"
    layer, spec, builder = layer_of(vc, name, kw, cls, cuda_device)
    qlens = [1, 1, 1, 70, 5, 200]
    lens = [300, 1, 77, 70, 400, 333]
    b = mod_ref.Batch(lens, qlens, HQ, HKV, kind=kind, seed=91)
    # vLLM's own shape and page size of this cache
    shape = cls.get_kv_cache_shape(b.kc.shape[0], BS, HKV, D, dtype)
    assert shape[1:] == tuple(b.kc.shape)
    assert spec.page_size_bytes * b.kc.shape[0] == 2 * b.kc.numel() * b.kc.element_size()
    kv = torch.stack([b.kc, b.vc])
    layer.kv_cache = kv
    if kind != "16bit":
        layer._k_scale, layer._v_scale = b.scales["k_scale"], b.scales["v_scale"]
    # the step's rows and slots: the last qlens tokens of each sequence
    new = torch.cat([torch.arange(sum(lens[:i]) + n - q, sum(lens[:i + 1])) for i, (n, q) in enumerate(zip(lens, qlens))])
    k, v, slots = b.rows_k[new].to(cuda_device), b.rows_v[new].to(cuda_device), b.slots[new].to(cuda_device)
    starts = b.starts.to(cuda_device)

    def run(n_seqs):
        T = int(b.starts[n_seqs])
        cm = CommonAttentionMetadata(
            query_start_loc=starts[:n_seqs + 1], query_start_loc_cpu=b.starts[:n_seqs + 1], seq_lens=b.lens[:n_seqs],
            num_reqs=n_seqs, num_actual_tokens=T, max_query_len=max(qlens[:n_seqs]), max_seq_len=max(lens[:n_seqs]),
            block_table_tensor=b.table[:n_seqs], slot_mapping=slots[:T], causal=True)
        md = builder.build(0, cm)

        def step():
            with set_forward_context({name: md}, vc, slot_mapping={name: cm.slot_mapping}):
                return layer(b.q[:T].flatten(1), k[:T].flatten(1), v[:T].flatten(1)).view(-1, HQ, D)

        return step, md

    before = kv.clone()
    step, _ = run(len(lens))
    out = step()
    torch.cuda.synchronize()
    assert torch.equal(kv.view(torch.uint8), before.view(torch.uint8))  # the rows that were there, stored again
    # (the prefill rounds its weights to the query's type, over a cache of any kind)
    ro, rl, otol, ltol = mod_ref.attention(b.q, b.ks, b.vs, b.starts, b.scale, mod, b.dtype, True)
    no_lse = torch.zeros_like(rl)
    mod_ref.check(out, no_lse, (ro, no_lse, otol, ltol))
    # the decode rows alone, captured and replayed on other queries
    step, _ = run(3)
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    b.q[:3] = torch.randn(3, HQ, D, generator=torch.Generator().manual_seed(92)).to(b.q.dtype)
    g.replay()
    torch.cuda.synchronize()
    ro, rl, otol, ltol = (x[:3] if x.dim() == 3 else x[:, :3] for x in b.reference(mod))
    no_lse = torch.zeros_like(rl)
    mod_ref.check(captured, no_lse, (ro, no_lse, otol, ltol))
