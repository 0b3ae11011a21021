"""Torch-facing ops over libps_attn.so.

These functions mirror the two GPU calls vLLM's FlashAttention backend makes
per decoder layer and keep their argument meaning:

* :func:`kv_append` -- ``reshape_and_cache_flash(key, value, key_cache,
  value_cache, slot_mapping, ...)`` (``vllm/_custom_ops.py:2591-2610``);
* :func:`paged_attention` -- ``flash_attn_varlen_func(q, k_cache, v_cache, out,
  cu_seqlens_q, max_seqlen_q, seqused_k, max_seqlen_k, softmax_scale,
  causal=True, block_table=...)`` as called at
  ``vllm/v1/attention/backends/flash_attn.py:796-817``.  It dispatches to
  :func:`paged_decode` (``max_seqlen_q == 1``) or :func:`chunked_prefill`.

Tensors stay on the device; the work is enqueued on the current CUDA stream;
nothing here synchronises or allocates except :class:`DecodeWorkspace`
construction (and :func:`dequant_gather` without ``out``).  Score modifiers (tanh cap, distance bias,
sliding window, document and prefix masks) are a :class:`ScoreMod` passed to
the attention calls; a 4-bit cache (:func:`nvfp4_cache_shape`) is recognised by
its shape.  All validation failures raise :class:`ps_attn._lib.PSError` or
``ValueError``; there is no non-CUDA path.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib

_DTYPES = {
    torch.float16: _lib.PS_DTYPE_FP16,
    torch.bfloat16: _lib.PS_DTYPE_BF16,
    torch.float32: _lib.PS_DTYPE_FP32,
}


def _stream_ptr(device: torch.device) -> int:
    # the raw handle, without the Stream object that current_stream() builds
    # (1.5 us of a small call's host time)
    return torch._C._cuda_getCurrentRawStream(device.index if device.index is not None
                                              else torch.cuda.current_device())


def _require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("ps_attn ops take CUDA tensors only (no CPU path)")


FP8_CACHE_DTYPES = (torch.uint8, torch.float8_e4m3fn)


def is_fp8_cache(cache: torch.Tensor) -> bool:
    """An fp8 (e4m3) KV cache: uint8 codes or torch.float8_e4m3fn."""
    return cache.dtype in FP8_CACHE_DTYPES


NVFP4_ROW_BYTES = _lib.PS_NVFP4_ROW_BYTES


def nvfp4_cache_shape(num_blocks: int, block_size: int, num_kv_heads: int, head_size: int = 128) -> tuple:
    """Shape of one half (K or V) of a 4-bit KV cache, a ``torch.uint8`` tensor:
    ``(num_blocks, num_kv_heads, block_size, 72)``.  The last two dimensions are
    an opaque sequence of 1152-byte tiles of 16 tokens (e2m1 codes and one e4m3
    scale per 16 dims; ``csrc/nvfp4.cuh``); :func:`kv_append` writes it,
    :func:`paged_decode` and :func:`dequant_gather` read it."""
    if head_size != 128:
        raise ValueError(f"nvfp4 caches hold head_size 128 (got {head_size})")
    if block_size <= 0 or block_size % 16:
        raise ValueError(f"block_size {block_size} must be a positive multiple of 16")
    return (num_blocks, num_kv_heads, block_size, NVFP4_ROW_BYTES)


def is_nvfp4_cache(cache: torch.Tensor, head_size: int = 128) -> bool:
    """A half of a 4-bit KV cache for rows of ``head_size`` elements (an fp8
    cache's last dimension is the head size itself)."""
    return (cache.dtype == torch.uint8 and cache.dim() == 4 and cache.shape[-1] == NVFP4_ROW_BYTES
            and head_size == 128)


def _check_nvfp4(key_cache: torch.Tensor, value_cache: torch.Tensor) -> None:
    strides = key_cache.stride()
    if value_cache.dtype != torch.uint8 or key_cache.shape != value_cache.shape or strides != value_cache.stride():
        raise ValueError("nvfp4: key_cache and value_cache must have the same dtype, shape and strides")
    if key_cache.shape[2] % 16:
        raise ValueError("nvfp4: block_size must be a multiple of 16")
    if strides[3] != 1 or strides[2] != NVFP4_ROW_BYTES:
        raise ValueError("nvfp4: the (block_size, 72) part of a cache must be contiguous")


def _launch(device: torch.device, fn, *args) -> None:
    """Call a C entry point with ``device`` current (the library launches on the
    current device)."""
    if device.index is None or torch._C._cuda_getDevice() == device.index:
        _lib.check(fn(*args))
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args))


@dataclass(frozen=True)
class ScoreMod:
    """Score modifiers of an attention call (``ps_score_mod``).

    With i a query row's position in its sequence and j a key's, the score
    ``z = softmax_scale * q.k`` becomes ``softcap * tanh(z / softcap)`` (if
    ``softcap > 0``), then ``z - alibi_slopes[h] * |i - j|``, over the keys
    ``max(0, i - window_left, key_start[row]) <= j <= max(i, prefix_lens[b] - 1)``
    below the sequence's length.  A row that sees no key gives 0 and LSE -inf.

    alibi_slopes: float32 [Hq]; window_left: -1 for no window (vLLM's
    ``sliding_window - 1``); key_start: int32, one entry per query row, the
    first key of the row's document; prefix_lens: int32 [B], the first keys of
    the sequence, which the rows before them see too, as far as the window and
    ``key_start`` let them (prefill; no effect on a decode row, which sees no
    key behind its own).  Keys past a row's range may hold anything; keys that
    one row of a sequence sees and another does not must hold finite values.
    """

    softcap: float = 0.0
    alibi_slopes: torch.Tensor | None = None
    window_left: int = -1
    key_start: torch.Tensor | None = None
    prefix_lens: torch.Tensor | None = None

    def _struct(self, q: torch.Tensor, num_seqs: int) -> "_lib.ScoreMod":
        m = _lib.ScoreMod()
        cap = float(self.softcap)
        if not 0.0 <= cap < float("inf"):
            raise ValueError(f"softcap must be finite and >= 0 (got {self.softcap})")
        m.logits_soft_cap = cap
        w = int(self.window_left)
        m.window_left = -1 if w < 0 else min(w, 2 ** 31 - 1)

        def array(t, name, dtype, n, exact):
            if t is None:
                return None
            if t.dtype != dtype or t.dim() != 1 or not t.is_contiguous() or t.device != q.device:
                raise ValueError(f"{name} must be a contiguous 1-D {dtype} tensor on {q.device}")
            if t.shape[0] < n or (exact and t.shape[0] != n):
                raise ValueError(f"{name} has {t.shape[0]} entries, the call needs {n}")
            return t.data_ptr()

        m.alibi_slopes = array(self.alibi_slopes, "alibi_slopes", torch.float32, q.shape[1], True)
        m.key_start = array(self.key_start, "key_start", torch.int32, q.shape[0], False)
        m.prefix_lens = array(self.prefix_lens, "prefix_lens", torch.int32, num_seqs, True)
        return m


def _scale_ptr(scale):
    if scale is None:
        return None
    if scale.dtype != torch.float32 or not scale.is_cuda or scale.numel() != 1:
        raise ValueError("k_scale / v_scale must be one-element CUDA float32 tensors")
    return scale.data_ptr()


def kv_append(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
              value_cache: torch.Tensor, slot_mapping: torch.Tensor,
              status: torch.Tensor | None = None, k_scale: torch.Tensor | None = None,
              v_scale: torch.Tensor | None = None) -> None:
    """Write ``key``/``value`` rows into the paged cache at ``slot_mapping``.

    key, value: [T', Hkv, D] (T' >= len(slot_mapping)); key_cache,
    value_cache: [num_blocks, block_size, Hkv, D]; slot_mapping: int64 [T].
    Negative slots are skipped.  Bit-exact copy; for an fp8 cache (uint8 or
    float8_e4m3fn) the rows are stored as e4m3(x / k_scale) and
    e4m3(x / v_scale) (``reshape_and_cache_flash`` with kv_cache_dtype "fp8";
    scales: one-element float32 device tensors, None = 1); for an nvfp4 cache
    (uint8 :func:`nvfp4_cache_shape`) as e2m1 codes with an e4m3 scale per 16
    dims under the same per-tensor scales (``ps_kv_append_nvfp4``; no two rows
    may share a slot).
    """
    lib = _lib.load()
    _require_cuda(key, value, key_cache, value_cache, slot_mapping)
    if slot_mapping.dtype != torch.int64:
        raise ValueError("slot_mapping must be int64")
    if key.dim() == 3 and is_nvfp4_cache(key_cache, key.shape[-1]):
        _append_nvfp4(lib, key, value, key_cache, value_cache, slot_mapping, status, k_scale, v_scale)
        return
    fp8 = is_fp8_cache(key_cache)
    if fp8:
        if value_cache.dtype != key_cache.dtype or key.dtype != value.dtype or \
                key.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("fp8 cache: fp16/bf16 key and value rows, both caches fp8")
    elif key.dtype != key_cache.dtype or value.dtype != value_cache.dtype or key.dtype != value.dtype:
        raise ValueError("key/value/cache dtypes must match")
    if key_cache.stride() != value_cache.stride() or key_cache.shape != value_cache.shape:
        raise ValueError("key_cache and value_cache must have the same shape and strides")
    if key.stride(-1) != 1 or value.stride(-1) != 1 or key_cache.stride(-1) != 1:
        raise ValueError("last dimension must be contiguous")
    if not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous")
    T = slot_mapping.shape[0]
    if key.shape[0] < T or value.shape[0] < T:
        raise ValueError("key/value have fewer rows than slot_mapping")
    nb, bs, hkv, d = key_cache.shape
    if key.shape[1:] != (hkv, d) or value.shape[1:] != (hkv, d):
        raise ValueError(f"key/value shape {tuple(key.shape)} does not match cache {tuple(key_cache.shape)}")
    if fp8:
        _launch(key.device, lib.ps_kv_append_fp8,
                key.data_ptr(), key.stride(0), key.stride(1),
                value.data_ptr(), value.stride(0), value.stride(1),
                key_cache.data_ptr(), value_cache.data_ptr(),
                key_cache.stride(0), key_cache.stride(1), key_cache.stride(2), nb,
                slot_mapping.data_ptr(), T, hkv, d, bs, _DTYPES[key.dtype],
                _scale_ptr(k_scale), _scale_ptr(v_scale),
                status.data_ptr() if status is not None else None,
                _stream_ptr(key.device))
        return
    _launch(key.device, lib.ps_kv_append,
            key.data_ptr(), key.stride(0), key.stride(1),
            value.data_ptr(), value.stride(0), value.stride(1),
            key_cache.data_ptr(), value_cache.data_ptr(),
            key_cache.stride(0), key_cache.stride(1), key_cache.stride(2), nb,
            slot_mapping.data_ptr(), T, hkv, d, bs, key.element_size(),
            status.data_ptr() if status is not None else None,
            _stream_ptr(key.device))


def _append_nvfp4(lib, key, value, key_cache, value_cache, slot_mapping, status, k_scale, v_scale) -> None:
    _check_nvfp4(key_cache, value_cache)
    if key.dtype != value.dtype or key.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("nvfp4 cache: fp16/bf16 key and value rows of one dtype")
    k_st, k_sh, k_sd = key.stride()
    v_st, v_sh, v_sd = value.stride() if value.dim() == 3 else (0, 0, 0)
    if k_sd != 1 or v_sd != 1 or not slot_mapping.is_contiguous():
        raise ValueError("key/value rows and slot_mapping must be contiguous")
    nb, hkv, bs, _ = key_cache.shape
    s_block, s_head = key_cache.stride()[:2]
    T = slot_mapping.shape[0]
    if key.shape[0] < T or value.shape[0] < T:
        raise ValueError("key/value have fewer rows than slot_mapping")
    if key.shape[1:] != (hkv, 128) or value.shape[1:] != (hkv, 128):
        raise ValueError(f"key/value shape {tuple(key.shape)} does not match {hkv} kv heads of 128")
    _launch(key.device, lib.ps_kv_append_nvfp4,
            key.data_ptr(), k_st, k_sh, value.data_ptr(), v_st, v_sh,
            key_cache.data_ptr(), value_cache.data_ptr(), s_block, s_head, nb,
            slot_mapping.data_ptr(), T, hkv, 128, bs, _DTYPES[key.dtype], _scale_ptr(k_scale),
            _scale_ptr(v_scale), status.data_ptr() if status is not None else None, _stream_ptr(key.device))


def rope_kv_append(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                   positions: torch.Tensor, cos_sin_cache: torch.Tensor, is_neox: bool,
                   key_cache: torch.Tensor, value_cache: torch.Tensor,
                   slot_mapping: torch.Tensor, status: torch.Tensor | None = None) -> None:
    """Rotary embedding of ``query``/``key`` in place, then the KV append of the
    rotated key and ``value`` (``do_rope_and_kv_cache_update``'s contract).

    query [T, Hq*D] or [T, Hq, D]; key, value [T, Hkv*D] or [T, Hkv, D];
    positions int64 [T]; cos_sin_cache [max_position, rotary_dim] (fp32 or the
    model dtype; cos half then sin half); caches [num_blocks, block_size, Hkv,
    D]; slot_mapping int64 [T] (negative: no cache write).  Bit-identical to
    vLLM's torch-native rotary embedding followed by ``kv_append``.
    """
    lib = _lib.load()
    _require_cuda(query, key, value, positions, cos_sin_cache, key_cache, value_cache, slot_mapping)
    nb, bs, hkv, d = key_cache.shape
    T = slot_mapping.shape[0]
    if positions.dtype != torch.int64 or slot_mapping.dtype != torch.int64:
        raise ValueError("positions and slot_mapping must be int64")
    if positions.numel() < T or not positions.is_contiguous() or not slot_mapping.is_contiguous():
        raise ValueError("positions must hold a position per token; both contiguous")
    q3 = query.view(query.shape[0], -1, d)
    k3 = key.view(key.shape[0], -1, d)
    v3 = value.view(value.shape[0], -1, d)
    if k3.shape[1] != hkv or v3.shape[1] != hkv or q3.shape[0] < T or k3.shape[0] < T:
        raise ValueError("query/key/value shapes do not match the cache")
    dtype = query.dtype
    if dtype not in (torch.bfloat16, torch.float16) or key.dtype != dtype or value.dtype != dtype \
            or key_cache.dtype != dtype or value_cache.dtype != dtype:
        raise ValueError("query, key, value and caches must share one fp16/bf16 dtype")
    if cos_sin_cache.dtype not in (torch.float32, dtype) or cos_sin_cache.stride(-1) != 1:
        raise ValueError("cos_sin_cache must be fp32 or the model dtype, rows contiguous")
    if key_cache.stride() != value_cache.stride() or key_cache.stride(-1) != 1:
        raise ValueError("key_cache and value_cache must share strides, last dim contiguous")
    if q3.stride(-1) != 1 or k3.stride(-1) != 1 or v3.stride(-1) != 1:
        raise ValueError("last dimension must be contiguous")
    pr = _lib.RopeAppendProblem()
    pr.query = q3.data_ptr()
    pr.query_stride_token, pr.query_stride_head = q3.stride(0), q3.stride(1)
    pr.key = k3.data_ptr()
    pr.key_stride_token, pr.key_stride_head = k3.stride(0), k3.stride(1)
    pr.value = v3.data_ptr()
    pr.value_stride_token, pr.value_stride_head = v3.stride(0), v3.stride(1)
    pr.key_cache = key_cache.data_ptr()
    pr.value_cache = value_cache.data_ptr()
    pr.cache_stride_block, pr.cache_stride_slot, pr.cache_stride_head = key_cache.stride()[:3]
    pr.num_blocks = nb
    pr.block_size = bs
    pr.slot_mapping = slot_mapping.data_ptr()
    pr.positions = positions.data_ptr()
    pr.cos_sin_cache = cos_sin_cache.data_ptr()
    pr.cos_sin_stride = cos_sin_cache.stride(0)
    pr.max_position = cos_sin_cache.shape[0]
    pr.cos_sin_dtype = _DTYPES[cos_sin_cache.dtype]
    pr.rotary_dim = cos_sin_cache.shape[-1]
    pr.is_neox = int(bool(is_neox))
    pr.num_tokens = T
    pr.num_q_heads = q3.shape[1]
    pr.num_kv_heads = hkv
    pr.head_size = d
    pr.dtype = _DTYPES[dtype]
    if status is not None:
        pr.status = status.data_ptr()
    _launch(query.device, lib.ps_rope_kv_append, ctypes.byref(pr), _stream_ptr(query.device))


class DecodeWorkspace:
    """Fixed-size device workspace for :func:`paged_decode`.

    Sized for ``max_num_seqs`` once (independent of sequence lengths, so one
    buffer serves every step and every CUDA-graph replay) and zeroed at
    creation; the kernel leaves its counters at zero.  Serves calls with
    ``num_kv_heads`` kv heads only: the counters' place depends on them.  ``status()`` reads and
    ``clear_status()`` resets the device status word (PS_DEV_* bits).
    """

    def __init__(self, max_num_seqs: int, num_q_heads: int, num_kv_heads: int,
                 head_size: int, device: torch.device | str | int | None = None,
                 cascade: bool = False):
        lib = _lib.load()
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        if dev.type != "cuda":
            raise ValueError("DecodeWorkspace lives on a CUDA device")
        with torch.cuda.device(dev):
            nbytes = lib.ps_paged_decode_workspace_size(max_num_seqs, num_q_heads, num_kv_heads, head_size)
            if cascade:  # serves both kinds of call: the larger size
                nbytes = max(nbytes, lib.ps_paged_decode_cascade_workspace_size(
                    max_num_seqs, num_q_heads, num_kv_heads, head_size))
        if nbytes < 0:
            _lib.check(_lib.PS_ERR_INVALID_ARGUMENT)
        self.cascade = cascade
        self.max_num_seqs = max_num_seqs
        self.num_q_heads = num_q_heads
        self.num_kv_heads = num_kv_heads
        self.nbytes = int(nbytes)
        self.buffer = torch.zeros(self.nbytes, dtype=torch.uint8, device=dev)

    def status(self) -> int:
        return int(self.buffer[:4].view(torch.int32).item())

    def clear_status(self) -> None:
        self.buffer[:4].zero_()


_WS_CACHE: dict = {}       # (device, stream, heads, kind) -> workspace of the stream's own calls
_WS_CAPTURES: dict = {}    # (device, stream) -> (capture, {(heads, kind): workspace}) of the stream's last capture


def get_workspace(num_seqs: int, num_q_heads: int, num_kv_heads: int, head_size: int,
                  device: torch.device, cascade: bool = False) -> DecodeWorkspace:
    """The workspace of calls on ``device``'s current stream, per (heads, kind), grown to the largest batch seen.

    Calls of one stream run one after the other, so they can share it.  A call
    that is captured into a CUDA graph gets a workspace of that graph's: it lives
    in the graph's memory pool and is zeroed by each replay, so that neither a
    larger batch later on, nor another graph, nor the stream's own calls touch it."""
    lib = _lib.load()
    stream = _stream_ptr(device)
    key = (num_q_heads, num_kv_heads, head_size, cascade)
    capture = lib.ps_stream_capture_id(stream)
    if capture:
        of, kept = _WS_CAPTURES.get((device.index, stream), (0, None))
        if of != capture:
            kept = {}
            _WS_CAPTURES[device.index, stream] = (capture, kept)
    else:
        kept, key = _WS_CACHE, (device.index, stream) + key
    ws = kept.get(key)
    if ws is None or ws.max_num_seqs < num_seqs:
        cap = max(num_seqs, 256 if ws is None else 2 * ws.max_num_seqs)
        if cascade:
            cap = min(cap, CASCADE_MAX_SEQS)
        ws = DecodeWorkspace(cap, num_q_heads, num_kv_heads, head_size, device, cascade=cascade)
        kept[key] = ws
    return ws


CASCADE_MAX_SEQS = 2048
PLAN_HEADER_WORDS = 32


class CascadePlan:
    """Device buffer of a shared-prefix plan (``ps_cascade_plan_build``).

    Sized for up to ``max_num_seqs`` sequences and zeroed once; rebuilt in
    place by :func:`cascade_plan` for each batch (once per step, shared by all
    layers).  ``num_seqs`` is the batch the current contents describe.
    """

    def __init__(self, max_num_seqs: int, device: torch.device | str | int | None = None):
        lib = _lib.load()
        if not 0 <= max_num_seqs <= CASCADE_MAX_SEQS:
            raise ValueError(f"cascade plans hold at most {CASCADE_MAX_SEQS} sequences")
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        nbytes = lib.ps_cascade_plan_bytes(max(max_num_seqs, 1))
        if nbytes < 0:
            _lib.check(_lib.PS_ERR_INVALID_ARGUMENT)
        self.max_num_seqs = max_num_seqs
        self.nbytes = int(nbytes)
        self.buffer = torch.zeros(self.nbytes // 4, dtype=torch.int32, device=dev)
        self.num_seqs = 0

    def views(self) -> dict:
        """The plan's arrays for the batch it was last built for (device tensors)."""
        B = self.num_seqs
        gm = max(1, B // 2)
        w = self.buffer
        o = PLAN_HEADER_WORDS
        return {
            "num_groups": w[0:1],
            "seq_group": w[o:o + B],
            "group_first": w[o + B:o + B + gm],
            "group_size": w[o + B + gm:o + B + 2 * gm],
            "group_pages": w[o + B + 2 * gm:o + B + 3 * gm],
            "shared_pages": w[o + B + 3 * gm:o + 2 * B + 3 * gm],
        }


def cascade_plan(block_table: torch.Tensor, seq_lens: torch.Tensor, num_q_heads: int,
                 num_kv_heads: int, block_size: int, query_start_loc: torch.Tensor | None = None,
                 min_shared_pages: int = 8, plan: CascadePlan | None = None) -> CascadePlan:
    """Find groups of adjacent decode sequences with identical leading pages.

    Enqueued on the current stream (no host synchronisation).  The result is
    valid for any later :func:`paged_decode` call on the same block_table,
    seq_lens and query_start_loc; pass it as ``cascade=``.
    """
    lib = _lib.load()
    _require_cuda(block_table, seq_lens, query_start_loc)
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise ValueError("block_table and seq_lens must be int32")
    if block_table.stride(-1) != 1 or not seq_lens.is_contiguous():
        raise ValueError("block_table rows and seq_lens must be contiguous")
    B = seq_lens.shape[0]
    if plan is None:
        plan = CascadePlan(B, seq_lens.device)
    elif plan.max_num_seqs < B:
        raise ValueError(f"plan sized for {plan.max_num_seqs} sequences < {B}")
    pr = _lib.PagedProblem()
    pr.block_table = block_table.data_ptr()
    pr.block_table_stride = block_table.stride(0)
    pr.max_blocks_per_seq = block_table.shape[1]
    pr.seq_lens = seq_lens.data_ptr()
    pr.query_start_loc = query_start_loc.data_ptr() if query_start_loc is not None else None
    pr.num_seqs = B
    pr.num_q_heads = num_q_heads
    pr.num_kv_heads = num_kv_heads
    pr.head_size = 128
    pr.block_size = block_size
    _launch(seq_lens.device, lib.ps_cascade_plan_build, ctypes.byref(pr), int(min_shared_pages),
            plan.buffer.data_ptr(), plan.nbytes, _stream_ptr(seq_lens.device))
    plan.num_seqs = B
    return plan


def _problem(q, key_cache, value_cache, block_table, seq_lens, query_start_loc,
             softmax_scale, out, lse, status=None, k_scale=None, v_scale=None) -> _lib.PagedProblem:
    _require_cuda(q, key_cache, value_cache, block_table, seq_lens, out, query_start_loc, lse)
    # (shapes and strides are read once each: a read costs 0.1-0.2 us of a small call)
    dtype = q.dtype
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"attention dtype {dtype} unsupported (fp16/bf16)")
    rows, hq, dq = q.shape
    q_st, q_sh, q_sd = q.stride()
    out_rows, out_heads, out_d = out.shape
    o_st, o_sh, o_sd = out.stride()
    cache_dtype = key_cache.dtype
    fp4 = is_nvfp4_cache(key_cache, dq)
    fp8 = cache_dtype in FP8_CACHE_DTYPES and not fp4
    if fp4:
        _check_nvfp4(key_cache, value_cache)
        if out.dtype != dtype:
            raise ValueError("nvfp4 cache: out must have the query dtype")
    elif fp8:
        if value_cache.dtype != cache_dtype or out.dtype != dtype:
            raise ValueError("fp8 cache: both caches fp8, out in the query dtype")
    elif cache_dtype != dtype or value_cache.dtype != dtype or out.dtype != dtype:
        raise ValueError("q, caches and out must share one dtype")
    strides = key_cache.stride()
    if strides != value_cache.stride() or key_cache.shape != value_cache.shape:
        raise ValueError("key_cache and value_cache must have the same shape and strides")
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise ValueError("block_table and seq_lens must be int32")
    if query_start_loc is not None and query_start_loc.dtype != torch.int32:
        raise ValueError("query_start_loc must be int32")
    table_rows, table_cols = block_table.shape
    table_st, table_sd = block_table.stride()
    if table_sd != 1 or not seq_lens.is_contiguous():
        raise ValueError("block_table rows and seq_lens must be contiguous")
    if q_sd != 1 or o_sd != 1 or strides[3] != 1:
        raise ValueError("last dimension must be contiguous")
    nb, bs, hkv, d = key_cache.shape
    s_block, s_slot, s_head = strides[:3]
    if fp4:
        hkv, bs, d = bs, hkv, dq
        s_slot, s_head = s_head, s_slot
    if d != dq:
        raise ValueError(f"q has head size {dq}, the cache {d}")
    if out_rows < rows or out_heads != hq or out_d != dq:
        raise ValueError("out must have q's heads and head size, and no fewer rows than q")
    l_sh = l_st = 0
    if lse is not None:
        lse_heads, lse_rows = lse.shape
        if lse.dtype != torch.float32 or lse_heads < hq or lse_rows < rows:
            raise ValueError("lse must be float32 [num_q_heads, num_tokens]")
        l_sh, l_st = lse.stride()
    # (the kernels read a table row and an offset, or a query row, per sequence)
    num_seqs = seq_lens.shape[0]
    if table_rows < num_seqs:
        raise ValueError(f"block_table has {table_rows} rows for {num_seqs} sequences")
    if query_start_loc is None:
        if rows < num_seqs:
            raise ValueError(f"q has {rows} rows for {num_seqs} sequences")
    elif query_start_loc.shape[0] <= num_seqs or not query_start_loc.is_contiguous():
        raise ValueError(f"query_start_loc must be contiguous, with {num_seqs + 1} entries")
    if status is not None and (status.dtype != torch.int32 or not status.is_cuda):
        raise ValueError("status must be a CUDA int32 tensor")
    # packed in one go: setting the fields one by one costs a small call 8 us
    return _lib.PagedProblem.from_buffer_copy(_lib.PAGED_PROBLEM_STRUCT.pack(
        q.data_ptr(), q_st, q_sh, key_cache.data_ptr(), value_cache.data_ptr(), s_block, s_slot, s_head, nb,
        block_table.data_ptr(), table_st, table_cols, seq_lens.data_ptr(),
        query_start_loc.data_ptr() if query_start_loc is not None else 0, num_seqs,
        out.data_ptr(), o_st, o_sh, lse.data_ptr() if lse is not None else 0, l_sh, l_st,
        hq, hkv, d, bs, _DTYPES[dtype], float(softmax_scale), rows,
        status.data_ptr() if status is not None else 0,
        0, 0, 0, 0, 0, 0, 0,  # new_key .. slot_mapping: set by the caller
        _lib.PS_KV_NVFP4 if fp4 else _lib.PS_KV_FP8_E4M3 if fp8 else _lib.PS_KV_AUTO,
        _scale_ptr(k_scale) or 0, _scale_ptr(v_scale) or 0))


def paged_decode(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                 block_table: torch.Tensor, seq_lens: torch.Tensor, softmax_scale: float,
                 out: torch.Tensor, lse: torch.Tensor | None = None,
                 query_start_loc: torch.Tensor | None = None,
                 workspace: DecodeWorkspace | None = None,
                 new_key: torch.Tensor | None = None, new_value: torch.Tensor | None = None,
                 slot_mapping: torch.Tensor | None = None,
                 cascade: CascadePlan | None = None, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None, out_address: int | None = None,
                 head_gather: "_lib.HeadGatherProblem | None" = None,
                 score_mod: ScoreMod | None = None) -> torch.Tensor:
    """Decode attention, one query row per sequence, written into ``out``.

    q/out: [T, Hq, D]; caches [num_blocks, block_size, Hkv, D]; block_table
    int32 [B, P]; seq_lens int32 [B] (including the new token);
    query_start_loc int32 [B+1] or None (row b for sequence b); lse fp32
    [Hq, T] or None (natural log).  Calls that can overlap on the GPU must not
    share a workspace (the default one is shared by the calls of a stream, or of a
    captured graph: :func:`get_workspace`).

    ``new_key``/``new_value`` [T, Hkv, D] + ``slot_mapping`` int64 [T] fuse the
    KV append of the decode tokens into the same launch (same result as
    :func:`kv_append` followed by this call without them).

    ``cascade``: a :class:`CascadePlan` built by :func:`cascade_plan` for this
    batch; shared prefixes are then read once per group pass (same outputs).
    The workspace must then be a cascade workspace.

    fp8 caches (uint8 codes or float8_e4m3fn): attention over code * k_scale
    and code * v_scale (one-element float32 device tensors, None = 1); the
    fused append stores e4m3(x / scale).

    ``out_address``: write the output rows to this device address instead,
    contiguous [T, Hq, D] in ``out``'s dtype (``out`` then only supplies the
    dtype and shape) -- a peer-memory slab for :mod:`ps_attn.sharding`'s
    NVLink head gather.

    ``head_gather``: a filled ``ps_head_gather_problem`` -- this call is then
    one rank's part of a KV-head-sharded group and runs
    ``ps_paged_decode_head_gather`` (the group's rows land in
    ``head_gather.out`` on every rank; ``out`` only supplies shape and dtype).
    Used by :class:`ps_attn.sharding.FusedHeadGather`.

    nvfp4 caches (uint8, :func:`nvfp4_cache_shape`): attention over e2m1 *
    block scale * k_scale (v_scale); the fused append stores what
    :func:`kv_append` stores.

    ``score_mod``: a :class:`ScoreMod` (any cache dtype, with the fused append;
    not with ``cascade`` or ``head_gather``).  Pages below a sequence's visible
    range are neither read nor looked up.
    """
    lib = _lib.load()
    B = seq_lens.shape[0]
    fp4 = is_nvfp4_cache(key_cache, q.shape[-1])
    if (fp4 or score_mod is not None) and (cascade is not None or head_gather is not None):
        raise ValueError("nvfp4 caches and score modifiers take neither a cascade plan nor the fused head gather")
    hkv, d = (key_cache.shape[1], q.shape[2]) if fp4 else (key_cache.shape[2], key_cache.shape[3])
    if workspace is None:
        workspace = get_workspace(B, q.shape[1], hkv, d, q.device, cascade=cascade is not None)
    elif workspace.max_num_seqs < B:
        raise ValueError(f"workspace sized for {workspace.max_num_seqs} sequences < {B}")
    elif workspace.num_kv_heads not in (None, hkv):
        # partial rows of one head count would lie on the counters of another
        raise ValueError(f"workspace made for {workspace.num_kv_heads} kv heads, the call has {hkv}")
    if cascade is not None and cascade.num_seqs != B:
        raise ValueError(f"cascade plan built for {cascade.num_seqs} sequences, call has {B}")
    pr = _problem(q, key_cache, value_cache, block_table, seq_lens, query_start_loc,
                  softmax_scale, out, lse, k_scale=k_scale, v_scale=v_scale)
    if out_address is not None:
        if out_address % 16:
            raise ValueError("out_address must be 16-byte aligned")
        pr.out = out_address
        pr.out_stride_token, pr.out_stride_head = q.shape[1] * q.shape[2], q.shape[2]
    if new_key is not None:
        _require_cuda(new_key, new_value, slot_mapping)
        if new_value is None or slot_mapping is None:
            raise ValueError("fused append needs new_key, new_value and slot_mapping")
        if slot_mapping.dtype != torch.int64 or not slot_mapping.is_contiguous():
            raise ValueError("slot_mapping must be contiguous int64")
        if new_key.dtype != q.dtype or new_value.dtype != q.dtype:
            raise ValueError("new key/value must have the query dtype")
        if new_key.shape[1:] != (hkv, d) or new_value.shape[1:] != (hkv, d):
            raise ValueError("new key/value shape does not match the cache")
        if new_key.stride(-1) != 1 or new_value.stride(-1) != 1:
            raise ValueError("last dimension must be contiguous")
        if min(slot_mapping.shape[0], new_key.shape[0], new_value.shape[0]) < q.shape[0]:
            raise ValueError("fused append needs a key/value row and a slot per query row")
        pr.new_key = new_key.data_ptr()
        pr.new_key_stride_token, pr.new_key_stride_head = new_key.stride(0), new_key.stride(1)
        pr.new_value = new_value.data_ptr()
        pr.new_value_stride_token, pr.new_value_stride_head = new_value.stride(0), new_value.stride(1)
        pr.slot_mapping = slot_mapping.data_ptr()
    if head_gather is not None:
        if cascade is not None or out_address is not None:
            raise ValueError("the fused head gather runs the plain decode into its own output")
        _launch(q.device, lib.ps_paged_decode_head_gather, ctypes.byref(pr), workspace.buffer.data_ptr(),
                workspace.nbytes, ctypes.byref(head_gather), _stream_ptr(q.device))
    elif cascade is not None:
        _launch(q.device, lib.ps_paged_decode_cascade, ctypes.byref(pr), cascade.buffer.data_ptr(),
                cascade.nbytes, workspace.buffer.data_ptr(), workspace.nbytes, _stream_ptr(q.device))
    elif score_mod is not None:
        mod = score_mod._struct(q, B)
        _launch(q.device, lib.ps_paged_decode_mod, ctypes.byref(pr), ctypes.byref(mod),
                workspace.buffer.data_ptr(), workspace.nbytes, _stream_ptr(q.device))
    else:
        _launch(q.device, lib.ps_paged_decode, ctypes.byref(pr), workspace.buffer.data_ptr(),
                workspace.nbytes, _stream_ptr(q.device))
    return out


def dequant_gather(key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                   seq_lens: torch.Tensor, max_pages: int, dtype: torch.dtype,
                   k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                   status: torch.Tensor | None = None, out: tuple | None = None):
    """The pages ``seq_lens`` covers of an fp8 or nvfp4 cache, dequantized into a
    16-bit scratch cache: returns (key, value [B * max_pages, bs, Hkv, D] of
    ``dtype``, block table [B, max_pages] int32 into them).  Pages past a
    sequence's length are left uninitialised (never read).  Without scales
    the scratch holds the e4m3 values (nvfp4: code * block scale) exactly
    (attend over it with the scales); with them, code * scale rounded to
    ``dtype``.  ``out``: the (key, value) or (key, value, block table) of an
    earlier call of this shape to write into instead of new tensors, contiguous;
    the third result is then its block table (None for a pair): a caller that
    keeps the scratch keeps the table, which does not change."""
    lib = _lib.load()
    _require_cuda(key_cache, value_cache, block_table, seq_lens)
    if not is_fp8_cache(key_cache) or value_cache.dtype != key_cache.dtype:
        raise ValueError("dequant_gather reads an fp8 or nvfp4 cache")
    B = seq_lens.shape[0]
    nb, bs, hkv, d = key_cache.shape
    fp4 = is_nvfp4_cache(key_cache)
    if fp4:
        hkv, bs, d = bs, hkv, 128
    dev = key_cache.device
    if out is None:
        kd = torch.empty(B * max_pages, bs, hkv, d, dtype=dtype, device=dev)
        vd = torch.empty_like(kd)
    else:
        kd, vd = out[:2]
        for x in (kd, vd):
            if tuple(x.shape) != (B * max_pages, bs, hkv, d) or x.dtype != dtype or x.device != dev \
                    or not x.is_contiguous():
                raise ValueError(f"out must be contiguous [{B * max_pages}, {bs}, {hkv}, {d}] {dtype} on {dev}")
    if out is None:
        bt = torch.arange(B * max_pages, dtype=torch.int32, device=dev).view(B, max_pages)
    else:
        bt = out[2] if len(out) > 2 else None
    if B == 0 or max_pages == 0:
        return kd, vd, bt
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"scratch dtype {dtype} unsupported (fp16/bf16)")
    if key_cache.stride() != value_cache.stride() or key_cache.shape != value_cache.shape:
        raise ValueError("key_cache and value_cache must have the same shape and strides")
    if block_table.dtype != torch.int32 or seq_lens.dtype != torch.int32:
        raise ValueError("block_table and seq_lens must be int32")
    if block_table.shape[0] < B:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for {B} sequences")
    if block_table.stride(-1) != 1 or not seq_lens.is_contiguous() or key_cache.stride(-1) != 1:
        raise ValueError("block_table rows, seq_lens and the caches' last dimension must be contiguous")
    if status is not None and (status.dtype != torch.int32 or not status.is_cuda):
        raise ValueError("status must be a CUDA int32 tensor")
    if fp4:
        _check_nvfp4(key_cache, value_cache)
        s_block, s_head, s_slot = key_cache.stride()[:3]
    else:
        s_block, s_slot, s_head = key_cache.stride()[:3]
    pr = _lib.PagedProblem.from_buffer_copy(_lib.PAGED_PROBLEM_STRUCT.pack(
        0, 0, 0, key_cache.data_ptr(), value_cache.data_ptr(), s_block, s_slot, s_head, nb,
        block_table.data_ptr(), block_table.stride(0), block_table.shape[1], seq_lens.data_ptr(), 0, B,
        0, 0, 0, 0, 0, 0, hkv, hkv, d, bs, _DTYPES[dtype], 1.0, 0,
        status.data_ptr() if status is not None else 0, 0, 0, 0, 0, 0, 0, 0,
        _lib.PS_KV_NVFP4 if fp4 else _lib.PS_KV_FP8_E4M3, _scale_ptr(k_scale) or 0, _scale_ptr(v_scale) or 0))
    _launch(dev, lib.ps_kv_dequant_gather, ctypes.byref(pr), max_pages, kd.data_ptr(), vd.data_ptr(),
            _stream_ptr(dev))
    return kd, vd, bt


def merge_attn_states(output: torch.Tensor, prefix_output: torch.Tensor, prefix_lse: torch.Tensor,
                      suffix_output: torch.Tensor, suffix_lse: torch.Tensor,
                      output_lse: torch.Tensor | None = None) -> torch.Tensor:
    """vLLM's ``merge_attn_states`` (``vllm/v1/attention/ops/merge_attn_states.py:9``):
    two partial attentions of the same rows over disjoint keys, outputs
    [T, H, D] and LSEs [H, T] (fp32, contiguous), into ``output`` (may alias
    an input) and ``output_lse``."""
    lib = _lib.load()
    _require_cuda(output, prefix_output, prefix_lse, suffix_output, suffix_lse, output_lse)
    T, H, D = output.shape
    for t in (prefix_output, suffix_output):
        if t.dtype != output.dtype or tuple(t.shape) != (T, H, D) or t.stride(-1) != 1:
            raise ValueError("prefix/suffix outputs must match output [T, H, D]")
    for t in (prefix_lse, suffix_lse) + ((output_lse,) if output_lse is not None else ()):
        if t.dtype != torch.float32 or tuple(t.shape) != (H, T) or not t.is_contiguous():
            raise ValueError("LSEs must be contiguous float32 [H, T]")
    _launch(output.device, lib.ps_merge_attn_states,
            prefix_output.data_ptr(), prefix_output.stride(0), prefix_output.stride(1), prefix_lse.data_ptr(),
            suffix_output.data_ptr(), suffix_output.stride(0), suffix_output.stride(1), suffix_lse.data_ptr(),
            output.data_ptr(), output.stride(0), output.stride(1),
            output_lse.data_ptr() if output_lse is not None else None,
            T, H, D, _DTYPES[output.dtype], _stream_ptr(output.device))
    return output


def chunked_prefill(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                    block_table: torch.Tensor, seq_lens: torch.Tensor,
                    query_start_loc: torch.Tensor, softmax_scale: float, out: torch.Tensor,
                    lse: torch.Tensor | None = None,
                    status: torch.Tensor | None = None,
                    workspace: "DecodeWorkspace | None" = None,
                    k_scale: torch.Tensor | None = None,
                    v_scale: torch.Tensor | None = None,
                    score_mod: ScoreMod | None = None) -> torch.Tensor:
    """Causal (bottom-right) varlen attention over the paged cache; any q_len >= 1.

    ``k_scale``/``v_scale`` (one-element float32 device tensors): the cache
    is read as K * k_scale, V * v_scale -- attention over the unscaled
    scratch of :func:`dequant_gather` with an fp8 cache's scales.

    ``query_start_loc`` [B+1] holds absolute row offsets into ``q``/``out``
    (a slice of a larger batch's offsets is fine).  ``status`` (int32 [1],
    optional) receives PS_DEV_* bits from device-side checks.  With a
    ``workspace`` (a :class:`DecodeWorkspace` serves) the work units are
    handed out dynamically (``ps_chunked_prefill_ws``).

    ``score_mod``: a :class:`ScoreMod`; its ``key_start`` is indexed like the
    rows of ``q``, its ``prefix_lens`` like ``seq_lens``.  KV tiles that no row
    of a pair of 128-row tiles sees are skipped.
    """
    lib = _lib.load()
    if query_start_loc is None:
        raise ValueError("chunked_prefill needs query_start_loc")
    pr = _problem(q, key_cache, value_cache, block_table, seq_lens, query_start_loc,
                  softmax_scale, out, lse, status, k_scale=k_scale, v_scale=v_scale)
    if score_mod is not None:
        mod = score_mod._struct(q, seq_lens.shape[0])
        _launch(q.device, lib.ps_chunked_prefill_mod, ctypes.byref(pr), ctypes.byref(mod),
                workspace.buffer.data_ptr() if workspace is not None else None,
                workspace.nbytes if workspace is not None else 0, _stream_ptr(q.device))
    elif workspace is not None:
        _launch(q.device, lib.ps_chunked_prefill_ws, ctypes.byref(pr), workspace.buffer.data_ptr(),
                workspace.nbytes, _stream_ptr(q.device))
    else:
        _launch(q.device, lib.ps_chunked_prefill, ctypes.byref(pr), _stream_ptr(q.device))
    return out


def paged_attention(q, key_cache, value_cache, out, query_start_loc, max_query_len, seq_lens,
                    softmax_scale, block_table, lse=None, workspace=None, score_mod=None,
                    k_scale=None, v_scale=None):
    """``flash_attn_varlen_func``'s paged, causal call shape: route by ``max_query_len``.
    ``k_scale`` / ``v_scale``: an fp8 or nvfp4 cache's (single-row calls), or those of the
    cache that 16-bit pages were gathered from."""
    if max_query_len <= 1:
        return paged_decode(q, key_cache, value_cache, block_table, seq_lens, softmax_scale, out,
                            lse=lse, query_start_loc=query_start_loc, workspace=workspace,
                            score_mod=score_mod, k_scale=k_scale, v_scale=v_scale)
    return chunked_prefill(q, key_cache, value_cache, block_table, seq_lens, query_start_loc,
                           softmax_scale, out, lse=lse, score_mod=score_mod, k_scale=k_scale,
                           v_scale=v_scale)
