// Launches of the paged split-KV decode: plain (16-bit and fp8 caches),
// shared-prefix (cascade) and with the head all-gather fused in.  The kernel
// is in paged_decode_impl.cuh; its instantiations with score modifiers are in
// paged_decode_mod.cu.
#include "paged_decode_impl.cuh"

int64_t ps_decode_partial_slots(int num_seqs, int num_kv_heads, int sm_count, int cascade, int fp8, int fp4) {
  // slot = global warp index + unit index; units: (sequence, kv head) and, in
  // cascade mode, at most one prefix segment per (sequence, kv head) more
  const int64_t units = static_cast<int64_t>(num_seqs) * num_kv_heads * (cascade ? 2 : 1);
  return static_cast<int64_t>(sm_count) * ps::kDecodeCtasPerSm *
             (fp4 ? ps::kDecodeFp4Warps : fp8 ? ps::kDecodeFp8Warps : ps::kDecodeWarps) + units;
}

namespace ps {
// Plain decode (no cascade plan): cache dtype x I/O dtype x query-column tiles.
template <bool kGather>
static int launch_plain(const DecodeParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap,
                        int dtype_bf16, int sm_count, cudaStream_t stream, int fp8_cache, int nt) {
  if (fp8_cache) {
    if (dtype_bf16)
      return nt == 1 ? launch_t<true, 1, false, true, kGather>(p, kmap, vmap, sm_count, stream)
                     : launch_t<true, 2, false, true, kGather>(p, kmap, vmap, sm_count, stream);
    return nt == 1 ? launch_t<false, 1, false, true, kGather>(p, kmap, vmap, sm_count, stream)
                   : launch_t<false, 2, false, true, kGather>(p, kmap, vmap, sm_count, stream);
  }
  if (dtype_bf16)
    return nt == 1 ? launch_t<true, 1, false, false, kGather>(p, kmap, vmap, sm_count, stream)
                   : launch_t<true, 2, false, false, kGather>(p, kmap, vmap, sm_count, stream);
  return nt == 1 ? launch_t<false, 1, false, false, kGather>(p, kmap, vmap, sm_count, stream)
                 : launch_t<false, 2, false, false, kGather>(p, kmap, vmap, sm_count, stream);
}
}  // namespace ps

int ps_launch_paged_decode(const ps::DecodeParams& p, const CUtensorMap& kmap,
                           const CUtensorMap& vmap, int dtype_bf16, int sm_count,
                           cudaStream_t stream, int fp8_cache) {
  const int nt = p.group <= 8 ? 1 : 2;
  if (p.cas_num_groups != nullptr && !fp8_cache && p.gather_world == 0) {
    // cascade: group <= 8 (checked by the caller)
    return dtype_bf16 ? ps::launch_t<true, 1, true>(p, kmap, vmap, sm_count, stream)
                      : ps::launch_t<false, 1, true>(p, kmap, vmap, sm_count, stream);
  }
  if (p.gather_world > 0)  // plain decode only (checked by the caller)
    return ps::launch_plain<true>(p, kmap, vmap, dtype_bf16, sm_count, stream, fp8_cache, nt);
  return ps::launch_plain<false>(p, kmap, vmap, dtype_bf16, sm_count, stream, fp8_cache, nt);
}
