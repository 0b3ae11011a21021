// Launches of the paged split-KV decode with score modifiers: tanh cap, bias
// that falls with the distance, sliding window, document mask.  The kernel is
// paged_decode_impl.cuh's in its kModded mode: the page-head list holds only
// the units from each sequence's first visible key on, so a sliding window of
// window_left = W (W + 1 keys) reads at most (W + 15) / 16 + 1 pages of a sequence
// however long it is.
#include "paged_decode_impl.cuh"

namespace ps {
template <bool kBF16, bool kFP8>
static int launch_mod(const DecodeParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap, int sm_count,
                      cudaStream_t stream) {
  return p.group <= 8 ? launch_t<kBF16, 1, false, kFP8, false, true>(p, kmap, vmap, sm_count, stream)
                      : launch_t<kBF16, 2, false, kFP8, false, true>(p, kmap, vmap, sm_count, stream);
}
}  // namespace ps

int ps_launch_paged_decode_mod(const ps::DecodeParams& p, const CUtensorMap& kmap, const CUtensorMap& vmap,
                               int dtype_bf16, int sm_count, cudaStream_t stream, int fp8_cache) {
  if (fp8_cache)
    return dtype_bf16 ? ps::launch_mod<true, true>(p, kmap, vmap, sm_count, stream)
                      : ps::launch_mod<false, true>(p, kmap, vmap, sm_count, stream);
  return dtype_bf16 ? ps::launch_mod<true, false>(p, kmap, vmap, sm_count, stream)
                    : ps::launch_mod<false, false>(p, kmap, vmap, sm_count, stream);
}
