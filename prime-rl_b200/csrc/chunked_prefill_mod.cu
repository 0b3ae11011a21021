// Launch of the chunked prefill with score modifiers (the kernel:
// chunked_prefill_impl.cuh).  The cap and the bias each cost instructions on every
// score, so each has its own instantiation; the masks are one.
#include "chunked_prefill_impl.cuh"

namespace ps {
template <bool kBF16>
static int launch_mod(const PrefillParams& p, const CUtensorMap& qmap, const CUtensorMap& kmap,
                      const CUtensorMap& vmap, int grid, cudaStream_t stream) {
  const bool cap = p.mod.cap_log2 > 0.f, bias = p.mod.slopes != nullptr;
  if (cap && bias) return launch_prefill_t<kBF16, true, true, true>(p, qmap, kmap, vmap, grid, stream);
  if (cap) return launch_prefill_t<kBF16, true, true, false>(p, qmap, kmap, vmap, grid, stream);
  if (bias) return launch_prefill_t<kBF16, true, false, true>(p, qmap, kmap, vmap, grid, stream);
  return launch_prefill_t<kBF16, true, false, false>(p, qmap, kmap, vmap, grid, stream);
}
}  // namespace ps

int ps_launch_chunked_prefill_mod(const ps::PrefillParams& p, const CUtensorMap& qmap,
                                  const CUtensorMap& kmap, const CUtensorMap& vmap, int dtype_bf16,
                                  int grid, cudaStream_t stream) {
  return dtype_bf16 ? ps::launch_mod<true>(p, qmap, kmap, vmap, grid, stream)
                    : ps::launch_mod<false>(p, qmap, kmap, vmap, grid, stream);
}
