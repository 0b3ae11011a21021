// Launch of the chunked prefill.  The kernel is in chunked_prefill_impl.cuh; its
// instantiations with score modifiers are in chunked_prefill_mod.cu.
#include "chunked_prefill_impl.cuh"

int ps_launch_chunked_prefill(const ps::PrefillParams& p, const CUtensorMap& qmap,
                              const CUtensorMap& kmap, const CUtensorMap& vmap, int dtype_bf16,
                              int grid, cudaStream_t stream) {
  if (p.k_scale != nullptr || p.v_scale != nullptr)
    return dtype_bf16 ? ps::launch_prefill_t<true, false, false, false, true>(p, qmap, kmap, vmap, grid, stream)
                      : ps::launch_prefill_t<false, false, false, false, true>(p, qmap, kmap, vmap, grid, stream);
  return dtype_bf16 ? ps::launch_prefill_t<true>(p, qmap, kmap, vmap, grid, stream)
                    : ps::launch_prefill_t<false>(p, qmap, kmap, vmap, grid, stream);
}
