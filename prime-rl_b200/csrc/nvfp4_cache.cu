// Writing rows into a 4-bit (nvfp4) paged cache and reading pages back into a
// 16-bit scratch cache.  The format is described in nvfp4.cuh.
#include "nvfp4.cuh"
#include "ps_launch.h"

namespace ps {

// Append.  One thread per 8 dims of a (token, head) row of K or V; a CTA
// takes kFp4AppendTokens tokens per step and issues all their loads before the
// first quotient, so a step waits on memory once.
constexpr int kFp4AppendTokens = 4;

template <bool kBF16>
__global__ void __launch_bounds__(256) kv_append_nvfp4_kernel(const AppendArgs a, const float* k_scale,
                                                              const float* v_scale) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int U = kFp4AppendTokens;
  const float ks = k_scale ? __ldg(k_scale) : 1.f;
  const float vs = v_scale ? __ldg(v_scale) : 1.f;
  const int per_tensor = a.num_heads * 16;
  const int per_token = 2 * per_tensor;  // a multiple of 32: warps stay whole
  for (int64_t t0 = static_cast<int64_t>(blockIdx.x) * U; t0 < a.num_tokens;
       t0 += static_cast<int64_t>(gridDim.x) * U) {
    const int n = static_cast<int>(min(static_cast<int64_t>(U), a.num_tokens - t0));
    for (int j = threadIdx.x; j < per_token; j += blockDim.x) {
      const bool is_v = j >= per_tensor;
      const int r = is_v ? j - per_tensor : j;
      const int h = r >> 4, c = r & 15;
      const char* src = (is_v ? a.value + h * a.val_sh : a.key + h * a.key_sh) + c * 16;
      const int64_t st = is_v ? a.val_st : a.key_st;
      int64_t slot[U];
      uint4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        slot[u] = u < n ? __ldg(a.slot_mapping + t0 + u) : -1;
        v[u] = u < n ? __ldg(reinterpret_cast<const uint4*>(src + (t0 + u) * st)) : make_uint4(0u, 0u, 0u, 0u);
      }
      char* base = (is_v ? a.value_cache : a.key_cache) + h * a.c_shead;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (slot[u] < 0 || slot[u] >= a.num_slots) continue;  // (the same for the whole CTA)
        uint32_t word, scale;
        quantize8_nvfp4<kBF16>(v[u], is_v ? vs : ks, word, scale);
        const int64_t blk = slot[u] / a.block_size;
        const int off = static_cast<int>(slot[u] - blk * a.block_size);
        char* tile = base + blk * a.c_sblock + (off >> 4) * kFp4TileBytes;
        *reinterpret_cast<uint32_t*>(tile + fp4_word_offset(is_v, off & 15, c)) = word;
        if ((c & 1) == 0) tile[fp4_scale_offset(is_v, off & 15, c >> 1)] = static_cast<char>(scale);
      }
    }
    if (threadIdx.x < n && __ldg(a.slot_mapping + t0 + threadIdx.x) >= a.num_slots)
      set_status(a.status, PS_DEV_SLOT_OUT_OF_RANGE);
  }
}

// Gather: the pages a batch of sequences covers, as 16-bit values (code *
// block scale is exact in either 16-bit type; times the tensor's scale it is
// rounded once).  A warp takes one tile: its 1152 bytes are read as 16-byte
// words and written as rows of the scratch block [slot][head][128].
template <bool kBF16>
__global__ void __launch_bounds__(256) kv_dequant_gather_nvfp4_kernel(const DequantArgs a, int num_heads,
                                                                      int64_t c_shead) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float ks = a.k_scale ? __ldg(a.k_scale) : 1.f;
  const float vs = a.v_scale ? __ldg(a.v_scale) : 1.f;
  const int lane = threadIdx.x & 31;
  const int spb = a.block_size >> 4;
  const int per_block = spb * num_heads * 2;
  const int64_t units = static_cast<int64_t>(a.num_seqs) * a.max_pages * per_block;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t u = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; u < units; u += step) {
    const int64_t page = u / per_block;  // b * max_pages + p
    int rest = static_cast<int>(u - page * per_block);
    const int which = rest & 1;
    rest >>= 1;
    const int sub = rest / num_heads, h = rest - sub * num_heads;
    const int b = static_cast<int>(page / a.max_pages);
    const int p = static_cast<int>(page - static_cast<int64_t>(b) * a.max_pages);
    const int L = __ldg(a.seq_lens + b);
    if (static_cast<int64_t>(p) * a.block_size >= L) continue;
    if (p >= a.max_blocks_per_seq) {
      if (rest == 0 && which == 0 && lane == 0) set_status(a.status, PS_DEV_BAD_METADATA);
      continue;
    }
    const int blk = __ldg(a.block_table + static_cast<int64_t>(b) * a.bt_stride + p);
    if (blk < 0 || blk >= a.num_blocks) {
      if (rest == 0 && which == 0 && lane == 0) set_status(a.status, PS_DEV_BLOCK_OUT_OF_RANGE);
      continue;
    }
    const char* tile = (which ? a.value_cache : a.key_cache) + blk * a.c_sblock + h * c_shead + sub * kFp4TileBytes;
    const float s = which ? vs : ks;
    char* out = (which ? a.out_value : a.out_key) +
                ((page * a.block_size + sub * 16) * num_heads + h) * 256;
    const int64_t row = static_cast<int64_t>(num_heads) * 256;
    const uint4 w0 = __ldg(reinterpret_cast<const uint4*>(tile) + lane);
    const uint4 w1 = __ldg(reinterpret_cast<const uint4*>(tile + 512) + lane);
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const uint32_t w[4] = {m ? w1.x : w0.x, m ? w1.y : w0.y, m ? w1.z : w0.z, m ? w1.w : w0.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // K: token 8m + g, dims 32t + 8i ..; V: token 8(i / 2) + 2t + i % 2, dims 64m + 8g ..
        const int r = which ? (i >> 1) * 8 + 2 * t + (i & 1) : 8 * m + g;
        const int c = which ? 8 * m + g : 4 * t + i;
        const __half_raw sr = __nv_cvt_fp8_to_halfraw(
            static_cast<__nv_fp8_storage_t>(__ldg(tile + fp4_scale_offset(which != 0, r, c >> 1))), __NV_E4M3);
        const __half2 s2 = __half2half2(__half(sr));
        uint32_t x[4], o[4];
        e2m1x8_to_f16x2x4(w[i], x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = __half22float2(__hmul2(as_half2(x[k]), s2));
          o[k] = pack2<kBF16>(f.x * s, f.y * s);
        }
        *reinterpret_cast<uint4*>(out + r * row + c * 16) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
  }
}

}  // namespace ps

int ps_launch_kv_append_nvfp4(const ps::AppendArgs& a, const float* k_scale, const float* v_scale,
                              int dtype_bf16, int sm_count, cudaStream_t stream) {
  if (a.num_tokens == 0) return 0;
  int64_t blocks = (a.num_tokens + ps::kFp4AppendTokens - 1) / ps::kFp4AppendTokens;
  const int64_t cap = static_cast<int64_t>(sm_count) * 8;
  if (blocks > cap) blocks = cap;
  if (dtype_bf16)
    ps::kv_append_nvfp4_kernel<true><<<static_cast<int>(blocks), 256, 0, stream>>>(a, k_scale, v_scale);
  else
    ps::kv_append_nvfp4_kernel<false><<<static_cast<int>(blocks), 256, 0, stream>>>(a, k_scale, v_scale);
  return static_cast<int>(cudaGetLastError());
}

int ps_launch_kv_dequant_gather_nvfp4(const ps::DequantArgs& a, int num_heads, int64_t c_shead, int dtype_bf16,
                                      int sm_count, cudaStream_t stream) {
  const int64_t units = static_cast<int64_t>(a.num_seqs) * a.max_pages * (a.block_size / 16) * num_heads * 2;
  if (units == 0) return 0;
  int64_t g = (units + 7) / 8;
  const int64_t cap = 8LL * sm_count;
  if (g > cap) g = cap;
  if (dtype_bf16)
    ps::kv_dequant_gather_nvfp4_kernel<true><<<static_cast<unsigned>(g), 256, 0, stream>>>(a, num_heads, c_shead);
  else
    ps::kv_dequant_gather_nvfp4_kernel<false><<<static_cast<unsigned>(g), 256, 0, stream>>>(a, num_heads, c_shead);
  return static_cast<int>(cudaGetLastError());
}
