// Writing rows into a 4-bit (nvfp4) paged cache and reading pages back into a
// 16-bit scratch cache.  The format is described in nvfp4.cuh.
#include <climits>

#include "nvfp4.cuh"
#include "ps_launch.h"

namespace ps {

// Append.  Tokens are taken 16 at a time.  A thread has dims 8c .. 8c + 7 of one
// (K or V, head) and four of the tokens; their rows are loaded before the
// first quotient.  Where the 16 tokens' slots are consecutive, as a prompt's
// are, thread t of a page takes page positions 2t, 2t + 1, 2t + 8, 2t + 9: their V
// words are 16 consecutive bytes of the tile (8 where the tokens straddle two
// pages), and the two t of a warp fill a 32-byte sector.
// 16,384 tokens of 8 heads (86 MB): 32 us, 2.7 TB/s -- 19 us of it the rows' loads
// and their latency, 6 the stores, 8 the quantization.  64 registers (four CTAs per
// SM) against 79: 33 against 37 us.
constexpr int kFp4AppendGroup = 16;

template <bool kBF16>
__global__ void __launch_bounds__(256, 4) kv_append_nvfp4_kernel(const AppendArgs a, const float* k_scale,
                                                              const float* v_scale) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  constexpr int N = kFp4AppendGroup;
  const float ks = k_scale ? __ldg(k_scale) : 1.f;
  const float vs = v_scale ? __ldg(v_scale) : 1.f;
  const int lane = threadIdx.x & 31;
  const int per_group = 2 * a.num_heads * 64;            // threads: (K or V, head, t, c); whole warps
  const int chunks = (per_group + 255) / 256;            // of a CTA's size
  const int64_t groups = (a.num_tokens + N - 1) / N;
  for (int64_t u = blockIdx.x; u < groups * chunks; u += gridDim.x) {
    const int64_t group = u / chunks;
    const int chunk = static_cast<int>(u - group * chunks);
    const int64_t t0 = group * N;
    const int n = static_cast<int>(min(static_cast<int64_t>(N), a.num_tokens - t0));
    int64_t slot = lane < n ? __ldg(a.slot_mapping + t0 + lane) : -1;
    if (slot >= a.num_slots) {
      if (chunk == 0 && threadIdx.x < 32) set_status(a.status, PS_DEV_SLOT_OUT_OF_RANGE);
      slot = -1;
    }
    // lane i: byte offset of token i's tile in its head's part of a cache half
    // (one division per token and warp; a 64-bit one only in pools that need it)
    const int64_t s = max(slot, static_cast<int64_t>(0));
    const int64_t blk = a.num_slots <= INT_MAX ? static_cast<int64_t>(static_cast<uint32_t>(s) / static_cast<uint32_t>(a.block_size))
                                                 : s / a.block_size;
    const int64_t tile_off = blk * a.c_sblock + (static_cast<int>(s - blk * a.block_size) >> 4) * kFp4TileBytes;
    const int64_t slot0 = __shfl_sync(0xffffffffu, slot, 0);
    const bool run = __all_sync(0xffffffffu, lane >= N || (slot0 >= 0 && slot == slot0 + lane));
    const int j = chunk * 256 + threadIdx.x;
    if (j >= per_group) continue;  // (whole warps)
    const int c = j & 15, t = (j >> 4) & 3, rest = j >> 6;
    const bool is_v = rest >= a.num_heads;
    const int h = is_v ? rest - a.num_heads : rest;
    const char* src = (is_v ? a.value + h * a.val_sh : a.key + h * a.key_sh) + c * 16;
    const int64_t st = is_v ? a.val_st : a.key_st;
    const int shift = run ? static_cast<int>(slot0 & 15) : 0;
    int pos[4];  // page position of each token, < 0: not stored
    char* tile[4];
    uint4 v[4];
    char* base = (is_v ? a.value_cache : a.key_cache) + h * a.c_shead;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = (2 * t + (q & 1) + 8 * (q >> 1) - shift) & (N - 1);  // token of this page position
      pos[q] = __shfl_sync(0xffffffffu, slot < 0 ? -1 : static_cast<int>(slot & 15), i);
      tile[q] = base + __shfl_sync(0xffffffffu, tile_off, i);
      v[q] = i < n ? __ldg(reinterpret_cast<const uint4*>(src + (t0 + i) * st)) : make_uint4(0u, 0u, 0u, 0u);
    }
    uint32_t word[4], scale[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) quantize8_nvfp4<kBF16>(v[q], is_v ? vs : ks, word[q], scale[q]);
    if (is_v && run) {
      // positions 2t, 2t + 1 (q = 0, 1) and 2t + 8, 2t + 9: one page's, or the ends of two
      const int w_off = (c >> 3) * 512 + ((c & 7) * 4 + t) * 16;
      const int s_off = kFp4CodeBytes + ((c >> 1) & 3) * 32 + t * 8 + (c >> 3) * 4;
      if (tile[0] == tile[1] && tile[0] == tile[2] && tile[0] == tile[3]) {
        *reinterpret_cast<uint4*>(tile[0] + w_off) = make_uint4(word[0], word[1], word[2], word[3]);
        if ((c & 1) == 0)
          *reinterpret_cast<uint32_t*>(tile[0] + s_off) =
              scale[0] | (scale[1] << 8) | (scale[2] << 16) | (scale[3] << 24);
      } else {
#pragma unroll
        for (int q = 0; q < 4; q += 2) {
          if (tile[q] == tile[q + 1]) {
            *reinterpret_cast<uint2*>(tile[q] + w_off + q * 4) = make_uint2(word[q], word[q + 1]);
            if ((c & 1) == 0)
              *reinterpret_cast<uint16_t*>(tile[q] + s_off + q) = static_cast<uint16_t>(scale[q] | (scale[q + 1] << 8));
          } else {
#pragma unroll
            for (int i = q; i < q + 2; ++i) {
              *reinterpret_cast<uint32_t*>(tile[i] + w_off + i * 4) = word[i];
              if ((c & 1) == 0) tile[i][s_off + i] = static_cast<char>(scale[i]);
            }
          }
        }
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (pos[q] < 0) continue;
        *reinterpret_cast<uint32_t*>(tile[q] + fp4_word_offset(is_v, pos[q], c)) = word[q];
        if ((c & 1) == 0) tile[q][fp4_scale_offset(is_v, pos[q], c >> 1)] = static_cast<char>(scale[q]);
      }
    }
  }
}

// Gather: the pages a batch of sequences covers, as 16-bit values (code *
// block scale is exact in either 16-bit type; times the tensor's scale it is
// rounded once).  A warp takes the K and the V tile of one (page, head): all
// its loads are issued before the first conversion, and every store fills
// whole sectors of the scratch block's rows [slot][head][128].
template <bool kBF16>
__device__ __forceinline__ uint4 fp4_word_values(uint32_t word, __half2 block_scale, float s) {
  uint32_t x[4], o[4];
  e2m1x8_to_f16x2x4(word, x);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = __half22float2(__hmul2(as_half2(x[k]), block_scale));
    o[k] = pack2<kBF16>(f.x * s, f.y * s);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <bool kBF16>
__global__ void __launch_bounds__(256) kv_dequant_gather_nvfp4_kernel(const DequantArgs a, int num_heads,
                                                                      int64_t c_shead) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float ks = a.k_scale ? __ldg(a.k_scale) : 1.f;
  const float vs = a.v_scale ? __ldg(a.v_scale) : 1.f;
  const int lane = threadIdx.x & 31;
  const int spb = a.block_size >> 4;
  const int per_block = spb * num_heads;
  const int64_t units = static_cast<int64_t>(a.num_seqs) * a.max_pages * per_block;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  const int64_t row = static_cast<int64_t>(num_heads) * 256;
  const int g = lane >> 2, t = lane & 3;
  for (int64_t u = (static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5; u < units; u += step) {
    const int64_t page = u / per_block;  // b * max_pages + p
    const int rest = static_cast<int>(u - page * per_block);
    const int sub = rest / num_heads, h = rest - sub * num_heads;
    const int b = static_cast<int>(page / a.max_pages);
    const int p = static_cast<int>(page - static_cast<int64_t>(b) * a.max_pages);
    const int L = __ldg(a.seq_lens + b);
    if (static_cast<int64_t>(p) * a.block_size >= L) continue;
    if (p >= a.max_blocks_per_seq) {
      if (rest == 0 && lane == 0) set_status(a.status, PS_DEV_BAD_METADATA);
      continue;
    }
    const int blk = __ldg(a.block_table + static_cast<int64_t>(b) * a.bt_stride + p);
    if (blk < 0 || blk >= a.num_blocks) {
      if (rest == 0 && lane == 0) set_status(a.status, PS_DEV_BLOCK_OUT_OF_RANGE);
      continue;
    }
    const int64_t tile = blk * a.c_sblock + h * c_shead + sub * kFp4TileBytes;
    const char* kt = a.key_cache + tile;
    const char* vt = a.value_cache + tile;
    const int64_t first = ((page * a.block_size + sub * 16) * num_heads + h) * 256;
    // K: token 8m + g, dims 32i + 8t ..; V: tokens 2t, 2t + 1, 2t + 8, 2t + 9, dims 64m + 8g ..
    uint32_t kw[2][4], vw[2][4];
    uint2 ksc[2];
    uint32_t vsc[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        kw[m][i] = __ldg(reinterpret_cast<const uint32_t*>(kt + (8 * m + g) * 64 + i * 16 + t * 4));
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(vt + m * 512) + lane);
      vw[m][0] = w.x;
      vw[m][1] = w.y;
      vw[m][2] = w.z;
      vw[m][3] = w.w;
      ksc[m] = __ldg(reinterpret_cast<const uint2*>(kt + kFp4CodeBytes + (8 * m + g) * 8));
      vsc[m] = __ldg(reinterpret_cast<const uint32_t*>(vt + kFp4CodeBytes + (g >> 1) * 32 + t * 8 + m * 4));
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // block 2i + t / 2 of the token's eight
        const uint32_t two = ((i < 2 ? ksc[m].x : ksc[m].y) >> (i & 1) * 16) & 0xffffu;
        const uint32_t s2 = e4m3x2_to_f16x2(two);
        const __half2 s = t & 2 ? __high2half2(as_half2(s2)) : __low2half2(as_half2(s2));
        *reinterpret_cast<uint4*>(a.out_key + first + (8 * m + g) * row + i * 64 + t * 16) =
            fp4_word_values<kBF16>(kw[m][i], s, ks);
      }
      uint32_t s01, s23;
      e4m3x4_to_f16x2x2(vsc[m], s01, s23);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 pair = as_half2(i < 2 ? s01 : s23);
        *reinterpret_cast<uint4*>(a.out_value + first + ((i >> 1) * 8 + 2 * t + (i & 1)) * row + m * 128 + g * 16) =
            fp4_word_values<kBF16>(vw[m][i], i & 1 ? __high2half2(pair) : __low2half2(pair), vs);
      }
    }
  }
}

}  // namespace ps

int ps_launch_kv_append_nvfp4(const ps::AppendArgs& a, const float* k_scale, const float* v_scale,
                              int dtype_bf16, int sm_count, cudaStream_t stream) {
  if (a.num_tokens == 0) return 0;
  int64_t blocks = (a.num_tokens + ps::kFp4AppendGroup - 1) / ps::kFp4AppendGroup * ((2 * a.num_heads * 64 + 255) / 256);
  // (16 CTAs per SM, four of them resident: 32 us for the tokens above, 33 with 8 or 4)
  const int64_t cap = static_cast<int64_t>(sm_count) * 16;
  if (blocks > cap) blocks = cap;
  if (dtype_bf16)
    ps::kv_append_nvfp4_kernel<true><<<static_cast<int>(blocks), 256, 0, stream>>>(a, k_scale, v_scale);
  else
    ps::kv_append_nvfp4_kernel<false><<<static_cast<int>(blocks), 256, 0, stream>>>(a, k_scale, v_scale);
  return static_cast<int>(cudaGetLastError());
}

int ps_launch_kv_dequant_gather_nvfp4(const ps::DequantArgs& a, int num_heads, int64_t c_shead, int dtype_bf16,
                                      int sm_count, cudaStream_t stream) {
  const int64_t units = static_cast<int64_t>(a.num_seqs) * a.max_pages * (a.block_size / 16) * num_heads;
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
