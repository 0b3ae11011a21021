// The 4-bit ("nvfp4") KV-cache format: e2m1 codes with one e4m3 scale per 16
// dims and one fp32 scale per tensor; an element's value is
//   e2m1(code) * e4m3(block scale) * tensor scale.
// The counterpart of vLLM's kv_cache_dtype "nvfp4", whose rows take the same
// 72 bytes per token and head (64 of codes, 8 of scales; vllm/utils/
// torch_utils.py nvfp4_kv_cache_full_dim).
//
// Layout: a cache half is [num_blocks][num_kv_heads][block_size][72] bytes, in
// which the 16 tokens of a page of one head are one contiguous 1152-byte tile
// (copied 16 bytes a lane), ordered for the decode's tensor-core fragments so that
// a lane's operands are two 16-byte shared-memory loads:
//   K tile: codes of token r, dims d, d + 1 (d even; d in the low nibble) at
//           r * 64 + d / 2; scale of block k at 1024 + r * 8 + k.  A lane
//           takes 32 consecutive dims of a token, so it needs two scales.
//   V tile: token r = 8a + 2t + e, dims 64m + 8g .. + 7 are one 4-byte word at
//           m * 512 + (4g + t) * 16 + a * 8 + e * 4; the scale of block
//           4m + k at 1024 + k * 32 + t * 8 + m * 4 + a * 2 + e.
// Writing one token touches whole 4-byte words only, so tokens of a page can
// be appended by different threads without read-modify-write.
#pragma once

#include <cuda_fp4.h>

#include "ps_common.cuh"

namespace ps {

constexpr int kFp4TileBytes = 1152;      // 16 tokens of one head: 1024 of codes, 128 of scales
constexpr int kFp4CodeBytes = 1024;

// Offsets in a tile of the 4-byte word of dims 8c .. 8c + 7 and of the scale
// of block k, token r.
__device__ __forceinline__ int fp4_word_offset(bool value, int r, int c) {
  if (!value) return r * 64 + c * 4;
  return (c >> 3) * 512 + ((c & 7) * 4 + ((r & 7) >> 1)) * 16 + (r >> 3) * 8 + (r & 1) * 4;
}
__device__ __forceinline__ int fp4_scale_offset(bool value, int r, int k) {
  if (!value) return kFp4CodeBytes + r * 8 + k;
  return kFp4CodeBytes + (k & 3) * 32 + ((r & 7) >> 1) * 8 + (k >> 2) * 4 + (r >> 3) * 2 + (r & 1);
}

// Four bytes of code pairs to four f16x2 (low half from the low nibble).
// Every e2m1 value is exact in f16.
__device__ __forceinline__ void e2m1x8_to_f16x2x4(uint32_t v, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(v));
}

__device__ __forceinline__ uint32_t hmul2_u32(uint32_t a, __half2 b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ __half2 as_half2(uint32_t a) { return *reinterpret_cast<const __half2*>(&a); }

// e2m1 codes of eight values times m, in order from the low nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float2 (&f)[4], float m) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(f[0].x * m), "f"(f[0].y * m), "f"(f[1].x * m), "f"(f[1].y * m), "f"(f[2].x * m), "f"(f[2].y * m),
        "f"(f[3].x * m), "f"(f[3].y * m));
  return w;
}

// Warp-collective: eight model-dtype elements of a row per lane, lanes 2i and
// 2i + 1 holding one 16-dim block, to codes and the block's scale.
//   scale = e4m3(max|x| / (6 g)), codes = e2m1(x / (scale * g))
// -- quotients and products rounded to fp32, then to the nearest code, ties to
// even, saturating (a quotient, not a product with a reciprocal: 16-bit
// inputs land on ties of e2m1, which a rounded reciprocal would move).  A
// block whose scale rounds to zero stores zeros; a block with a NaN stores a
// NaN scale, so that reading it gives NaN as from a 16-bit cache.
//
// Only next to a tie are the divisions carried out: a product with an
// approximate reciprocal is within 2^-21 of the quotient, so where that product
// a little reduced and a little enlarged gives the same codes, the quotient
// gives them too.  (With a division for each element the append was 200
// instructions for 8 elements, and bound by them.)
constexpr float kNearLo = 1.f - 1.f / (1 << 19), kNearHi = 1.f + 1.f / (1 << 19);

template <bool kBF16>
__device__ __forceinline__ uint32_t max2_abs_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  a &= 0x7fff7fffu;
  b &= 0x7fff7fffu;
  if constexpr (kBF16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <bool kBF16>
__device__ __forceinline__ void quantize8_nvfp4(uint4 v, float g, uint32_t& word, uint32_t& scale) {
  // the block's largest magnitude, in the rows' own type (NaN if it has one)
  uint32_t m = max2_abs_nan<kBF16>(max2_abs_nan<kBF16>(v.x, v.y), max2_abs_nan<kBF16>(v.z, v.w));
  m = max2_abs_nan<kBF16>(m, __shfl_xor_sync(0xffffffffu, m, 1));
  const float2 mm = unpack2<kBF16>(m);
  float amax;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(amax) : "f"(mm.x), "f"(mm.y));
  const float six_g = __fmul_rn(6.f, g);
  const bool usual = six_g > 1e-30f && six_g < 1e30f;
  const float near = amax * rcp_approx(six_g);
  const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(near * kNearLo, near * kNearHi), __NV_SATFINITE, __NV_E4M3);
  scale = two & 0xffu;
  // (below 2^-9 a flushed subnormal could hide a tie)
  if (!usual || scale != two >> 8 || (near < 1e-30f && amax > 0.f))
    scale = __nv_cvt_float_to_fp8(__fdiv_rn(amax, six_g), __NV_SATFINITE, __NV_E4M3);
  if (amax != amax) scale = 0x7f;
  const __half_raw s16 = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(scale), __NV_E4M3);
  const float d = __fmul_rn(__half2float(__half(s16)), g);
  word = 0;
  if (d > 0.f) {
    const float2 f[4] = {unpack2<kBF16>(v.x), unpack2<kBF16>(v.y), unpack2<kBF16>(v.z), unpack2<kBF16>(v.w)};
    uint32_t hi = 1;
    if (d > 1e-30f && d < 1e30f) {
      const float inv = rcp_approx(d);
      word = e2m1x8(f, inv * kNearLo);
      hi = e2m1x8(f, inv * kNearHi);
    }
    if (word != hi) {
      word = 0;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
        const float2 x = unpack2<kBF16>(w);
        const uint32_t c = __nv_cvt_float2_to_fp4x2(make_float2(__fdiv_rn(x.x, d), __fdiv_rn(x.y, d)), __NV_E2M1,
                                                    cudaRoundNearest);
        word |= (c & 0xffu) << (8 * i);
      }
    }
  }
}

}  // namespace ps
