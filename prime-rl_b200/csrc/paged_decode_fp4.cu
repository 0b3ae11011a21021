// Paged split-KV decode over a 4-bit (nvfp4) cache, plain or with score
// modifiers.  Work list, split records and the fused combine are
// paged_decode_impl.cuh's; this file has the page format's loads and math.
//
// A page-head is 2304 bytes (K tile + V tile) against 8192 in 16 bits, so
// what bounds the kernel is the instruction stream that turns codes into
// tensor-core operands (each warp's own: 57 % of the issue slots are taken), not HBM.
// Hence:
//   - the unit of work is four pages of one (sequence, kv head): one wait, one
//     maximum and one rescale per unit; four more warps of a CTA do the copying;
//   - the tile layout (nvfp4.cuh) is the fragment order: a lane's K codes are
//     two 16-byte loads and its V codes two more, without ldmatrix;
//   - K: the reduction dims of the 8 MMA steps are permuted so that a lane
//     meets 32 consecutive dims of a token, i.e. two block scales (one
//     conversion per token) -- the query fragments carry the same permutation;
//   - V: two tokens' words are interleaved nibble by nibble (two shifts and two
//     selects per eight values) before the conversion, so that each
//     converted pair is already an MMA operand (consecutive tokens of a dim);
//   - e2m1 * e4m3 has 6 significant bits and lies in [2^-10, 2688]: the block
//     scale multiplies in f16 exactly, and every MMA operand but the query and
//     P is exact.  The query is scaled by a power of two per head into [-2, 2]
//     so that no 16-bit query overflows f16; the power goes into the score
//     scale.  P is rounded to f16 (2^-11).
// 40 sequences of 2k-32k tokens, 64 / 8 heads (459 MB): 112 us, 4.1 TB/s, 63 % of the
// measured copy rate; without the conversions, the scaling and the nibble
// interleaving 23 % less, without the MMAs 1 %.  64 of 1k-4k, 16 / 8 heads (158 MB):
// 48 us; one of 1,531: 13 us.
#include "nvfp4.cuh"
#include "paged_decode_impl.cuh"

namespace ps {

constexpr int kFp4Stages = kDecodeFp4Stages;
constexpr int kFp4Warps = kDecodeFp4Warps;   // streaming warps
// Pages of one unit: a unit costs a warp 180 instructions besides 260 a page, and
// four pages are what two stages of eight warps leave room for (units of two
// pages: 161 us where four take 134, before the copying warps).
constexpr int kFp4UnitPages = 4;
constexpr int kFp4StageBytes = 2 * kFp4UnitPages * kFp4TileBytes;  // K tiles, then V tiles
static_assert(kFp4UnitPages % 2 == 0, "the scale rows of a unit are copied four tiles at a time");
static_assert(kFp4StageBytes % 128 == 0, "stage alignment");
// Four more warps copy for the streaming warps, two each.  Copying is addresses and
// shuffles with little to overlap them, 1,000 of the 4,400 cycles a unit took a
// warp that did both.  Registers: 384 threads start with 168 each; the
// streaming warps take the copying warps' share (256 * 216 + 128 * 72 = 384 * 168).
constexpr int kFp4CopyWarps = 4, kFp4Feeds = kFp4Warps / kFp4CopyWarps;
constexpr int kFp4Threads = (kFp4Warps + kFp4CopyWarps) * 32;
constexpr int kFp4StreamRegs = 216, kFp4CopyRegs = 72;
static_assert(kFp4Warps == 8, "two warpgroups of streaming warps, one of copying warps");
static_assert(256 * kFp4StreamRegs + 128 * kFp4CopyRegs <= 384 * 168, "the launch's registers");

// 16 bytes global -> shared, asynchronous, through L2 only.
__device__ __forceinline__ void cp_async16(uint32_t smem_dst, const void* gsrc, uint64_t policy) {
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(smem_dst),
               "l"(reinterpret_cast<uint64_t>(gsrc)), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t smem_dst, const void* gsrc) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(gsrc))
               : "memory");
}
// This thread's arrival on `bar`, once its asynchronous copies so far are done.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Query slot: unpadded rows (they are read once per segment, and the padding
// would cost the 16-column kernel the room of its sequence table).
constexpr int kFp4QRowBytes = kHeadDim * 2;
template <int NT>
__host__ __device__ constexpr int fp4_qslot_bytes() {
  return 8 * NT * kFp4QRowBytes;
}
template <int NT>
__host__ __device__ constexpr int fp4_smem_bytes_before_table() {
  // stages | per-warp query slots | full and empty barriers
  return kFp4Warps * kFp4Stages * (kFp4StageBytes + fp4_qslot_bytes<NT>() + 16);
}

// Position in the list.  A segment (sequence, kv head) of P units takes P +
// kFp4SegCost positions, the last of them empty: what its end and the next
// segment's start cost a warp (partial rows, counter, query fragments: 4,000
// cycles, a unit 4,400), so that the equal cut also gives equal times to warps
// with more segment ends.  40 sequences of 2k-32k tokens, 64 / 8 heads: 120.4 us
// without, 117.3 with 1, 119.0 with 2, 120.7 with 4.
#ifndef PS_DECODE_FP4_SEG_COST
#define PS_DECODE_FP4_SEG_COST 1
#endif
constexpr int kFp4SegCost = PS_DECODE_FP4_SEG_COST;
struct Fp4Cursor {
  int b, h, p, P, off;
  int64_t v;  // position in the list
};

template <bool kMod, int kUnitTokens>
__device__ __forceinline__ void fp4_sequence(Fp4Cursor& c, const DecodeParams& p, const int* prefix) {
  c.P = seq_pages(prefix, c.b) - kFp4SegCost;
  c.off = 0;
  if constexpr (kMod) c.off = mod_first_unit(p, c.b, __ldg(p.seq_lens + c.b), kUnitTokens);
}

// Step to the next unit; c.v >= end afterwards (and nothing else of c valid)
// when there is none before `end`.
template <bool kMod, int kUnitTokens>
__device__ __forceinline__ void fp4_next(Fp4Cursor& c, const DecodeParams& p, const int* prefix, int64_t end) {
  ++c.v;
  if (++c.p < c.P) return;
  c.v += kFp4SegCost - (c.p - c.P);  // (a cursor placed on an empty position is past P already)
  c.p = 0;
  if (c.v >= end || ++c.h < p.num_kv_heads) return;
  c.h = 0;
  do ++c.b;
  while (seq_pages(prefix, c.b) == 0);
  fp4_sequence<kMod, kUnitTokens>(c, p, prefix);
}

// The segment that position v lies in and v's place there, which may be one of
// its empty positions (p >= P).
template <bool kMod, int kUnitTokens>
__device__ __forceinline__ Fp4Cursor fp4_locate(int64_t v, const DecodeParams& p, const int* prefix) {
  Fp4Cursor c;
  int lo = 0, hi = p.num_seqs - 1;  // largest b with prefix[b] * Hkv <= v
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (static_cast<int64_t>(prefix[mid]) * p.num_kv_heads <= v)
      lo = mid;
    else
      hi = mid - 1;
  }
  c.b = lo;
  c.v = v;
  const int V = seq_pages(prefix, lo);
  const int64_t r = v - static_cast<int64_t>(prefix[lo]) * p.num_kv_heads;
  c.h = static_cast<int>(r / V);
  c.p = static_cast<int>(r - static_cast<int64_t>(c.h) * V);
  fp4_sequence<kMod, kUnitTokens>(c, p, prefix);
  return c;
}

// First unit at or after position v; v < end <= the list's length.
template <bool kMod, int kUnitTokens>
__device__ __forceinline__ Fp4Cursor fp4_seek(int64_t v, int64_t end, const DecodeParams& p, const int* prefix) {
  Fp4Cursor c = fp4_locate<kMod, kUnitTokens>(v, p, prefix);
  if (c.p >= c.P) {  // an empty position: the next segment's first unit
    --c.v;
    --c.p;
    fp4_next<kMod, kUnitTokens>(c, p, prefix, end);
  }
  return c;
}

__device__ __forceinline__ SplitSeg fp4_split(const Fp4Cursor& c, int num_kv_heads, int64_t Qc) {
  const int64_t seg0 = c.v - c.p;
  SplitSeg g = {c.b, c.h, static_cast<int64_t>(c.b) * num_kv_heads + c.h, seg0 / Qc, 0};
  g.nsplit = static_cast<int>((seg0 + c.P - 1) / Qc - g.first_w + 1);
  return g;
}

// The copying side of one streaming warp (kept by a copying warp).  Its list
// positions are [pc.v, end).
struct Fp4Feed {
  Fp4Cursor pc;  // next unit to copy
  int64_t end;
  int k;         // units copied so far
  int pseg;      // segments started so far
  // Block-table entries are held 64 at a time, [bt_e0, bt_e0 + 64) of sequence
  // bt_b: the second half is loaded when the first comes into use, so that
  // only a new sequence waits for its entries.
  int bt_b, bt_e0, bt_reg, bt_next;
};

// Copy the next unit into its stage: two 512-byte warp copies of codes per tile,
// and one warp copy for the scale rows (128 bytes) of four tiles.  Pages past the
// sequence or below the visible range are neither copied nor looked up (their
// tokens are masked).  (Bulk copies, one per tile, cost 140 cycles each to
// issue: their operands are uniform, so lanes take turns.)
template <int NT, bool kMod>
__device__ __forceinline__ void fp4_copy_unit(Fp4Feed& f, const DecodeParams& p, uint8_t* wsm, uint8_t* wq,
                                              uint64_t* full, const int* prefix, uint64_t spb_inv, uint64_t kv_policy,
                                              int lane) {
  constexpr int D = kFp4Stages;
  constexpr int kUP = kFp4UnitPages;
  constexpr int SB = kFp4StageBytes;
  const Fp4Cursor& c = f.pc;
  const int spb = p.block_size / kPageTokens;
  const int stage = f.k % D;
  // page / spb without a division: spb is in [1, 16] and a page index below
  // 2^27, so the 2^32-scaled reciprocal, rounded up, is exact
  auto block_of = [&](int page) { return static_cast<int>((static_cast<uint64_t>(page) * spb_inv) >> 32); };
  auto entry = [&](int b, int idx) {
    return idx < p.max_blocks_per_seq ? __ldg(p.block_table + b * p.bt_stride + idx) : 0;
  };
  const int pg0 = (c.p + c.off) * kUP;
  int npg = kUP;
  if (c.p == c.P - 1) {  // only a sequence's last unit can be short
    const int L = max(__ldg(p.seq_lens + c.b), 0);
    npg = min(kUP, min((L + kPageTokens - 1) / kPageTokens, p.max_blocks_per_seq * spb) - pg0);
  }
  int skip = 0;
  if constexpr (kMod) skip = mod_skip_pages(p, c.b, pg0, c.p == 0);
  const int e0 = block_of(pg0);
  if (c.b != f.bt_b || e0 < f.bt_e0) {  // (another kv head starts over)
    f.bt_b = c.b;
    f.bt_e0 = e0;
    f.bt_reg = entry(c.b, e0 + lane);
    f.bt_next = entry(c.b, e0 + 32 + lane);
  } else if (e0 >= f.bt_e0 + 32) {
    f.bt_e0 += 32;
    f.bt_reg = f.bt_next;
    f.bt_next = entry(c.b, f.bt_e0 + 32 + lane);
  }
  // lane u < kUP: byte offset of page u's tile in either cache half
  const int pg = pg0 + min(lane, npg - 1), e = block_of(pg);
  // (shuffles take the lane index modulo 32)
  const int b_lo = __shfl_sync(0xffffffffu, f.bt_reg, e - f.bt_e0);
  const int b_hi = __shfl_sync(0xffffffffu, f.bt_next, e - f.bt_e0);
  int blk = e - f.bt_e0 < 32 ? b_lo : b_hi;
  if (blk < 0 || blk >= p.num_blocks) {
    if (lane >= skip && lane < npg) set_status(p.status, PS_DEV_BLOCK_OUT_OF_RANGE);
    blk = 0;
  }
  const int64_t tile = blk * p.c_sblock + c.h * p.c_shead + (pg - e * spb) * kFp4TileBytes;
  const char* kbase = static_cast<const char*>(p.key_cache);
  const char* vbase = static_cast<const char*>(p.value_cache);
  const uint32_t dst = smem_u32(wsm + stage * SB) + lane * 16;
#pragma unroll
  for (int u = 0; u < kUP; ++u) {
    const int64_t off = __shfl_sync(0xffffffffu, tile, u) + lane * 16;
    if (u >= skip && u < npg) {
      cp_async16(dst + u * kFp4TileBytes, kbase + off, kv_policy);
      cp_async16(dst + u * kFp4TileBytes + 512, kbase + off + 512, kv_policy);
      cp_async16(dst + (kUP + u) * kFp4TileBytes, vbase + off, kv_policy);
      cp_async16(dst + (kUP + u) * kFp4TileBytes + 512, vbase + off + 512, kv_policy);
    }
  }
#pragma unroll
  for (int i = 0; i < 2 * kUP; i += 4) {  // tile i + lane / 8 of K tiles, then V tiles
    const int x = i + (lane >> 3), u = x < kUP ? x : x - kUP;
    const int64_t off = __shfl_sync(0xffffffffu, tile, u) + kFp4CodeBytes + (lane & 7) * 16;
    if (u >= skip && u < npg)
      cp_async16(smem_u32(wsm + stage * SB) + x * kFp4TileBytes + kFp4CodeBytes + (lane & 7) * 16,
                 (x < kUP ? kbase : vbase) + off, kv_policy);
  }
  if (f.k == 0 || c.p == 0) {  // a segment starts for this warp: its query rows
    const int qrow = p.qsl ? __ldg(p.qsl + c.b) : c.b;
    const uint16_t* q =
        reinterpret_cast<const uint16_t*>(p.q) + qrow * p.q_st + static_cast<int64_t>(c.h) * p.group * p.q_sh;
    const uint32_t qdst = smem_u32(wq + (f.pseg % D) * fp4_qslot_bytes<NT>());
    for (int i = lane; i < p.group * 16; i += 32)
      cp_async16(qdst + i * 16, q + (i >> 4) * p.q_sh + (i & 15) * 8);
    ++f.pseg;
  }
  cp_async_arrive(full + stage);
  ++f.k;
  fp4_next<kMod, kUP * kPageTokens>(f.pc, p, prefix, f.end);
}

// A copying warp: keeps the rings of kFp4Feeds streaming warps full.
template <int NT, bool kMod>
__device__ __forceinline__ void fp4_copy_warp(const DecodeParams& p, const Tables& tb, int64_t total, int64_t gw0,
                                              uint8_t* smem, uint8_t* qslots, uint64_t* full, uint64_t* empty,
                                              int first, int lane) {
  constexpr int D = kFp4Stages;
  constexpr int kUnitTokens = kFp4UnitPages * kPageTokens;
  const int spb = p.block_size / kPageTokens;
  const uint64_t spb_inv = ((1ull << 32) + spb - 1) / spb;
  const uint64_t kv_policy = l2_policy_evict_first();
  Fp4Feed f[kFp4Feeds];
#pragma unroll
  for (int i = 0; i < kFp4Feeds; ++i) {
    const int64_t start = min(total, (gw0 + i) * tb.Qc);
    f[i].end = min(total, start + tb.Qc);
    f[i].k = f[i].pseg = f[i].bt_e0 = f[i].bt_reg = f[i].bt_next = 0;
    f[i].bt_b = -1;
    f[i].pc.v = f[i].end;
    if (start < f[i].end) f[i].pc = fp4_seek<kMod, kUnitTokens>(start, f[i].end, p, tb.prefix);
  }
  long long since = clock64();
  while (true) {
    bool more = false, copied = false;
#pragma unroll
    for (int i = 0; i < kFp4Feeds; ++i) {
      if (f[i].pc.v >= f[i].end) continue;
      more = true;
      const int ring = (first + i) * D;
      const int use = f[i].k / D;  // earlier uses of the stage, the last of which must have been released
      int free = 1;
      if (use > 0) {
        if (lane == 0) free = mbar_test(empty + ring + f[i].k % D, static_cast<uint32_t>((use - 1) & 1));
        free = __shfl_sync(0xffffffffu, free, 0);
        __syncwarp();  // lane 0's acquire orders the whole warp's copies
      }
      if (!free) continue;
      fp4_copy_unit<NT, kMod>(f[i], p, smem + ring * kFp4StageBytes, qslots + ring * fp4_qslot_bytes<NT>(),
                              full + ring, tb.prefix, spb_inv, kv_policy, lane);
      copied = true;
    }
    if (!more) break;
    if (copied) {
      since = clock64();
    } else if (clock64() - since > kWaitLimitCycles) {
      if (lane == 0) set_status(p.status, PS_DEV_WAIT_TIMEOUT);
      break;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// A streaming warp attends over the units of list positions [start, end).
template <bool kBF16, int NT, bool kMod>
__device__ __forceinline__ void stream_range_fp4(const DecodeParams& p, const Tables& tb, int64_t start, int64_t end,
                                                 int64_t gw, uint8_t* wsm, uint8_t* wq, uint64_t* full,
                                                 uint64_t* empty, int lane) {
  constexpr int kRec = 8 * NT;
  constexpr int D = kFp4Stages;
  constexpr int kUP = kFp4UnitPages;
  constexpr int kUnitTokens = kUP * kPageTokens;
  constexpr int SB = kFp4StageBytes;
  const int Hkv = p.num_kv_heads;
  const int group = p.group;
  const float k_scale = p.k_scale ? __ldg(p.k_scale) : 1.f;
  const float v_scale = p.v_scale ? __ldg(p.v_scale) : 1.f;
  const float scale_log2 = p.scale_log2 * k_scale;
  Fp4Cursor cc = fp4_seek<kMod, kUnitTokens>(start, end, p, tb.prefix);  // next unit to attend over

  const int g = lane >> 2, t = lane & 3;
  uint32_t qf[NT][8][2];
  float o[NT][8][4];
  float m[NT][2], l[NT][2];
  float sc[NT][2];     // score scale of this lane's head columns (exp2 domain)
  float slope[NT][2];  // score modifiers: bias slopes (times log2 e)
  int L = 0, key_low = 0, cseg = 0;
  int pending = 0;  // merges this warp owes: 1 its first segment's, 2 its last one's
  const bool fused = p.new_key != nullptr;
  uint4 new_row = make_uint4(0u, 0u, 0u, 0u);
  int64_t new_slot = -1;

  for (int k = 0; cc.v < end; ++k) {
    const int stage = k % D;
    uint8_t* st = wsm + stage * SB;
    if (!mbar_wait_bounded(full + stage, static_cast<uint32_t>((k / D) & 1))) {
      if (lane == 0) set_status(p.status, PS_DEV_WAIT_TIMEOUT);
      return;
    }

    // ---- segment start: query fragments, reset state ---------------------------
    if (k == 0 || cc.p == 0) {
      L = __ldg(p.seq_lens + cc.b);
      if constexpr (kMod) key_low = mod_key_low(p, cc.b, L);
      if (fused) {
        const int qrow = p.qsl ? __ldg(p.qsl + cc.b) : cc.b;
        new_slot = __ldg(p.slot_mapping + qrow);
        const int c = lane & 15;
        const uint16_t* src = lane < 16
            ? reinterpret_cast<const uint16_t*>(p.new_key) + qrow * p.nk_st + cc.h * p.nk_sh
            : reinterpret_cast<const uint16_t*>(p.new_value) + qrow * p.nv_st + cc.h * p.nv_sh;
        new_row = __ldg(reinterpret_cast<const uint4*>(src) + c);
      }
      const uint8_t* qs = wq + (cseg % D) * fp4_qslot_bytes<NT>();
      ++cseg;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        // head nt*8 + g; MMA step ks reduces dims 32t + 4ks .. + 3 of each lane
        const bool ok = nt * 8 + g < group;
        const uint4* row = reinterpret_cast<const uint4*>(qs + (nt * 8 + g) * kFp4QRowBytes + t * 64);
        float2 f[8][2];
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 w = ok ? row[i] : make_uint4(0u, 0u, 0u, 0u);
          f[2 * i][0] = unpack2<kBF16>(w.x);
          f[2 * i][1] = unpack2<kBF16>(w.y);
          f[2 * i + 1][0] = unpack2<kBF16>(w.z);
          f[2 * i + 1][1] = unpack2<kBF16>(w.w);
        }
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          mx = fmaxf(mx, fmaxf(fmaxf(fabsf(f[ks][0].x), fabsf(f[ks][0].y)),
                               fmaxf(fabsf(f[ks][1].x), fabsf(f[ks][1].y))));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // mx in [2^e, 2^(e+1)): the head's query is multiplied by 2^-e
        const int ex = min(max(__float_as_int(mx) >> 23, 1), 253);
        const float down = __int_as_float((254 - ex) << 23), up = __int_as_float(ex << 23);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          qf[nt][ks][0] = pack2<false>(f[ks][0].x * down, f[ks][0].y * down);
          qf[nt][ks][1] = pack2<false>(f[ks][1].x * down, f[ks][1].y * down);
        }
        // this lane's score columns are heads nt*8 + 2t, + 1: lane 4 * head has
        // that head's power (the raw score times it is the dot product)
        sc[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t);
        sc[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if constexpr (kMod) {
            const int col = nt * 8 + 2 * t + j;
            slope[nt][j] = p.mod.slopes != nullptr && col < group
                               ? __ldg(p.mod.slopes + cc.h * group + col) * 1.4426950408889634f
                               : 0.f;
          } else {
            sc[nt][j] *= scale_log2;
          }
          m[nt][j] = -INFINITY;
          l[nt][j] = 0.f;
        }
#pragma unroll
        for (int mi = 0; mi < 8; ++mi)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][mi][c] = 0.f;
      }
    }

    const int tok0 = (cc.p + cc.off) * kUnitTokens;
    const int valid = min(kUnitTokens, L - tok0);
    const int below = kMod ? key_low - tok0 : 0;

    // ---- fused append: the sequence's last unit carries the new token -------
    if (fused && cc.p == cc.P - 1 && new_slot >= 0) {
      const int pos = L - 1;
      const int bidx = pos / p.block_size;
      // (a length past the table, or a slot past the pool, is reported and not stored)
      const int64_t want =
          bidx < p.max_blocks_per_seq && new_slot < p.num_blocks * p.block_size
              ? static_cast<int64_t>(__ldg(p.block_table + cc.b * p.bt_stride + bidx)) * p.block_size +
                    (pos - bidx * p.block_size)
              : -1;
      if (new_slot == want) {
        // lanes 0-15: K dims 8c .. 8c + 7, lanes 16-31: V; into this stage's
        // copy of the tile and into the cache, as ps_kv_append_nvfp4 stores them
        const bool is_v = lane >= 16;
        const int c = lane & 15, r = pos & (kPageTokens - 1), u = (pos - tok0) / kPageTokens;
        uint32_t word, scale;
        quantize8_nvfp4<kBF16>(new_row, is_v ? v_scale : k_scale, word, scale);
        const int64_t blk = new_slot / p.block_size;
        const int off = static_cast<int>(new_slot - blk * p.block_size);
        uint8_t* tile = st + ((is_v ? kUP : 0) + u) * kFp4TileBytes;
        uint8_t* dst = static_cast<uint8_t*>(is_v ? p.value_cache : p.key_cache) + blk * p.c_sblock +
                       cc.h * p.c_shead + (off >> 4) * kFp4TileBytes;
        const int wo = fp4_word_offset(is_v, r, c);
        *reinterpret_cast<uint32_t*>(tile + wo) = word;
        *reinterpret_cast<uint32_t*>(dst + wo) = word;
        if ((c & 1) == 0) {
          const int so = fp4_scale_offset(is_v, r, c >> 1);
          tile[so] = static_cast<uint8_t>(scale);
          dst[so] = static_cast<uint8_t>(scale);
        }
      } else if (lane == 0) {
        set_status(p.status, PS_DEV_BAD_METADATA);
      }
      __syncwarp();
    }

    // ---- S^T = K Q^T --------------------------------------------------------------
    float s[kUP][NT][4];
#pragma unroll
    for (int u = 0; u < kUP; ++u) {
      // two accumulators, so that an MMA does not wait for the one before it
      float s1[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[u][nt][c] = s1[nt][c] = 0.f;
      const uint8_t* kt = st + u * kFp4TileBytes;
      // tokens g and g + 8, dims 32t .. 32t + 31
      const uint4 ka = *reinterpret_cast<const uint4*>(kt + lane * 16);
      const uint4 kb = *reinterpret_cast<const uint4*>(kt + 512 + lane * 16);
      const uint32_t sa = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(kt + kFp4CodeBytes + lane * 2));
      const uint32_t sb = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(kt + kFp4CodeBytes + 64 + lane * 2));
#pragma unroll
      for (int w = 0; w < 4; ++w) {  // 8 dims of each token: MMA steps 2w, 2w + 1
        const uint32_t wa = w == 0 ? ka.x : w == 1 ? ka.y : w == 2 ? ka.z : ka.w;
        const uint32_t wb = w == 0 ? kb.x : w == 1 ? kb.y : w == 2 ? kb.z : kb.w;
        const __half2 s_a = w < 2 ? __low2half2(as_half2(sa)) : __high2half2(as_half2(sa));
        const __half2 s_b = w < 2 ? __low2half2(as_half2(sb)) : __high2half2(as_half2(sb));
        uint32_t xa[4], xb[4];
        e2m1x8_to_f16x2x4(wa, xa);
        e2m1x8_to_f16x2x4(wb, xb);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xa[i] = hmul2_u32(xa[i], s_a);
          xb[i] = hmul2_u32(xb[i], s_b);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma_16816<false>(s[u][nt], xa[0], xb[0], xa[1], xb[1], qf[nt][2 * w][0], qf[nt][2 * w][1]);
          mma_16816<false>(s1[nt], xa[2], xb[2], xa[3], xb[3], qf[nt][2 * w + 1][0], qf[nt][2 * w + 1][1]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[u][nt][c] += s1[nt][c];
    }

    // ---- online softmax, one max / rescale per unit --------------------------------
    const bool edge = valid < kUnitTokens || below > 0;
    uint32_t pb[kUP][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int u = 0; u < kUP; ++u) {
        const int i0 = u * kPageTokens + g, i1 = i0 + 8;
        if constexpr (kMod) {
          const float d0 = static_cast<float>(tok0 + i0 - (L - 1)), d1 = d0 + 8.f;
          if (p.mod.cap_log2 > 0.f) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              s[u][nt][c] = mod_score<true>(p.mod, s[u][nt][c] * sc[nt][c & 1], scale_log2, slope[nt][c & 1],
                                            c < 2 ? d0 : d1);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              s[u][nt][c] = mod_score<false>(p.mod, s[u][nt][c] * sc[nt][c & 1], scale_log2, slope[nt][c & 1],
                                             c < 2 ? d0 : d1);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) s[u][nt][c] *= sc[nt][c & 1];
        }
        if (edge) {
          if (i0 >= valid || i0 < below) s[u][nt][0] = s[u][nt][1] = -INFINITY;
          if (i1 >= valid || i1 < below) s[u][nt][2] = s[u][nt][3] = -INFINITY;
        }
      }
      float alpha[2], mref[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = fmaxf(s[0][nt][j], s[0][nt][j + 2]);
#pragma unroll
        for (int u = 1; u < kUP; ++u) mx = fmaxf(mx, fmaxf(s[u][nt][j], s[u][nt][j + 2]));
        mx = warp_max_xor(mx, 0);
        const float mnew = fmaxf(m[nt][j], mx);
        mref[j] = kMod && mnew == -INFINITY ? 0.f : mnew;
        alpha[j] = ex2(m[nt][j] - mref[j]);  // m = -inf -> 0
        m[nt][j] = mnew;
        l[nt][j] *= alpha[j];
      }
#pragma unroll
      for (int u = 0; u < kUP; ++u) {
        const float p0 = ex2(s[u][nt][0] - mref[0]);
        const float p1 = ex2(s[u][nt][1] - mref[1]);
        const float p2 = ex2(s[u][nt][2] - mref[0]);
        const float p3 = ex2(s[u][nt][3] - mref[1]);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        pb[u][nt][0] = movmatrix_t(pack2<false>(p0, p1));
        pb[u][nt][1] = movmatrix_t(pack2<false>(p2, p3));
      }
      if (alpha[0] != 1.f || alpha[1] != 1.f) {
#pragma unroll
        for (int mi = 0; mi < 8; ++mi) {
          o[nt][mi][0] *= alpha[0];
          o[nt][mi][1] *= alpha[1];
          o[nt][mi][2] *= alpha[0];
          o[nt][mi][3] *= alpha[1];
        }
      }
    }

    // ---- O^T += V^T P^T: output tile 4m + j has dims 64m + 8g + 2j (row g) and
    // + 1 (row g + 8); the lane's tokens are 2t, 2t + 1, 2t + 8, 2t + 9 ----------
#pragma unroll
    for (int u = 0; u < kUP; ++u) {
      const uint8_t* vt = st + (kUP + u) * kFp4TileBytes;
      const uint2 sv = *reinterpret_cast<const uint2*>(vt + kFp4CodeBytes + (g >> 1) * 32 + t * 8);
      uint32_t m01 = 0xffffffffu, m23 = 0xffffffffu;
      if (edge) {  // P is 0 there: keep stale scales (NaN codes among them) out
        const int i = u * kPageTokens + 2 * t;
        auto out = [&](int x) { return x >= valid || x < below; };
        m01 = (out(i) ? 0u : 0xffffu) | (out(i + 1) ? 0u : 0xffff0000u);
        m23 = (out(i + 8) ? 0u : 0xffffu) | (out(i + 9) ? 0u : 0xffff0000u);
      }
#pragma unroll
      for (int mq = 0; mq < 2; ++mq) {
        const uint4 w = *reinterpret_cast<const uint4*>(vt + mq * 512 + lane * 16);
        uint32_t s01, s23;
        e4m3x4_to_f16x2x2(mq ? sv.y : sv.x, s01, s23);
        s01 &= m01;
        s23 &= m23;
        constexpr uint32_t kLo = 0x0f0f0f0fu;
        uint32_t e01[4], d01[4], e23[4], d23[4];  // even and odd dims of the token pairs
        e2m1x8_to_f16x2x4((w.x & kLo) | ((w.y << 4) & ~kLo), e01);
        e2m1x8_to_f16x2x4(((w.x >> 4) & kLo) | (w.y & ~kLo), d01);
        e2m1x8_to_f16x2x4((w.z & kLo) | ((w.w << 4) & ~kLo), e23);
        e2m1x8_to_f16x2x4(((w.z >> 4) & kLo) | (w.w & ~kLo), d23);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a0 = hmul2_u32(e01[j], as_half2(s01)), a1 = hmul2_u32(d01[j], as_half2(s01));
          const uint32_t a2 = hmul2_u32(e23[j], as_half2(s23)), a3 = hmul2_u32(d23[j], as_half2(s23));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_16816<false>(o[nt][4 * mq + j], a0, a1, a2, a3, pb[u][nt][0], pb[u][nt][1]);
        }
      }
    }
    __syncwarp();

    // ---- the stage may be filled again ----------------------------------------
    if (lane == 0) mbar_arrive(empty + stage);

    // ---- segment end: finalize ---------------------------------------------------
    const Fp4Cursor at = cc;
    fp4_next<kMod, kUnitTokens>(cc, p, tb.prefix, end);
    if (at.p == at.P - 1 || cc.v >= end) {
      const int b = at.b, h = at.h;
      const SplitSeg sg = fp4_split(at, Hkv, tb.Qc);
      const int nsplit = sg.nsplit;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float lt = warp_sum_xor_4_8_16(l[nt][j]);
          const bool zero = (lt == 0.f) || (lt != lt);
          const float inv = zero ? 0.f : v_scale / lt;
          const float lse = zero ? -INFINITY : (m[nt][j] + __log2f(lt)) * 0.6931471805599453f;
          const int col = nt * 8 + 2 * t + j;
          if (col >= group) continue;
          if (nsplit == 1) {
            const int qrow = p.qsl ? __ldg(p.qsl + b) : b;
            const int qh = h * group + col;
            char* ob = static_cast<char*>(p.out) + (qrow * p.o_st + qh * p.o_sh + 8 * g) * 2;
#pragma unroll
            for (int mq = 0; mq < 2; ++mq) {
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                w[i] = pack2<kBF16>(o[nt][4 * mq + i][j] * inv, o[nt][4 * mq + i][j + 2] * inv);
              *reinterpret_cast<uint4*>(ob + mq * 128) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (g == 0 && p.lse) p.lse[qh * p.lse_sh + qrow * p.lse_st] = lse;
          } else {
            const int64_t slot = gw + sg.unit;
            float4* po = reinterpret_cast<float4*>(slot_o<kRec>(p, slot, col) + 8 * g);
#pragma unroll
            for (int mq = 0; mq < 2; ++mq)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                po[mq * 16 + i] = make_float4(o[nt][4 * mq + 2 * i][j] * inv, o[nt][4 * mq + 2 * i][j + 2] * inv,
                                              o[nt][4 * mq + 2 * i + 1][j] * inv, o[nt][4 * mq + 2 * i + 1][j + 2] * inv);
            if (g == 0) *slot_lse<kRec>(p, slot, col) = lse;
          }
        }
      if (nsplit > 1 && count_record(p, sg, gw, lane)) pending |= at.v - at.p < start ? 1 : 2;
    }
  }
  for (int i = 1; i <= 2; ++i)
    if (pending & i) {
      const Fp4Cursor c = fp4_locate<kMod, kUnitTokens>(i == 1 ? start : end - 1, p, tb.prefix);
      merge_split<kBF16, kRec, false>(p, fp4_split(c, Hkv, tb.Qc), gw, lane);
    }
}

template <bool kBF16, int NT, bool kMod>
__global__ void __launch_bounds__(kFp4Threads, 1) paged_decode_fp4_kernel(const __grid_constant__ DecodeParams p) {
  constexpr int D = kFp4Stages, W = kFp4Warps;
  constexpr int kUP = kFp4UnitPages, kUnitTokens = kUP * kPageTokens, SB = kFp4StageBytes;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* qslots = smem + W * D * SB;
  uint64_t* full = reinterpret_cast<uint64_t*>(qslots + W * D * fp4_qslot_bytes<NT>());
  uint64_t* empty = full + W * D;
  int* prefix = reinterpret_cast<int*>(empty + W * D);
  __shared__ int s_warp_tot[kFp4Threads / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int B = p.num_seqs, Hkv = p.num_kv_heads;
  const int spb = p.block_size / kPageTokens;
  if (tid < W * D) {
    mbar_init(full + tid, 32);  // every lane of the copying warp
    mbar_init(empty + tid, 1);
    fence_mbar_init();
  }
  // the launch overlaps the previous kernel in the stream up to here
  asm volatile("griddepcontrol.wait;" ::: "memory");

  Tables tb = {};
  tb.prefix = prefix;

  // ---- prologue: units per sequence and their exclusive prefix sum -------------
  const int per = (B + blockDim.x - 1) / blockDim.x;
  const int b_lo = min(B, tid * per), b_hi = min(B, b_lo + per);
  auto units_of = [&](int b) {
    const int P = (own_pages_of(p, b, spb) + kUP - 1) / kUP;
    int real = P;
    if constexpr (kMod)
      real = P > 0 ? max(0, P - mod_first_unit(p, b, __ldg(p.seq_lens + b), kUnitTokens)) : 0;
    return real > 0 ? real + kFp4SegCost : 0;  // list positions per kv head
  };
  int bad = 0, local = 0;
  for (int b = b_lo; b < b_hi; ++b) {
    const int L = __ldg(p.seq_lens + b);
    const int qlen = p.qsl ? __ldg(p.qsl + b + 1) - __ldg(p.qsl + b) : 1;
    if (qlen == 1)
      bad |= L < 0 || (max(L, 0) + kPageTokens - 1) / kPageTokens > p.max_blocks_per_seq * spb;
    else
      bad |= qlen != 0;  // multi-token queries belong to the prefill kernel
    local += units_of(b);
  }
  int total_units;
  int run = block_exclusive_scan(local, s_warp_tot, &total_units);
  for (int b = b_lo; b < b_hi; ++b) {
    prefix[b] = run;
    run += units_of(b);
  }
  if (tid == 0) prefix[B] = total_units;
  const int any_bad = __syncthreads_or(bad);
  if (tid == 0 && any_bad) set_status(p.status, PS_DEV_BAD_METADATA);
  const int64_t total = static_cast<int64_t>(total_units) * Hkv;
  const int64_t nwarps = static_cast<int64_t>(gridDim.x) * W;
  tb.Qc = max(static_cast<int64_t>(1), (total + nwarps - 1) / nwarps);

  // ---- empty sequences (q_len 1, seq_len 0): zero output, LSE -inf ---------------
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + tid; i < static_cast<int64_t>(B) * p.num_q_heads;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int b = static_cast<int>(i / p.num_q_heads);
    if (prefix[b + 1] != prefix[b]) continue;
    const int qh = static_cast<int>(i - static_cast<int64_t>(b) * p.num_q_heads);
    if (p.qsl && __ldg(p.qsl + b + 1) - __ldg(p.qsl + b) != 1) continue;
    const int qrow = p.qsl ? __ldg(p.qsl + b) : b;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<char*>(p.out) + (qrow * p.o_st + qh * p.o_sh) * 2);
    for (int d = 0; d < 16; ++d) dst[d] = make_uint4(0u, 0u, 0u, 0u);
    if (p.lse) p.lse[qh * p.lse_sh + qrow * p.lse_st] = -INFINITY;
  }

  // (the scan's barriers order the mbarriers' initialisation)
  if (warp >= W) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp4CopyRegs));
    const int first = (warp - W) * kFp4Feeds;
    if (first < W)
      fp4_copy_warp<NT, kMod>(p, tb, total, static_cast<int64_t>(blockIdx.x) * W + first, smem, qslots, full, empty,
                              first, lane);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp4StreamRegs));
    const int64_t gw = static_cast<int64_t>(blockIdx.x) * W + warp;
    const int64_t start = min(total, gw * tb.Qc), end = min(total, start + tb.Qc);
    if (start < end)
      stream_range_fp4<kBF16, NT, kMod>(p, tb, start, end, gw, smem + warp * D * SB,
                                        qslots + warp * D * fp4_qslot_bytes<NT>(), full + warp * D, empty + warp * D,
                                        lane);
  }
}

template <bool kBF16, int NT, bool kMod>
static int launch_fp4(const DecodeParams& p, int sm_count, cudaStream_t stream) {
  constexpr int base = fp4_smem_bytes_before_table<NT>();
  static_assert(base + (kDecodeMaxSeqs + 1) * 4 + 256 <= 232448, "shared memory");
  static bool configured[64] = {false};  // the attribute is per function and per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= 64) return static_cast<int>(cudaErrorInvalidDevice);
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(paged_decode_fp4_kernel<kBF16, NT, kMod>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               base + (kDecodeMaxSeqs + 1) * 4);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sm_count);
  cfg.blockDim = dim3(kFp4Threads);
  cfg.dynamicSmemBytes = base + static_cast<size_t>(p.num_seqs + 1) * 4;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_decode_fp4_kernel<kBF16, NT, kMod>, p);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}

template <bool kBF16, bool kMod>
static int launch_fp4_group(const DecodeParams& p, int sm_count, cudaStream_t stream) {
  return p.group <= 8 ? launch_fp4<kBF16, 1, kMod>(p, sm_count, stream)
                      : launch_fp4<kBF16, 2, kMod>(p, sm_count, stream);
}

}  // namespace ps

int ps_launch_paged_decode_fp4(const ps::DecodeParams& p, int dtype_bf16, int sm_count, cudaStream_t stream,
                               int modded) {
  if (modded)
    return dtype_bf16 ? ps::launch_fp4_group<true, true>(p, sm_count, stream)
                      : ps::launch_fp4_group<false, true>(p, sm_count, stream);
  return dtype_bf16 ? ps::launch_fp4_group<true, false>(p, sm_count, stream)
                    : ps::launch_fp4_group<false, false>(p, sm_count, stream);
}
