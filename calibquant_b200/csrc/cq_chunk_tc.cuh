// Tiles of packed or full-precision keys and values as operands of tcgen05.mma, for the chunk attention and the key weights.
//
// A tile is 128 x 128 numbers of 16 bits: two panels of [128 rows][128 bytes], 128-byte swizzled.  Packed keys have a channel per row and
// tokens along it, packed values a token per row and channels along it: in both a 32-bit word of codes is eight numbers = one 16-byte
// chunk of a row, and four words share scale and minimum.  Full-precision rows have a token per row.
#pragma once

#include "cq_chunk.cuh"
#include "cq_ptx.cuh"
#include "cq_tc.cuh"

namespace cq {
namespace chunk {

constexpr int PANEL_BYTES = 128 * 128;
constexpr int TILE_BYTES = 2 * PANEL_BYTES;

// 16-byte chunk c (0..15) of row r
__device__ __forceinline__ uint32_t chunk_at(uint32_t tile, int r, int c) {
  return tile + (uint32_t)((c >> 3) * PANEL_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// What one lane holds of a packed tile: 32 codes of a row (one group) and their scale and minimum.
struct Unit {
  uint4 w;
  uint16_t scale, mn;
};

template <bool BF16>
__device__ __forceinline__ float number(uint16_t bits) {
  return BF16 ? __uint_as_float((uint32_t)bits << 16) : __half2float(__ushort_as_half(bits));
}

// Two numbers as 16-bit pairs whose sum they are: hi is the number cut off, lo the rest rounded.  A value scale * code + minimum has
// up to 16 bits in all cases but those where the minimum is hundreds of scales away from zero, and is exact then.
template <bool BF16>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  if (BF16) {
    hi = ptx::prmt(__float_as_uint(a), __float_as_uint(b), 0x7632);
    const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(rb), "f"(ra));
  } else {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(b), "f"(a));
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(b - h.y), "f"(a - h.x));
  }
}

// code N (0..7) of a word as the float 16 + code
template <int N>
__device__ __forceinline__ float code16(uint32_t w) {
  constexpr int sh = 19 - 4 * N;
  const uint32_t s = sh >= 0 ? w << (sh >= 0 ? sh : 0) : w >> (sh < 0 ? -sh : 0);
  return __uint_as_float((s & 0x00780000u) | 0x41800000u);
}

// Eight keys of a channel, scale * code + minimum exactly in fp32, as chunks of the two tiles whose sum they are.
template <bool BF16>
__device__ __forceinline__ void keys_of_word(uint32_t w, float s, float off, uint32_t (&hi)[4], uint32_t (&lo)[4]) {      // off = minimum - 16 scale
  split_pair<BF16>(fmaf(code16<0>(w), s, off), fmaf(code16<1>(w), s, off), hi[0], lo[0]);
  split_pair<BF16>(fmaf(code16<2>(w), s, off), fmaf(code16<3>(w), s, off), hi[1], lo[1]);
  split_pair<BF16>(fmaf(code16<4>(w), s, off), fmaf(code16<5>(w), s, off), hi[2], lo[2]);
  split_pair<BF16>(fmaf(code16<6>(w), s, off), fmaf(code16<7>(w), s, off), hi[3], lo[3]);
}

// Eight values of a token, scale * code + minimum rounded once, in the order 0 4 1 5 2 6 3 7 (codes four nibbles apart come out of a
// word as a pair).
template <bool BF16>
__device__ __forceinline__ void values_of_word(uint32_t w, uint32_t s2, uint32_t m2, uint32_t (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t c = ((w >> (4 * j)) & 0x000f000fu) | (BF16 ? 0x43004300u : 0x64006400u);      // 128 + code, 1024 + code
    if (BF16) {
      uint32_t t;
      asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(t) : "r"(c), "r"(0x43004300u));
      asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(v[j]) : "r"(t), "r"(s2), "r"(m2));
    } else {
      uint32_t t;
      asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(t) : "r"(c), "r"(0x64006400u));
      v[j] = ptx::hfma2_u32(t, s2, m2);
    }
  }
}
// the same order for a chunk of full-precision values
__device__ __forceinline__ void order_values(uint4& x) {
  const uint32_t a = x.x, b = x.y, c = x.z, d = x.w;      // (0,1) (2,3) (4,5) (6,7)
  x = make_uint4(ptx::prmt(a, c, 0x5410), ptx::prmt(a, c, 0x7632), ptx::prmt(b, d, 0x5410), ptx::prmt(b, d, 0x7632));
}

// ---- units: lane = (row 8 u + lane / 4, group lane % 4), u = 0..15 of a tile -------------------------------------------------------
// `tile` counts tiles of 128 visual tokens; what lies behind the last token is zero.
__device__ __forceinline__ void load_k_unit(const Params& p, int64_t bh, int tile, int u, int lane, Unit& x) {
  const int g = tile * 4 + (lane & 3), groups = p.t_vis >> 5;
  const int64_t at = (bh * 128 + u * 8 + (lane >> 2)) * groups + g;
  x.w = make_uint4(0, 0, 0, 0);
  x.scale = x.mn = 0;
  if (g < groups) {
    x.w = reinterpret_cast<const uint4*>(p.k_code)[at];
    x.scale = static_cast<const uint16_t*>(p.k_scale)[at];
    x.mn = static_cast<const uint16_t*>(p.k_mn)[at];
  }
}
__device__ __forceinline__ void load_v_unit(const Params& p, int64_t bh, int tile, int u, int lane, bool live, Unit& x) {
  const int t = tile * 128 + u * 8 + (lane >> 2);
  const int64_t at = (bh * p.t_vis + t) * 4 + (lane & 3);
  x.w = make_uint4(0, 0, 0, 0);
  x.scale = x.mn = 0;
  if (t < p.t_vis && live) {
    x.w = reinterpret_cast<const uint4*>(p.v_code)[at];
    x.scale = static_cast<const uint16_t*>(p.v_scale)[at];
    x.mn = static_cast<const uint16_t*>(p.v_mn)[at];
  }
}
// Chunk order of a lane: lanes of groups 2 and 3 write their words in the order 2 3 0 1, so that the 16-byte stores of eight lanes
// (two rows, four groups) fall on different banks.
template <bool BF16>
__device__ __forceinline__ void store_k_unit(uint32_t hi_tile, uint32_t lo_tile, const Unit& x, int u, int lane) {
  const int r = u * 8 + (lane >> 2), g = lane & 3, flip = g & 2;
  const uint32_t w[4] = {flip ? x.w.z : x.w.x, flip ? x.w.w : x.w.y, flip ? x.w.x : x.w.z, flip ? x.w.y : x.w.w};
  const float s = number<BF16>(x.scale), off = fmaf(-16.f, s, number<BF16>(x.mn));
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t hi[4], lo[4];
    keys_of_word<BF16>(w[k], s, off, hi, lo);
    const int c = g * 4 + (k ^ flip);
    sts128(chunk_at(hi_tile, r, c), hi[0], hi[1], hi[2], hi[3]);
    sts128(chunk_at(lo_tile, r, c), lo[0], lo[1], lo[2], lo[3]);
  }
}
template <bool BF16>
__device__ __forceinline__ void store_v_unit(uint32_t tile, const Unit& x, int u, int lane) {
  const int r = u * 8 + (lane >> 2), g = lane & 3, flip = g & 2;
  const uint32_t w[4] = {flip ? x.w.z : x.w.x, flip ? x.w.w : x.w.y, flip ? x.w.x : x.w.z, flip ? x.w.y : x.w.w};
  const uint32_t s2 = x.scale * 0x10001u, m2 = x.mn * 0x10001u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint32_t v[4];
    values_of_word<BF16>(w[k], s2, m2, v);
    sts128(chunk_at(tile, r, g * 4 + (k ^ flip)), v[0], v[1], v[2], v[3]);
  }
}

// Instruction descriptor with the majors of both operands (0: K, 1: M or N contiguous).
inline uint32_t idesc_of(int is_bf16, int a_mn, int b_mn, int m, int n) { return tc::make_idesc(is_bf16, b_mn, m, n) | (uint32_t)a_mn << 15; }

}  // namespace chunk
}  // namespace cq
