// Tiles of packed or full-precision keys and values as operands of tcgen05.mma, for the chunk attention and the key weights.
//
// A tile is 128 x 128 numbers of 16 bits: two panels of [128 rows][128 bytes], 128-byte swizzled.  Packed keys have a channel per row and
// tokens along it, packed values a token per row and channels along it: in both a 32-bit word of codes is eight numbers = one 16-byte
// chunk of a row, and four words share scale and minimum.  Full-precision rows have a token per row.
#pragma once

#include <cuda.h>

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

__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
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

// (x0, x1) = (a0, a1) * (b0, b1) + (c0, c1)
__device__ __forceinline__ void fma_pair(float& x0, float& x1, float a0, float a1, float b0, float b1, float c0, float c1) {
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(x0), "=f"(x1) : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}
// (s0, s1) += (a0, a1)
__device__ __forceinline__ void add_pair(float& s0, float& s1, float a0, float a1) {
  asm("{\n\t.reg .b64 ra, rs;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rs, {%0, %1};\n\tadd.rn.f32x2 rs, rs, ra;\n\tmov.b64 {%0, %1}, rs;\n\t}"
      : "+f"(s0), "+f"(s1) : "f"(a0), "f"(a1));
}

// Two numbers as 16-bit pairs whose sum they are: hi is the number cut off, lo the rest rounded.  bfloat16: a value scale * code + minimum of
// up to 16 bits is exact, which it has unless the minimum is hundreds of scales away from zero; others are off by 2^-16 of themselves at most.
// fp16: 22 bits, but none below 2^-24, so that a value is off by 2^-25 at most: 2^-15 of a key of 2^-10, nothing of one from 2^-3 on.
template <bool BF16>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  if (BF16) {
    hi = ptx::prmt(__float_as_uint(a), __float_as_uint(b), 0x7632);
    fma_pair(a, b, __uint_as_float(__float_as_uint(a) & 0xffff0000u), __uint_as_float(__float_as_uint(b) & 0xffff0000u), -1.f, -1.f, a, b);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(b), "f"(a));
  } else {
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(b), "f"(a));
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    fma_pair(a, b, h.x, h.y, -1.f, -1.f, a, b);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(b), "f"(a));
  }
}

// Code N (0..7) of a word as the float 128 + code
template <int N>
__device__ __forceinline__ float code128(uint32_t w) {
  constexpr int sh = 16 - 4 * N;
  const uint32_t s = sh >= 0 ? w << (sh >= 0 ? sh : 0) : w >> (sh < 0 ? -sh : 0);
  return __uint_as_float((s & 0x000f0000u) | 0x43000000u);
}
// Eight keys of a channel, scale * code + minimum in fp32, as chunks of the two tiles whose sum they are; off = minimum - 128 scale.  The
// products are exact, the offset is unless the minimum is thousands of times smaller than the scale (then 2^-17 scales off).
template <bool BF16>
__device__ __forceinline__ void keys_of_word(uint32_t w, float s, float off, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  float k[8];
  fma_pair(k[0], k[1], code128<0>(w), code128<1>(w), s, s, off, off);
  fma_pair(k[2], k[3], code128<2>(w), code128<3>(w), s, s, off, off);
  fma_pair(k[4], k[5], code128<4>(w), code128<5>(w), s, s, off, off);
  fma_pair(k[6], k[7], code128<6>(w), code128<7>(w), s, s, off, off);
#pragma unroll
  for (int j = 0; j < 4; ++j) split_pair<BF16>(k[2 * j], k[2 * j + 1], hi[j], lo[j]);
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
  const float s = number<BF16>(x.scale), off = fmaf(-128.f, s, number<BF16>(x.mn));
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

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(ptx::smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(void* dst, const void* tmap, int c0, int c1, int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(ptx::smem_u32(dst)), "l"(tmap), "r"(c0), "r"(c1), "r"(c2), "r"(ptx::smem_u32(bar))
      : "memory");
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static const EncodeTiled fn = []() -> EncodeTiled {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Queries [B,L,Hq,128] as a map (channel, head, query, batch row) whose box is 64 channels of the heads of a KV head for
// `queries` queries: rows of 128 bytes in query-major order, the panel layout above.
inline bool query_map(CUtensorMap* m, const cq_chunk_args* a, int queries) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[4] = {128, (cuuint64_t)a->n_q_heads, (cuuint64_t)a->q_len, (cuuint64_t)a->batch};
  const int64_t step[3] = {a->q_strides[2], a->q_strides[1], a->q_strides[0]};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] == 1 ? 256 : (cuuint64_t)step[i] * 2;      // an extent of one: any
  const cuuint32_t box[4] = {64, (cuuint32_t)(a->n_q_heads / a->n_kv_heads), (cuuint32_t)queries, 1}, one[4] = {1, 1, 1, 1};
  return encode(m, a->dtype == CQ_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(a->q), dims,
                strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Instruction descriptor with the majors of both operands (0: K, 1: M or N contiguous).
inline uint32_t idesc_of(int is_bf16, int a_mn, int b_mn, int m, int n) { return tc::make_idesc(is_bf16, b_mn, m, n) | (uint32_t)a_mn << 15; }

}  // namespace chunk
}  // namespace cq
