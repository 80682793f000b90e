// The chunk attention and the key weights for few rows (up to 16 of a KV head: single tokens, drafts): what counts is how fast codes are
// unpacked, so they go from global memory to registers and from there, as operands, into the warp MMA (m16n8k16); no tile is built.
//
// A CTA goes over tiles of eight groups of 32 keys, a group for each of its eight warps.  Keys are the M side, query rows the N side (NT blocks of eight):
//   S^T = K Q^T       A = codes (16 keys x 16 channels, pairs along the channels), exact as they are; B = query * scale, which changes with
//                     the group and is the sum of two 16-bit numbers (the product rounded, and what an fma finds missing);
//                     the minima come in as a product of their own.  In bfloat16 that is exact.  In fp16 the queries are scaled by a power of
//                     two per row and the scales by one per group: what is lost is below 2^-24, where the largest product of a row and group
//                     lies between 2^13 and 2^15 (2^8 at least where all of a group's scales are below 2^-9, but not subnormal).
//                     The group's power costs 1.6 % (16 requests x 3328 + 193 keys: 37.1 -> 37.7 us, weights 20.7 -> 21.1).
//   O^T += V^T P^T    A = values (16 channels x 16 keys, pairs along the keys), scale * code + minimum rounded once; B = probabilities,
//                     transposed from the layout of S^T by movmatrix.
// Which key (channel) a lane's row of A is, is free to choose: lane (g, c) takes the codes of word g % 4 of its group, the lower or the
// upper four by g / 4.  So it loads one word per channel (key), half of which it uses, and a byte permute of two words leaves the pairs of
// four A registers: one operation per code.  Register j = 2 * block + half of a lane stands for key (channel) index_of(g, j).
// Each warp has a softmax of its own (running maximum and sum), merged in shared memory at the end.  Up to eight CTAs of a KV head are a cluster
// and merge through each other's shared memory, more by the combine launch.  One request of 256 + 23 keys, which two CTAs share that way:
// 7.9 us, 10.2 with one (14 000 cycles: 2600 until the queries are there, 4400 full-precision keys, 3600 packed ones, 2700 merge).
// Bound: instruction issue (0.55 a cycle and scheduler): about 1000 a group, of which 128 codes a lane of keys and as many of values take two each.
// 16 requests x 8 heads x 3328 + 193 keys, four rows, bfloat16: 38 us (2.1 TB/s; the tile kernel 77), the weights of the keys 22.3; 8 x 32 768
// keys: 126 us (fp16 129.5), where the decode step, which rounds scores to the type and unpacks codes with two operations a pair, takes 93.
// On the way: every lane its own words from global memory 60, scales multiplied into the codes 55, one or two groups a TMA request 51, whole
// rows 48, one address under eight exclusive ors 45.
// TMA brings the codes of the next tile in while one is worked on, whole 128-byte rows (with the 16 or 32 bytes of one or two groups a
// request, the requests were the bound).
#include <math.h>

#include <type_traits>

#include "cq_chunk_few.cuh"
#include "cq_chunk_tc.cuh"

namespace cq {
namespace chunk {
namespace few {

using namespace ptx;

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr float LOG2E = 1.4426950408889634f, SCALE = 0.08838834764831845f;
constexpr int Q_LOG2 = 7, SCALE_LOG2 = 6;      // fp16: the largest of a row's queries lies in [2^7, 2^8), of a group's scales in [2^6, 2^7)

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// of fp16 pairs
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hmax2_abs(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b & 0x7fff7fffu));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  if (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16) mma_bf16(d, a0, a1, a2, a3, b0, b1);
  else mma_f16(d, a0, a1, a2, a3, b0, b1);
}
// codes j of two words (their lower or upper halves side by side in z) as a pair of numbers
template <bool BF16>
__device__ __forceinline__ uint32_t code_pair(uint32_t z, int j) {
  return sub2<BF16>(((z >> (4 * j)) & 0x000f000fu) | (BF16 ? 0x43004300u : 0x64006400u), BF16 ? 0x43004300u : 0x64006400u);
}
// Place within a group of 32 of row g (0..7) of register j = 2 * block + half
__device__ __forceinline__ int index_of(int g, int j) { return (g & 3) * 8 + (g >> 2) * 4 + j; }

// Shared memory of block `rank` of the cluster, at the same place as this block's
__device__ __forceinline__ uint32_t peer(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float peer_f32(uint32_t addr, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float4 peer_f32x4(uint32_t addr, int rank) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer(addr, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A tile: codes [channel][32 words] and [two keys][32 words] (128-byte swizzle), scales and minima of the values [key][4].
struct __align__(1024) Stage {
  uint32_t k[128][32];
  uint32_t v[128][32];
  uint2 vs[256], vm[256];
};
struct __align__(1024) KeyStage {
  uint32_t k[128][32];
};
// Scales and minima of a tile's keys: [scale, minimum][group][channel]
struct __align__(16) Scales {
  uint16_t x[2][8][128];
};
constexpr uint32_t WAIT_TRIES = 1u << 22;
template <bool WEIGHTS> using StageOf = typename std::conditional<WEIGHTS, KeyStage, Stage>::type;

template <bool BF16, bool MASK, int NT, bool WEIGHTS>
__global__ void __launch_bounds__(THREADS, NT == 1 || WEIGHTS ? 2 : 1) few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ FewParams a) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const Params& p = a.p;
  constexpr int ROWS = 8 * NT;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* dyn_s = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);      // stages [2], scales [2]; at the end results
                                                                                           // [warp][row][128], [warp][row][2]
  __shared__ __align__(8) uint64_t bar[2];
  float* merge_s = reinterpret_cast<float*>(dyn_s);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int hk = blockIdx.x % p.hkv, b = blockIdx.x / p.hkv, part = blockIdx.y;
  const int64_t bh = blockIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  const int live = live_tokens(p), groups = p.t_vis >> 5;
  // tiles: full-precision ones first (of what is to be written, for weights), under which the codes of the first visual one come in
  const int nf = (int)(((WEIGHTS ? a.capacity : (int64_t)live) + 255) >> 8), tiles = nf + ((groups + 7) >> 3), per = (tiles + (int)gridDim.y - 1) / (int)gridDim.y;
  const int t0 = min(tiles, part * per), t1 = min(tiles, t0 + per);
  const uint32_t half_sel = g >> 2 ? 0x7632 : 0x5410;
  const int v_row = index_of(2 * c, 0) >> 1, v_base = (warp * 16 + v_row) * 32 + (v_row & 7) * 4 + (g & 3);

  // ---- the queries, as the B operand: channels 2c, 2c+1 (+8) of row g of block nt
  uint32_t q[NT][8][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = nt * 8 + g, i = r / p.n_rep;
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_st + (int64_t)(hk * p.n_rep + r - i * p.n_rep) * p.q_sh + 2 * c;
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
#pragma unroll
      for (int e = 0; e < 2; ++e) q[nt][ks][e] = r < p.rows ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + e * 8) : 0u;
  }
  float unit[NT][2];      // of the scores of rows 2c, 2c + 1: 1 / sqrt(128), times what fp16 queries were divided by
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    unit[nt][0] = unit[nt][1] = SCALE;
    if (!BF16) {
      float top = 0.f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&q[nt][ks][e]));
          top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
        }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int exponent = top > 0.f && top < INFINITY ? max(ilogbf(top) - Q_LOG2, -30) : 0;      // -30 .. 8
      const __half down = __float2half_rn(exp2f((float)-(exponent / 2))), down2 = __float2half_rn(exp2f((float)-(exponent - exponent / 2)));
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          __half2 v = *reinterpret_cast<const __half2*>(&q[nt][ks][e]);
          v = __hmul2(__hmul2(v, __half2half2(down)), __half2half2(down2));
          q[nt][ks][e] = *reinterpret_cast<const uint32_t*>(&v);
        }
#pragma unroll
      for (int e = 0; e < 2; ++e) unit[nt][e] = SCALE * exp2f((float)__shfl_sync(0xffffffffu, exponent, (2 * c + e) * 4));
    }
  }
  // rows 2c, 2c+1 of each block: full-precision tokens that they see, log-sum-exp (weights)
  int limit[NT][2];
  float lse[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = nt * 8 + 2 * c + e, i = r / p.n_rep;
      limit[nt][e] = live - p.q_len + i + 1;
      lse[nt][e] = INFINITY;
      if (WEIGHTS && r < p.rows) {
        const float v = p.lse[((int64_t)b * p.hq + hk * p.n_rep + r - i * p.n_rep) * p.q_len + i];
        lse[nt][e] = v == -INFINITY ? INFINITY : v;      // such a row adds nothing
      }
    }

  using St = StageOf<WEIGHTS>;
  St* stages = reinterpret_cast<St*>(dyn_s);
  Scales* scales = reinterpret_cast<Scales*>(dyn_s + 2 * sizeof(St));
  if (tid == 0) {
    mbar_init(&bar[0], 1);
    mbar_init(&bar[1], 1);
    mbar_fence_init();
  }
  const auto request = [&](int t) {             // codes of tile t; one thread
    if (t >= t1 || t < nf) return;
    const int first = (t - nf) * 256;
    St& st = stages[(t - t0) & 1];
    uint64_t* full = &bar[(t - t0) & 1];
    const int keys = min(256, p.t_vis - first);
    mbar_expect_tx(full, sizeof(st.k) + (WEIGHTS ? 0 : 16384 + 16 * keys));
    tma_load_2d(st.k, &tm_k, first / 8, (int)(bh * 128), full);
    if constexpr (!WEIGHTS) {
      const int64_t tok = bh * p.t_vis + first;
      tma_load_3d(st.v, &tm_v, 0, first / 2, (int)bh, full);
      bulk_load_1d(st.vs, static_cast<const char*>(p.v_scale) + tok * 8, 8 * keys, full);
      bulk_load_1d(st.vm, static_cast<const char*>(p.v_mn) + tok * 8, 8 * keys, full);
    }
  };
  // Scales (threads 0-127) or minima (128-255) of a channel of tile t: one load where the pitch of a channel allows it
  uint32_t sc[4];
  const auto fetch_scales = [&](int t) {
    if (t >= t1 || t < nf) return;
    const uint16_t* src = static_cast<const uint16_t*>(tid < 128 ? p.k_scale : p.k_mn) + (bh * 128 + (tid & 127)) * groups + (t - nf) * 8;
    if (groups % 8 == 0) {
      const uint4 v = *reinterpret_cast<const uint4*>(src);
      sc[0] = v.x; sc[1] = v.y; sc[2] = v.z; sc[3] = v.w;
    } else {
      const int n = groups - (t - nf) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[i] = 2 * i < n ? src[2 * i] : 0u;
        if (2 * i + 1 < n) sc[i] |= (uint32_t)src[2 * i + 1] << 16;
      }
    }
  };
  const auto put_scales = [&](int t) {
    if (t >= t1 || t < nf) return;
    uint16_t* dst = &scales[(t - t0) & 1].x[tid >> 7][0][tid & 127];
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i * 128] = (uint16_t)(sc[i >> 1] >> (16 * (i & 1)));
  };

  float m_ref[NT][2], l_run[NT][2], o[8][NT][4];      // rows 2c, 2c+1; o: channel block, as the A rows are ordered
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) { m_ref[nt][e] = -INFINITY; l_run[nt][e] = 0.f; }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;

  __syncthreads();
  bool ok = true;
  if (tid == 0) request(t0);
  fetch_scales(t0);
  put_scales(t0);
  fetch_scales(t0 + 1);
  for (int t = t0; t < t1; ++t) {
    __syncthreads();                            // the tile before has been read, this one's scales are there
    if (tid == 0) request(t + 1);
    put_scales(t + 1);
    fetch_scales(t + 2);
    const bool vis = t >= nf;
    // this warp's 32 keys: first one in cache order, how many there are
    const int key0 = vis ? ((t - nf) * 8 + warp) * 32 : p.t_vis + (t * 8 + warp) * 32;
    const int there = vis ? min(32, p.t_vis - key0) : min(32, live - (key0 - p.t_vis));
    const St& st = stages[(t - t0) & 1];
    const uint32_t (*sc_s)[64] = reinterpret_cast<const uint32_t (*)[64]>(scales[(t - t0) & 1].x);      // [scale or minimum, group][channel pair]
    if (vis) {                                  // after a time-out too, so that no copy is under way when the block ends
      const int use = (t - max(t0, nf)) >> 1;    // visual tiles that came through this stage before
      if (!mbar_wait_bounded(&bar[(t - t0) & 1], use & 1, ok ? WAIT_TRIES : 1024u)) {
        ok = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) lse[nt][e] = l_run[nt][e] = NAN;      // and so are the results
      }
    }
    if (there <= 0 && !(WEIGHTS && !vis && key0 - p.t_vis < a.capacity)) continue;

    float mask[2][2];
    bool dead = false;
    if (MASK) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = index_of(g, j);
        mask[j >> 1][j & 1] = k < there ? Elem<T>::to_f(static_cast<const T*>(p.mask)[b * p.mask_sb + mask_index(p, key0 + k)]) : -INFINITY;
      }
      dead = __any_sync(0xffffffffu, mask[0][0] == -INFINITY || mask[0][1] == -INFINITY || mask[1][0] == -INFINITY || mask[1][1] == -INFINITY);
    }

    // ---- scores: s[block][nt]: key index_of(g, 2 * block + (e >> 1)), row 2c + (e & 1)
    float s[2][NT][4], small[2][NT][4];
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[mb][nt][e] = small[mb][nt][e] = 0.f;
    if (vis) {
      // fp16: the group's scales times a power of two, so that the products are as far from either end of the range as they can be
      uint32_t up2 = 0;
      float down = 1.f;
      if (!BF16) {
        const uint32_t x = hmax2_abs(sc_s[warp][lane], sc_s[warp][lane + 32]);
        const int field = (int)(__reduce_max_sync(0xffffffffu, max(x & 0xffffu, x >> 16)) >> 10);      // 2^(field - 15), or below 2^-14
        const int k = min(SCALE_LOG2 + 15 - field, 15);                                                // -10 .. 15
        up2 = (uint32_t)(k + 15) << 10;
        up2 |= up2 << 16;
        down = __uint_as_float((uint32_t)(127 - k) << 23);
      }
      float minima[NT][4];                      // the same in every row
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) minima[nt][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        uint32_t s2[2] = {sc_s[warp][ks * 8 + c], sc_s[warp][ks * 8 + c + 4]};
        if (!BF16) {
          s2[0] = hmul2(s2[0], up2);
          s2[1] = hmul2(s2[1], up2);
        }
        const int row = ks * 16 + 2 * c, quad = (warp ^ (2 * c)) * 4 + (g & 3), quad1 = quad ^ 4;
        const uint32_t za = prmt(st.k[row][quad], st.k[row + 1][quad1], half_sel), zb = prmt(st.k[row + 8][quad], st.k[row + 9][quad1], half_sel);
        uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            constexpr uint32_t zero = 0x80008000u;      // -0: what is added to a product and leaves its sign
            hi[nt][e] = fma2<BF16>(q[nt][ks][e], s2[e], zero);
            lo[nt][e] = fma2<BF16>(q[nt][ks][e], s2[e], hi[nt][e] ^ 0x80008000u);
          }
#pragma unroll
        for (int mb = 0; mb < 2; ++mb) {
          const uint32_t c0 = code_pair<BF16>(za, 2 * mb), c1 = code_pair<BF16>(za, 2 * mb + 1), c2 = code_pair<BF16>(zb, 2 * mb), c3 = code_pair<BF16>(zb, 2 * mb + 1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma<BF16>(s[mb][nt], c0, c1, c2, c3, hi[nt][0], hi[nt][1]);
            mma<BF16>(small[mb][nt], c0, c1, c2, c3, lo[nt][0], lo[nt][1]);
          }
        }
        const uint32_t m0 = sc_s[8 + warp][ks * 8 + c], m1 = sc_s[8 + warp][ks * 8 + c + 4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma<BF16>(minima[nt], m0, 0u, m1, 0u, q[nt][ks][0], q[nt][ks][1]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float own = minima[nt][e];
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) {
            if (BF16) {
              s[mb][nt][e] += small[mb][nt][e] + own;
              s[mb][nt][e + 2] += small[mb][nt][e + 2] + own;
            } else {
              s[mb][nt][e] = fmaf(s[mb][nt][e] + small[mb][nt][e], down, own);
              s[mb][nt][e + 2] = fmaf(s[mb][nt][e + 2] + small[mb][nt][e + 2], down, own);
            }
          }
        }
    } else if (there > 0) {
      const T* src = static_cast<const T*>(p.k_fp) + b * p.fp_sb + hk * p.fp_sh + (int64_t)(key0 - p.t_vis) * 128 + 2 * c;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        uint32_t f[4][2];                       // [j][channels 2c.. or 2c+8..]
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            f[j][e] = index_of(g, j) < there ? *reinterpret_cast<const uint32_t*>(src + (int64_t)index_of(g, j) * 128 + ks * 16 + e * 8) : 0u;
#pragma unroll
        for (int mb = 0; mb < 2; ++mb)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<BF16>(s[mb][nt], f[2 * mb][0], f[2 * mb + 1][0], f[2 * mb][1], f[2 * mb + 1][1], q[nt][ks][0], q[nt][ks][1]);
      }
    }
    // natural units, masks; a visual group is whole
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[mb][nt][e] *= unit[nt][e & 1];
          if (MASK) s[mb][nt][e] = mask[mb][e >> 1] == -INFINITY ? -INFINITY : s[mb][nt][e] + mask[mb][e >> 1];
        }
    if (!vis) {
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = index_of(g, 2 * mb + (e >> 1));
            if (k >= there || key0 - p.t_vis + k >= limit[nt][e & 1]) s[mb][nt][e] = -INFINITY;
          }
    }

    if constexpr (WEIGHTS) {
      float w[4] = {};                          // key index_of(g, j), over this lane's rows, then the other lanes'
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) w[j] += ex2_approx((s[j >> 1][nt][(j & 1) * 2 + e] - lse[nt][e]) * LOG2E);
        w[j] += __shfl_xor_sync(0xffffffffu, w[j], 1);
        w[j] += __shfl_xor_sync(0xffffffffu, w[j], 2);
      }
      if (c == 0) {
        const int64_t first = vis ? bh * p.t_vis + key0 : bh * a.capacity + key0 - p.t_vis;
        const float* in = vis ? a.vis_in : a.fp_in;
        float* out = vis ? a.vis : a.fp;
        const int end = vis ? there : (int)min((int64_t)32, a.capacity - (key0 - p.t_vis));
        const int k = index_of(g, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (k + j < end) out[first + k + j] = (in ? in[first + k + j] : 0.f) + w[j];
      }
      continue;
    }

    // ---- softmax of the warp's keys so far
    bool grow_any = false;
    float top[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
        top[nt][e] = fmaxf(x, m_ref[nt][e]);
        grow_any |= top[nt][e] - m_ref[nt][e] > 5.5f;      // a row keeps its reference until the true maximum is e^5.5 above it
      }
    if (__any_sync(0xffffffffu, grow_any)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float alpha = top[nt][e] == -INFINITY ? 1.f : ex2_approx((m_ref[nt][e] - top[nt][e]) * LOG2E);
          m_ref[nt][e] = top[nt][e];
          l_run[nt][e] *= alpha;
#pragma unroll
          for (int i = 0; i < 8; ++i) { o[i][nt][e] *= alpha; o[i][nt][e + 2] *= alpha; }
        }
    }
    uint32_t pb[2][NT][2];                      // probabilities, B operand: [k step][nt][half]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float m0 = m_ref[nt][0] == -INFINITY ? 0.f : m_ref[nt][0], m1 = m_ref[nt][1] == -INFINITY ? 0.f : m_ref[nt][1];
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float e0 = ex2_approx((s[mb][nt][2 * h] - m0) * LOG2E), e1 = ex2_approx((s[mb][nt][2 * h + 1] - m1) * LOG2E);
          l_run[nt][0] += e0;
          l_run[nt][1] += e1;
          pb[mb][nt][h] = movmatrix_trans(pack16<BF16>(e0, e1));
        }
    }

    // ---- values
    if (vis) {
     if constexpr (!WEIGHTS) {
      // Where the words of key index_of(2c, 0) are, for each of the eight values that the swizzle's exclusive or may take: those of key
      // index_of(2c + e, 2 kt + h) and channel group grp are 4 e + kt rows on, under (h ^ e) * 4 + (grp ^ kt)
      const uint32_t* at[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) at[i] = &st.v[0][0] + (v_base ^ (i * 4));
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        uint2 vs[2][2], vm[2][2];               // scales and minima of keys 2c, 2c+1 of both halves, all four groups of channels
        int tok[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            tok[h][e] = index_of(2 * c + e, 2 * kt + h);
            vs[h][e] = st.vs[warp * 32 + tok[h][e]];
            vm[h][e] = st.vm[warp * 32 + tok[h][e]];
            // a key that takes no part: zeros, whatever its values are
            if (MASK && dead && Elem<T>::to_f(static_cast<const T*>(p.mask)[b * p.mask_sb + mask_index(p, key0 + tok[h][e])]) == -INFINITY)
              vs[h][e] = vm[h][e] = make_uint2(0, 0);
          }
#pragma unroll
        for (int grp = 0; grp < 4; ++grp) {
          uint32_t s2[2], m2[2], z[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t sel = grp & 1 ? 0x7632 : 0x5410;
            s2[h] = grp < 2 ? prmt(vs[h][0].x, vs[h][1].x, sel) : prmt(vs[h][0].y, vs[h][1].y, sel);
            m2[h] = grp < 2 ? prmt(vm[h][0].x, vm[h][1].x, sel) : prmt(vm[h][0].y, vm[h][1].y, sel);
            z[h] = prmt(at[h * 4 + (grp ^ kt)][kt * 32], at[(h ^ 1) * 4 + (grp ^ kt)][kt * 32 + 128], half_sel);
          }
#pragma unroll
          for (int mb = 0; mb < 2; ++mb) {
            const uint32_t a0 = fma2<BF16>(code_pair<BF16>(z[0], 2 * mb), s2[0], m2[0]), a1 = fma2<BF16>(code_pair<BF16>(z[0], 2 * mb + 1), s2[0], m2[0]);
            const uint32_t a2 = fma2<BF16>(code_pair<BF16>(z[1], 2 * mb), s2[1], m2[1]), a3 = fma2<BF16>(code_pair<BF16>(z[1], 2 * mb + 1), s2[1], m2[1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<BF16>(o[grp * 2 + mb][nt], a0, a1, a2, a3, pb[kt][nt][0], pb[kt][nt][1]);
          }
        }
      }
     }
    } else {
      // rows of full-precision values, transposed block by block: a lane loads the channel pairs of rows 2c and 2c+1 of A
      const T* src = static_cast<const T*>(p.v_fp) + b * p.fp_sb + hk * p.fp_sh + (int64_t)(key0 - p.t_vis) * 128;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        bool use[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) use[h] = index_of(g, 2 * kt + h) < there && !(MASK && mask[kt][h] == -INFINITY);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t av[2][2];                    // [half of the keys][channel half]
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const T* row = src + (int64_t)index_of(g, 2 * kt + h) * 128 + (j >> 1) * 32 + 2 * (j & 1);
            const uint32_t w0 = use[h] ? *reinterpret_cast<const uint32_t*>(row + index_of(2 * c, 0)) : 0u;
            const uint32_t w1 = use[h] ? *reinterpret_cast<const uint32_t*>(row + index_of(2 * c + 1, 0)) : 0u;
            av[h][0] = movmatrix_trans(prmt(w0, w1, 0x5410));
            av[h][1] = movmatrix_trans(prmt(w0, w1, 0x7632));
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma<BF16>(o[j][nt], av[0][0], av[0][1], av[1][0], av[1][1], pb[kt][nt][0], pb[kt][nt][1]);
        }
      }
    }
  }
  if (!__all_sync(0xffffffffu, ok) && lane == 0) atomicExch(a.status, CQ_ERR_TIMEOUT);
  if constexpr (WEIGHTS) return;

  // ---- the warps' results, over scales and stages
  __syncthreads();
  float* ml_s = merge_s + WARPS * ROWS * 128;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = l_run[nt][e];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int r = nt * 8 + 2 * c + e;
      if (g == 0) {
        ml_s[(warp * ROWS + r) * 2] = m_ref[nt][e];
        ml_s[(warp * ROWS + r) * 2 + 1] = l;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) merge_s[(warp * ROWS + r) * 128 + (i >> 1) * 32 + index_of(g, 2 * (i & 1) + h)] = o[i][nt][e + 2 * h];
    }
  __syncthreads();
  float* own_s = ml_s + WARPS * ROWS * 2;       // the block's result, for the others of its cluster: [row][128, maximum, sum, 2 unused]
  const auto result = [&](int r, float m, float l, const float (&x)[4]) {
    const int i = r / p.n_rep;
    const int64_t h = hk * p.n_rep + r - i * p.n_rep;
    const float inv = l != l ? l : l > 0.f ? 1.f / l : 0.f;
    T* dst = static_cast<T*>(p.out) + b * p.o_sb + i * p.o_st + h * p.o_sh + lane * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<BF16>(x[0] * inv, x[1] * inv), pack16<BF16>(x[2] * inv, x[3] * inv));
    if (p.lse && lane == 0) p.lse[(b * (int64_t)p.hq + h) * p.q_len + i] = l != l ? l : l > 0.f ? m + logf(l) : -INFINITY;
  };
  for (int r = warp; r < min(ROWS, p.rows); r += WARPS) {
    float m = -INFINITY, l = 0.f, x[4] = {};
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, ml_s[(w * ROWS + r) * 2]);
    for (int w = 0; w < WARPS; ++w) {
      const float mw = ml_s[(w * ROWS + r) * 2];
      const float lw = ml_s[(w * ROWS + r) * 2 + 1];
      if (mw == -INFINITY && lw == lw) continue;
      const float f = ex2_approx((mw - m) * LOG2E);
      const float4 v = *reinterpret_cast<const float4*>(merge_s + (w * ROWS + r) * 128 + lane * 4);
      l = fmaf(lw, f, l);
      x[0] = fmaf(v.x, f, x[0]); x[1] = fmaf(v.y, f, x[1]); x[2] = fmaf(v.z, f, x[2]); x[3] = fmaf(v.w, f, x[3]);
    }
    if (gridDim.y == 1) {
      result(r, m, l, x);
    } else if (a.cluster) {
      float* own = own_s + r * 132;
      *reinterpret_cast<float4*>(own + lane * 4) = make_float4(x[0], x[1], x[2], x[3]);
      if (lane == 0) { own[128] = m; own[129] = l; }
    } else {
      const int64_t at = (bh * p.rows + r) * a.parts + part;
      *reinterpret_cast<float4*>(a.part_o + at * 128 + lane * 4) = make_float4(x[0], x[1], x[2], x[3]);
      if (lane == 0) a.part_ml[at] = make_float2(m, l);
    }
  }
  if (!a.cluster) return;
  // the blocks of a KV head are a cluster: block r % parts merges row r, in the order of the blocks
  cluster_sync();
  for (int r = part + warp * a.parts; r < min(ROWS, p.rows); r += WARPS * a.parts) {
    const uint32_t own = smem_u32(own_s + r * 132);
    float m = -INFINITY, l = 0.f, x[4] = {};
    for (int s = 0; s < a.parts; ++s) m = fmaxf(m, peer_f32(own + 512, s));
    for (int s = 0; s < a.parts; ++s) {
      const float ms = peer_f32(own + 512, s), ls = peer_f32(own + 516, s);
      if (ms == -INFINITY && ls == ls) continue;
      const float f = ex2_approx((ms - m) * LOG2E);
      const float4 v = peer_f32x4(own + lane * 16, s);
      l = fmaf(ls, f, l);
      x[0] = fmaf(v.x, f, x[0]); x[1] = fmaf(v.y, f, x[1]); x[2] = fmaf(v.z, f, x[2]); x[3] = fmaf(v.w, f, x[3]);
    }
    result(r, m, l, x);
  }
  cluster_sync();                               // nobody leaves while its memory is read
}

// Packed codes as a map of 32-bit words: `words` of a row, `rows` rows, `heads` of those (0: a map of two dimensions); a box of box_words x box_rows
static bool code_map(CUtensorMap* m, const void* base, int64_t words, int64_t rows, int64_t heads, int box_words, int box_rows, CUtensorMapSwizzle swizzle) {
  if (!base || words == 0 || rows == 0) {      // no packed keys: a map that nothing uses
    *m = CUtensorMap{};
    return true;
  }
  const EncodeTiled encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)words, (cuuint64_t)rows, (cuuint64_t)heads}, strides[2] = {(cuuint64_t)words * 4, (cuuint64_t)(words * rows) * 4};
  const cuuint32_t box[3] = {(cuuint32_t)box_words, (cuuint32_t)box_rows, 1}, one[3] = {1, 1, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_INT32, heads ? 3 : 2, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16, bool MASK, int NT, bool WEIGHTS>
static int run(const FewParams& p, int batch, cudaStream_t st) {
  CUtensorMap tk, tv;
  if (!code_map(&tk, p.p.k_code, p.p.t_vis / 8, 128 * (int64_t)batch * p.p.hkv, 0, 32, 128, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !code_map(&tv, p.p.v_code, 32, p.p.t_vis / 2, (int64_t)batch * p.p.hkv, 32, 128, CU_TENSOR_MAP_SWIZZLE_128B))
    return CQ_ERR_LAUNCH;
  constexpr int stages = 1024 + 2 * (int)(sizeof(Scales) + sizeof(StageOf<WEIGHTS>)), results = WEIGHTS ? 0 : 1024 + 8 * NT * (WARPS * 130 + 132) * (int)sizeof(float);
  constexpr int smem = stages > results ? stages : results;
  if (smem > 24 * 1024) {
    static bool configured[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return CQ_ERR_LAUNCH;
    if (!configured[dev]) {
      if (cudaFuncSetAttribute(few_kernel<BF16, MASK, NT, WEIGHTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return CQ_ERR_LAUNCH;
      configured[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch * p.p.hkv), p.parts);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1; attr[1].val.clusterDim.y = p.cluster ? p.parts : 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.cluster ? 2 : 1;
  return launched(cudaLaunchKernelEx(&cfg, few_kernel<BF16, MASK, NT, WEIGHTS>, tk, tv, p));
}

}  // namespace few

// CTAs per KV head: two an SM (one for the attention of more than eight rows), in whole rounds; a CTA costs about a tile of 256 keys beside its own.
// The blocks of an attention's KV head, up to FEW_CLUSTER, merge their results as a cluster; more take a second launch.
int few_parts(int64_t heads, int64_t t_vis, int64_t fp_keys, bool one, bool merged) {
  const int64_t slots = (int64_t)sm_count() * (one ? 1 : 2), tiles = (t_vis + 255) / 256 + (fp_keys + 255) / 256;
  double cost = 1e300;
  int best = 1;
  for (int s = 1; s <= 64 && s <= tiles; ++s) {
    const int64_t per = (tiles + s - 1) / s;
    if ((tiles + per - 1) / per != s) continue;      // leaves a part empty
    const double c = (double)((heads * s + slots - 1) / slots) * (per + 1.0) + (!merged || s == 1 ? 0.0 : s <= FEW_CLUSTER ? 0.25 : 1.5);
    if (c < cost) { cost = c; best = s; }
  }
  return best;
}

int few_run(const FewParams& p, int batch, bool bf16, bool weights, cudaStream_t st) {
  using few::run;
#define CQ_NT(B, M, W) (p.p.rows <= 8 ? run<B, M, 1, W>(p, batch, st) : run<B, M, 2, W>(p, batch, st))
#define CQ_M(B, W) (p.p.mask ? CQ_NT(B, true, W) : CQ_NT(B, false, W))
  if (weights) return bf16 ? CQ_M(true, true) : CQ_M(false, true);
  return bf16 ? CQ_M(true, false) : CQ_M(false, false);
#undef CQ_M
#undef CQ_NT
}

}  // namespace chunk
}  // namespace cq
