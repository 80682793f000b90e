// Attention of several new tokens over [system | visual (4-bit group format) | text] on the 5th-generation tensor cores.
//
// Rows are (query, head) pairs of one KV head, query major.  A tile holds as many whole queries as 128 rows take (a TMEM lane per row),
// and a CTA works on one KV head of one request with two tiles A and B:
//   PAIR    A and B are adjacent tiles and share every key tile (more queries than one tile takes);
//   else    A and B are the SAME rows and take the even and the odd key tiles, two partial results.
// The keys of a CTA are a part of the request's key tiles, visual ones first (`parts` on the grid); partial results are merged by
// combine_kernel.  Roles:
//   warps 0-3 / 4-7  softmax of A / B: thread = row; running maximum and sum, probabilities back to tensor memory
//   warps 8-15       operands: codes from global memory (requested a tile ahead), unpacked into 16-bit tiles in shared memory: two
//                    buffers of keys (two terms each) and one of values, two where there is one query tile; full-precision
//                    rows into the same layout
//   warp 16          issues the products
// S = Q K^T with packed keys as two 16-bit terms, whose sum is scale * code + minimum but for what split_pair says, so scores carry hardly a
// rounding but that of fp32 sums; O += P V with P in tensor memory.  S_A [0,128) S_B [128,256) O_A [256,384) O_B [384,512) TMEM columns.
// Key tiles that six or more row blocks would unpack are unpacked once, by chunk_unpack_kernel, into images of the shared-memory tiles (96 KB per
// 128 visual tokens), which the attention then loads in bulk.
//
// What bounds it.  With images: 48 products of 64 cycles a key tile and pair of query tiles; measured 4100 cycles (8 x 1024 queries on
// 3328 + 1280 keys, bfloat16, at 1.75 GHz under the power cap: 596 us, and 56 for the images at 4.2 TB/s; 684 to 690 in a row).  What is above is the chain of one query tile
// (S -> softmax, 1900 cycles -> P V -> next S) that the other one does not cover.  Without images: the same chain beside warps that unpack
// (39 instructions per word of eight keys, twice rounded), and instructions that do not come in time: with the two halves of a row's scores as
// a loop instead of two copies of the code 73.5 -> 66 us (37 queries of four padded requests on 6656 tokens), 112 -> 98 (40 of 16 on
// 3328); quarters, or a loop over the warp's two units, gave nothing more.  With images for one row block too: 101.
// Taken for granted by neither: a slot or tile as an index instead of a constant costs the issuing lane 104 cycles a product (917 -> 1036 us
// when the slot became a switch, 676 with constants); a ring of five slots held up the keys (980 -> 945).
// Every wait is bounded; one that runs out sets CQ_ERR_TIMEOUT in the workspace's first word, and the CTA ends once the copies and products that it
// started have (another bounded wait), with NaN for the rows whose results did not come.
#include <float.h>
#include <math.h>

#include <type_traits>

#include "cq_chunk_few.cuh"
#include "cq_chunk_tc.cuh"

namespace cq {
namespace chunk {

using namespace ptx;
using namespace tc;

constexpr int PRODUCERS = 8;
// Threads and registers.  Without images: 8 softmax warps, 8 producers, the issuer's warpgroup; 256 x 104 + 256 x 88 + 128 x 96 = the launch's
// 640 x 96.  With images: 8 softmax warps, which hold a row's 128 scores at once, and the issuer's warpgroup; 256 x 184 + 128 x 128
// = 63 488 of the launch's 384 x 168.
template <bool IMAGE> struct Roles {
  static constexpr int MMA_WARP = IMAGE ? 8 : 16, THREADS = IMAGE ? 384 : 640;
  static constexpr int SOFTMAX_REGS = IMAGE ? 184 : 104, CONTROL_REGS = IMAGE ? 128 : 96, PRODUCER_REGS = 88;
};
constexpr int SMEM_BYTES = 7 * TILE_BYTES + 1024;
constexpr uint32_t WAIT_TRIES = 1u << 22, DRAIN_TRIES = 1u << 16;      // the latter for what is still under way after a wait that ran out
constexpr long long WAIT_CYCLES = 1ll << 30;
constexpr float LOG2E = 1.4426950408889634f;

struct AttnParams {
  Params p;
  int tile_queries, tile_rows;      // of a tile
  int parts;                 // partial results per row (1: the kernel writes the output itself)
  float scale;               // 1 / sqrt(128)
  uint32_t idesc_kmajor, idesc_mn;
  unsigned char* image;      // unpacked tiles, see unpack_kernel
  int image_fp_tiles;
  float* part_o;             // [batch][KV head][row][part][128]
  float2* part_ml;           // [batch][KV head][row][part]: maximum and sum
  int* status;
};

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// register split between warpgroups; every warp of a group runs it
template <int N> __device__ __forceinline__ void setmaxnreg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void setmaxnreg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// barrier among the four softmax warps of a tile that also tells whether any thread passed `flag`
__device__ __forceinline__ bool tile_any(int id, bool flag) {
  uint32_t out;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbar.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(out) : "r"((uint32_t)flag), "r"(id) : "memory");
  return out != 0;
}

// Key tiles of a CTA: visual tiles [0, nv), full-precision ones [nv, n_all); this CTA's are [t0, t0 + n).
struct Range {
  int nv, t0, n;
};

// Unpacked tiles of a KV head as they lie in shared memory, one after the other: per visual tile both terms of the keys and the values, per
// full-precision tile keys and values.
__host__ __device__ __forceinline__ size_t image_bytes(int nv, int nf) { return (size_t)(3 * nv + 2 * nf) * TILE_BYTES; }

// whether a key's mask lets it take part (its values are not looked at otherwise)
template <bool BF16, bool MASK>
__device__ __forceinline__ bool takes_part(const Params& p, int b, int key) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  return !MASK || Elem<T>::to_f(static_cast<const T*>(p.mask)[b * p.mask_sb + mask_index(p, key)]) != -INFINITY;
}

// A full-precision tile, rows that are not live (values: or that the mask takes out) as zeros; 256 threads.
template <bool BF16, bool MASK>
__device__ __forceinline__ void fill_fp_tile(const Params& p, const void* base, int b, int hk, int t_first, int live, bool values, uint32_t dst, int ptid) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const T* src = static_cast<const T*>(base) + b * p.fp_sb + hk * p.fp_sh;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    uint4 v[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int t = t_first + (half * 4 + it) * 16 + (ptid >> 4);
      v[it] = make_uint4(0, 0, 0, 0);
      if (t < live) {
        v[it] = *reinterpret_cast<const uint4*>(src + (int64_t)t * 128 + (ptid & 15) * 8);
        if (values && !takes_part<BF16, MASK>(p, b, p.t_vis + t)) v[it] = make_uint4(0, 0, 0, 0);
      }
      if (values) order_values(v[it]);
    }
#pragma unroll
    for (int it = 0; it < 4; ++it)
      sts128(chunk_at(dst, (half * 4 + it) * 16 + (ptid >> 4), ptid & 15), v[it].x, v[it].y, v[it].z, v[it].w);
  }
}

__device__ __forceinline__ void bulk_store_1d(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

// Unpacks every key tile once, for calls whose rows would have the attention unpack it many times: a CTA per tile.
template <bool BF16, bool MASK>
__global__ void __launch_bounds__(256) chunk_unpack_kernel(const __grid_constant__ AttnParams a) {
  const Params& p = a.p;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t s0 = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nv = (p.t_vis + 127) >> 7, tile = blockIdx.x;
  const int hk = blockIdx.y % p.hkv, b = blockIdx.y / p.hkv;
  const int64_t bh = (int64_t)b * p.hkv + hk;
  pdl_launch_dependents();
  pdl_wait();
  const int live = live_tokens(p);
  unsigned char* dst = a.image + bh * image_bytes(nv, a.image_fp_tiles);
  int n;
  if (tile < nv) {
    Unit k[2], v[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int key = tile * 128 + (warp + 8 * u) * 8 + (lane >> 2);
      load_k_unit(p, bh, tile, warp + 8 * u, lane, k[u]);
      load_v_unit(p, bh, tile, warp + 8 * u, lane, key < p.t_vis && takes_part<BF16, MASK>(p, b, key), v[u]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      store_k_unit<BF16>(s0, s0 + TILE_BYTES, k[u], warp + 8 * u, lane);
      store_v_unit<BF16>(s0 + 2 * TILE_BYTES, v[u], warp + 8 * u, lane);
    }
    dst += (size_t)tile * 3 * TILE_BYTES;
    n = 3;
  } else {
    const int t_first = (tile - nv) * 128;
    if (t_first >= live) return;
    fill_fp_tile<BF16, MASK>(p, p.k_fp, b, hk, t_first, live, false, s0, tid);
    fill_fp_tile<BF16, MASK>(p, p.v_fp, b, hk, t_first, live, true, s0 + TILE_BYTES, tid);
    dst += image_bytes(nv, tile - nv);
    n = 2;
  }
  fence_proxy_async_smem();
  __syncthreads();
  if (tid == 0) {
    bulk_store_1d(dst, s0, n * TILE_BYTES);
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
}

template <bool BF16, bool MASK, bool PAIR, bool IMAGE>
__global__ void __launch_bounds__(Roles<IMAGE>::THREADS, 1) chunk_attn_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ AttnParams a) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const Params& p = a.p;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  static_assert(PAIR || !IMAGE, "images are for many rows");
  constexpr int QT = PAIR ? 2 : 1, MMA_WARP = Roles<IMAGE>::MMA_WARP;      // query tiles
  const uint32_t q_s = smem_u32(smem), k_s = q_s + QT * TILE_BYTES, v_s = k_s + 4 * TILE_BYTES;      // keys: [buffer][large terms, small ones]
  // bar_q (once); bar_k / bar_v[buffer] full, bar_kfree / bar_vfree read; bar_s[X] scores of X ready; bar_p[X][half] probabilities of keys 0-63 / 64-127 stored;
  // bar_pv[X] the tile's P V done; bar_end all products done
  __shared__ __align__(8) uint64_t bar_q, bar_k[2], bar_kfree[2], bar_v[2], bar_vfree[2], bar_s[2], bar_p[2][2], bar_pv[2], bar_end;
  __shared__ uint32_t tmem_base_s;
  __shared__ __align__(16) T mask_s[MASK ? 2 : 1][MASK ? 2 : 1][MASK ? 128 : 8];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hk = blockIdx.y % p.hkv, b = blockIdx.y / p.hkv, part = blockIdx.z;
  const int64_t bh = (int64_t)b * p.hkv + hk;
  const int i0 = ((int)gridDim.x - 1 - (int)blockIdx.x) * (PAIR ? 2 : 1) * a.tile_queries;      // first query; those that see most keys first

  if (tid == 0) {
    mbar_init(&bar_q, 1 + (IMAGE ? 1 : PRODUCERS));
    for (int x = 0; x < 2; ++x) {
      mbar_init(&bar_k[x], IMAGE ? 1 : PRODUCERS);
      mbar_init(&bar_kfree[x], 1);
      mbar_init(&bar_v[x], IMAGE ? 1 : PRODUCERS);
      mbar_init(&bar_vfree[x], 1);
      mbar_init(&bar_s[x], 1);
      mbar_init(&bar_p[x][0], 128);
      mbar_init(&bar_p[x][1], 128);
      mbar_init(&bar_pv[x], 1);
    }
    mbar_init(&bar_end, 1);
    mbar_fence_init();
  }
  pdl_launch_dependents();
  pdl_wait();
  const int live = live_tokens(p);
  if (warp == MMA_WARP) tmem_alloc(&tmem_base_s, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  Range k;
  {
    const int last = min(i0 + (PAIR ? 2 : 1) * a.tile_queries, p.q_len) - 1;
    const int n_fp = max(0, live - p.q_len + last + 1);      // full-precision tokens that the last query sees
    k.nv = (p.t_vis + 127) >> 7;
    const int n_all = k.nv + ((n_fp + 127) >> 7), grid_parts = gridDim.z, per = (n_all + grid_parts - 1) / grid_parts;
    k.t0 = min(n_all, part * per);
    k.n = min(n_all, k.t0 + per) - k.t0;
  }

  // rows of a query tile that hold no query are zeros; TMA brings the others
  const auto clear_q = [&](int thread, int threads) {
    for (int c = a.tile_rows * 8 + thread; c < 128 * 8; c += threads)
      for (int s = 0; s < 2 * QT; ++s) sts128(q_s + s * PANEL_BYTES + c * 16, 0, 0, 0, 0);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bar_q);
  };

  if (!IMAGE && warp >= 8 && warp < MMA_WARP) {
    // ================= operands =================
    setmaxnreg_dec<Roles<IMAGE>::PRODUCER_REGS>();
    const int pw = warp - 8, ptid = tid - 256;
    bool ok = true;
    clear_q(ptid, 256);

    Unit ku[2], vu[2];                        // requested: the warp's two units
    bool taken[2] = {true, true};
    const auto request_k = [&](int j) {
      const int tile = k.t0 + j;
      if (j < k.n && tile < k.nv) {
        load_k_unit(p, bh, tile, pw, lane, ku[0]);
        load_k_unit(p, bh, tile, pw + 8, lane, ku[1]);
      }
    };
    const auto request_v = [&](int j) {
      const int tile = k.t0 + j;
      if (j < k.n && tile < k.nv) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int key = tile * 128 + (pw + 8 * u) * 8 + (lane >> 2);
          load_v_unit(p, bh, tile, pw + 8 * u, lane, true, vu[u]);
          if (MASK) taken[u] = key < p.t_vis && takes_part<BF16, MASK>(p, b, key);      // looked at when the unit is stored
        }
      }
    };
    const auto wait_free = [&](uint64_t* bar, int use) {      // the buffer's use-th use is about to start
      if (ok && use > 0) ok = mbar_wait_bounded(bar, (use - 1) & 1, WAIT_TRIES);
      ok = __all_sync(0xffffffffu, ok);
    };
    const auto publish = [&](uint64_t* bar) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    request_k(0);
    request_v(0);
    // Keys one tile ahead of values: scores come first.  What the next use needs is requested behind the fence, which would wait for
    // it.  One copy of this code: with two tiles requested ahead and the loop written out twice instructions were missing
    for (int j = -1; j < k.n && ok; ++j) {
      if (j + 1 < k.n) {
        const int tile = k.t0 + j + 1, buf = (j + 1) & 1;
        const uint32_t hi = k_s + buf * 2 * TILE_BYTES, lo = hi + TILE_BYTES;
        wait_free(&bar_kfree[buf], (j + 1) >> 1);
        if (!ok) break;
        if (tile < k.nv) {
          store_k_unit<BF16>(hi, lo, ku[0], pw, lane);
          store_k_unit<BF16>(hi, lo, ku[1], pw + 8, lane);
        } else {
          fill_fp_tile<BF16, MASK>(p, p.k_fp, b, hk, (tile - k.nv) * 128, live, false, hi, ptid);
        }
        publish(&bar_k[buf]);
        request_k(j + 2);
      }
      if (j >= 0) {
        const int tile = k.t0 + j, buf = PAIR ? 0 : j & 1;
        const uint32_t dst = v_s + buf * TILE_BYTES;
        wait_free(&bar_vfree[buf], PAIR ? j : j >> 1);
        if (!ok) break;
        if (tile < k.nv) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
            if (MASK && !taken[u]) { vu[u].w = make_uint4(0, 0, 0, 0); vu[u].scale = vu[u].mn = 0; }
          store_v_unit<BF16>(dst, vu[0], pw, lane);
          store_v_unit<BF16>(dst, vu[1], pw + 8, lane);
        } else {
          fill_fp_tile<BF16, MASK>(p, p.v_fp, b, hk, (tile - k.nv) * 128, live, true, dst, ptid);
        }
        publish(&bar_v[buf]);
        request_v(j + 1);
      }
    }
    if (!ok && lane == 0) atomicExch(a.status, CQ_ERR_TIMEOUT);
  } else if (warp >= MMA_WARP) {
    // ================= products =================
    setmaxnreg_dec<Roles<IMAGE>::CONTROL_REGS>();
    if (warp == MMA_WARP) {
    // The whole warp runs the loop and one elected lane issues.  Loop bounds and tile numbers come out of a shuffle, so that the compiler
    // knows them to be the warp's: operands that it holds per lane cost the issuing lane 104 cycles a product, of which the pipe takes 64.
    const auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const Range kr = k;
    const Range k = {uniform(kr.nv), uniform(kr.t0), uniform(kr.n)};
    const uint32_t lead = elect_one();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    constexpr uint32_t tile16 = TILE_BYTES >> 4;
    const uint64_t qd = smem_desc(q_s, 16, 1024), kd = smem_desc(k_s, 16, 1024), kmd = smem_desc(k_s, PANEL_BYTES, 1024), vd = smem_desc(v_s, PANEL_BYTES, 1024);
    bool ok = true;
    const auto all = [](bool r) { return __all_sync(0xffffffffu, r) != 0; };
    if (lead) {
      mbar_expect_tx(&bar_q, 256 * a.tile_rows * QT);
      for (int s = 0; s < 2 * QT; ++s)      // both halves of the channels; queries past the end are zeros
        tma_load_4d(q_s + s * PANEL_BYTES, &tm_q, (s & 1) * 64, hk * p.n_rep, i0 + (s >> 1) * a.tile_queries, b, &bar_q);
    }
    const auto commit = [&](uint64_t* bar) { if (lead) umma_commit(bar); };
    using C0 = std::integral_constant<int, 0>;
    using C1 = std::integral_constant<int, 1>;
    // tile and buffer are constants of the code
    const auto take_k = [&](auto bc, int j) {
      constexpr int buf = decltype(bc)::value;
      ok = ok && all(mbar_wait_bounded(&bar_k[buf], (j >> 1) & 1, WAIT_TRIES));
      tc_fence_after();
    };
    const auto issue_s = [&](auto xc, auto bc, int j) {      // S_x = Q_x K^T of key tile j
      constexpr int x = decltype(xc)::value, buf = decltype(bc)::value;
      constexpr uint32_t q0 = PAIR && x ? tile16 : 0, hi = 2 * buf * tile16, lo = hi + tile16;
      if (!lead) return;
      const uint32_t d = tm + (uint32_t)x * 128u;
      if (k.t0 + j < k.nv) {                                 // the small terms first: sums are cut off, not rounded
#pragma unroll
        for (int ks = 0; ks < 16; ++ks) {
          const uint32_t qo = (uint32_t)((((ks & 7) >> 2) * PANEL_BYTES + (ks & 3) * 32) >> 4);
          umma(d, desc_at(qd, q0 + qo), desc_at(kmd, (ks < 8 ? lo : hi) + (ks & 7) * 128), a.idesc_mn, ks > 0);
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t qo = (uint32_t)(((ks >> 2) * PANEL_BYTES + (ks & 3) * 32) >> 4);
          umma(d, desc_at(qd, q0 + qo), desc_at(kd, hi + qo), a.idesc_kmajor, ks > 0);
        }
      }
      umma_commit(&bar_s[x]);
    };
    // O_x += P_x V, the probabilities of keys 0-63 first; `count` key tiles of x before
    const auto pv = [&](auto xc, auto vc, int count) {
      constexpr int x = decltype(xc)::value, buf = decltype(vc)::value;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        ok = ok && all(mbar_wait_cycles(&bar_p[x][half], count & 1, WAIT_CYCLES));
        if (!ok) return;
        tc_fence_after();
        if (lead) {
#pragma unroll
          for (int ks = 4 * half; ks < 4 * half + 4; ++ks)
            umma_ts(tm + 256u + (uint32_t)x * 128u, tm + (uint32_t)x * 128u + (uint32_t)ks * 8u, desc_at(vd, buf * tile16 + ks * 128), a.idesc_mn,
                    (ks > 0 || count > 0) ? 1u : 0u);
        }
      }
      commit(&bar_pv[x]);
    };
    ok = all(mbar_wait_bounded(&bar_q, 0, WAIT_TRIES));
    if (PAIR) {
      if (k.n > 0) {
        take_k(C0{}, 0);
        if (ok) { issue_s(C0{}, C0{}, 0); issue_s(C1{}, C0{}, 0); commit(&bar_kfree[0]); }
      }
      const auto step = [&](auto next, int j) {              // next: the buffer of key tile j + 1
        constexpr int nb = decltype(next)::value;
        if (j >= k.n || !ok) return;
        const bool more = j + 1 < k.n;
        ok = all(mbar_wait_bounded(&bar_v[0], j & 1, WAIT_TRIES));
        if (ok) pv(C0{}, C0{}, j);
        if (more && ok) take_k(next, j + 1);
        if (more && ok) issue_s(C0{}, next, j + 1);
        if (ok) pv(C1{}, C0{}, j);
        if (!ok) return;
        commit(&bar_vfree[0]);
        if (more) {
          issue_s(C1{}, next, j + 1);
          commit(&bar_kfree[nb]);
        }
      };
      for (int j = 0; j < k.n && ok; j += 2) {
        step(C1{}, j);
        step(C0{}, j + 1);
      }
    } else {
      const auto first = [&](auto xc) {                      // x, its buffers and key tile are one number here
        constexpr int x = decltype(xc)::value;
        if (x >= k.n || !ok) return;
        take_k(xc, x);
        if (ok) { issue_s(xc, xc, x); commit(&bar_kfree[x]); }
      };
      const auto step = [&](auto xc, int j) {
        constexpr int x = decltype(xc)::value;
        if (j >= k.n || !ok) return;
        ok = all(mbar_wait_bounded(&bar_v[x], (j >> 1) & 1, WAIT_TRIES));
        if (ok) pv(xc, xc, j >> 1);
        if (!ok) return;
        commit(&bar_vfree[x]);
        if (j + 2 >= k.n) return;
        take_k(xc, j + 2);
        if (ok) { issue_s(xc, xc, j + 2); commit(&bar_kfree[x]); }
      };
      first(C0{});
      first(C1{});
      for (int j = 0; j < k.n && ok; j += 2) {
        step(C0{}, j);
        step(C1{}, j + 1);
      }
    }
    commit(&bar_end);
    ok = all(mbar_wait_bounded(&bar_end, 0, ok ? WAIT_TRIES : DRAIN_TRIES)) && ok;
    if (!ok) {
      mbar_wait_bounded(&bar_q, 0, DRAIN_TRIES);
      if (lead) atomicExch(a.status, CQ_ERR_TIMEOUT);
    }
    __syncwarp();
    } else if (IMAGE && warp == MMA_WARP + 1) {
      // ================= operands from the images =================
      clear_q(lane, 32);
      if (lane == 0) {
        const unsigned char* src = a.image + bh * image_bytes(k.nv, a.image_fp_tiles);
        bool ok = true;
        int ks = 0, vs = 0;                       // loads requested
        const auto load_k = [&](int j) {
          if (j >= k.n || !ok) return;
          const int tile = k.t0 + j, buf = j & 1;
          if (j >= 2) ok = mbar_wait_bounded(&bar_kfree[buf], ((j >> 1) - 1) & 1, WAIT_TRIES);
          if (!ok) return;
          const uint32_t bytes = (tile < k.nv ? 2 : 1) * TILE_BYTES;
          mbar_expect_tx(&bar_k[buf], bytes);
          bulk_load_1d(smem + (QT + 2 * buf) * TILE_BYTES, src + (tile < k.nv ? (size_t)tile * 3 * TILE_BYTES : image_bytes(k.nv, tile - k.nv)), bytes, &bar_k[buf]);
          ks = j + 1;
        };
        load_k(0);
        for (int j = 0; j < k.n && ok; ++j) {
          load_k(j + 1);
          if (ok && j > 0) ok = mbar_wait_bounded(&bar_vfree[0], (j - 1) & 1, WAIT_TRIES);
          if (!ok) break;
          const int tile = k.t0 + j;
          mbar_expect_tx(&bar_v[0], TILE_BYTES);
          bulk_load_1d(smem + (QT + 4) * TILE_BYTES, src + (tile < k.nv ? (size_t)(3 * tile + 2) * TILE_BYTES : image_bytes(k.nv, tile - k.nv) + TILE_BYTES),
                       TILE_BYTES, &bar_v[0]);
          vs = j + 1;
        }
        // whoever reads them may have given up: the last ones have to be there before the CTA ends
        const auto arrived = [&](uint64_t* bar, int use) { ok = mbar_wait_bounded(bar, use & 1, ok ? WAIT_TRIES : DRAIN_TRIES) && ok; };
        for (int j = max(0, ks - 2); j < ks; ++j) arrived(&bar_k[j & 1], j >> 1);
        if (vs > 0) arrived(&bar_v[0], vs - 1);
        if (!ok) atomicExch(a.status, CQ_ERR_TIMEOUT);
      }
      __syncwarp();
    }
  } else {
    // ================= softmax: thread = row =================
    setmaxnreg_inc<Roles<IMAGE>::SOFTMAX_REGS>();
    const int x = warp >> 2, quarter = warp & 3, r_in = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + (uint32_t)x * 128u + lane_off, tO = tmem + 256u + (uint32_t)x * 128u + lane_off;
    const int q_first = i0 + (PAIR ? x * a.tile_queries : 0), i_in = r_in / p.n_rep, i = q_first + i_in;
    const bool valid_row = r_in < a.tile_rows && i < p.q_len;
    const int limit = live - p.q_len + i + 1;                     // full-precision tokens that the row sees
    const int n_x = PAIR ? k.n : (k.n + 1 - x) >> 1;
    // Units of the reference: without a mask, scores as the tensor core gives them; with one they are scaled and masked first (a mask of
    // the type's lowest value times log2 e would leave fp32's range).  `factor` makes powers of two of either.
    const float factor = MASK ? LOG2E : a.scale * LOG2E;
    bool ok = true;
    float m_ref = -INFINITY, l_run = 0.f;
    const auto mask_of = [&](int j) {                              // of column r_in of this tile's j-th key tile
      const int tile = k.t0 + (PAIR ? j : 2 * j + x);
      const int key = tile < k.nv ? tile * 128 + r_in : p.t_vis + (tile - k.nv) * 128 + r_in;
      if (j >= n_x || (tile < k.nv ? key >= p.t_vis : key - p.t_vis >= live)) return Elem<T>::from_f(-INFINITY);
      return static_cast<const T*>(p.mask)[b * p.mask_sb + mask_index(p, key)];
    };
    const auto lim_tile = [&](int tile) { return tile < k.nv ? p.t_vis - tile * 128 : live - (tile - k.nv) * 128; };      // keys that are there
    T mask_next = MASK ? mask_of(0) : Elem<T>::from_f(0.f);
    for (int j = 0; j < n_x; ++j) {
      const int tile = k.t0 + (PAIR ? j : 2 * j + x);
      const int lim = min(128, tile < k.nv ? p.t_vis - tile * 128 : limit - (tile - k.nv) * 128);      // columns from lim on are not seen
      const T* mk = mask_s[MASK ? x : 0][MASK ? j & 1 : 0];
      bool masked = false;                    // some mask of the tile is not zero; most tiles of a padded request have none
      if (MASK) {
        mask_s[x][j & 1][r_in] = mask_next;
        masked = tile_any(1 + x, Elem<T>::to_f(mask_next) != 0.f && r_in < lim_tile(tile));
        mask_next = mask_of(j + 1);
      }
      const bool need = __any_sync(0xffffffffu, lim < 128);
      if (ok) ok = mbar_wait_cycles(&bar_s[x], j & 1, WAIT_CYCLES);
      tc_fence_after();
      const auto shown = [&](int cc, uint32_t (&s)[32]) {          // 32 scores with the mask
        if (MASK && masked) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const uint2 m4 = *reinterpret_cast<const uint2*>(mk + cc * 32 + c);
            const uint16_t m16[4] = {(uint16_t)m4.x, (uint16_t)(m4.x >> 16), (uint16_t)m4.y, (uint16_t)(m4.y >> 16)};
            const float m[4] = {number<BF16>(m16[0]), number<BF16>(m16[1]), number<BF16>(m16[2]), number<BF16>(m16[3])};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[c + e] = m[e] == -INFINITY ? 0xff800000u : __float_as_uint(fmaf(__uint_as_float(s[c + e]), a.scale, m[e]));
          }
        }
        if (need) {
#pragma unroll
          for (int c = 0; c < 32; ++c)
            if (cc * 32 + c >= lim) s[c] = 0xff800000u;
        }
      };
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      uint32_t s[IMAGE ? 4 : 2][32];          // with images the row's 128 scores, read once
      const auto read = [&](int half) {
        tmem_ld32_nowait(tS + half * 64, s[IMAGE ? half * 2 : 0]);
        tmem_ld32_nowait(tS + half * 64 + 32, s[IMAGE ? half * 2 + 1 : 1]);
      };
      if (IMAGE) read(0);
      if (IMAGE) read(1);
#pragma unroll (IMAGE ? 2 : 1)
      for (int half = 0; half < 2; ++half) {
        if (!IMAGE) read(half);
        if (!IMAGE || half == 0) tmem_ld_wait();
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t (&v)[32] = s[IMAGE ? half * 2 + cc : cc];
          shown(half * 2 + cc, v);
#pragma unroll
          for (int c = 0; c < 32; c += 2) mx4[(c >> 1) & 3] = max3(mx4[(c >> 1) & 3], __uint_as_float(v[c]), __uint_as_float(v[c + 1]));
        }
      }
      const float top = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), m_true = fmaxf(m_ref, MASK && !masked ? top * a.scale : top);
      // a row keeps its reference until the true maximum is 2^8 above it (probabilities stay below 256), or for the first time
      const bool grow = (m_true - m_ref) * factor > 8.f;
      if (j > 0 && __any_sync(0xffffffffu, grow)) {
        if (ok) ok = mbar_wait_bounded(&bar_pv[x], (j - 1) & 1, WAIT_TRIES);
        tc_fence_after();
        const float alpha = grow ? exp2f((m_ref - m_true) * factor) : 1.f;
#pragma unroll 1
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t r[32];
          tmem_ld32(tO + cc * 32, r);
#pragma unroll
          for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * alpha);
          tmem_st32(tO + cc * 32, r);
        }
        l_run *= alpha;
      }
      if (grow) m_ref = m_true;
      // A row that has seen nothing but keys at the type's lowest value has a reference whose multiple may leave fp32's range, and the hidden
      // keys of a tile without a mask are at -infinity: what is added to those stays finite
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref, neg = fminf(-m_use * factor, FLT_MAX);
      float rs[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll (IMAGE ? 2 : 1)
      for (int half = 0; half < 2; ++half) {
        uint32_t w[32];
        if (!IMAGE) {
          read(half);
          tmem_ld_wait();
        }
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          uint32_t (&v)[32] = s[IMAGE ? half * 2 + cc : cc];
          if (!IMAGE) shown(half * 2 + cc, v);
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            float e0 = __uint_as_float(v[c]), e1 = __uint_as_float(v[c + 1]);
            if (MASK && masked) {
              e0 = (e0 - m_use) * factor;
              e1 = (e1 - m_use) * factor;
            } else {
              fma_pair(e0, e1, e0, e1, a.scale * LOG2E, a.scale * LOG2E, neg, neg);
            }
            e0 = ex2_approx(e0);
            e1 = ex2_approx(e1);
            add_pair(rs[c & 2], rs[(c & 2) + 1], e0, e1);
            w[cc * 16 + (c >> 1)] = pack16<BF16>(e0, e1);
          }
        }
        tmem_st32(tS + half * 32, w);               // over scores that have been read
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&bar_p[x][half]);
      }
      l_run += (rs[0] + rs[1]) + (rs[2] + rs[3]);
    }
    // without a key tile no product was waited for, and the queries may still be on their way to where the results are staged
    if (ok) ok = n_x > 0 ? mbar_wait_bounded(&bar_pv[x], (n_x - 1) & 1, WAIT_TRIES) : mbar_wait_bounded(&bar_q, 0, WAIT_TRIES);
    ok = __all_sync(0xffffffffu, ok);
    if (!ok) {
      mbar_wait_bounded(&bar_q, 0, DRAIN_TRIES);
      if (lane == 0) atomicExch(a.status, CQ_ERR_TIMEOUT);
    }
    tc_fence_after();
    const int h = hk * p.n_rep + r_in - i_in * p.n_rep;
    const float nat = MASK ? 1.f : a.scale;         // reference maximum in natural units
    if (a.parts == 1) {
      // the tile's rows through its query tile in shared memory (no product reads that any more), then 16 lanes a row
      const bool bad = !ok || l_run != l_run;       // no result, or a key or query that is not a number
      const float inv = bad ? NAN : l_run > 0.f ? 1.f / l_run : 0.f;
      if (valid_row && p.lse) p.lse[((int64_t)b * p.hq + h) * p.q_len + i] = bad ? NAN : l_run > 0.f ? m_ref * nat + logf(l_run) : -INFINITY;
      const uint32_t stage = q_s + (uint32_t)x * TILE_BYTES;
      const bool sums = n_x > 0 && ok;
#pragma unroll 1
      for (int cc = 0; cc < 4; ++cc) {
        uint32_t r[32];
        if (sums) tmem_ld32(tO + cc * 32, r);
#pragma unroll
        for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(sums ? __uint_as_float(r[c]) * inv : inv);
#pragma unroll
        for (int c = 0; c < 32; c += 8) {           // columns 0 4 1 5 2 6 3 7 of eight channels
          const auto f = [&](int e) { return __uint_as_float(r[c + e]); };
          sts128(chunk_at(stage, r_in, cc * 4 + (c >> 3)), pack16<BF16>(f(0), f(2)), pack16<BF16>(f(4), f(6)), pack16<BF16>(f(1), f(3)),
                 pack16<BF16>(f(5), f(7)));
        }
      }
      __syncwarp();
      for (int it = 0; it < 16; ++it) {
        const int rr = quarter * 32 + it * 2 + (lane >> 4), ii = rr / p.n_rep;
        if (rr < a.tile_rows && q_first + ii < p.q_len) {
          const uint4 v = lds128(chunk_at(stage, rr, lane & 15));
          T* dst = static_cast<T*>(p.out) + b * p.o_sb + (int64_t)(q_first + ii) * p.o_st + (int64_t)(hk * p.n_rep + rr - ii * p.n_rep) * p.o_sh;
          *reinterpret_cast<uint4*>(dst + (lane & 15) * 8) = v;
        }
      }
    } else if (__any_sync(0xffffffffu, valid_row)) {
      // a partial result, the channels in their order
      const int64_t at = (bh * p.rows + (int64_t)i * p.n_rep + (h - hk * p.n_rep)) * a.parts + (PAIR ? part : 2 * part + x);
      if (valid_row) a.part_ml[at] = make_float2(ok ? (n_x > 0 ? m_ref * nat : -INFINITY) : 0.f, ok ? l_run : NAN);
      if (n_x > 0 && ok) {
#pragma unroll 1
        for (int cc = 0; cc < 4; ++cc) {
          uint32_t r[32];
          tmem_ld32(tO + cc * 32, r);
          if (valid_row) {
            float4* dst = reinterpret_cast<float4*>(a.part_o + at * 128 + cc * 32);
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
              const auto f = [&](int e) { return __uint_as_float(r[c + e]); };
              dst[c >> 2] = make_float4(f(0), f(2), f(4), f(6));
              dst[(c >> 2) + 1] = make_float4(f(1), f(3), f(5), f(7));
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

// Merge of a row's partial results: a warp per row, a lane per four channels.
template <bool BF16>
__global__ void __launch_bounds__(256) chunk_combine_kernel(AttnParams a, int64_t all_rows) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const Params& p = a.p;
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  pdl_wait();
  if (at >= all_rows) return;
  const float2* ml = a.part_ml + at * a.parts;
  float m = -INFINITY;
  bool bad = false;
  for (int s = 0; s < a.parts; ++s) {
    const float2 v = ml[s];
    bad |= v.y != v.y;
    if (v.y > 0.f) m = fmaxf(m, v.x);
  }
  float l = 0.f, o[4] = {};
  for (int s = 0; s < a.parts; ++s) {
    const float2 v = ml[s];
    if (!(v.y > 0.f)) continue;
    const float f = exp2f((v.x - m) * LOG2E);
    const float4 x = *reinterpret_cast<const float4*>(a.part_o + (at * a.parts + s) * 128 + lane * 4);
    l = fmaf(v.y, f, l);
    o[0] = fmaf(x.x, f, o[0]); o[1] = fmaf(x.y, f, o[1]); o[2] = fmaf(x.z, f, o[2]); o[3] = fmaf(x.w, f, o[3]);
  }
  const float inv = bad ? NAN : l > 0.f ? 1.f / l : 0.f;
  const int row = (int)(at % p.rows), i = row / p.n_rep;
  const int64_t bh = at / p.rows, b = bh / p.hkv, h = (bh % p.hkv) * p.n_rep + row % p.n_rep;
  T* dst = static_cast<T*>(p.out) + b * p.o_sb + i * p.o_st + h * p.o_sh + lane * 4;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack16<BF16>(o[0] * inv, o[1] * inv), pack16<BF16>(o[2] * inv, o[3] * inv));
  if (p.lse && lane == 0) p.lse[(b * p.hq + h) * p.q_len + i] = bad ? NAN : l > 0.f ? m + logf(l) : -INFINITY;
}

// 3328 visual tokens, images against unpacking in the kernel: 300 queries of 8 requests (5 row blocks) 290 against 282 us, 400 (7 blocks) 371
// against 380, 150 (3 blocks) 192 against 167.
constexpr int IMAGE_BLOCKS = 6;

// ---- host ---------------------------------------------------------------------------------------------------------
struct Plan {
  bool few, pair, image, cluster;      // few: cq_chunk_few.cu; cluster: it merges its parts itself
  int queries, row_blocks, grid_parts, parts;      // queries of a tile
};
// Split of the key tiles: as many CTAs as fill the SMs, in whole rounds where there are several; a CTA costs about three key tiles beside
// its own (its start, and its partial result).
static Plan make_plan(const cq_chunk_args* a) {
  Plan pl;
  const int64_t rows = (int64_t)a->q_len * (a->n_q_heads / a->n_kv_heads);
  pl.few = rows <= FEW_ROWS;
  pl.pair = pl.image = pl.cluster = false;
  if (pl.few) {
    pl.queries = pl.row_blocks = 0;
    pl.grid_parts = pl.parts = few_parts((int64_t)a->batch * a->n_kv_heads, a->t_vis, a->t_fp, rows > 8, true);
    pl.cluster = pl.parts > 1 && pl.parts <= FEW_CLUSTER;
    return pl;
  }
  pl.queries = 128 / (a->n_q_heads / a->n_kv_heads);
  pl.pair = a->q_len > pl.queries;
  const int block = pl.queries * (pl.pair ? 2 : 1);
  pl.row_blocks = (a->q_len + block - 1) / block;
  const int64_t items = (int64_t)a->batch * a->n_kv_heads * pl.row_blocks;
  const int tiles = (a->t_vis + 127) / 128 + (a->t_fp + 127) / 128, sms = sm_count();
  int best = 1;
  double cost = 1e300;
  for (int s = 1; s <= 64 && s <= tiles; ++s) {
    const int per = (tiles + s - 1) / s;
    if (s > 1 && (tiles + per - 1) / per != s) continue;      // leaves a part empty
    const double c = (double)((items * s + sms - 1) / sms) * (per * (pl.pair ? 2 : 1) + 3 + (s > 1 && pl.pair ? 2 : 0));
    if (c < cost) { cost = c; best = s; }
  }
  // Key tiles that several row blocks would unpack are unpacked once, if their images take a gigabyte at most
  pl.image = pl.row_blocks >= IMAGE_BLOCKS && (size_t)a->batch * a->n_kv_heads * image_bytes((a->t_vis + 127) / 128, (a->t_fp + 127) / 128) <= (size_t)1 << 30;
  pl.grid_parts = best;
  pl.parts = pl.pair ? best : 2 * best;
  return pl;
}
// The status word's 256 bytes, the images, the partial results.
static size_t images_of(const cq_chunk_args* a, const Plan& pl) {
  return pl.image ? (size_t)a->batch * a->n_kv_heads * image_bytes((a->t_vis + 127) / 128, (a->t_fp + 127) / 128) : 0;
}
static size_t workspace_bytes(const cq_chunk_args* a, const Plan& pl) {
  const size_t rows = (size_t)a->batch * a->n_q_heads * a->q_len;
  return 256 + images_of(a, pl) + (pl.parts == 1 || pl.cluster ? 0 : rows * pl.parts * (128 * sizeof(float) + sizeof(float2)));
}

template <bool BF16>
static int launch_combine(const AttnParams& p, int batch, cudaStream_t st) {
  if (p.parts == 1) return CQ_OK;
  const int64_t rows = (int64_t)batch * p.p.hkv * p.p.rows;
  return launched(launch_pdl(chunk_combine_kernel<BF16>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, p, rows));
}

template <bool BF16, bool MASK, bool PAIR, bool IMAGE>
static int launch_attn(const CUtensorMap& tm, const AttnParams& p, const Plan& pl, int batch, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return CQ_ERR_LAUNCH;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(chunk_attn_kernel<BF16, MASK, PAIR, IMAGE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(chunk_unpack_kernel<BF16, MASK>, cudaFuncAttributeMaxDynamicSharedMemorySize, 3 * TILE_BYTES + 1024) != cudaSuccess)
      return CQ_ERR_LAUNCH;
    configured[dev] = true;
  }
  const dim3 grid(pl.row_blocks, batch * p.p.hkv, pl.grid_parts);
  if (IMAGE) {
    const dim3 tiles((p.p.t_vis + 127) / 128 + p.image_fp_tiles, batch * p.p.hkv);
    if (const int rc = launched(launch_pdl(chunk_unpack_kernel<BF16, MASK>, tiles, dim3(256), 3 * TILE_BYTES + 1024, st, p))) return rc;
  }
  if (const int rc = launched(launch_pdl(chunk_attn_kernel<BF16, MASK, PAIR, IMAGE>, grid, dim3(Roles<IMAGE>::THREADS), SMEM_BYTES, st, tm, p))) return rc;
  return launch_combine<BF16>(p, batch, st);
}

static bool attn_valid(const cq_chunk_args* a) {
  if (!valid(a) || !a->out || !aligned16(a->out) || !a->v_fp || !aligned16(a->v_fp)) return false;
  const int extent[3] = {a->batch, a->q_len, a->n_q_heads};
  for (int i = 0; i < 3; ++i)
    if (a->out_strides[i] % 8 || (extent[i] > 1 && a->out_strides[i] <= 0)) return false;
  return !a->t_vis || (a->v_code && a->v_scale && a->v_mn && aligned16(a->v_code) && aligned16(a->v_scale) && aligned16(a->v_mn));
}
static bool attn_supported(const cq_chunk_args* a) {
  return supported(a) && (int64_t)a->batch * a->n_kv_heads <= 65535;
}

}  // namespace chunk
}  // namespace cq

using namespace cq;

extern "C" size_t cq_chunk_attn_workspace_bytes(const cq_chunk_args* a) {
  if (!chunk::attn_valid(a) || !chunk::attn_supported(a)) return 0;
  return chunk::workspace_bytes(a, chunk::make_plan(a));
}

extern "C" int cq_chunk_attn(const cq_chunk_args* a, void* workspace, size_t workspace_bytes, void* stream) {
  if (!chunk::attn_valid(a)) return CQ_ERR_BAD_ARG;
  if (!chunk::attn_supported(a)) return CQ_ERR_UNSUPPORTED;
  const chunk::Plan pl = chunk::make_plan(a);
  if (!workspace || !aligned16(workspace) || workspace_bytes < chunk::workspace_bytes(a, pl)) return CQ_ERR_WORKSPACE;
  if (a->batch == 0) return CQ_OK;
  chunk::AttnParams p = {};
  p.p = chunk::make_params(a);
  p.parts = pl.parts;
  p.scale = 0.08838834764831845f;
  p.tile_queries = pl.queries; p.tile_rows = pl.queries * p.p.n_rep;
  const int bf16 = a->dtype == CQ_DTYPE_BF16;
  p.idesc_kmajor = chunk::idesc_of(bf16, 0, 0, 128, 128);
  p.idesc_mn = chunk::idesc_of(bf16, 0, 1, 128, 128);
  const size_t rows = (size_t)a->batch * a->n_q_heads * a->q_len;
  p.status = static_cast<int*>(workspace);
  p.image = static_cast<unsigned char*>(workspace) + 256;
  p.image_fp_tiles = (a->t_fp + 127) / 128;
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256 + chunk::images_of(a, pl));
  p.part_ml = reinterpret_cast<float2*>(p.part_o + rows * pl.parts * 128);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (pl.few) {
    chunk::FewParams f = {};
    f.p = p.p; f.part_o = p.part_o; f.part_ml = p.part_ml; f.status = p.status; f.parts = pl.parts; f.cluster = pl.cluster;
    const int rc = chunk::few_run(f, a->batch, bf16, false, st);
    if (rc || pl.cluster) return rc;
    return bf16 ? chunk::launch_combine<true>(p, a->batch, st) : chunk::launch_combine<false>(p, a->batch, st);
  }
  CUtensorMap tm;
  if (!chunk::query_map(&tm, a, pl.queries)) return CQ_ERR_LAUNCH;
#define CQ_RUN(B, M) (pl.image ? chunk::launch_attn<B, M, true, true>(tm, p, pl, a->batch, st) : \
                      pl.pair ? chunk::launch_attn<B, M, true, false>(tm, p, pl, a->batch, st) : chunk::launch_attn<B, M, false, false>(tm, p, pl, a->batch, st))
  if (bf16) return a->mask ? CQ_RUN(true, true) : CQ_RUN(true, false);
  return a->mask ? CQ_RUN(false, true) : CQ_RUN(false, false);
#undef CQ_RUN
}
