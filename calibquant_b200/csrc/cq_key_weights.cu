// How much attention the queries of a chunk paid to each key: column sums of exp(score - log-sum-exp), on tcgen05.
//
// The scores are formed the other way round than for the attention, S^T = K Q^T: a TMEM lane per key, so that a key's sum over the queries
// stays in one thread and no exchange is needed.  A CTA holds two key tiles of 128 (packed keys as two 16-bit terms, as there) and
// goes over the query rows of their KV head in blocks of NB.  Roles:
//   warps 0-15  the key tiles, once; then the sums: a thread has a key and every other 32 (16) of a block's rows, warps 0-3, 8-11 tile 0,
//               4-7, 12-15 tile 1
//   warp 16     issues the products
//   warp 17     has TMA bring the query blocks into two slots
// A block is the query heads of the KV head for as many queries as NB rows hold: a row of a block is the same head for every block.
// Bound: 64 products of 64 cycles per pair of packed key tiles and 256 rows, and the 2 x 128 x 128 exponentials of a block of 128 rows, which
// take the special-function units as long as its products take the tensor cores (2048 cycles) and run beside them; 2750 cycles a block
// measured.  8 x 1024 queries on 3328 + 1280 keys, bfloat16: 455 us alone, 460 in a row of launches, of which 10 % are
// the CTAs' starts (key tiles, first block).  Trials, on a GPU where this form took 422: half the products 407, no exponentials 385.  Keys in tensor memory as the products' other
// operand (nothing but queries read from shared memory), four query slots, a quarter of the exponentials by a polynomial: 410 to 424, and 4 us
// more for 20 to 100 queries, whose key tiles go through shared memory first.  Scores in halves of 64 rows: 474.
// The rows' log-sum-exp come by cp.async one chunk ahead, both key tiles are requested before one is unpacked: 41 -> 39 us (2 x 517
// queries on 1312 + 600), 28.6 -> 26.7 (300 on 3328 + 360).
// TMEM: tile X's scores in columns X * 256 + buffer * 128.  Where the key tiles are fewer than the SMs, the rows are cut into parts whose
// sums finish_kernel adds in their order.
#include <cuda.h>
#include <math.h>

#include <type_traits>

#include "cq_chunk_few.cuh"
#include "cq_chunk_tc.cuh"

namespace cq {
namespace chunk {

using namespace ptx;
using namespace tc;

namespace kw {

constexpr int WORKERS = 16, MMA_WARP = 16, TMA_WARP = 17, THREADS = 18 * 32;
constexpr int LSE_BLOCKS = 16;             // blocks whose rows' log-sum-exp are in shared memory at a time
constexpr int SMEM_BYTES = 6 * TILE_BYTES + 1024;
constexpr uint32_t WAIT_TRIES = 1u << 22, DRAIN_TRIES = 1u << 16;      // the latter for what is still under way after a wait that ran out
constexpr long long WAIT_CYCLES = 1ll << 30;
constexpr float LOG2E = 1.4426950408889634f;

struct WeightParams {
  Params p;
  const float *vis_in, *fp_in;
  float *vis, *fp;
  int64_t capacity;          // full-precision weights per (batch row, KV head)
  int64_t batch;
  int parts, block_rows, block_queries;      // block_rows = block_queries * n_rep <= NB
  float* part;               // [part][batch][KV head][t_vis + capacity]
  float scale;
  uint32_t idesc_kmajor, idesc_mn;
  int* status;
};

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void worker_barrier() { asm volatile("bar.sync 1, 512;" ::: "memory"); }
// result of key `key` (cache order [visual | fp]) of KV head bh
__device__ __forceinline__ void put(const WeightParams& a, int64_t bh, int64_t key, float w) {
  const int64_t vis = bh * a.p.t_vis + key, fp = bh * a.capacity + key - a.p.t_vis;
  if (key < a.p.t_vis) a.vis[vis] = (a.vis_in ? a.vis_in[vis] : 0.f) + w;
  else a.fp[fp] = (a.fp_in ? a.fp_in[fp] : 0.f) + w;
}

template <bool BF16, bool MASK, int NB>
__global__ void __launch_bounds__(THREADS, 1) key_weights_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ WeightParams a) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  const Params& p = a.p;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const uint32_t k_s = smem_u32(smem), q_s = k_s + 4 * TILE_BYTES;      // key tiles [X][hi, lo], query slots
  // bar_k the key tiles are there; bar_q/free[slot] query blocks; bar_d/dfree[X][buffer] scores ready / read; bar_end all products done
  __shared__ __align__(8) uint64_t bar_k, bar_q[2], bar_free[2], bar_d[2][2], bar_dfree[2][2], bar_end;
  __shared__ uint32_t tmem_base_s;
  __shared__ __align__(16) float lse_s[2][LSE_BLOCKS * NB];
  __shared__ float half_s[256];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hk = blockIdx.y % p.hkv, b = blockIdx.y / p.hkv;
  const int64_t bh = (int64_t)b * p.hkv + hk;
  pdl_launch_dependents();
  pdl_wait();
  const int live = live_tokens(p), nv = (p.t_vis + 127) >> 7;
  // first key of tile X; keys of a tile that are there; first row that sees one of them
  const int tile0 = (int)blockIdx.x * 2;
  const auto first_key = [&](int x) { return tile0 + x < nv ? (tile0 + x) * 128 : p.t_vis + (tile0 + x - nv) * 128; };
  const auto alive = [&](int x) { return tile0 + x < nv || (tile0 + x - nv) * 128 < live; };
  const auto first_row = [&](int t) { return (int64_t)max(0, t - live + p.q_len) * p.n_rep; };      // of full-precision token t
  const int blocks_all = (p.q_len + a.block_queries - 1) / a.block_queries, per = (blocks_all + (int)gridDim.z - 1) / (int)gridDim.z;
  int blk0 = min(blocks_all, (int)blockIdx.z * per);
  const int blk1 = min(blocks_all, blk0 + per);
  if (tile0 >= nv) blk0 = max(blk0, (int)min((int64_t)blk1, first_row((tile0 - nv) * 128) / a.block_rows));
  const int n_x = !alive(0) ? 0 : alive(1) ? 2 : 1, nb = n_x ? blk1 - blk0 : 0;

  if (tid == 0) {
    mbar_init(&bar_k, WORKERS);
    mbar_init(&bar_end, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&bar_q[s], 1);
      mbar_init(&bar_free[s], 1);
      for (int x = 0; x < 2; ++x) {
        mbar_init(&bar_d[x][s], 1);
        mbar_init(&bar_dfree[x][s], 256);
      }
    }
    mbar_fence_init();
  }
  if (warp == MMA_WARP) tmem_alloc(&tmem_base_s, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  if (warp == TMA_WARP) {
    // ================= query blocks =================
    if (lane == 0) {
      bool ok = true;
      int n = 0;
      for (; n < nb; ++n) {
        const int s = n & 1;
        // rows of a block that no query fills are zeros for good: written before bar_k
        if (n >= 2) ok = mbar_wait_bounded(&bar_free[s], ((n >> 1) - 1) & 1, WAIT_TRIES);
        if (!ok) break;
        mbar_expect_tx(&bar_q[s], 256 * a.block_rows);
        const int i0 = (blk0 + n) * a.block_queries;
        tma_load_4d(q_s + s * TILE_BYTES, &tm_q, 0, hk * p.n_rep, i0, b, &bar_q[s]);
        tma_load_4d(q_s + s * TILE_BYTES + PANEL_BYTES, &tm_q, 64, hk * p.n_rep, i0, b, &bar_q[s]);
      }
      // whoever reads them may have given up: the last two blocks have to be there before the CTA ends
      for (int m = max(0, n - 2); m < n; ++m) ok = mbar_wait_bounded(&bar_q[m & 1], (m >> 1) & 1, ok ? WAIT_TRIES : DRAIN_TRIES) && ok;
      if (!ok) atomicExch(a.status, CQ_ERR_TIMEOUT);
    }
    __syncwarp();
  } else if (warp == MMA_WARP) {
    // ================= products =================
    // loop bounds come out of a shuffle, so that the compiler knows them to be the warp's and keeps the operands in uniform registers
    const auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const int nb_lane = nb, n_x_lane = n_x;
    const int nb = uniform(nb_lane), n_x = uniform(n_x_lane);
    const uint32_t lead = elect_one();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    constexpr uint32_t tile16 = TILE_BYTES >> 4;
    const uint64_t kd = smem_desc(k_s, 16, 1024), md = smem_desc(k_s, PANEL_BYTES, 1024), qd = smem_desc(q_s, 16, 1024);
    const auto all = [](bool r) { return __all_sync(0xffffffffu, r) != 0; };
    // slot and tile as constants: with both as indices the issuing lane's address arithmetic held up the tensor pipe
    const auto issue = [&](auto xc, auto sc, bool packed) {
      constexpr int x = decltype(xc)::value, s = decltype(sc)::value;
      if (lead) {
        if (packed) {
          // its small terms first: sums are cut off, not rounded
#pragma unroll
          for (int ks = 0; ks < 16; ++ks) {
            constexpr uint32_t lo = (2 * x + 1) * tile16, hi = 2 * x * tile16;
            const uint32_t qo = (uint32_t)((((ks & 7) >> 2) * PANEL_BYTES + (ks & 3) * 32) >> 4);
            umma(tm + (uint32_t)(x * 256 + s * 128), desc_at(md, (ks < 8 ? lo : hi) + (ks & 7) * 128), desc_at(qd, s * tile16 + qo), a.idesc_mn, ks > 0);
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const uint32_t qo = (uint32_t)(((ks >> 2) * PANEL_BYTES + (ks & 3) * 32) >> 4);
            umma(tm + (uint32_t)(x * 256 + s * 128), desc_at(kd, 2 * x * tile16 + qo), desc_at(qd, s * tile16 + qo), a.idesc_kmajor, ks > 0);
          }
        }
        umma_commit(&bar_d[x][s]);
      }
    };
    const bool packed0 = uniform(tile0 < nv), packed1 = uniform(tile0 + 1 < nv);
    bool ok = nb == 0 || all(mbar_wait_bounded(&bar_k, 0, WAIT_TRIES));
    const auto block = [&](auto sc, int n) {
      constexpr int s = decltype(sc)::value;
      ok = all(mbar_wait_bounded(&bar_q[s], (n >> 1) & 1, WAIT_TRIES));
      if (ok && n >= 2) ok = all(mbar_wait_cycles(&bar_dfree[0][s], ((n >> 1) - 1) & 1, WAIT_CYCLES));
      if (!ok) return;
      tc_fence_after();
      issue(std::integral_constant<int, 0>{}, sc, packed0);
      if (n_x > 1) {
        if (n >= 2) ok = all(mbar_wait_cycles(&bar_dfree[1][s], ((n >> 1) - 1) & 1, WAIT_CYCLES));
        if (!ok) return;
        tc_fence_after();
        issue(std::integral_constant<int, 1>{}, sc, packed1);
      }
      if (lead) umma_commit(&bar_free[s]);
    };
    for (int n = 0; n < nb && ok; n += 2) {
      block(std::integral_constant<int, 0>{}, n);
      if (n + 1 < nb && ok) block(std::integral_constant<int, 1>{}, n + 1);
    }
    if (lead) umma_commit(&bar_end);
    ok = all(mbar_wait_bounded(&bar_end, 0, ok ? WAIT_TRIES : DRAIN_TRIES)) && ok;
    if (!ok && lead) atomicExch(a.status, CQ_ERR_TIMEOUT);
    __syncwarp();
  } else {
    // rows' log-sum-exp of the blocks from n0 on, on their way; what adds nothing -inf
    const auto request_lse = [&](int n0, int buf) {
      for (int c = tid; c < LSE_BLOCKS * NB; c += 512) {
        const int r = c % NB, i = (blk0 + n0 + c / NB) * a.block_queries + r / p.n_rep;
        if (r < a.block_rows && n0 + c / NB < nb && i < p.q_len)
          cp_async4(&lse_s[buf][c], p.lse + ((int64_t)b * p.hq + hk * p.n_rep + r % p.n_rep) * p.q_len + i);
        else
          lse_s[buf][c] = -INFINITY;
      }
    };
    // minus them in units of the exponent (with a mask: as they are); a row that adds nothing: an argument of -inf
    const auto take_lse = [&](int buf) {
      cp_async_wait();
      for (int c = tid; c < LSE_BLOCKS * NB; c += 512) {
        const float v = lse_s[buf][c];
        lse_s[buf][c] = v == -INFINITY ? (MASK ? INFINITY : -INFINITY) : MASK ? v : -v * LOG2E;
      }
    };
    if (nb > 0) request_lse(0, 0);
    // ================= the key tiles =================
    if (nb > 0) {
      Unit u[2];
#pragma unroll
      for (int x = 0; x < 2; ++x)
        if (x < n_x && tile0 + x < nv) load_k_unit(p, bh, tile0 + x, warp, lane, u[x]);
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x >= n_x) break;
        const uint32_t hi = k_s + x * 2 * TILE_BYTES, lo = hi + TILE_BYTES;
        if (tile0 + x < nv) {
          store_k_unit<BF16>(hi, lo, u[x], warp, lane);
        } else {
          const T* src = static_cast<const T*>(p.k_fp) + b * p.fp_sb + hk * p.fp_sh;
#pragma unroll
          for (int it = 0; it < 4; ++it) {
            const int r = it * 32 + (tid >> 4), t = (tile0 + x - nv) * 128 + r;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (t < live) w = *reinterpret_cast<const uint4*>(src + (int64_t)t * 128 + (tid & 15) * 8);
            sts128(chunk_at(hi, r, tid & 15), w.x, w.y, w.z, w.w);
          }
        }
      }
      // rows of a block that no query fills
      for (int c = a.block_rows * 8 + tid; c < NB * 8; c += 512)
        for (int s = 0; s < 4; ++s) sts128(q_s + s * PANEL_BYTES + c * 16, 0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar_k);
    }
    // ================= sums: thread = key =================
    constexpr int COLS = NB / 4;                                        // columns at a time; a half takes the even or the odd ones of four
    const int x = (warp >> 2) & 1, half = warp >> 3, r_in = (warp & 3) * 32 + lane;
    const int64_t key = first_key(x) + r_in;
    const bool vis = tile0 + x < nv;
    const int t = (int)(key - p.t_vis);                                 // full-precision token
    const bool there = vis ? key < p.t_vis : t < live;
    float m = 0.f;
    if (MASK && there) m = Elem<T>::to_f(static_cast<const T*>(p.mask)[b * p.mask_sb + mask_index(p, (int)key)]);
    const int64_t rmin = vis ? 0 : first_row(t);                        // the first row that sees the key
    const uint32_t tD = tmem + (uint32_t)x * 256u + ((uint32_t)((warp & 3) * 32) << 16);
    const float c1 = a.scale * LOG2E;
    bool ok = true;
    float acc[4] = {};
    for (int n0 = 0; n0 < nb; n0 += LSE_BLOCKS) {
      const int buf = (n0 / LSE_BLOCKS) & 1;
      take_lse(buf);
      worker_barrier();                       // nobody reads the other half any more
      if (n0 + LSE_BLOCKS < nb) request_lse(n0 + LSE_BLOCKS, buf ^ 1);
      if (x >= n_x) continue;
      for (int n = n0; n < min(nb, n0 + LSE_BLOCKS); ++n) {
        const int s = n & 1;
        if (ok) ok = mbar_wait_cycles(&bar_d[x][s], (n >> 1) & 1, WAIT_CYCLES);
        tc_fence_after();
        uint32_t d[2][COLS];
        if constexpr (COLS == 32) {
          tmem_ld32_nowait(tD + s * 128 + half * 32, d[0]);
          tmem_ld32_nowait(tD + s * 128 + half * 32 + 64, d[1]);
        } else {
          tmem_ld8_nowait(tD + s * 128 + half * 8, d[0]);
          tmem_ld8_nowait(tD + s * 128 + half * 8 + 16, d[1]);
        }
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(&bar_dfree[x][s]);
        const int64_t hidden = rmin - (int64_t)(blk0 + n) * a.block_rows;      // columns below are not seen
        const auto sum = [&](auto diagonal) {
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const int col0 = cc * 2 * COLS + half * COLS;
            const float* l_s = &lse_s[buf][(n - n0) * NB + col0];
#pragma unroll
            for (int c = 0; c < COLS; c += 4) {
              const float4 l = *reinterpret_cast<const float4*>(l_s + c);
              const float f[4] = {__uint_as_float(d[cc][c]), __uint_as_float(d[cc][c + 1]), __uint_as_float(d[cc][c + 2]), __uint_as_float(d[cc][c + 3])};
              float e[4];
              if (MASK) {
                e[0] = (fmaf(f[0], a.scale, m) - l.x) * LOG2E;
                e[1] = (fmaf(f[1], a.scale, m) - l.y) * LOG2E;
                e[2] = (fmaf(f[2], a.scale, m) - l.z) * LOG2E;
                e[3] = (fmaf(f[3], a.scale, m) - l.w) * LOG2E;
              } else {
                fma_pair(e[0], e[1], f[0], f[1], c1, c1, l.x, l.y);
                fma_pair(e[2], e[3], f[2], f[3], c1, c1, l.z, l.w);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                e[i] = ex2_approx(e[i]);
                if (decltype(diagonal)::value && col0 + c + i < hidden) e[i] = 0.f;
              }
              add_pair(acc[0], acc[1], e[0], e[1]);
              add_pair(acc[2], acc[3], e[2], e[3]);
            }
          }
        };
        if (__any_sync(0xffffffffu, hidden > 0)) sum(std::true_type{});
        else sum(std::false_type{});
      }
    }
    if (!__all_sync(0xffffffffu, ok) && lane == 0) atomicExch(a.status, CQ_ERR_TIMEOUT);
    float w = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    if (!ok) w = NAN;
    if (half == 1) half_s[x * 128 + r_in] = w;
    worker_barrier();
    if (half == 0) {
      w += half_s[x * 128 + r_in];
      if (!there || (MASK && m == -INFINITY)) w = 0.f;
      const int64_t end = vis ? p.t_vis : p.t_vis + a.capacity;
      if (key < end) {
        if (a.parts == 1) put(a, bh, key, w);
        else a.part[((int64_t)blockIdx.z * a.batch * p.hkv + bh) * (p.t_vis + a.capacity) + key] = w;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

// sums of the parts, in their order
__global__ void __launch_bounds__(256) key_weights_finish_kernel(WeightParams a) {
  const int64_t key = (int64_t)blockIdx.x * 256 + threadIdx.x, bh = blockIdx.y, keys = a.p.t_vis + a.capacity;
  pdl_wait();
  if (key >= keys) return;
  float w = 0.f;
  for (int s = 0; s < a.parts; ++s) w += a.part[((int64_t)s * gridDim.y + bh) * keys + key];
  put(a, bh, key, w);
}

// ---- host ---------------------------------------------------------------------------------------------------------
struct Plan {
  int nb, queries, pairs, parts;      // queries of a block
};
static Plan make_plan(const cq_chunk_args* a, int64_t capacity) {
  Plan pl;
  const int64_t rows = (int64_t)a->q_len * (a->n_q_heads / a->n_kv_heads);
  const int n_rep = a->n_q_heads / a->n_kv_heads;
  pl.nb = rows <= 32 ? 32 : 128;
  pl.queries = pl.nb / n_rep;
  pl.pairs = (int)(((a->t_vis + 127) / 128 + (capacity + 127) / 128 + 1) / 2);
  // CTAs for the keys alone leave SMs idle: rows in parts, each of four blocks at least
  const int64_t ctas = (int64_t)a->batch * a->n_kv_heads * pl.pairs, blocks = (a->q_len + pl.queries - 1) / pl.queries;
  int64_t parts = ctas > 0 ? sm_count() / ctas : 1;
  if (parts > blocks / 4) parts = blocks / 4;
  pl.parts = (int)(parts < 1 ? 1 : parts > 16 ? 16 : parts);
  return pl;
}
static size_t bytes_of(const cq_chunk_args* a, int64_t capacity, const Plan& pl) {
  return 256 + (pl.parts > 1 ? (size_t)pl.parts * a->batch * a->n_kv_heads * (a->t_vis + capacity) * sizeof(float) : 0);
}

template <bool BF16, bool MASK, int NB>
static int run(const CUtensorMap& tm, const WeightParams& p, const Plan& pl, cudaStream_t st) {
  static bool configured[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return CQ_ERR_LAUNCH;
  if (!configured[dev]) {
    if (cudaFuncSetAttribute(key_weights_kernel<BF16, MASK, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) return CQ_ERR_LAUNCH;
    configured[dev] = true;
  }
  const unsigned bh = (unsigned)(p.batch * p.p.hkv);
  if (const int rc = launched(launch_pdl(key_weights_kernel<BF16, MASK, NB>, dim3(pl.pairs, bh, pl.parts), dim3(THREADS), SMEM_BYTES, st, tm, p))) return rc;
  if (pl.parts == 1) return CQ_OK;
  return launched(launch_pdl(key_weights_finish_kernel, dim3((unsigned)((p.p.t_vis + p.capacity + 255) / 256), bh), dim3(256), 0, st, p));
}

}  // namespace kw
}  // namespace chunk
}  // namespace cq

using namespace cq;

static bool weights_supported(const cq_chunk_args* a, int64_t capacity) {
  return chunk::supported(a) && a->t_vis + capacity < (1ll << 30) && (int64_t)a->batch * a->n_kv_heads <= 65535;
}

extern "C" size_t cq_key_weights_workspace_bytes(const cq_chunk_args* a, int64_t w_capacity) {
  if (!chunk::valid(a) || !a->lse || w_capacity < a->t_fp || !weights_supported(a, w_capacity)) return 0;
  return chunk::kw::bytes_of(a, w_capacity, chunk::kw::make_plan(a, w_capacity));
}

extern "C" int cq_key_weights(const cq_chunk_args* a, const float* w_vis_in, const float* w_fp_in, float* w_vis, float* w_fp,
                              int64_t w_capacity, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace chunk::kw;
  if (!chunk::valid(a) || !a->lse || (a->t_vis && !w_vis) || !w_fp || w_capacity < a->t_fp) return CQ_ERR_BAD_ARG;
  for (const float* w : {w_vis_in, w_fp_in, (const float*)w_vis, (const float*)w_fp})
    if (reinterpret_cast<uintptr_t>(w) % 4) return CQ_ERR_BAD_ARG;
  if (!weights_supported(a, w_capacity)) return CQ_ERR_UNSUPPORTED;
  const Plan pl = make_plan(a, w_capacity);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!workspace || !aligned16(workspace) || workspace_bytes < bytes_of(a, w_capacity, pl)) return CQ_ERR_WORKSPACE;
  if (a->batch == 0) return CQ_OK;
  const int bf16 = a->dtype == CQ_DTYPE_BF16;
  if ((int64_t)a->q_len * (a->n_q_heads / a->n_kv_heads) <= chunk::FEW_ROWS) {
    chunk::FewParams f = {};
    f.p = chunk::make_params(a);
    f.vis_in = w_vis_in; f.fp_in = w_fp_in; f.vis = w_vis; f.fp = w_fp; f.capacity = w_capacity;
    f.status = static_cast<int*>(workspace);
    f.parts = chunk::few_parts((int64_t)a->batch * a->n_kv_heads, a->t_vis, w_capacity, false, false);
    return chunk::few_run(f, a->batch, bf16, true, st);
  }
  WeightParams p = {};
  p.p = chunk::make_params(a);
  p.vis_in = w_vis_in; p.fp_in = w_fp_in; p.vis = w_vis; p.fp = w_fp;
  p.capacity = w_capacity; p.batch = a->batch; p.parts = pl.parts;
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + 256);
  p.scale = 0.08838834764831845f;
  p.block_queries = pl.queries; p.block_rows = pl.queries * p.p.n_rep;
  CUtensorMap tm;
  if (!chunk::query_map(&tm, a, pl.queries)) return CQ_ERR_LAUNCH;
  p.idesc_kmajor = chunk::idesc_of(bf16, 0, 0, 128, pl.nb);
  p.idesc_mn = chunk::idesc_of(bf16, 1, 0, 128, pl.nb);
  p.status = static_cast<int*>(workspace);
#define CQ_RUN(B, M) (pl.nb == 32 ? run<B, M, 32>(tm, p, pl, st) : run<B, M, 128>(tm, p, pl, st))
  if (bf16) return a->mask ? CQ_RUN(true, true) : CQ_RUN(true, false);
  return a->mask ? CQ_RUN(false, true) : CQ_RUN(false, false);
#undef CQ_RUN
}
