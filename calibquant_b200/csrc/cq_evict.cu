// Eviction by weight: of the units of a (batch row, KV head) -- groups of 32 packed visual tokens, or single full-precision tokens --
// the `keep` with the largest weight stay, in their order, and move to a smaller cache unchanged.
//
// Selection: the weights become integers whose order is the weights' order (the bits of the number, all of them flipped for a negative one, the
// sign bit for any other; -0 as +0, NaN above infinity).  Up to a thread's number of units are ranked by counting those above; of more, the
// value of the keep-th largest is found eight bits at a time from a histogram of the units that agree with it so far, until all that
// agree stay.  A unit stays if it is above that value, or equal to it and among the first of the equal ones that fill the rest.  A group's weight is the sum of its 32 weights in 64
// bits, in their order: exact, whatever the order, as long as the largest of them is at most 2^24 times the smallest one above zero.  Only counts are
// added atomically: the result depends on nothing but the weights.
// Bound: HBM, and before it the selection, which every CTA waits for.  A group's keys are 16 bytes of 128 rows: a quarter of the groups kept
// reads two thirds of the rows' 64-byte pieces and all of the scales, 261 MB for 8 x 8 heads of 32 768 tokens (40 us at the copy rate, 62
// measured; four CTAs an SM, each selecting for itself: 82).  16 x 8 heads of 4099 full-precision tokens, a quarter kept: 35 us, 4 TB/s (31 behind one another).
// One launch: every CTA of a (batch row, KV head) finds the selection itself and moves its share of the cache.
#include "cq_common.cuh"
#include "cq_ptx.cuh"

namespace cq {
namespace evict {

constexpr int THREADS = 512, BINS = 256;
constexpr int MAX_GROUPS = 16384, MAX_TOKENS = 24576;      // keys and places of all of them: 192 KB
constexpr int MAX_SMEM = 192 * 1024;

// order-preserving bits
__device__ __forceinline__ uint64_t ordered(double v) {
  if (v != v) return ~0ull;
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);      // -0 + 0 = +0
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ uint32_t ordered(float v) {
  if (v != v) return ~0u;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b >> 31 ? ~b : b | 1u << 31;
}

struct Shared {
  int hist[BINS];
  int scan[THREADS / 32][2];
  int digit, above;
};

// Sum of x over the threads before this one, and over all of them.
__device__ __forceinline__ int2 block_prefix(int x, int* total, int (*scan)[2], int which) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) scan[warp][which] = inc;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    const int v = scan[w][which];
    before += w < warp ? v : 0;
    all += v;
  }
  *total = all;
  return make_int2(before + inc - x, all);
}

// list[0 .. keep-1] = the units with the keep largest keys of key[0 .. n-1], ascending; all threads.
template <typename Key>
__device__ __forceinline__ void select(const Key* key, int n, int keep, int* list, Shared& s) {
  if (n <= THREADS) {
    const int i = threadIdx.x;
    bool stays = false;
    if (i < n) {
      const Key own = key[i];
      int above = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) above += key[j] > own || (key[j] == own && j < i);
      stays = above < keep;
    }
    int total;
    const int at = block_prefix(stays, &total, s.scan, 0).x;
    if (stays) list[at] = i;
    __syncthreads();
    return;
  }
  Key prefix = 0, mask = 0;
  int rest = keep;                               // how many of the units that agree with the prefix stay
  for (int shift = 8 * (int)sizeof(Key) - 8; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < BINS; i += THREADS) s.hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += THREADS) {
      const Key k = key[i];
      if ((k & mask) == prefix) atomicAdd(&s.hist[(int)(k >> shift) & (BINS - 1)], 1);
    }
    __syncthreads();
    if (threadIdx.x < 32) {                      // the digit with fewer than `rest` units above it and at least `rest` from it on
      int c[8], sum = 0;
      for (int i = 0; i < 8; ++i) sum += c[i] = s.hist[BINS - 1 - (threadIdx.x * 8 + i)];
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, inc, o);
        if ((int)threadIdx.x >= o) inc += up;
      }
      int above = inc - sum;
      if (above < rest && inc >= rest) {
        int i = 0;
        while (above + c[i] < rest) above += c[i++];
        s.digit = BINS - 1 - ((int)threadIdx.x * 8 + i);
        s.above = above;
      }
    }
    __syncthreads();
    prefix |= (Key)s.digit << shift;
    mask |= (Key)(BINS - 1) << shift;
    rest -= s.above;
    const bool whole = s.hist[s.digit] == rest;      // all that agree so far stay
    __syncthreads();
    if (whole) break;
  }
  // each thread a run of consecutive units, so that the places are ascending
  const int run = (n + THREADS - 1) / THREADS, i0 = min(n, (int)threadIdx.x * run), i1 = min(n, i0 + run);
  int above = 0, equal = 0;
  for (int i = i0; i < i1; ++i) {
    above += (key[i] & mask) > prefix;
    equal += (key[i] & mask) == prefix;
  }
  int total;
  int ties = block_prefix(equal, &total, s.scan, 0).x;
  int place = block_prefix(above, &total, s.scan, 1).x + min(ties, rest);
  for (int i = i0; i < i1; ++i) {
    const Key k = key[i] & mask;
    if (k > prefix) list[place++] = i;
    else if (k == prefix && ties++ < rest) list[place++] = i;
  }
  __syncthreads();
}

template <int WORDS> struct Codes;      // of a channel and group
template <> struct Codes<1> { using T = uint32_t; };
template <> struct Codes<2> { using T = uint2; };
template <> struct Codes<4> { using T = uint4; };

struct Groups {
  const void* k_code; const uint16_t *k_scale, *k_mn;
  const uint4* v_code; const uint4 *v_scale, *v_mn;
  const float4* weights;
  void* k_code_out; uint16_t *k_scale_out, *k_mn_out;
  uint4* v_code_out; uint4 *v_scale_out, *v_mn_out;
  float4* w_out;
  int64_t* kept;
  int groups, keep;
};

// WORDS (= bits) 32-bit words of codes per channel and group
template <int WORDS>
__global__ void __launch_bounds__(THREADS) groups_kernel(Groups p) {
  using C = typename Codes<WORDS>::T;
  extern __shared__ uint64_t key[];
  __shared__ Shared s;
  int* list = reinterpret_cast<int*>(key + p.groups);
  const int64_t bh = blockIdx.y;
  const int keep = p.keep, groups = p.groups, lane = threadIdx.x & 31;
  const float4* w = p.weights + bh * groups * 8;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  for (int g = threadIdx.x; g < groups; g += THREADS) {
    float4 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = w[(int64_t)g * 8 + i];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) { sum += v[i].x; sum += v[i].y; sum += v[i].z; sum += v[i].w; }
    key[g] = ordered(sum);
  }
  __syncthreads();
  select(key, groups, keep, list, s);
  // A warp takes a channel of the keys (32 groups at a time, side by side in the result) or the values and weights of a group
  const int warps = (int)gridDim.x * (THREADS / 32);
  for (int item = (int)blockIdx.x * (THREADS / 32) + ((int)threadIdx.x >> 5); item < 128 + keep; item += warps) {
    if (item < 128) {
      const int64_t from = (bh * 128 + item) * groups, to = (bh * 128 + item) * keep;
      const C* src = static_cast<const C*>(p.k_code) + from;
      C* dst = static_cast<C*>(p.k_code_out) + to;
      for (int j0 = 0; j0 < keep; j0 += 128) {
        C c[4];
        uint16_t sc[4], mn[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = j0 + u * 32 + lane;
          if (j < keep) {
            const int g = list[j];
            c[u] = src[g];
            sc[u] = p.k_scale[from + g];
            mn[u] = p.k_mn[from + g];
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int j = j0 + u * 32 + lane;
          if (j < keep) {
            dst[j] = c[u];
            p.k_scale_out[to + j] = sc[u];
            p.k_mn_out[to + j] = mn[u];
          }
        }
      }
    } else {
      const int j = item - 128, g = list[j];
      const int64_t from = bh * groups + g, to = bh * keep + j;
      uint4 c[WORDS];
#pragma unroll
      for (int i = 0; i < WORDS; ++i) c[i] = p.v_code[from * 32 * WORDS + i * 32 + lane];      // 32 tokens of WORDS 16-byte pieces
      const uint4 sm = lane < 16 ? p.v_scale[from * 16 + lane] : p.v_mn[from * 16 + lane - 16];
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (lane < 8) x = w[(int64_t)g * 8 + lane];
#pragma unroll
      for (int i = 0; i < WORDS; ++i) p.v_code_out[to * 32 * WORDS + i * 32 + lane] = c[i];
      if (lane < 16) p.v_scale_out[to * 16 + lane] = sm;
      else p.v_mn_out[to * 16 + lane - 16] = sm;
      if (lane < 8) p.w_out[to * 8 + lane] = x;
      if (lane == 0) p.kept[to] = g;
    }
  }
}

struct Tokens {
  const uint4 *k, *v;
  int64_t sb, sh;                              // in 16-byte units
  const float* weights;
  int64_t w_stride;
  uint4 *k_out, *v_out;
  float* w_out;
  int64_t* kept;
  int heads, t_fp, keep, t_sys, recent;
};

__global__ void __launch_bounds__(THREADS) tokens_kernel(Tokens p) {
  extern __shared__ uint32_t key32[];
  __shared__ Shared s;
  int* list = reinterpret_cast<int*>(key32 + p.t_fp);
  const int64_t bh = blockIdx.y;
  const float* w = p.weights + bh * p.w_stride;
  ptx::pdl_launch_dependents();
  ptx::pdl_wait();
  // among the tokens that need not stay
  const int n = p.t_fp - p.t_sys - p.recent, m = p.keep - p.t_sys - p.recent;
  for (int t = threadIdx.x; t < n; t += THREADS) key32[t] = ordered(w[p.t_sys + t]);
  __syncthreads();
  if (m > 0) select(key32, n, m, list, s);
  const uint4 *k = p.k + (bh / p.heads) * p.sb + (bh % p.heads) * p.sh, *v = p.v + (bh / p.heads) * p.sb + (bh % p.heads) * p.sh;
  const int64_t out = bh * p.keep;
  const auto source = [&](int j) { return j < p.t_sys ? j : j < p.t_sys + m ? p.t_sys + list[j - p.t_sys] : p.t_fp - (p.keep - j); };
  // half a warp takes a token's row, four of them at a time
  const int half = ((int)blockIdx.x * THREADS + (int)threadIdx.x) >> 4, halves = (int)gridDim.x * (THREADS / 16), c = threadIdx.x & 15;
  for (int j0 = half; j0 < p.keep; j0 += 4 * halves) {
    uint4 kx[4], vx[4];
    int t[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + u * halves;
      if (j < p.keep) {
        t[u] = source(j);
        kx[u] = k[(int64_t)t[u] * 16 + c];
        vx[u] = v[(int64_t)t[u] * 16 + c];
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = j0 + u * halves;
      if (j < p.keep) {
        p.k_out[(out + j) * 16 + c] = kx[u];
        p.v_out[(out + j) * 16 + c] = vx[u];
        if (c == 0) {
          p.w_out[out + j] = w[t[u]];
          p.kept[out + j] = t[u];
        }
      }
    }
  }
}

// CTAs per (batch row, KV head): as many as PER_SM an SM hold at once, at least 16 KB to move for each
constexpr int PER_SM = 2;
static int slices(int64_t rows, int64_t bytes) {
  const int64_t fill = PER_SM * sm_count() / rows, work = (bytes + 16383) / 16384, n = fill < work ? fill : work;
  return (int)(n > 0 ? n : 1);
}

template <typename... K, typename... A>
static int run(void (*kern)(K...), dim3 grid, size_t smem, cudaStream_t st, A... args) {
  // 48 KB need not be asked for, of which the kernels' own variables (Shared, above 1 KB) take their part
  static_assert(sizeof(Shared) <= 2048, "what is left of 48 KB");
  if (smem > 46 * 1024 && cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM) != cudaSuccess) {
    (void)cudaGetLastError();
    return CQ_ERR_LAUNCH;
  }
  return launched(launch_pdl(kern, grid, dim3(THREADS), smem, st, args...));
}

}  // namespace evict
}  // namespace cq

using namespace cq;

extern "C" int cq_evict_groups(const int32_t* k_code, const void* k_scale, const void* k_mn, const int32_t* v_code, const void* v_scale,
                               const void* v_mn, const float* weights, int batch, int heads, int head_dim, int t_vis, int keep,
                               int bits, int group_size, int32_t* k_code_out, void* k_scale_out, void* k_mn_out, int32_t* v_code_out,
                               void* v_scale_out, void* v_mn_out, float* w_out, int64_t* kept, void* stream) {
  if (batch < 0 || heads <= 0 || t_vis <= 0 || t_vis % kGroup || keep <= 0 || keep > t_vis / kGroup) return CQ_ERR_BAD_ARG;
  for (const void* q : {(const void*)k_code, k_scale, k_mn, (const void*)v_code, v_scale, v_mn, (const void*)weights, (const void*)k_code_out,
                        (const void*)k_scale_out, (const void*)k_mn_out, (const void*)v_code_out, (const void*)v_scale_out,
                        (const void*)v_mn_out, (const void*)w_out, (const void*)kept})
    if (!q || !aligned16(q)) return CQ_ERR_BAD_ARG;
  const int groups = t_vis / kGroup;
  const size_t smem = (size_t)groups * 8 + (size_t)keep * 4;
  if (head_dim != kHeadDim || group_size != kGroup || (bits != 1 && bits != 2 && bits != 4) || groups > evict::MAX_GROUPS ||
      (int64_t)batch * heads > 65535)
    return CQ_ERR_UNSUPPORTED;
  if (batch == 0) return CQ_OK;
  evict::Groups p = {k_code, static_cast<const uint16_t*>(k_scale), static_cast<const uint16_t*>(k_mn), reinterpret_cast<const uint4*>(v_code),
                     static_cast<const uint4*>(v_scale), static_cast<const uint4*>(v_mn), reinterpret_cast<const float4*>(weights), k_code_out,
                     static_cast<uint16_t*>(k_scale_out), static_cast<uint16_t*>(k_mn_out), reinterpret_cast<uint4*>(v_code_out),
                     static_cast<uint4*>(v_scale_out), static_cast<uint4*>(v_mn_out), reinterpret_cast<float4*>(w_out), kept, groups, keep};
  const int64_t rows = (int64_t)batch * heads;
  const dim3 grid(evict::slices(rows, (int64_t)keep * 32 * (32 * bits + 32)), (unsigned)rows);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (bits == 1) return evict::run(evict::groups_kernel<1>, grid, smem, st, p);
  if (bits == 2) return evict::run(evict::groups_kernel<2>, grid, smem, st, p);
  return evict::run(evict::groups_kernel<4>, grid, smem, st, p);
}

extern "C" int cq_evict_tokens(const void* k, const void* v, int64_t stride_b, int64_t stride_h, const float* weights, int64_t w_stride,
                               int batch, int heads, int head_dim, int t_fp, int keep, int t_sys, int recent, void* k_out,
                               void* v_out, float* w_out, int64_t* kept, void* stream) {
  if (batch < 0 || heads <= 0 || t_fp <= 0 || keep <= 0 || keep > t_fp || t_sys < 0 || recent < 0 || (int64_t)t_sys + recent > keep ||
      stride_b % 8 || stride_h % 8 || w_stride < t_fp)
    return CQ_ERR_BAD_ARG;
  for (const void* q : {k, v, (const void*)k_out, (const void*)v_out})
    if (!q || !aligned16(q)) return CQ_ERR_BAD_ARG;
  if (!weights || !w_out || !kept || reinterpret_cast<uintptr_t>(weights) % 4 || reinterpret_cast<uintptr_t>(w_out) % 4 || reinterpret_cast<uintptr_t>(kept) % 8)
    return CQ_ERR_BAD_ARG;
  const size_t smem = (size_t)t_fp * 4 + (size_t)(keep - t_sys - recent) * 4;
  if (head_dim != kHeadDim || t_fp > evict::MAX_TOKENS || (int64_t)batch * heads > 65535)
    return CQ_ERR_UNSUPPORTED;
  if (batch == 0) return CQ_OK;
  evict::Tokens p = {static_cast<const uint4*>(k), static_cast<const uint4*>(v), stride_b / 8, stride_h / 8, weights, w_stride,
                     static_cast<uint4*>(k_out), static_cast<uint4*>(v_out), w_out, kept, heads, t_fp, keep, t_sys, recent};
  const int64_t rows = (int64_t)batch * heads;
  const dim3 grid(evict::slices(rows, (int64_t)keep * 512), (unsigned)rows);
  return evict::run(evict::tokens_kernel, grid, smem, static_cast<cudaStream_t>(stream), p);
}
