// How much attention each key got: the simplest form.  A warp per eight keys, a lane holds four channels; scores are summed over the
// lanes.  All arithmetic in fp32.
#include <math.h>

#include "cq_chunk.cuh"

namespace cq {
namespace chunk {

constexpr int WARPS = 8;

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  using T2 = typename Elem<T>::T2;
  const float2 a = Elem<T>::to_f2(*reinterpret_cast<const T2*>(&w.x)), b = Elem<T>::to_f2(*reinterpret_cast<const T2*>(&w.y));
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}

// Keys key0 .. key0+7 in cache order [visual | fp], this lane's channels 4*lane .. +3; keys past the end are zeros.
template <typename T>
__device__ __forceinline__ void load_keys(const Params& p, int b, int hk, int key0, int n_keys, int lane, float (&k)[8][4]) {
  if (key0 < p.t_vis) {
    const int64_t row = ((int64_t)b * p.hkv + hk) * 128 + lane * 4;
    for (int c = 0; c < 4; ++c) {
      const uint32_t w = p.k_code[(row + c) * (p.t_vis / 8) + key0 / 8];
      const float s = Elem<T>::to_f(static_cast<const T*>(p.k_scale)[(row + c) * (p.t_vis / 32) + key0 / 32]);
      const float m = Elem<T>::to_f(static_cast<const T*>(p.k_mn)[(row + c) * (p.t_vis / 32) + key0 / 32]);
      for (int j = 0; j < 8; ++j) k[j][c] = fmaf((float)((w >> (4 * j)) & 15u), s, m);
    }
  } else {
    for (int j = 0; j < 8; ++j) {
      if (key0 + j < n_keys)
        load4(static_cast<const T*>(p.k_fp) + b * p.fp_sb + hk * p.fp_sh + (int64_t)(key0 + j - p.t_vis) * 128 + lane * 4, k[j]);
      else
        for (int c = 0; c < 4; ++c) k[j][c] = 0.f;
    }
  }
}

// logits of a row against eight keys; -inf where a key takes no part
template <typename T>
__device__ __forceinline__ void logits(const Params& p, int b, int key0, int limit, const float (&q)[4], const float (&k)[8][4], float (&s)[8]) {
  for (int j = 0; j < 8; ++j) {
    float x = q[0] * k[j][0] + q[1] * k[j][1] + q[2] * k[j][2] + q[3] * k[j][3];
    x = warp_sum(x) * 0.08838834764831845f;
    const int key = key0 + j;
    if (key >= limit) {
      x = -INFINITY;
    } else if (p.mask) {
      const float m = Elem<T>::to_f(static_cast<const T*>(p.mask)[b * p.mask_sb + mask_index(p, key)]);
      x = m == -INFINITY ? -INFINITY : x + m;
    }
    s[j] = x;
  }
}

template <typename T>
__global__ void __launch_bounds__(WARPS * 32) key_weights_kernel(Params p, const float* vis_in, const float* fp_in, float* vis, float* fp,
                                                                 int64_t capacity) {
  const int lane = threadIdx.x & 31, key0 = (blockIdx.x * WARPS + (threadIdx.x >> 5)) * 8, hk = blockIdx.y, b = blockIdx.z;
  const int live = live_tokens(p), n_keys = p.t_vis + live;
  if (key0 >= p.t_vis + capacity) return;
  float w[8] = {};
  if (key0 < n_keys) {
    float k[8][4];
    load_keys<T>(p, b, hk, key0, n_keys, lane, k);
    for (int row = 0; row < p.rows; ++row) {
      const int i = row / p.n_rep, h = hk * p.n_rep + row % p.n_rep;
      const float lse = p.lse[((int64_t)b * p.hq + h) * p.q_len + i];
      if (lse == -INFINITY) continue;
      float q[4], s[8];
      load4(static_cast<const T*>(p.q) + b * p.q_sb + i * p.q_st + h * p.q_sh + lane * 4, q);
      logits<T>(p, b, key0, p.t_vis + max(0, live - p.q_len + i + 1), q, k, s);
      for (int j = 0; j < 8; ++j)
        if (s[j] != -INFINITY) w[j] += expf(s[j] - lse);
    }
  }
  if (lane == 0) {
    const int64_t bh = (int64_t)b * p.hkv + hk;
    for (int j = 0; j < 8; ++j) {
      const int key = key0 + j;
      if (key < p.t_vis)
        vis[bh * p.t_vis + key] = (vis_in ? vis_in[bh * p.t_vis + key] : 0.f) + w[j];
      else if (key < p.t_vis + capacity)
        fp[bh * capacity + key - p.t_vis] = (fp_in ? fp_in[bh * capacity + key - p.t_vis] : 0.f) + w[j];
    }
  }
}

}  // namespace chunk
}  // namespace cq

using namespace cq;

extern "C" size_t cq_key_weights_workspace_bytes(const cq_chunk_args* a) {
  return chunk::valid(a) && a->lse && chunk::supported(a) ? 256 : 0;
}

extern "C" int cq_key_weights(const cq_chunk_args* a, const float* w_vis_in, const float* w_fp_in, float* w_vis, float* w_fp,
                              int64_t w_capacity, void* workspace, size_t workspace_bytes, void* stream) {
  if (!chunk::valid(a) || !a->lse || (a->t_vis && !w_vis) || !w_fp || w_capacity < a->t_fp) return CQ_ERR_BAD_ARG;
  if (!chunk::supported(a) || a->t_vis + w_capacity >= (1ll << 30)) return CQ_ERR_UNSUPPORTED;
  if (!workspace || workspace_bytes < cq_key_weights_workspace_bytes(a)) return CQ_ERR_WORKSPACE;
  if (a->batch == 0) return CQ_OK;
  const chunk::Params p = chunk::make_params(a);
  const dim3 grid((unsigned)((p.t_vis + w_capacity + chunk::WARPS * 8 - 1) / (chunk::WARPS * 8)), p.hkv, a->batch);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a->dtype == CQ_DTYPE_BF16)
    chunk::key_weights_kernel<__nv_bfloat16><<<grid, chunk::WARPS * 32, 0, st>>>(p, w_vis_in, w_fp_in, w_vis, w_fp, w_capacity);
  else
    chunk::key_weights_kernel<__half><<<grid, chunk::WARPS * 32, 0, st>>>(p, w_vis_in, w_fp_in, w_vis, w_fp, w_capacity);
  return check_launch();
}
