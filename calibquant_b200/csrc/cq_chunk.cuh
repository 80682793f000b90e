// What the chunk attention and the key weights share: arguments as the kernels take them.
#pragma once

#include "cq_common.cuh"

namespace cq {
namespace chunk {

struct Params {
  int hq, hkv, n_rep, q_len, t_vis, t_fp, t_sys;
  int rows;                                     // query rows of a KV head, row = query * n_rep + head
  const void* q;
  int64_t q_sb, q_st, q_sh;
  const uint32_t* k_code;
  const void *k_scale, *k_mn;
  const uint32_t* v_code;
  const void *v_scale, *v_mn;
  const void *k_fp, *v_fp;
  int64_t fp_sb, fp_sh;
  const void* mask;
  int64_t mask_sb;
  void* out;
  int64_t o_sb, o_st, o_sh;
  float* lse;
  const int32_t* t_fp_dev;
};

// Live full-precision tokens; the new tokens are the last q_len of them.
__device__ __forceinline__ int live_tokens(const Params& p) {
  if (!p.t_fp_dev) return p.t_fp;
  const int n = *p.t_fp_dev;
  return max(0, min(n, p.t_fp));
}

inline bool valid(const cq_chunk_args* a) {
  if (!a || a->batch < 0 || a->n_q_heads <= 0 || a->n_kv_heads <= 0 || a->n_q_heads % a->n_kv_heads || a->q_len <= 0 || a->t_vis < 0 ||
      a->t_fp < a->q_len || a->t_sys < 0 || a->t_sys > a->t_fp || a->reserved != 0 || (a->dtype != CQ_DTYPE_F16 && a->dtype != CQ_DTYPE_BF16))
    return false;
  if (!a->q || !a->k_fp || !aligned16(a->q) || !aligned16(a->k_fp) || a->fp_stride_b % 8 || a->fp_stride_h % 8) return false;
  for (int i = 0; i < 3; ++i)
    if (a->q_strides[i] % 8 || a->q_strides[i] < 0) return false;
  if ((a->q_strides[0] == 0 && a->batch > 1) || (a->q_strides[1] == 0 && a->q_len > 1) || (a->q_strides[2] == 0 && a->n_q_heads > 1)) return false;
  if (a->mask && reinterpret_cast<uintptr_t>(a->mask) % 2) return false;
  if (reinterpret_cast<uintptr_t>(a->lse) % 4 || reinterpret_cast<uintptr_t>(a->t_fp_dev) % 4) return false;
  if (a->t_vis && (!a->k_code || !a->k_scale || !a->k_mn || !aligned16(a->k_code) || !aligned16(a->k_scale) || !aligned16(a->k_mn))) return false;
  return true;
}
inline bool supported(const cq_chunk_args* a) {
  return a->head_dim == kHeadDim && a->group_size == kGroup && a->bits == 4 && a->t_vis % kGroup == 0 &&
         a->batch <= 65535 && a->n_kv_heads <= 65535 && a->n_q_heads / a->n_kv_heads <= 128 &&
         (int64_t)a->q_len * (a->n_q_heads / a->n_kv_heads) < (1ll << 30) && (int64_t)a->t_vis + a->t_fp < (1ll << 30);
}

inline Params make_params(const cq_chunk_args* a) {
  Params p = {};
  p.hq = a->n_q_heads; p.hkv = a->n_kv_heads; p.n_rep = a->n_q_heads / a->n_kv_heads; p.q_len = a->q_len;
  p.t_vis = a->t_vis; p.t_fp = a->t_fp; p.t_sys = a->t_sys; p.rows = p.n_rep * a->q_len;
  p.q = a->q; p.q_sb = a->q_strides[0]; p.q_st = a->q_strides[1]; p.q_sh = a->q_strides[2];
  p.k_code = reinterpret_cast<const uint32_t*>(a->k_code); p.k_scale = a->k_scale; p.k_mn = a->k_mn;
  p.v_code = reinterpret_cast<const uint32_t*>(a->v_code); p.v_scale = a->v_scale; p.v_mn = a->v_mn;
  p.k_fp = a->k_fp; p.v_fp = a->v_fp; p.fp_sb = a->fp_stride_b; p.fp_sh = a->fp_stride_h;
  p.mask = a->mask; p.mask_sb = a->mask_stride_b;
  p.out = a->out; p.o_sb = a->out_strides[0]; p.o_st = a->out_strides[1]; p.o_sh = a->out_strides[2];
  p.lse = a->lse; p.t_fp_dev = a->t_fp_dev;
  return p;
}

// Place in the mask (key order [sys | visual | text]) of key `key` in cache order [visual | fp].
__device__ __forceinline__ int mask_index(const Params& p, int key) {
  const int t = key - p.t_vis;
  return t < 0 ? p.t_sys + key : (t < p.t_sys ? t : p.t_vis + t);
}

}  // namespace chunk
}  // namespace cq
