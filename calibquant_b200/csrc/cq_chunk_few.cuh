// Few rows (cq_chunk_few.cu): what the entry points of the chunk attention and of the key weights call.
#pragma once

#include "cq_chunk.cuh"

namespace cq {
namespace chunk {

constexpr int FEW_ROWS = 16, FEW_CLUSTER = 8;

struct FewParams {
  Params p;
  int parts;                                   // CTAs per KV head
  float* part_o;                               // attention, parts > 1: [batch][KV head][row][part][128] and maximum, sum
  float2* part_ml;
  const float *vis_in, *fp_in;                 // weights
  float *vis, *fp;
  int64_t capacity;
  int* status;
  int cluster;                                 // attention: the parts of a KV head merge as a cluster, part_o and part_ml are not used
};

int few_parts(int64_t heads, int64_t t_vis, int64_t fp_keys, bool one, bool merged);
int few_run(const FewParams& p, int batch, bool bf16, bool weights, cudaStream_t st);

}  // namespace chunk
}  // namespace cq
