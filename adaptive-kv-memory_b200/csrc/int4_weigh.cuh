// Shared pieces of the kernels that weigh the cached tokens (int4_weigh.cu says what they compute).
#pragma once

#include "int4.cuh"

namespace akv {

constexpr int kWeighRows = 1024;   // call rows of one launch

struct WeighParams {
  akv_int4_cache c;
  const int32_t* rows;
  const int32_t* n_new;
  int row0, R;  // call rows [row0, row0 + R) of this launch
  int M, Hq;
  const uint16_t* q;
  int64_t q_sr, q_sh, q_sm;
  const float* lse;
  float scale;
  float* weights;
  int64_t w_stride;
  int bf16;
  // many queries: prepared query tiles, the CTAs' meta records and part sums
  uint8_t* tiles;
  int4* meta;
  float* part;
  int* status;
};

// the new tokens of call row row0 + e; 0 for a row that an earlier call row names
AKV_DEV int weigh_new(const WeighParams& P, int e, const Int4Row& r) {
  if (P.rows)
    for (int s = 0; s < P.row0 + e; ++s)
      if (P.rows[s] == r.seq) {
        set_status(P.status, AKV_ERR_SHAPE);
        return 0;
      }
  return r.n_new;
}

// Many queries, on the fifth-generation tensor cores (int4_weigh_many.cu).
size_t weigh_many_workspace(int R, int M, int Hq, int kv_heads, int head_dim, int n_groups);
int weigh_many(WeighParams P, int R, void* workspace, cudaStream_t st);

}  // namespace akv
