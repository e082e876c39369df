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

// Lengths and new tokens of the launch's call rows, the latter 0 for a row that
// an earlier call row names.  Every row's sequence sets a bit of `names`, a second
// one if the first was set; only rows whose sequence has that one look through
// the rows before them.  (Bits stand for sequences mod 32,768.)  Rows that each
// looked through all before them took 1,024 named rows of 300 tokens 238 us; so 32,
// unnamed 28.  All threads of the block; `names` is free again behind a barrier.
constexpr int kNameWords = 1024;
constexpr int kNameBytes = 2 * kNameWords * 4;

AKV_DEV void weigh_lengths(const WeighParams& P, uint32_t* names, int* s_len, int* s_new) {
  const bool named = P.rows && P.row0 + P.R > 1;
  for (int e = threadIdx.x; e < P.R; e += blockDim.x) {
    const Int4Row r = int4_row(P.c, P.rows, P.n_new, P.row0 + e, P.M, P.status);
    s_len[e] = r.len;
    s_new[e] = r.n_new;
  }
  if (!named) return;
  const int words = min(kNameWords, (P.c.max_seqs + 31) / 32);
  for (int k = threadIdx.x; k < words; k += blockDim.x) names[k] = names[kNameWords + k] = 0u;
  __syncthreads();
  for (int s = threadIdx.x; s < P.row0 + P.R; s += blockDim.x) {
    const int seq = __ldg(P.rows + s);
    if (static_cast<unsigned>(seq) >= static_cast<unsigned>(P.c.max_seqs)) continue;
    const uint32_t bit = 1u << (seq & 31), word = seq / 32 % kNameWords;
    if (atomicOr(names + word, bit) & bit) atomicOr(names + kNameWords + word, bit);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < P.R; e += blockDim.x) {
    const int seq = __ldg(P.rows + P.row0 + e);
    if (static_cast<unsigned>(seq) >= static_cast<unsigned>(P.c.max_seqs)) continue;
    if (!(names[kNameWords + seq / 32 % kNameWords] >> (seq & 31) & 1u)) continue;
    bool again = false;
#pragma unroll 8
    for (int s = 0; s < P.row0 + e; ++s) again |= __ldg(P.rows + s) == seq;
    if (again) {
      set_status(P.status, AKV_ERR_SHAPE);
      s_new[e] = 0;
    }
  }
}

// Many queries, on the fifth-generation tensor cores (int4_weigh_many.cu).
size_t weigh_many_workspace(int R, int M, int Hq, int kv_heads, int head_dim, int n_groups);
int weigh_many(WeighParams P, int R, void* workspace, cudaStream_t st);

}  // namespace akv
