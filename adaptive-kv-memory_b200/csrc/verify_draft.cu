// Verification of drafted tokens (speculative decoding).
//
// Draft j of a sequence is accepted while u_j * q_j(x_j) < p_j(x_j); the next
// token comes from max(P - Q, 0) at the first rejected position (which leaves
// the target's distribution unchanged), or from P after the last draft.  The
// draw is the inverse CDF of one given uniform.  Probabilities count whole
// units of 2^-40, so every sum is an exact integer whatever the order of its
// additions, and the drawn token depends on the inputs alone.  (Float sums
// would move a boundary of the CDF by a unit in the last place of their total:
// over a 150K vocabulary that changes a token every hundred draws or so.)
//
// Bound by memory: one target and one draft row per sequence.  A cluster of
// CTAs takes a sequence, each a contiguous part of the vocabulary: sums first,
// exchanged through distributed shared memory, then the part that holds the
// goal finds its warp's range and reads that range (from L2) once more.
#include <cooperative_groups.h>

#include "int4.cuh"

namespace akv {

namespace cg = cooperative_groups;

constexpr int kVerifyCluster = 8;
constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;

struct VerifyParams {
  const void* target;
  int64_t t_sb, t_sj;
  const void* draft;
  int64_t d_sb, d_sj;
  const int64_t* tokens;
  const int32_t* n_draft;
  const float* accept_u;
  const float* sample_u;
  int K, vocab;
  int32_t* accepted;
  int64_t* out;
  int* status;
};

template <int DT>
struct ProbElem {
  using type = uint16_t;
  AKV_DEV static float get(uint16_t u) { return elem_to_float<DT == AKV_BF16>(u); }
};
template <>
struct ProbElem<AKV_FP32> {
  using type = float;
  AKV_DEV static float get(float u) { return u; }
};

// whole units of 2^-40; fmaxf turns NaN into 0
AKV_DEV int64_t prob_units(float p) { return __float2ll_rn(fminf(fmaxf(p, 0.f), 1.f) * 1099511627776.f); }

AKV_DEV uint64_t warp_sum_u64(uint64_t x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}

template <int DT, bool DRAFT>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(VerifyParams P) {
  using E = ProbElem<DT>;
  using T = typename E::type;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ uint64_t s_w[kVerifyWarps], s_p[kVerifyWarps];  // per warp: units of the difference, of the target
  __shared__ uint64_t s_sum[2];
  __shared__ int s_acc;
  const int b = blockIdx.y, part = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const T* target = static_cast<const T*>(P.target) + b * P.t_sb;
  const T* draft = DRAFT ? static_cast<const T*>(P.draft) + b * P.d_sb : nullptr;
  const int64_t* tok = P.tokens + static_cast<int64_t>(b) * P.K;
  int n = P.n_draft ? P.n_draft[b] : P.K;
  n = n < 0 ? 0 : (n > P.K ? P.K : n);

  // the first rejected draft; every CTA of the cluster finds it for itself
  if (warp == 0) {
    int acc = n;
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + lane;
      bool ok = true;
      if (j < n) {
        const int64_t x = tok[j];
        if (x < 0 || x >= P.vocab) {
          set_status(P.status, AKV_ERR_SHAPE);
          ok = false;
        } else {
          const double p = E::get(target[j * P.t_sj + x]);
          double q = 1.0;
          if constexpr (DRAFT) q = E::get(draft[j * P.d_sj + x]);
          ok = static_cast<double>(P.accept_u[static_cast<int64_t>(b) * P.K + j]) * q < p;
        }
      }
      const unsigned no = __ballot_sync(~0u, !ok);
      if (no) {
        acc = j0 + __ffs(no) - 1;
        break;
      }
    }
    if (lane == 0) s_acc = acc;
  }
  __syncthreads();
  const int acc = s_acc;
  const T* prow = target + acc * P.t_sj;
  const bool residual = acc < n;
  const T* qrow = DRAFT && residual ? draft + acc * P.d_sj : nullptr;
  // without a draft distribution all of q is on the drafted token
  const int64_t hot = !DRAFT && residual ? tok[acc] : -1;
  auto weight = [&](int x, uint64_t& full) -> uint64_t {
    const int64_t p = prob_units(E::get(prow[x]));
    full = p;
    if constexpr (DRAFT) {
      if (qrow) {
        const int64_t d = p - prob_units(E::get(qrow[x]));
        return d > 0 ? d : 0;
      }
    } else if (x == hot) {
      return 0;
    }
    return p;
  };

  // this CTA's part, a contiguous range for each warp
  const int per_warp = (P.vocab + kVerifyCluster * kVerifyWarps - 1) / (kVerifyCluster * kVerifyWarps);
  const int first = (part * kVerifyWarps + warp) * per_warp;
  const int end = min(first + per_warp, P.vocab);
  uint64_t sum_w = 0, sum_p = 0;
  for (int x = first + lane; x < end; x += 32) {
    uint64_t f;
    sum_w += weight(x, f);
    sum_p += f;
  }
  sum_w = warp_sum_u64(sum_w);
  sum_p = warp_sum_u64(sum_p);
  if (lane == 0) {
    s_w[warp] = sum_w;
    s_p[warp] = sum_p;
  }
  __syncthreads();
  if (t < 2) {
    const uint64_t* s = t ? s_p : s_w;
    uint64_t a = 0;
    for (int w = 0; w < kVerifyWarps; ++w) a += s[w];
    s_sum[t] = a;
  }
  cluster.sync();
  uint64_t before[2] = {0, 0}, total[2] = {0, 0};
#pragma unroll
  for (int r = 0; r < kVerifyCluster; ++r) {
    const uint64_t* o = cluster.map_shared_rank(s_sum, r);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (r < part) before[k] += o[k];
      total[k] += o[k];
    }
  }
  cluster.sync();  // no CTA leaves while another reads its sums
  const int pick = total[0] ? 0 : 1;  // an empty difference draws from the target itself
  const uint64_t all = pick ? total[1] : total[0];
  int64_t* out = P.out + static_cast<int64_t>(b) * (P.K + 1);
  if (part == 0) {
    for (int j = t; j <= P.K; j += kVerifyThreads)
      if (j != acc) out[j] = j < acc ? tok[j] : -1;
    if (t == 0) {
      P.accepted[b] = acc;
      if (!all) out[acc] = -1;
    }
  }
  if (!all) return;
  const float u = fminf(fmaxf(P.sample_u[b], 0.f), 0.99999994f);
  const uint64_t u24 = static_cast<uint64_t>(u * 16777216.f);
  const uint64_t goal = (all >> 24) * u24 + (((all & 0xFFFFFFull) * u24) >> 24);
  uint64_t base = pick ? before[1] : before[0];
  if (goal < base || goal - base >= s_sum[pick]) return;  // another CTA's part
  // the warp range that holds the goal
  const uint64_t* s = pick ? s_p : s_w;
  int w = 0;
  while (goal - base >= s[w]) base += s[w++];
  const int f0 = (part * kVerifyWarps + w) * per_warp, f1 = min(f0 + per_warp, P.vocab);
  __syncthreads();  // s_w / s_p are reused below
  for (int x0 = f0; x0 < f1; x0 += kVerifyThreads) {
    const int x = x0 + t;
    uint64_t mine = 0, f = 0;
    if (x < f1) {
      mine = weight(x, f);
      if (pick) mine = f;
    }
    uint64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(~0u, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) s_w[warp] = inc;
    __syncthreads();
    uint64_t pre = base, sum = 0;
    for (int k = 0; k < kVerifyWarps; ++k) {
      if (k < warp) pre += s_w[k];
      sum += s_w[k];
    }
    inc += pre;
    if (mine && inc > goal && inc - mine <= goal) out[acc] = x;
    base += sum;
    if (base > goal) return;
    __syncthreads();
  }
}

}  // namespace akv

using namespace akv;

template <int DT>
static cudaError_t verify_launch(const VerifyParams& p, int B, bool draft, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(kVerifyCluster, B);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = kVerifyCluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return draft ? cudaLaunchKernelEx(&cfg, verify_kernel<DT, true>, p) : cudaLaunchKernelEx(&cfg, verify_kernel<DT, false>, p);
}

extern "C" int akv_verify_draft(const void* target, int64_t t_sb, int64_t t_sj, const void* draft, int64_t d_sb,
                                int64_t d_sj, const int64_t* tokens, const int32_t* n_draft, const float* accept_u,
                                const float* sample_u, int B, int K, int vocab, int dtype, int32_t* accepted,
                                int64_t* out, int* status, void* stream) {
  if (B < 0 || K < 0 || vocab <= 0 || vocab > (1 << 23)) return AKV_ERR_SHAPE;  // 2^23 units of 2^40 stay below 2^63
  if (dtype != AKV_FP32 && dtype != AKV_FP16 && dtype != AKV_BF16) return AKV_ERR_UNSUPPORTED;
  if (B > 65535) return AKV_ERR_UNSUPPORTED;
  if (B == 0) return AKV_OK;
  if (!target || !sample_u || !accepted || !out || (K && (!tokens || !accept_u))) return AKV_ERR_NULL;
  const uintptr_t mask = dtype == AKV_FP32 ? 3 : 1;
  if ((reinterpret_cast<uintptr_t>(target) | reinterpret_cast<uintptr_t>(draft)) & mask) return AKV_ERR_ALIGN;
  VerifyParams p{target, t_sb, t_sj, draft, d_sb, d_sj, tokens, n_draft, accept_u, sample_u, K, vocab, accepted, out,
                 status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  const bool d = draft != nullptr;
  if (dtype == AKV_FP32) e = verify_launch<AKV_FP32>(p, B, d, st);
  else if (dtype == AKV_FP16) e = verify_launch<AKV_FP16>(p, B, d, st);
  else e = verify_launch<AKV_BF16>(p, B, d, st);
  return e == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}
