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
//
// A probability's units are taken as hi * 2^23 + lo with hi = rint(p * 2^17)
// and lo = rint((p - hi * 2^-17) * 2^40), each by one addition that leaves the
// integer in a float's low bits (a conversion to 64-bit integers costs several
// times as much), two probabilities at a time.  The remainder is exact and
// hi * 2^23 even, so this is rint(p * 2^40), ties to even.  max(P - Q, 0) is
// units(max(p, q)) - units(q), because units() is monotone: no comparison of
// the two-part numbers.
//
// Measured (151,936 fp32 probabilities, draft and target, inputs from DRAM,
// launches of a graph): 64 sequences 23.1 us (3.4 TB/s of the 78 MB, 1.9 times
// the bytes' time: all CTAs go through accept, sums, exchange and draw in step,
// and only the sums stream), one sequence 7.8 us, all latency: accept 1.4, sums
// 1.5, two cluster exchanges 2.5, draw 1, launch.
#include <cooperative_groups.h>

#include <type_traits>

#include "int4.cuh"

namespace akv {

namespace cg = cooperative_groups;

constexpr int kVerifyCluster = 8;
// Threads of a CTA.  One sequence is a chain of latencies (accept, sums,
// exchange, draw) that more threads shorten; many sequences want several of
// their CTAs on an SM, so that one's loads cover another's chain.
constexpr int kVerifyFew = 512, kVerifyMany = 256;
constexpr int kVerifyManyFrom = 24;  // sequences

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

// Units of 2^-40 of two probabilities in [0, 1]: the bits of 2^23 + hi and of
// 1.5 * 2^23 + lo.
struct Units2 {
  int hi[2], lo[2];
};
constexpr int kHiBits = 0x4B000000, kLoBits = 0x4B400000;

AKV_DEV uint64_t f2_all(float x) { return f2_make(x, x); }

AKV_DEV Units2 prob_units(float p0, float p1) {
  const uint64_t p = f2_make(p0, p1);
  const uint64_t a = f2_fma(p, f2_all(131072.f), f2_all(8388608.f));
  // a - 2^23 is exact, so its product by 2^-17 is the rounded part of p
  const uint64_t part = f2_fma(a, f2_all(1.f / 131072.f), f2_all(-64.f));
  const uint64_t rest = f2_fma(part, f2_all(-1.f), p);
  const uint64_t b = f2_fma(rest, f2_all(1099511627776.f), f2_all(12582912.f));
  const float2 h = f2_split(a), l = f2_split(b);
  return Units2{{__float_as_int(h.x), __float_as_int(h.y)}, {__float_as_int(l.x), __float_as_int(l.y)}};
}

// NaN and less than 0 count as 0, more than 1 as 1
AKV_DEV float prob(float p) { return __saturatef(p); }

AKV_DEV uint64_t warp_sum_u64(uint64_t x) {
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
  return x;
}

// inclusive sum over the lanes
AKV_DEV uint64_t warp_scan_u64(uint64_t x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(~0u, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

template <int DT, bool DRAFT, int THREADS>
__global__ void __cluster_dims__(kVerifyCluster, 1, 1) __launch_bounds__(THREADS, THREADS == kVerifyMany ? 4 : 1)
    verify_kernel(VerifyParams P) {
  constexpr int WARPS = THREADS / 32;
  static_assert(WARPS <= 32, "a lane stands for a warp's sum");
  using E = ProbElem<DT>;
  using T = typename E::type;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ uint64_t s_w[WARPS];  // units in each warp's range
  __shared__ uint64_t s_sum, s_before, s_total;
  __shared__ int s_acc;
  const int b = blockIdx.y, part = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const T* target = static_cast<const T*>(P.target) + b * P.t_sb;
  const T* draft = DRAFT ? static_cast<const T*>(P.draft) + b * P.d_sb : nullptr;
  const int64_t* tok = P.tokens + static_cast<int64_t>(b) * P.K;
  int n = P.n_draft ? P.n_draft[b] : P.K;
  n = n < 0 ? 0 : (n > P.K ? P.K : n);

  const float u_last = fminf(fmaxf(P.sample_u[b], 0.f), 0.99999994f);
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
  // Weight of a token: units(max(p, q)) - units(q), which is max(P - Q, 0).
  // q is the draft's probability, without a draft distribution 1 on the hot
  // token; in the pass `over` the target itself (q = 0).
  auto weight = [&](int x, bool over) -> uint64_t {
    const float p = prob(E::get(prow[x]));
    float q = 0.f;
    if (!over) {
      if constexpr (DRAFT) q = qrow ? prob(E::get(qrow[x])) : 0.f;
      else q = x == hot ? 1.f : 0.f;
    }
    const Units2 u = prob_units(fmaxf(p, q), q);
    return (static_cast<int64_t>(u.hi[0] - u.hi[1]) << 23) + (u.lo[0] - u.lo[1]);
  };

  // this CTA's part, a contiguous range for each warp
  constexpr int VE = 16 / sizeof(T);  // elements of a 16-byte load
  int per_warp = (P.vocab + kVerifyCluster * WARPS - 1) / (kVerifyCluster * WARPS);
  per_warp = (per_warp + VE - 1) / VE * VE;
  const int first = min((part * WARPS + warp) * per_warp, P.vocab);
  const int end = min(first + per_warp, P.vocab);

  // sum of the weights of [first, end), without the hot token's correction
  auto range = [&](auto with_q) -> uint64_t {
    constexpr bool Q = decltype(with_q)::value;
    int64_t s_hi = 0, s_lo = 0;
    int hi = 0, lo = 0;  // of at most 64 elements, 2^23 each: flushed every round
    auto add2 = [&](float p0, float p1, float q0, float q1) {
      p0 = prob(p0), p1 = prob(p1);
      if constexpr (Q) {
        q0 = prob(q0), q1 = prob(q1);
        const Units2 p = prob_units(fmaxf(p0, q0), fmaxf(p1, q1)), q = prob_units(q0, q1);
        hi += p.hi[0] - q.hi[0];
        lo += p.lo[0] - q.lo[0];
        hi += p.hi[1] - q.hi[1];
        lo += p.lo[1] - q.lo[1];
      } else {
        const Units2 p = prob_units(p0, p1);
        hi += p.hi[0] - kHiBits;
        lo += p.lo[0] - kLoBits;
        hi += p.hi[1] - kHiBits;
        lo += p.lo[1] - kLoBits;
      }
    };
    auto flush = [&] {
      s_hi += hi;
      s_lo += lo;
      hi = lo = 0;
    };
    int x = first;
    if (((reinterpret_cast<uintptr_t>(prow) | (Q ? reinterpret_cast<uintptr_t>(qrow) : 0)) & 15) == 0) {
      constexpr int U = 4;
      for (; x + 32 * VE <= end; x += U * 32 * VE) {
        uint4 pv[U], qv[Q ? U : 1];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int at = x + (u * 32 + lane) * VE;
          pv[u] = make_uint4(0u, 0u, 0u, 0u);
          if constexpr (Q) qv[u] = pv[u];
          if (x + (u + 1) * 32 * VE <= end) {
            pv[u] = ldg_nc_v4(prow + at);
            if constexpr (Q) qv[u] = ldg_nc_v4(qrow + at);
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const T* pe = reinterpret_cast<const T*>(&pv[u]);
          const T* qe = reinterpret_cast<const T*>(&qv[Q ? u : 0]);
#pragma unroll
          for (int j = 0; j < VE; j += 2)
            add2(E::get(pe[j]), E::get(pe[j + 1]), Q ? E::get(qe[j]) : 0.f, Q ? E::get(qe[j + 1]) : 0.f);
        }
        flush();
      }
      x = first + (end - first) / (32 * VE) * (32 * VE);
    }
    constexpr int U = 8;
    for (; x < end; x += U * 32) {
      T pv[U], qv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = x + u * 32 + lane;
        pv[u] = T(0);
        qv[u] = T(0);
        if (at < end) {
          pv[u] = prow[at];
          if constexpr (Q) qv[u] = qrow[at];
        }
      }
#pragma unroll
      for (int u = 0; u < U; u += 2)
        add2(E::get(pv[u]), E::get(pv[u + 1]), Q ? E::get(qv[u]) : 0.f, Q ? E::get(qv[u + 1]) : 0.f);
      flush();
    }
    return static_cast<uint64_t>((s_hi << 23) + s_lo);
  };

  int64_t* out = P.out + static_cast<int64_t>(b) * (P.K + 1);
  // An empty difference (second pass) draws from the target itself.
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
    const bool over = pass == 1;
    uint64_t sum;
    if (DRAFT && qrow && !over) sum = range(std::integral_constant<bool, DRAFT>{});
    else sum = range(std::false_type{});
    if (!DRAFT && !over && hot >= first && hot < end && lane == 0) sum -= weight(static_cast<int>(hot), true);
    sum = warp_sum_u64(sum);
    if (lane == 0) s_w[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      const uint64_t a = warp_sum_u64(lane < WARPS ? s_w[lane] : 0);
      if (lane == 0) s_sum = a;
    }
    cluster.sync();
    if (warp == 0) {  // lane r: the cluster's CTA r
      const uint64_t v = lane < kVerifyCluster ? *cluster.map_shared_rank(&s_sum, lane) : 0;
      const uint64_t before = warp_sum_u64(lane < part ? v : 0), total = warp_sum_u64(v);
      if (lane == 0) {
        s_before = before;
        s_total = total;
      }
    }
    __syncthreads();
    cluster.barrier_arrive();  // no CTA reuses or leaves its sum while another reads it
    const uint64_t all = s_total;
    if (part == 0 && pass == 0) {
      for (int j = t; j <= P.K; j += THREADS)
        if (j != acc) out[j] = j < acc ? tok[j] : -1;
      if (t == 0) P.accepted[b] = acc;
    }
    if (part == 0 && t == 0 && over && !all) out[acc] = -1;
    const uint64_t u24 = static_cast<uint64_t>(u_last * 16777216.f);
    const uint64_t goal = (all >> 24) * u24 + (((all & 0xFFFFFFull) * u24) >> 24);
    uint64_t base = s_before;
    if (all && goal >= base && goal - base < s_sum) {  // the goal is in this CTA's part
      const uint64_t w_sum = lane < WARPS ? s_w[lane] : 0, w_inc = warp_scan_u64(w_sum);
      const int w = __ffs(__ballot_sync(~0u, base + w_inc > goal)) - 1;
      base += __shfl_sync(~0u, w_inc - w_sum, w);
      const int f0 = (part * WARPS + w) * per_warp, f1 = min(f0 + per_warp, P.vocab);
      for (int x0 = f0; x0 < f1 && base <= goal; x0 += THREADS) {
        const int x = x0 + t;
        const uint64_t mine = x < f1 ? weight(x, over) : 0;
        uint64_t inc = warp_scan_u64(mine);
        __syncthreads();  // the sums of warps are read above, and in the round before
        if (lane == 31) s_w[warp] = inc;
        __syncthreads();
        const uint64_t v = lane < WARPS ? s_w[lane] : 0, v_inc = warp_scan_u64(v);
        inc += base + __shfl_sync(~0u, v_inc - v, warp);
        if (mine && inc > goal && inc - mine <= goal) out[acc] = x;
        base += __shfl_sync(~0u, v_inc, 31);
      }
    }
    cluster.barrier_wait();
    if (all) break;
  }
}

}  // namespace akv

using namespace akv;

template <int DT, int THREADS>
static cudaError_t verify_launch(const VerifyParams& p, int B, cudaStream_t st) {
  const dim3 grid(kVerifyCluster, B);
  if (p.draft) verify_kernel<DT, true, THREADS><<<grid, THREADS, 0, st>>>(p);
  else verify_kernel<DT, false, THREADS><<<grid, THREADS, 0, st>>>(p);
  return cudaGetLastError();
}

// Measured (151,936 fp32 probabilities, draft and target, inputs from DRAM,
// launches of a graph; us with 512 / 256 threads): 1 sequence 7.8 / 10.5, 16
// 15.3 / 15.0, 24 17.2 / 15.6, 32 23.1 / 16.9, 64 39.7 / 23.1.
template <int DT>
static cudaError_t verify_launch(const VerifyParams& p, int B, cudaStream_t st) {
  return B >= kVerifyManyFrom ? verify_launch<DT, kVerifyMany>(p, B, st) : verify_launch<DT, kVerifyFew>(p, B, st);
}

extern "C" int akv_verify_draft(const akv_verify_args* a, void* stream) {
  if (!a) return AKV_ERR_NULL;
  if (a->B < 0 || a->K < 0 || a->vocab <= 0 || a->vocab > (1 << 23)) return AKV_ERR_SHAPE;  // 2^63 units
  if (a->dtype != AKV_FP32 && a->dtype != AKV_FP16 && a->dtype != AKV_BF16) return AKV_ERR_UNSUPPORTED;
  if (a->B > 65535) return AKV_ERR_UNSUPPORTED;
  if (a->B == 0) return AKV_OK;
  if (!a->target || !a->sample_u || !a->accepted || !a->out || (a->K && (!a->tokens || !a->accept_u)))
    return AKV_ERR_NULL;
  const uintptr_t mask = a->dtype == AKV_FP32 ? 3 : 1;
  if ((reinterpret_cast<uintptr_t>(a->target) | reinterpret_cast<uintptr_t>(a->draft)) & mask) return AKV_ERR_ALIGN;
  const VerifyParams p{a->target, a->t_sb,     a->t_sj,     a->draft,    a->d_sb, a->d_sj,     a->tokens,
                       a->n_draft, a->accept_u, a->sample_u, a->K,       a->vocab, a->accepted, a->out, a->status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->dtype == AKV_FP32) e = verify_launch<AKV_FP32>(p, a->B, st);
  else if (a->dtype == AKV_FP16) e = verify_launch<AKV_FP16>(p, a->B, st);
  else e = verify_launch<AKV_BF16>(p, a->B, st);
  return e == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}
