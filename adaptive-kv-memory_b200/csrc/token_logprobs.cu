// Log probabilities of given tokens, with entropy, rank and the top alternatives.
//
// Of a row x of logits, with M = max x, u = x - M, Z = sum e^u:
//   logprob = u[token] - ln Z     entropy = ln Z - sum(e^u u) / Z
//   rank    = 1 + the number of logits above the token's
// and the k largest logits, the lowest index first among equal ones.  One pass:
// a thread keeps the running maximum of what it has seen, Z and sum(e^u u)
// relative to it (in log2 units), and rescales both when the maximum moves.
// All sums are fp32.  In a batch where some u is -inf, u is clamped to -160 in
// log2 units, where e^u is 0 in fp32, so that it adds 0 and not 0 * -inf; a NaN
// stays one and shows in Z.
//
// Top alternatives: a warp holds the best 32 it has met, one a lane in
// descending order, as 64-bit keys (value's order << 32 | ~index): they decide
// ties, so the result depends on the inputs alone.  The lanes' maxima of the
// first batch, sorted, start the list; from then on a batch of up to 32 elements
// a lane is looked through only if its maximum reaches the k-th key, and of it the
// elements that do, a bit each, are inserted.  The lists of warps
// and CTAs are merged pairwise (maximum of one and the other reversed is the
// bitonic top half).
//
// Few rows are split over clusters of up to 8 CTAs.
//
// Bound by memory with fp32 logits (1,000 rows of 151,936: 102 us, 6.0 TB/s); with
// 16-bit ones, by the exponentials and some 6 instructions a logit between the
// loads: 4,093 rows 225 us, 5.5 TB/s, with the best alternative 276 us (the first
// batch's sort, new candidates of every warp, fewer CTAs); 248 and 290 to 303 in
// steady repetition.  One row of 151,936
// takes 5 us, with five alternatives 9.4; 64 rows of 32,003 5 and 8.
#include <cooperative_groups.h>

#include "int4.cuh"

namespace akv {

namespace cg = cooperative_groups;

constexpr int kLogpThreads = 256;
constexpr int kLogpWarps = kLogpThreads / 32;
constexpr int kLogpVecs = 4;         // 16-byte pieces of a thread's batch
constexpr int kLogpStages = 3;       // batches of the ring
constexpr int kLogpMaxTop = 32;
constexpr int kLogpMaxCluster = 8;
constexpr float kLog2E = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct LogpParams {
  const void* logits;
  int64_t row_stride;
  const int64_t* tokens;
  float* logprob;
  float* entropy;
  int32_t* rank;
  int64_t* top_tokens;
  float* top_logprobs;
  int vocab, top;
};

// max that gives NaN for NaN
AKV_DEV float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int DT>
struct LogitElem {  // two 16-bit logits a word
  using type = uint16_t;
  static constexpr int N = 8;  // logits of a 16-byte vector
  static constexpr uint32_t kNone = DT == AKV_BF16 ? 0xFF80FF80u : 0xFC00FC00u;  // -inf
  AKV_DEV static float get(uint16_t u) { return elem_to_float<DT == AKV_BF16>(u); }
  AKV_DEV static void unpack(uint32_t w, float (&x)[2]) {
    if constexpr (DT == AKV_BF16) {
      x[0] = __uint_as_float(w << 16);
      x[1] = __uint_as_float(w & 0xFFFF0000u);
    } else {
      const float2 f = __half22float2(u32_as_h2(w));
      x[0] = f.x, x[1] = f.y;
    }
  }
  AKV_DEV static uint32_t max_word(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (DT == AKV_BF16)
      asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  AKV_DEV static uint32_t min_word(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (DT == AKV_BF16)
      asm("min.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("min.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  AKV_DEV static float max_of(uint32_t w) {
    float x[2];
    unpack(w, x);
    return fmaxf(x[0], x[1]);
  }
  AKV_DEV static float min_of(uint32_t w) {
    float x[2];
    unpack(w, x);
    return fminf(x[0], x[1]);
  }
  // ones for the logits of a batch above x, which is a logit itself; counts up to 256 are exact
  AKV_DEV static int count_above(const uint32_t* w, int n, float x) {
    float c[2];
    if constexpr (DT == AKV_BF16) {
      const __nv_bfloat162 x2 = __float2bfloat162_rn(x);
      __nv_bfloat162 sum = __float2bfloat162_rn(0.f);
#pragma unroll
      for (int i = 0; i < n; ++i) sum = __hadd2(sum, __hgt2(*reinterpret_cast<const __nv_bfloat162*>(w + i), x2));
      const float2 f = __bfloat1622float2(sum);
      c[0] = f.x, c[1] = f.y;
    } else {
      const __half2 x2 = __float2half2_rn(x);
      __half2 sum = __float2half2_rn(0.f);
#pragma unroll
      for (int i = 0; i < n; ++i) sum = __hadd2(sum, __hgt2(u32_as_h2(w[i]), x2));
      const float2 f = __half22float2(sum);
      c[0] = f.x, c[1] = f.y;
    }
    return static_cast<int>(c[0] + c[1]);
  }
};
template <>
struct LogitElem<AKV_FP32> {
  using type = float;
  static constexpr int N = 4;
  static constexpr uint32_t kNone = 0xFF800000u;
  AKV_DEV static float get(float u) { return u; }
  AKV_DEV static uint32_t max_word(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  AKV_DEV static uint32_t min_word(uint32_t a, uint32_t b) {
    return __float_as_uint(fminf(__uint_as_float(a), __uint_as_float(b)));
  }
  AKV_DEV static float max_of(uint32_t w) { return __uint_as_float(w); }
  AKV_DEV static float min_of(uint32_t w) { return __uint_as_float(w); }
  AKV_DEV static int count_above(const uint32_t* w, int n, float x) {
    int c = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) c += __uint_as_float(w[i]) > x;
    return c;
  }
};

// 32-bit order of a logit (-0 as +0); never called for NaN
AKV_DEV uint32_t logit_order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
AKV_DEV float order_logit(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o); }

AKV_DEV uint64_t logit_key(float x, int index) {
  return static_cast<uint64_t>(logit_order(x)) << 32 | static_cast<uint32_t>(~index);
}

// What a part of a row comes to: maximum, and relative to it the sums of e^u and
// e^u u (u in log2 units).
struct LogpSums {
  float m, s, t;
};
AKV_DEV LogpSums join(LogpSums a, LogpSums b) {
  LogpSums r;
  r.m = max_nan(a.m, b.m);
  // a part without anything has s = t = 0; far below the other, it only has to vanish
  const float da = a.m == -INFINITY ? 0.f : fmaxf((a.m - r.m) * kLog2E, -1e4f);
  const float db = b.m == -INFINITY ? 0.f : fmaxf((b.m - r.m) * kLog2E, -1e4f);
  const float fa = exp2f(da), fb = exp2f(db);
  r.s = fa * a.s + fb * b.s;
  r.t = fa * fmaf(da, a.s, a.t) + fb * fmaf(db, b.s, b.t);
  return r;
}

// descending order over the lanes of any keys
AKV_DEV uint64_t bitonic_sort(uint64_t k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o; o >>= 1) {
      const uint64_t y = __shfl_xor_sync(~0u, k, o);
      const bool small = ((lane & o) != 0) != (size < 32 && (lane & size) != 0);
      k = small ? (k < y ? k : y) : (k > y ? k : y);
    }
  return k;
}

// descending order over the lanes of a bitonic sequence of keys
AKV_DEV uint64_t bitonic_merge(uint64_t k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t y = __shfl_xor_sync(~0u, k, o);
    k = (lane & o) ? (k < y ? k : y) : (k > y ? k : y);
  }
  return k;
}

// CTAs an SM.  With 16-bit logits and lists four leave too few registers (305 us
// for 4,093 x 151,936, three 276); with fp32 logits four fit (1,000 rows 102 us,
// three 110).
template <int DT, bool TOP>
constexpr int kLogpPerSm = TOP && DT != AKV_FP32 ? 3 : 4;

template <int DT, bool TOP>
__global__ void __launch_bounds__(kLogpThreads, kLogpPerSm<DT, TOP>) token_logprobs_kernel(const LogpParams P) {
  using E = LogitElem<DT>;
  using T = typename E::type;
  constexpr int W = kLogpVecs * 4;                 // words of a batch
  constexpr int PER = E::N / 4;                    // logits of a word
  __shared__ LogpSums s_sums[kLogpWarps];
  __shared__ int s_above[kLogpWarps];
  __shared__ uint64_t s_keys[TOP ? kLogpWarps : 1][32];

  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), rank = cluster.block_rank();
  const int row = blockIdx.x / C;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const T* x0 = static_cast<const T*>(P.logits) + row * P.row_stride;
  const int64_t token = P.tokens ? __ldg(P.tokens + row) : -1;
  const bool have = static_cast<uint64_t>(token) < static_cast<uint64_t>(P.vocab);
  const float mine = have ? E::get(__ldg(x0 + token)) : NAN;

  // 16-byte vectors from the first boundary on; what stands before and after them is taken one by one
  const int head = min(P.vocab, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) % 16 / sizeof(T)));
  const int n_vec = (P.vocab - head) / E::N;
  const int tail0 = head + n_vec * E::N;
  const int v0 = static_cast<int>(static_cast<int64_t>(n_vec) * rank / C);
  const int v1 = static_cast<int>(static_cast<int64_t>(n_vec) * (rank + 1) / C);
  const uint4* xv = reinterpret_cast<const uint4*>(x0 + head);

  LogpSums a{-INFINITY, 0.f, 0.f};
  float base = 0.f;  // the maximum, or 0 while there is none: -inf - base stays -inf
  int above = 0;
  uint64_t best = 0, least = 0;  // this lane's key; the k-th key of the warp

  auto raise = [&](float m) {
    if (a.m != -INFINITY) {
      const float d = fmaxf((a.m - m) * kLog2E, -1e4f), f = exp2f(d);
      a.t = f * fmaf(d, a.s, a.t);
      a.s *= f;
    }
    a.m = m;
    base = m;
  };
  auto add = [&](float x) {
    const float u = max_nan((x - base) * kLog2E, -160.f);
    const float e = fast_exp2(u);
    a.s += e;
    a.t = fmaf(e, u, a.t);
  };
  // one candidate of each lane (key 0: none) into the warp's list
  auto offer = [&](uint64_t key) {
    for (uint32_t who = __ballot_sync(~0u, key > least); who; who &= who - 1) {
      const uint64_t k = __shfl_sync(~0u, key, __ffs(who) - 1);
      if (k <= least) continue;
      const uint64_t up = __shfl_up_sync(~0u, best, 1);
      if (best < k) best = lane == 0 || up > k ? k : up;
      least = __shfl_sync(~0u, best, P.top - 1);
    }
  };

  // a thread copies what it reads itself, two batches ahead: nobody waits for anybody
  extern __shared__ uint4 ring[];  // [stage][piece][thread]
  int ahead = v0, into = 0;
  auto fetch = [&] {
#pragma unroll
    for (int j = 0; j < kLogpVecs; ++j) {
      const int at = ahead + j * kLogpThreads + t;
      if (at < v1) cp_async16(ring + (into * kLogpVecs + j) * kLogpThreads + t, xv + at);
    }
    cp_async_commit();
    ahead += kLogpVecs * kLogpThreads;
    into = into + 1 == kLogpStages ? 0 : into + 1;
  };
  for (int k = 1; k < kLogpStages; ++k) fetch();
  int stage = 0;
  for (int v = v0; v < v1; v += kLogpVecs * kLogpThreads) {
    fetch();
    cp_async_wait<kLogpStages - 1>();
    const uint4* mine4 = ring + stage * kLogpVecs * kLogpThreads + t;
    stage = stage + 1 == kLogpStages ? 0 : stage + 1;
    uint32_t w[W];
#pragma unroll
    for (int j = 0; j < kLogpVecs; ++j) {
      const int at = v + j * kLogpThreads + t;
      const uint4 q = at < v1 ? mine4[j * kLogpThreads] : make_uint4(E::kNone, E::kNone, E::kNone, E::kNone);
      w[4 * j] = q.x, w[4 * j + 1] = q.y, w[4 * j + 2] = q.z, w[4 * j + 3] = q.w;
    }
    uint32_t top = w[0], low = w[0];
#pragma unroll
    for (int i = 1; i < W; ++i) {
      top = E::max_word(top, w[i]);
      low = E::min_word(low, w[i]);
    }
    const float m = E::max_of(top);
    if (!(m <= a.m)) raise(m);
    if (__any_sync(~0u, (E::min_of(low) - base) * kLog2E == -INFINITY)) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        if constexpr (PER == 2) {
          float x[2];
          E::unpack(w[i], x);
          add(x[0]);
          add(x[1]);
        } else {
          add(__uint_as_float(w[i]));
        }
      }
    } else {
      const uint64_t back = f2_make(-base, -base), unit = f2_make(kLog2E, kLog2E);
      uint64_t s2 = 0, t2 = 0;
#pragma unroll
      for (int i = 0; i < W; i += 2 / PER) {
        float x[2];
        if constexpr (PER == 2) {
          E::unpack(w[i], x);
        } else {
          x[0] = __uint_as_float(w[i]), x[1] = __uint_as_float(w[i + 1]);
        }
        const uint64_t u2 = f2_mul(f2_add(f2_make(x[0], x[1]), back), unit);
        const float2 u = f2_split(u2);
        const uint64_t e2 = f2_make(fast_exp2(u.x), fast_exp2(u.y));
        s2 = f2_add(s2, e2);
        t2 = f2_fma(e2, u2, t2);
      }
      const float2 s = f2_split(s2), t2s = f2_split(t2);
      a.s += s.x + s.y;
      a.t += t2s.x + t2s.y;
    }
    if (m > mine) above += E::count_above(w, W, mine);
    if constexpr (TOP) {
      // the elements that reach `bar`, a bit each: word i's from PER * i on
      auto reach = [&](float bar) -> uint32_t {
        uint32_t bits = 0u;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          if (v + (i / 4) * kLogpThreads + t >= v1) continue;
          if constexpr (PER == 2) {
            float x[2];
            E::unpack(w[i], x);
            if (x[0] >= bar) bits |= 1u << (2 * i);
            if (x[1] >= bar) bits |= 2u << (2 * i);
          } else {
            if (__uint_as_float(w[i]) >= bar) bits |= 1u << i;
          }
        }
        return bits;
      };
      auto key_of = [&](int bit) -> uint64_t {
        const int i = bit / PER;
        const int c = head + (v + (i / 4) * kLogpThreads + t) * E::N + (i % 4) * PER + bit % PER;
        const T x = reinterpret_cast<const T*>(mine4 + (i / 4) * kLogpThreads)[(i % 4) * PER + bit % PER];
        return logit_key(E::get(x), c);
      };
      uint32_t done = 0u;
      if (v == v0) {
        const uint32_t bits = reach(m);
        done = bits & -bits;
        best = bitonic_sort(bits ? key_of(__ffs(bits) - 1) : 0);
        least = __shfl_sync(~0u, best, P.top - 1);
      }
      const bool look = m == m && logit_order(m) >= static_cast<uint32_t>(least >> 32);
      if (__any_sync(~0u, look)) {
        uint32_t bits = look ? reach(least ? order_logit(static_cast<uint32_t>(least >> 32)) : -INFINITY) & ~done : 0u;
        while (__any_sync(~0u, bits != 0u)) {
          offer(bits ? key_of(__ffs(bits) - 1) : 0);
          bits &= bits - 1;
        }
      }
    }
  }
  // the row's ends: fewer than 16 logits, by the first warp of the last CTA
  if (rank == C - 1 && warp == 0) {
    const int c = lane < head ? lane : tail0 + lane - head;
    const bool on = c < P.vocab;
    const float x = on ? E::get(x0[c]) : -INFINITY;
    if (!(x <= a.m)) raise(x);
    add(x);
    above += x > mine;
    if constexpr (TOP) offer(on && x == x ? logit_key(x, c) : 0);
  }

  // warps, then CTAs
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const LogpSums b{__shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o), __shfl_xor_sync(~0u, a.t, o)};
    // both lanes join in the same order
    a = (lane & o) ? join(b, a) : join(a, b);
  }
  above = __reduce_add_sync(~0u, above);
  if (lane == 0) {
    s_sums[warp] = a;
    s_above[warp] = above;
  }
  // the lists of the first n warps become the first one's
  auto merge_lists = [&](int n) {
    s_keys[warp][lane] = best;
    for (int o = 1; o < n; o *= 2) {
      __syncthreads();
      if (warp % (2 * o) == 0) {
        const uint64_t other = s_keys[warp + o][31 - lane];
        best = bitonic_merge(best > other ? best : other);
        s_keys[warp][lane] = best;
      }
    }
  };
  if constexpr (TOP) merge_lists(kLogpWarps);
  __syncthreads();
  if (t == 0) {
    for (int i = 1; i < kLogpWarps; ++i) {
      a = join(a, s_sums[i]);
      above += s_above[i];
    }
    s_sums[0] = a;
    s_above[0] = above;
  }
  cluster.sync();
  if constexpr (TOP) {
    if (rank == 0 && C > 1) {
      // warp i brings in CTA i's list: one at a time would be as many trips through the cluster
      if (warp > 0) best = warp < C ? cluster.map_shared_rank(&s_keys[0][0], warp)[lane] : 0;
      merge_lists(C);
    }
  }
  if (rank == 0 && warp == 0) {
    a = LogpSums{-INFINITY, 0.f, 0.f};
    above = 0;
    if (lane < C) {
      a = *cluster.map_shared_rank(&s_sums[0], lane);
      above = *cluster.map_shared_rank(&s_above[0], lane);
    }
#pragma unroll
    for (int o = 1; o < kLogpMaxCluster; o *= 2) {
      const LogpSums b{__shfl_xor_sync(~0u, a.m, o), __shfl_xor_sync(~0u, a.s, o), __shfl_xor_sync(~0u, a.t, o)};
      a = (lane & o) ? join(b, a) : join(a, b);
    }
    a = LogpSums{__shfl_sync(~0u, a.m, 0), __shfl_sync(~0u, a.s, 0), __shfl_sync(~0u, a.t, 0)};
    above = __reduce_add_sync(~0u, above);
    // no distribution: NaN or +inf among the logits, or all of them -inf
    const bool bad = !(fabsf(a.m) < INFINITY) || a.s != a.s;
    const float logz = logf(a.s);
    if (lane == 0) {
      P.logprob[row] = bad || !have ? NAN : (mine - a.m) - logz;
      P.entropy[row] = bad ? NAN : logz - a.t / a.s * kLn2;
      P.rank[row] = bad || !have ? 0 : above + 1;
    }
    if constexpr (TOP) {
      if (lane < P.top) {
        const float x = order_logit(static_cast<uint32_t>(best >> 32));
        P.top_tokens[static_cast<int64_t>(row) * P.top + lane] = bad ? -1 : static_cast<int>(~static_cast<uint32_t>(best));
        P.top_logprobs[static_cast<int64_t>(row) * P.top + lane] = bad ? NAN : (x - a.m) - logz;
      }
    }
  }
  cluster.sync();  // the first CTA has read the others' shared memory
}

template <int DT, bool TOP>
static int launch_logprobs(const LogpParams& p, int n, int cluster, cudaStream_t st) {
  constexpr int smem = kLogpStages * kLogpVecs * kLogpThreads * 16;
  // with the static arrays on top it is past the 48 KB that need no asking
  if (!ensure_dynamic_smem<token_logprobs_kernel<DT, TOP>>(smem + 1024)) return AKV_ERR_LAUNCH;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(n) * cluster);
  cfg.blockDim = dim3(kLogpThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<DT, TOP>, p) == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}

}  // namespace akv

using namespace akv;

extern "C" int akv_token_logprobs(const akv_logprobs_args* a, void* stream) {
  if (!a) return AKV_ERR_NULL;
  if (a->n < 0 || a->vocab <= 0 || a->top < 0 || a->top > kLogpMaxTop || a->top > a->vocab) return AKV_ERR_SHAPE;
  if (a->n > (1 << 28) || a->vocab > INT32_MAX - 64) return AKV_ERR_SHAPE;
  if (a->dtype != AKV_FP32 && a->dtype != AKV_FP16 && a->dtype != AKV_BF16) return AKV_ERR_UNSUPPORTED;
  if (a->n == 0) return AKV_OK;
  if (!a->logits || !a->tokens || !a->logprob || !a->entropy || !a->rank ||
      (a->top && (!a->top_tokens || !a->top_logprobs)))
    return AKV_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(a->logits) & (a->dtype == AKV_FP32 ? 3 : 1)) return AKV_ERR_ALIGN;
  LogpParams p{};
  p.logits = a->logits;
  p.row_stride = a->row_stride;
  p.tokens = a->tokens;
  p.logprob = a->logprob;
  p.entropy = a->entropy;
  p.rank = a->rank;
  p.top_tokens = a->top_tokens;
  p.top_logprobs = a->top_logprobs;
  p.vocab = a->vocab;
  p.top = a->top;
  // as many CTAs a row as fill the GPU, each with a batch's worth of logits at least
  const int batch = kLogpThreads * kLogpVecs * (a->dtype == AKV_FP32 ? 4 : 8);
  int cluster = 1;
  while (cluster < kLogpMaxCluster && a->n * cluster * 2 <= 148 * 4 && a->vocab > batch * cluster) cluster *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->dtype * 2 + (a->top > 0)) {
    case AKV_FP32 * 2: return launch_logprobs<AKV_FP32, false>(p, a->n, cluster, st);
    case AKV_FP32 * 2 + 1: return launch_logprobs<AKV_FP32, true>(p, a->n, cluster, st);
    case AKV_FP16 * 2: return launch_logprobs<AKV_FP16, false>(p, a->n, cluster, st);
    case AKV_FP16 * 2 + 1: return launch_logprobs<AKV_FP16, true>(p, a->n, cluster, st);
    case AKV_BF16 * 2: return launch_logprobs<AKV_BF16, false>(p, a->n, cluster, st);
    default: return launch_logprobs<AKV_BF16, true>(p, a->n, cluster, st);
  }
}
