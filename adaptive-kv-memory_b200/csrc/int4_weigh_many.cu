// Attention weight of the cached tokens from many queries (a prompt's chunk),
// on the fifth-generation tensor cores.  What is computed stands in
// int4_weigh.cu; here tokens are the MMA's 128 rows and queries its columns, so
// that a token's scale, zero and running sum are registers of one thread, and
// nothing is reduced across threads.
//
// A first kernel lays the queries out as MMA operands: tiles of N columns, one
// (new token, query head of the group) each, tokens outer, fp16 scaled by one
// power of two a tile (bf16: its largest element into [2^13, 2^14), exact unless
// 2^-38 of that; fp16 as it is), and for each column the group sums of q and
// -lse, both in units of the exponent.  The main kernel copies a tile at a time
// into a ring.  With S_g = q_g . (c_g - 8) from the tensor cores,
//   w += 2^(sum_g s'_g S_g + (z_g + 8 s_g) qs_g - lse),  s' = s * unit:
// two fp32 steps a group and column, an exponential, an addition.  A tile whose
// queries' largest elements lie further apart than 2^kManySpread scales each
// column by itself (its largest element to the same place), sums without lse and
// unit, and takes one step a column more: 2^(unit_column * sum - lse).  The case
// below with queries of such sizes takes 255, 294 and 426 us (one, two, four
// groups); units by column for every tile would take 211, 254 and 404.
//
// A unit is one (call row, 256 tokens): a warpgroup for each 128, whose codes
// stand in shared (D = 256: tensor) memory as the MMA's A, head after head.  The
// units' (head, query tile) pairs form one list that is cut into equal shares,
// one per CTA, from the lengths on the device; parts of a cut unit are joined in
// order by a third kernel.  While one warpgroup's exponentials run, the other's
// MMAs do.
//
// Bound by the chain of a tile (scores out of tensor memory, sums, exponentials,
// two barriers) with two warps a scheduler: 1,000 tokens of 32 / 8 heads of 128
// over 16K, 5e8 exponentials that alone would take 110 us, take 193 us with one
// group, 235 with two, 353 with four.  Sums of a column pair read as 16 bytes
// instead of 8 gave the same (362): the registers they pair up spill.
#include <type_traits>

#include "int4_weigh.cuh"
#include "umma.cuh"

namespace akv {

constexpr int kManySMs = 148;
constexpr int kManyTokens = 256;      // of a unit
constexpr int kManyThreads = 256 + 64;
constexpr float kManyLog2e = 1.4426950408889634f;
constexpr int kManySpread = 14;       // the smallest query of a tile keeps 2^-24 of its largest element

// Query columns of a tile: an MMA of up to 64 columns takes as long as one of 64
// (45 cycles; 32 columns are worth 16), so as many as the scores of all groups
// find room for in the tensor memory, the codes moved to shared memory for it:
// 1,000 tokens of 32 / 8 heads over 16K, groups of 32, 416 -> 357 us, of 64, 262
// -> 229.  With D = 256 the codes in shared memory would leave no ring.
constexpr int many_columns(int D, int G) { return D == 256 ? 128 / G : (G < 4 ? 128 : 64); }

template <int D, int G>
struct ManyShape {
  static constexpr bool SS = D <= 128;           // codes in shared memory
  static constexpr int N = many_columns(D, G);
  static constexpr int QB = N * D * 2;           // its operand
  static constexpr int META = N * (G + 1) * 4;   // per column pair: -lse, group sums
  static constexpr int OWN = QB + META + 16;     // the tile's unit; whether its columns have their own
  static constexpr int REC = OWN + N * 8;        // those, and -lse: per column pair
  static constexpr int STAGES = REC > 48 * 1024 ? 3 : 4;
  static constexpr int KG = D / G / 16;          // MMA steps of a group
  static constexpr int AB = SS ? 128 * D * 2 : 0;  // codes of a warpgroup
  static constexpr int OFF_A = STAGES * REC;
  static constexpr int OFF_BAR = OFF_A + 2 * AB;
  static constexpr int OFF_ROWS = OFF_BAR + 128;
  static constexpr int smem(int rows) { return OFF_ROWS + (2 * rows + 2) * 4 + (rows + 1) * 8; }
  // tensor memory of a warpgroup: codes, then scores
  static constexpr int T_A = 0, T_S = SS ? 0 : D / 2, T_WG = T_S + G * N;
  static_assert(2 * T_WG <= 512, "tensor memory");
  static_assert(OFF_BAR >= kNameBytes && REC % 16 == 0 && smem(kWeighRows) <= 227 * 1024, "shared memory");
};

// tiles of a call row's query columns
AKV_DEV int many_tiles(int n_new, int rep, int N) { return (n_new * rep + N - 1) / N; }

// ------------------------------------------------------------------ queries
template <int D, int G>
__global__ void __launch_bounds__(128) weigh_prepare_kernel(const WeighParams P) {
  using S = ManyShape<D, G>;
  constexpr int N = S::N;
  __shared__ uint32_t s_top[128 / N], s_low[128 / N];
  const int t = threadIdx.x, n = t % N, sub = t / N;
  const int H = P.c.kv_heads, rep = P.Hq / H, h = blockIdx.y, e = blockIdx.z, i = P.row0 + e;
  const int all = (P.M * rep + N - 1) / N;           // tiles that a row has room for
  const int qt = blockIdx.x * (128 / N) + sub;
  const Int4Row row = int4_row(P.c, P.rows, P.n_new, i, P.M, nullptr);
  const int rr = qt * N + n, m = rr / rep, hq = h * rep + rr - m * rep;
  const bool on = m < row.n_new;
  const uint16_t* src = P.q + i * P.q_sr + hq * P.q_sh + m * P.q_sm;
  const bool q16 = ((reinterpret_cast<uintptr_t>(P.q) & 15) | ((P.q_sr | P.q_sh | P.q_sm) & 7)) == 0;
  auto piece = [&](int c) -> uint4 {  // channels 8c .. 8c + 7
    if (!on) return make_uint4(0u, 0u, 0u, 0u);
    if (q16) return *reinterpret_cast<const uint4*>(src + 8 * c);
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = src[8 * c + 2 * k] | static_cast<uint32_t>(src[8 * c + 2 * k + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  if (t < 128 / N) s_top[t] = 0u, s_low[t] = 0x7FFFu;
  __syncthreads();
  uint32_t top = 0u;  // largest magnitude, as the 15 bits of the type
#pragma unroll 8
  for (int c = 0; c < D / 8; ++c) {
    const uint4 v = piece(c);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) top = max(top, max(w[k] & 0x7FFFu, w[k] >> 16 & 0x7FFFu));
  }
  const float lse = on ? __ldg(P.lse + (static_cast<int64_t>(i) * P.Hq + hq) * P.M + m) : -INFINITY;
  const bool counts = on && top < (P.bf16 ? 0x7F80u : 0x7C00u) && fabsf(lse) < INFINITY;
  if (P.bf16 && counts && top) {
    atomicMax(&s_top[sub], top);
    atomicMin(&s_low[sub], top);
  }
  __syncthreads();
  const bool own = static_cast<int>(s_top[sub] >> 7) - static_cast<int>(s_low[sub] >> 7) > kManySpread;
  const uint32_t most = own ? (counts ? top : 0u) : s_top[sub];
  int ex = 0;
  if (P.bf16 && most) ex = 13 - (static_cast<int>(most >> 7) - 127);
  ex = ex > 120 ? 120 : (ex < -120 ? -120 : ex);
  const float up = exp2f(static_cast<float>(ex));
  const float unit = ldexpf(P.scale * kManyLog2e, -ex);
  if (qt >= many_tiles(row.n_new, rep, N)) return;
  uint8_t* rec = P.tiles + ((static_cast<int64_t>(e) * H + h) * all + qt) * S::REC;
  float sum[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    sum[g] = 0.f;
#pragma unroll 8
    for (int c = g * (D / 8 / G); c < (g + 1) * (D / 8 / G); ++c) {
      const uint4 v = piece(c);
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
      if (P.bf16) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = pack_h2(__uint_as_float(w[k] << 16) * up, __uint_as_float(w[k] & 0xFFFF0000u) * up);
      }
      if (!counts) w[0] = w[1] = w[2] = w[3] = 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 f = __half22float2(u32_as_h2(w[k]));
        sum[g] += f.x + f.y;
      }
      // the order in which codes come out of a word
      *reinterpret_cast<uint4*>(rec + c * (N * 16) + n * 16) =
          make_uint4(prmt(w[0], w[2], 0x5410), prmt(w[0], w[2], 0x7632), prmt(w[1], w[3], 0x5410),
                     prmt(w[1], w[3], 0x7632));
    }
  }
  const float less = counts ? -lse * kManyLog2e : -INFINITY;
  float* meta = reinterpret_cast<float*>(rec + S::QB) + (n / 2) * 2 * (G + 1) + (n & 1);
  meta[0] = own ? 0.f : less;
#pragma unroll
  for (int g = 0; g < G; ++g) meta[2 + 2 * g] = own ? sum[g] : sum[g] * unit;
  float* mine = reinterpret_cast<float*>(rec + S::OWN) + (n / 2) * 4 + (n & 1);
  mine[0] = less;
  mine[2] = unit;
  if (n == 0) *reinterpret_cast<float2*>(rec + S::QB + S::META) = make_float2(own ? 1.f : unit, own ? 1.f : 0.f);
}

// ------------------------------------------------------------------ the list
// Part of a unit's list: query tiles [q0, q1) of one head.
struct ManyPart {
  int r, i, seq, len, n_new, tile, h, q0, q1;
  bool first, last;  // the unit's part in this CTA begins, ends here
  bool start, end;   // so does the unit
  int last_cta;
};

template <int N>
struct ManyWalk {
  const WeighParams* P;
  const int *len, *n_new;
  const int64_t* pref;
  int H, rep, r;
  int64_t share, begin, stop, pos;

  AKV_DEV static int first_tile(int base, int rep, int tile) {  // of a unit's query tiles: those before see none of it
    const int t0 = tile * kManyTokens;
    return t0 > base ? static_cast<int>(static_cast<int64_t>(t0 - base) * rep / N) : 0;
  }
  AKV_DEV static int64_t weight(int len, int n_new, int rep) {  // (unit, query tile) pairs of a row
    if (n_new <= 0 || len <= 0) return 0;
    const int qt = many_tiles(n_new, rep, N), units = (len + kManyTokens - 1) / kManyTokens, base = len - n_new;
    const int whole = base < 0 ? 0 : min(units, base / kManyTokens + 1);
    int64_t w = static_cast<int64_t>(whole) * qt;
    for (int u = whole; u < units; ++u) w += max(0, qt - first_tile(base, rep, u));
    return w;
  }
  AKV_DEV void init(const WeighParams* p, const int* l, const int* n, const int64_t* pr) {
    P = p, len = l, n_new = n, pref = pr;
    H = p->c.kv_heads;
    rep = p->Hq / H;
    const int64_t total = pref[p->R] * H;
    share = (total + gridDim.x - 1) / gridDim.x;
    if (share < 1) share = 1;
    begin = min(share * blockIdx.x, total);
    stop = min(begin + share, total);
    pos = begin;
    int lo = 0, hi = p->R;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (pref[mid] * H <= pos) lo = mid; else hi = mid;
    }
    r = lo;
  }
  AKV_DEV bool next(ManyPart& x) {
    if (pos >= stop) return false;
    while (pref[r + 1] * H <= pos) ++r;
    const int64_t at = pos - pref[r] * H;
    const int l = len[r], nn = n_new[r], base = l - nn, qt = many_tiles(nn, rep, N);
    const int whole = base < 0 ? 0 : min((l + kManyTokens - 1) / kManyTokens, base / kManyTokens + 1);
    int64_t off = at;  // within the unit
    int u, nq = qt;
    if (at < static_cast<int64_t>(whole) * qt * H) {
      u = static_cast<int>(at / (static_cast<int64_t>(qt) * H));
      off -= static_cast<int64_t>(u) * qt * H;
    } else {
      off -= static_cast<int64_t>(whole) * qt * H;
      for (u = whole;; ++u) {
        nq = max(0, qt - first_tile(base, rep, u));
        if (off < static_cast<int64_t>(nq) * H) break;
        off -= static_cast<int64_t>(nq) * H;
      }
    }
    const int64_t unit = pos - off, unit_end = unit + static_cast<int64_t>(nq) * H;
    x.r = r;
    x.i = P->row0 + r;
    x.seq = P->rows ? __ldg(P->rows + x.i) : x.i;
    x.len = l;
    x.n_new = nn;
    x.tile = u;
    x.h = static_cast<int>(off / nq);
    const int k = static_cast<int>(off % nq);
    const int n = static_cast<int>(min(static_cast<int64_t>(nq - k), stop - pos));
    x.q0 = qt - nq + k;
    x.q1 = x.q0 + n;
    x.first = pos == begin || off == 0;
    x.start = unit >= begin;
    pos += n;
    x.last = pos == stop || pos == unit_end;
    x.end = unit_end <= stop;
    x.last_cta = static_cast<int>((unit_end - 1) / share);
    return true;
  }
};

// the codes of a word as fp16 pairs c - 8 of channels (0, 4) (1, 5) (2, 6) (3, 7)
AKV_DEV void centred_codes(uint32_t w, uint32_t* c) {
  const uint32_t v = w >> 8;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(c[0]) : "r"(lop_magic<0x00F000F0u>(w)), "r"(0x2C002C00u), "r"(0xD480D480u));
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(c[1]) : "r"(lop_magic<0x000F000Fu>(w)), "r"(0xE408E408u));
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(c[2]) : "r"(lop_magic<0x00F000F0u>(v)), "r"(0x2C002C00u), "r"(0xD480D480u));
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(c[3]) : "r"(lop_magic<0x000F000Fu>(v)), "r"(0xE408E408u));
}

// ------------------------------------------------------------------ the kernel
template <int D, int G>
__global__ void __launch_bounds__(kManyThreads, 1) weigh_many_kernel(const WeighParams P) {
  using S = ManyShape<D, G>;
  constexpr int N = S::N;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  uint64_t *q_full = bars, *q_free = bars + 4, *a_ready = bars + 8, *s_full = bars + 10, *s_free = bars + 12;
  uint64_t* drained = bars + 14;
  int64_t* s_pref = reinterpret_cast<int64_t*>(smem + S::OFF_ROWS);
  int* s_len = reinterpret_cast<int*>(s_pref + P.R + 1);
  int* s_new = s_len + P.R;
  __shared__ uint32_t s_tmem;

  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int H = P.c.kv_heads, rep = P.Hq / H, all = (P.M * rep + N - 1) / N;
  if (t == 0) {
    for (int k = 0; k < S::STAGES; ++k) {
      mbar_init(q_full + k, 1);
      mbar_init(q_free + k, 1 + 8);
    }
    for (int k = 0; k < 2; ++k) {
      mbar_init(a_ready + k, 128);
      mbar_init(s_full + k, 1);
      mbar_init(s_free + k, 128);
    }
    mbar_init(drained, 1);
    fence_mbar_init();
    P.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  weigh_lengths(P, reinterpret_cast<uint32_t*>(smem), s_len, s_new);
  fence_proxy_async_shared();  // bulk copies follow where the rows' names stood
  for (int e = t; e < P.R; e += kManyThreads) s_pref[e + 1] = ManyWalk<N>::weight(s_len[e], s_new[e], rep);
  __syncthreads();
  if (warp == 0) {  // prefix sums
    int64_t base = 0;
    for (int e0 = 0; e0 < P.R; e0 += 32) {
      int64_t x = e0 + lane < P.R ? s_pref[e0 + lane + 1] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
      }
      if (e0 + lane < P.R) s_pref[e0 + lane + 1] = base + x;
      base += __shfl_sync(~0u, x, 31);
    }
    if (lane == 0) s_pref[0] = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  ManyWalk<N> walk;
  walk.init(&P, s_len, s_new, s_pref);
  ManyPart u{};
  bool ok = true;  // no bounded wait of this warp has run out

  if (warp < 8) {
    // ================================================================ weights
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      if (ok) ok = mbar_wait_warp(bar, phase, P.status);
      return ok;
    };
    constexpr Int4Layout L = int4_layout(D, G);
    constexpr int NW = D / 8;  // code words of a token
    const int wg = warp >> 2;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tA = tmem + lanes + wg * S::T_WG + S::T_A, tS = tmem + lanes + wg * S::T_WG + S::T_S;
    uint32_t kw[NW], kp[G];
    unsigned char* sA = smem + S::OFF_A + wg * S::AB + (t & 127) * 16;
    bool have = false;  // the thread's token is there, on a page
    auto fetch = [&](const ManyPart& x) {
      const int tok = x.tile * kManyTokens + t;
      const uint8_t* rec = nullptr;
      if (tok < x.len) {
        const int p = __ldg(P.c.table + x.seq * P.c.table_stride + tok / kBlockTokens);
        if (p >= 0 && p < P.c.n_pages) rec = P.c.pool + p * P.c.page_stride + x.h * P.c.head_stride;
        else set_status(P.status, AKV_ERR_SHAPE);
      }
      have = rec != nullptr;
      const int slot = tok % kBlockTokens;
#pragma unroll
      for (int k = 0; k < NW / 4; ++k) {
        const uint4 v = rec ? ldg_nc_v4(rec + L.kc + slot * (D / 2) + 16 * k) : make_uint4(0, 0, 0, 0);
        kw[4 * k] = v.x, kw[4 * k + 1] = v.y, kw[4 * k + 2] = v.z, kw[4 * k + 3] = v.w;
      }
#pragma unroll
      for (int k = 0; k < G; ++k) kp[k] = rec ? __ldg(reinterpret_cast<const uint32_t*>(rec + L.kp) + slot * G + k) : 0u;
    };
    uint32_t ph_s = 0, ph_q = 0;
    int st = 0;
    float total = 0.f;
    bool more = walk.next(u);
    if (more) fetch(u);
    while (more && ok) {
      // ---- this head's codes as the MMA's A: every S of the last part is out
      if constexpr (S::SS) {
#pragma unroll
        for (int k = 0; k < NW; ++k) {
          uint32_t c[4];
          centred_codes(kw[k], c);
          *reinterpret_cast<uint4*>(sA + k * (128 * 16)) = make_uint4(c[0], c[1], c[2], c[3]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < NW / 8; ++k) {
          uint32_t c[32];
#pragma unroll
          for (int j = 0; j < 8; ++j) centred_codes(kw[8 * k + j], c + 4 * j);
          tmem_st32u(tA + 32 * k, c);
        }
      }
      float s[G], mid[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float2 sz = __half22float2(u32_as_h2(kp[g]));
        s[g] = sz.x;
        mid[g] = fmaf(8.f, sz.x, sz.y);
      }
      const bool mine = have;
      if constexpr (S::SS) fence_proxy_async_shared();
      else tmem_wait_st();
      tc_fence_before();
      mbar_arrive(a_ready + wg);
      ManyPart nx;
      more = walk.next(nx);
      if (more) fetch(nx);

      const int tok = u.tile * kManyTokens + t;
      // Columns of the part's first tile that do not see the token, N fewer of each next one.  An
      // old token's difference passes 32 bits with many heads; the columns themselves are 2^30 at most.
      const int64_t see = static_cast<int64_t>(tok - (u.len - u.n_new)) * rep - static_cast<int64_t>(u.q0) * N;
      int hide = static_cast<int>(max(int64_t{0}, min(int64_t{1} << 30, see)));
      if (u.first) total = 0.f;
      for (int q = u.q0; q < u.q1; ++q, hide -= N) {
        if (!wait(q_full + st, ph_q)) break;
        const unsigned char* rec = smem + st * S::REC;
        const float2 tile = *reinterpret_cast<const float2*>(rec + S::QB + S::META);
        const float unit = tile.x;
        uint64_t s2[G], m2[G];
#pragma unroll
        for (int g = 0; g < G; ++g) {
          s2[g] = f2_make(s[g] * unit, s[g] * unit);
          m2[g] = f2_make(mid[g], mid[g]);
        }
        if (!wait(s_full + wg, ph_s)) break;
        ph_s ^= 1;
        tc_fence_after();
        const bool full = __all_sync(~0u, hide <= 0);
        uint64_t sum = 0;
        // with or without the columns' own units: a form for each, so that the usual one keeps its registers
        auto add = [&](auto own) {
#pragma unroll
          for (int c = 0; c < N / 32; ++c) {
            uint64_t y[16];
            const uint64_t* meta = reinterpret_cast<const uint64_t*>(rec + S::QB) + c * 16 * (G + 1);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if constexpr (G == 1) {
                const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(meta + 2 * k);
                y[k] = f2_fma(m2[0], v.y, v.x);
              } else {
                y[k] = meta[k * (G + 1)];
#pragma unroll
                for (int g = 0; g < G; ++g) y[k] = f2_fma(m2[g], meta[k * (G + 1) + 1 + g], y[k]);
              }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
              float x[32];
              tmem_ld32(tS + g * N + c * 32, x);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) y[k] = f2_fma(f2_make(x[2 * k], x[2 * k + 1]), s2[g], y[k]);
            }
            if constexpr (decltype(own)::value) {
              const ulonglong2* mine = reinterpret_cast<const ulonglong2*>(rec + S::OWN) + c * 16;
#pragma unroll
              for (int k = 0; k < 16; ++k) y[k] = f2_fma(y[k], mine[k].y, mine[k].x);
            }
            if (c == N / 32 - 1) {  // S is out
              tc_fence_before();
              mbar_arrive(s_free + wg);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float2 v = f2_split(y[k]);
              v.x = fast_exp2(v.x);
              v.y = fast_exp2(v.y);
              if (!full) {
                if (c * 32 + 2 * k < hide) v.x = 0.f;
                if (c * 32 + 2 * k + 1 < hide) v.y = 0.f;
              }
              sum = f2_add(sum, f2_make(v.x, v.y));
            }
          }
        };
        if (__any_sync(~0u, tile.y != 0.f)) add(std::true_type{});
        else add(std::false_type{});
        const float2 two = f2_split(sum);
        total += two.x + two.y;
        __syncwarp();
        if (lane == 0) mbar_arrive(q_free + st);
        if (++st == S::STAGES) st = 0, ph_q ^= 1;
      }
      if (!ok) break;
      if (u.last) {
        const float w = mine ? total : 0.f;
        if (u.start && u.end) {
          if (mine) P.weights[u.seq * P.w_stride + tok] += w;
        } else {
          P.part[(2 * static_cast<int64_t>(blockIdx.x) + (u.start ? 1 : 0)) * kManyTokens + t] = w;
          if (t == 0 && u.start) P.meta[blockIdx.x] = make_int4(u.r, u.tile, u.last_cta, 1);
        }
      }
      u = nx;
    }
  } else if (warp == 8) {
    // ================================================================ query tiles
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 1;  // a fresh barrier passes a wait for the phase before its first
      while (ok && walk.next(u)) {
        const uint8_t* src = P.tiles + (static_cast<int64_t>(u.r) * H + u.h) * all * S::REC;
        for (int q = u.q0; q < u.q1; ++q) {
          ok = mbar_wait(q_free + st, ph, P.status);
          if (!ok) break;
          mbar_arrive_expect_tx(q_full + st, S::REC);
          tma_load_1d(smem + st * S::REC, src + static_cast<int64_t>(q) * S::REC, S::REC, q_full + st);
          if (++st == S::STAGES) st = 0, ph ^= 1;
        }
      }
      if (!ok)  // a wait ran out: see the copies in flight land
        for (int k = 0; k < S::STAGES; ++k) {
          const int x = (st + k) % S::STAGES;
          mbar_wait(q_full + x, x >= st ? ph : ph ^ 1, P.status);
        }
    }
  } else {
    // ================================================================ MMA
    const uint32_t lead = elect_one();
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      if (ok) ok = mbar_wait_warp(bar, phase, P.status);
      return ok;
    };
    constexpr uint32_t IDESC = instr_desc(128, N, 0);
    const uint32_t base = smem_u32(smem), codes = desc_lo(base + S::OFF_A, 128 * 16);
    int st = 0;
    uint32_t ph_q = 0, ph_a = 0, ph_s = 1;
    while (ok && walk.next(u)) {
      wait(a_ready, ph_a);
      wait(a_ready + 1, ph_a);
      ph_a ^= 1;
      for (int q = u.q0; q < u.q1; ++q) {
        if (!wait(q_full + st, ph_q)) break;
        const uint32_t tile = desc_lo(base + st * S::REC, N * 16);
        for (int wg = 0; wg < 2; ++wg) {
          if (!wait(s_free + wg, ph_s)) break;
          tc_fence_after();
          const uint32_t tA = tmem + wg * S::T_WG + S::T_A, tS = tmem + wg * S::T_WG + S::T_S;
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int k = 0; k < S::KG; ++k) {
              const int step = g * S::KG + k;
              if constexpr (S::SS)
                umma_ss<desc_hi(128), desc_hi(128), IDESC>(tS + g * N, codes + wg * (S::AB / 16) + step * 256,
                                                           tile + step * 2 * N, k > 0 ? 1u : 0u, lead);
              else umma_ts<desc_hi(128), IDESC>(tS + g * N, tA + 8 * step, tile + step * 2 * N, k > 0 ? 1u : 0u, lead);
            }
          umma_commit(s_full + wg, lead);
        }
        if (!ok) break;
        ph_s ^= 1;
        umma_commit(q_free + st, lead);
        if (++st == S::STAGES) st = 0, ph_q ^= 1;
      }
    }
    if (!ok) {  // see what was issued end before the tensor memory goes
      umma_commit(drained, lead);
      mbar_wait(drained, 0, P.status);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// The parts of the unit whose first one CTA blockIdx.x holds, in order.
__global__ void __launch_bounds__(kManyTokens) weigh_join_kernel(const WeighParams P) {
  const int4 meta = P.meta[blockIdx.x];
  if (!meta.w) return;
  const Int4Row row = int4_row(P.c, P.rows, P.n_new, P.row0 + meta.x, P.M, nullptr);
  const int t = threadIdx.x, tok = meta.y * kManyTokens + t, c = blockIdx.x;
  if (tok >= row.len) return;
  float sum = __ldcg(P.part + (2 * static_cast<int64_t>(c) + 1) * kManyTokens + t);
  for (int k = c + 1; k <= meta.z; ++k) sum += __ldcg(P.part + 2 * static_cast<int64_t>(k) * kManyTokens + t);
  P.weights[row.seq * P.w_stride + tok] += sum;
}

namespace {

int64_t many_row_bytes(int M, int Hq, int kv_heads, int D, int G) {
  const int64_t N = many_columns(D, G), tiles = (static_cast<int64_t>(M) * (Hq / kv_heads) + N - 1) / N;
  return tiles * kv_heads * (N * D * 2 + N * (G + 3) * 4 + 16);
}
constexpr int64_t kManyRoom = 128 << 20;  // of prepared tiles of a launch, at least one row's
constexpr size_t kManyFixed = kManySMs * sizeof(int4) + 2 * kManySMs * kManyTokens * sizeof(float);

int many_rows(int R, int64_t row_bytes) {
  int64_t rows = kManyRoom / row_bytes;
  rows = rows < 1 ? 1 : (rows > kWeighRows ? kWeighRows : rows);
  return static_cast<int>(rows < R ? rows : R);
}

template <int D, int G>
int launch_many(const WeighParams& P, cudaStream_t st) {
  using S = ManyShape<D, G>;
  const int smem = S::smem(P.R);
  if (!ensure_dynamic_smem<weigh_many_kernel<D, G>>(smem)) return AKV_ERR_LAUNCH;
  const int rep = P.Hq / P.c.kv_heads;
  const int64_t blocks = (static_cast<int64_t>(P.M) * rep + 127) / 128;
  weigh_prepare_kernel<D, G><<<dim3(static_cast<unsigned>(blocks), P.c.kv_heads, P.R), 128, 0, st>>>(P);
  weigh_many_kernel<D, G><<<kManySMs, kManyThreads, smem, st>>>(P);
  weigh_join_kernel<<<kManySMs, kManyTokens, 0, st>>>(P);
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}

template <int D>
int many_by_group(const WeighParams& P, cudaStream_t st) {
  switch (D / P.c.group) {
    case 1: return launch_many<D, 1>(P, st);
    case 2: return launch_many<D, 2>(P, st);
    default: return launch_many<D, 4>(P, st);
  }
}

}  // namespace

size_t weigh_many_workspace(int R, int M, int Hq, int kv_heads, int head_dim, int n_groups) {
  const int64_t row = many_row_bytes(M, Hq, kv_heads, head_dim, n_groups);
  return kManyFixed + static_cast<size_t>(many_rows(R, row) * row);
}

int weigh_many(WeighParams P, int R, void* workspace, cudaStream_t st) {
  if (P.c.kv_heads > 65535) return AKV_ERR_UNSUPPORTED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  P.meta = reinterpret_cast<int4*>(ws);
  P.part = reinterpret_cast<float*>(ws + kManySMs * sizeof(int4));
  P.tiles = ws + kManyFixed;
  const int rows = many_rows(R, many_row_bytes(P.M, P.Hq, P.c.kv_heads, P.c.head_dim, P.c.head_dim / P.c.group));
  for (int r = 0; r < R; r += rows) {
    P.row0 = r;
    P.R = R - r < rows ? R - r : rows;
    const int e = P.c.head_dim == 64 ? many_by_group<64>(P, st)
                  : P.c.head_dim == 128 ? many_by_group<128>(P, st) : many_by_group<256>(P, st);
    if (e) return e;
  }
  return AKV_OK;
}

}  // namespace akv
