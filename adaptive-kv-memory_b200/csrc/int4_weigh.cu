// Attention weight that the tokens of the 4-bit paged cache receive.
//
//   weights[s][t] += sum over query heads h and new tokens m that see t of
//                    exp(q_hm . K_t * scale - lse_hm)
// with the log-sum-exp that attention returned, so each query's weights sum to
// 1 and nothing has to be normalised in a second pass.  Only the K half of the
// records is read.  With K_t = c s_tg + z_tg in channel group g,
//   q.K_t = sum_g s_tg (q_g . c_tg) + z_tg sum(q_g)
// the contraction runs on codes, and its accumulators, scales and sums are fp32:
// the only rounding before the exponential is fp32's.  A code's four bits, masked
// where they lie in a 16-bit word, are an fp16 subnormal, c 2^-24 in bits 0..3 and
// 16 c 2^-24 in bits 4..7, which the MMA multiplies exactly: one AND makes two
// operands.  The 16 is taken out of those channels' queries, the 2^24 goes into s.
// (Queries enter fp16 scaled per row by a power of two, exact unless 2^-24 of
// the row's largest.)
//
// A token's sum is formed by one thread set in a fixed order (heads, then
// queries), so a call repeated gives the same bits.
//
// Few queries: the pages of all rows form one list that is cut into equal
// shares, one per CTA that fits the SMs at once, from the lengths on the device.  A warp takes
// every fourth page of its share and streams the page's heads through its own
// ring of asynchronous copies (of threads: a bulk copy's barrier and issue cost a
// record of 2 KB more than its arithmetic); tokens are the MMA's rows, queries its columns.  The
// queries of up to kWeighUnits (head, 8 or 16 columns) units stand in shared
// memory as MMA fragments; more of them take the pages again.
//
// Bound by latency and issue: 16 x 32,768 tokens of 8 KV heads of 128, 285 MB of
// K codes, take 82 us, 44 at the memory's rate; a warp's record of 2 KB takes
// some 1,500 cycles at three warps a scheduler (four spill and measure 88).  One
// row of 4,096 tokens: 7.5 us.
#include <type_traits>

#include "int4_weigh.cuh"

namespace akv {

constexpr int kWeighWarps = 4;
constexpr int kWeighThreads = kWeighWarps * 32;
constexpr int kWeighUnits = 8;     // (head, column tile) units prepared at a time
template <int D>
constexpr int kWeighPerSm = D == 256 ? 2 : 3;  // CTAs an SM that the registers leave room for

template <int D, int G, int NT>
struct WeighShape {
  static constexpr int GS = D / G;
  static constexpr int BK = GS / 8;     // K bytes of a thread per token and group
  static constexpr int KS = D / 16;     // MMA steps
  static constexpr int ROWS = 8 * NT;   // query columns of a unit
  static constexpr int CODES = kBlockTokens * D / 2;
  static constexpr int PAIRS = kBlockTokens * G * 4;
  static constexpr int REC = CODES + PAIRS;
  static constexpr int STAGES = D == 256 ? 3 : 4;
  static constexpr int OFF_FRAG = kWeighWarps * STAGES * REC;
  static constexpr int FRAG = KS * NT * 32 * 8;
  // per unit: fragments, then group sums of q, exponent factors, minus lse, visible lengths
  static constexpr int OFF_QS = OFF_FRAG + kWeighUnits * FRAG;
  static constexpr int OFF_CQ = OFF_QS + kWeighUnits * ROWS * G * 4;
  static constexpr int OFF_L2 = OFF_CQ + kWeighUnits * ROWS * 4;
  static constexpr int OFF_SEE = OFF_L2 + kWeighUnits * ROWS * 4;
  static constexpr int OFF_PREF = OFF_SEE + kWeighUnits * ROWS * 4;
  static constexpr int smem(int rows) { return OFF_PREF + (3 * rows + 1) * 4; }
  static_assert(smem(kWeighRows) <= 226 * 1024, "shared memory");
  static_assert(OFF_FRAG >= kNameBytes, "the rows' names stand where the ring will");
};

// token of tile row g: see the attention kernel's bank note
AKV_DEV int weigh_token(int g) { return g ^ ((g >> 2) & 1); }

template <int BYTES>
AKV_DEV void weigh_lds(const uint8_t* p, uint32_t (&w)[BYTES < 4 ? 1 : BYTES / 4]) {
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = lds_v4(p + 16 * i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (BYTES == 8) {
    const uint2 v = lds_v2(p);
    w[0] = v.x, w[1] = v.y;
  } else if constexpr (BYTES == 4) {
    w[0] = lds_u32(p);
  } else {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
}

// Lengths of the call rows [row0, row0 + R) and their pages' prefix sums; a row
// without new tokens has none, nor has one that an earlier call row names.
AKV_DEV void weigh_rows(const WeighParams& P, uint32_t* names, int* s_pref, int* s_len, int* s_new, int* s_scan) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, n_warps = blockDim.x >> 5;
  weigh_lengths(P, names, s_len, s_new);
  int base = 0;
  for (int e0 = 0; e0 < P.R; e0 += blockDim.x) {
    __syncthreads();
    const int e = e0 + t;
    int x = e < P.R && s_new[e] > 0 ? (s_len[e] + kBlockTokens - 1) / kBlockTokens : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(~0u, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_scan[warp] = x;
    __syncthreads();
    int before = base, sum = base;
    for (int w = 0; w < n_warps; ++w) {
      if (w < warp) before += s_scan[w];
      sum += s_scan[w];
    }
    if (e < P.R) s_pref[e + 1] = before + x;
    base = sum;
  }
  if (t == 0) s_pref[0] = 0;
  __syncthreads();
}

template <int D, int G, int NT>
__global__ void __launch_bounds__(kWeighThreads, kWeighPerSm<D>) weigh_few_kernel(const WeighParams P) {
  using S = WeighShape<D, G, NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  float* s_qs = reinterpret_cast<float*>(smem + S::OFF_QS);   // [unit][G][ROWS]
  float* s_cq = reinterpret_cast<float*>(smem + S::OFF_CQ);
  float* s_l2 = reinterpret_cast<float*>(smem + S::OFF_L2);
  int* s_see = reinterpret_cast<int*>(smem + S::OFF_SEE);
  int* s_pref = reinterpret_cast<int*>(smem + S::OFF_PREF);
  int* s_len = s_pref + P.R + 1;
  int* s_new = s_len + P.R;
  __shared__ int s_scan[kWeighWarps];

  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int g = lane >> 2, q4 = lane & 3;
  const int H = P.c.kv_heads, rep = P.Hq / H;

  weigh_rows(P, reinterpret_cast<uint32_t*>(smem), s_pref, s_len, s_new, s_scan);

  const int total = s_pref[P.R];
  const int share = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  int pos = static_cast<int>(min(static_cast<int64_t>(share) * blockIdx.x, static_cast<int64_t>(total)));
  const int end = min(total, pos + share);
  int e = 0, hi = P.R;  // the last row that starts at or before pos
  while (hi - e > 1) {
    const int mid = (e + hi) / 2;
    if (s_pref[mid] <= pos) e = mid; else hi = mid;
  }

  uint8_t* ring = smem + warp * S::STAGES * S::REC;
  uint32_t stage = 0;

  while (pos < end) {
    while (s_pref[e + 1] <= pos) ++e;
    const int page0 = pos - s_pref[e];
    const int n_pages = min(s_pref[e + 1], end) - pos;
    const int i = P.row0 + e, len = s_len[e], n_new = s_new[e];
    const int seq = P.rows ? __ldg(P.rows + i) : i;
    const int32_t* table = P.c.table + seq * P.c.table_stride + page0;
    float* w_row = P.weights + seq * P.w_stride;
    const int mine = (n_pages - warp + kWeighWarps - 1) / kWeighWarps;  // pages warp, warp + 4, ...
    const int tiles = (n_new * rep + S::ROWS - 1) / S::ROWS, units = H * tiles;

    for (int u0 = 0; u0 < units; u0 += kWeighUnits) {
      const int u1 = min(units, u0 + kWeighUnits);
      const int h0 = u0 / tiles, heads = (u1 - 1) / tiles - h0 + 1;

      // a page's number, read one page ahead of its copies, checked when they start
      auto look = [&](int k) -> int { return k < mine ? __ldg(table + warp + k * kWeighWarps) : 0; };
      auto check = [&](int p) -> int {
        if (p >= 0 && p < P.c.n_pages) return p;
        set_status(P.status, AKV_ERR_SHAPE);
        return 0;  // a bad page is read as page 0; nothing of it is added
      };
      int next_k = 0, next_h = 0, next_p = check(look(0)), ahead = look(1);  // the next record to copy
      auto issue = [&](uint32_t st) {
        if (next_k < mine) {
          const uint8_t* rec = P.c.pool + next_p * P.c.page_stride + (h0 + next_h) * P.c.head_stride;
          uint8_t* to = ring + st * S::REC;
#pragma unroll
          for (int k = 0; k < D / 32; ++k)
            cp_async16(to + (k * 32 + lane) * 16, rec + int4_layout(D, G).kc + (k * 32 + lane) * 16);
          if (lane < G * 8) cp_async16(to + S::CODES + lane * 16, rec + int4_layout(D, G).kp + lane * 16);
          if (++next_h == heads) {
            next_h = 0;
            next_p = check(ahead);
            ahead = look(++next_k + 1);
          }
        }
        cp_async_commit();
      };
      for (int k = 0; k < S::STAGES; ++k) issue((stage + k) % S::STAGES);

      // ---- queries of the units as MMA operands
      __syncthreads();  // the previous units' are done with
      constexpr int PER = D / 32;
      static_assert(kWeighUnits * S::ROWS <= 32 * kWeighWarps, "a lane a column");
      const int columns = (u1 - u0) * S::ROWS;
      int64_t where = -1;  // lane c: the warp's c-th column's query
      {
        const int n = warp + lane * kWeighWarps, unit = n / S::ROWS;
        const int h = (u0 + unit) / tiles, rr = (u0 + unit) % tiles * S::ROWS + n % S::ROWS, m = rr / rep;
        const int hq = h * rep + rr - m * rep;
        if (n < columns) {
          float lse = -INFINITY;
          if (m < n_new) {
            where = i * P.q_sr + hq * P.q_sh + m * P.q_sm;
            lse = __ldg(P.lse + (static_cast<int64_t>(i) * P.Hq + hq) * P.M + m);
          }
          const bool counts = fabsf(lse) < INFINITY;
          s_l2[n] = counts ? -lse * 1.4426950408889634f : -INFINITY;
          s_see[n] = counts ? len - n_new + m + 1 : 0;
        }
      }
      __syncwarp();
      constexpr int BATCH = 4;  // columns whose loads fly together
      for (int n0 = 0; warp + n0 * kWeighWarps < columns; n0 += BATCH) {
        uint16_t raw[BATCH][PER];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
          const int64_t at = __shfl_sync(~0u, where, n0 + b);
#pragma unroll
          for (int k = 0; k < PER; ++k) raw[b][k] = at >= 0 ? P.q[at + lane * PER + k] : 0;
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
          const int n = warp + (n0 + b) * kWeighWarps, unit = n / S::ROWS, col = n % S::ROWS;
          if (n >= columns) break;
          float x[PER];
          uint32_t top = 0u;
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            x[k] = P.bf16 ? elem_to_float<true>(raw[b][k]) : elem_to_float<false>(raw[b][k]);
            top = max(top, __float_as_uint(x[k]) & 0x7FFFFFFFu);
          }
          top = __reduce_max_sync(~0u, top);
          const bool bad = top >= 0x7F800000u;
          int ex = 0;  // 2^ex brings the largest into [2^13, 2^14)
          if (top && !bad) ex = 13 - (static_cast<int>(top >> 23) - 127);
          ex = ex > 120 ? 120 : (ex < -120 ? -120 : ex);
          const float up = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
          uint16_t* frag = reinterpret_cast<uint16_t*>(smem + S::OFF_FRAG + unit * S::FRAG);
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            const int c = lane * PER + k;
            const float part = k & 1 ? 1.f : 16.f;  // even channels' codes are the high four bits
            const __half hv = __float2half_rn(bad ? 0.f : x[k] * up / part);
            sum += __half2float(hv) * part;
            const int gi = c / S::GS, r = c % S::GS, cc = r / (S::GS / 4), r2 = r % (S::GS / 4);
            int ks, half;
            if constexpr (S::BK >= 4) {
              ks = gi * (S::GS / 16) + (r2 / 8) * 2 + ((r2 >> 1) & 1);
              half = (r2 >> 2) & 1;
            } else {
              ks = gi;
              half = r2 >> 1;
            }
            const int reg = c & 1 ? 0 : 1;
            frag[(((ks * NT + col / 8) * 32 + (col % 8) * 4 + cc) * 2 + reg) * 2 + half] = __half_as_ushort(hv);
          }
          constexpr int GL = 32 / G;  // lanes of a group
#pragma unroll
          for (int o = 1; o < GL; o <<= 1) sum += __shfl_xor_sync(~0u, sum, o);
          if (lane % GL == 0) s_qs[(unit * G + lane / GL) * S::ROWS + col] = sum;
          if (lane == 0) {
            s_cq[n] = P.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
            if (bad) s_l2[n] = -INFINITY, s_see[n] = 0;
          }
        }
      }
      __syncthreads();

      // ---- this warp's pages: all heads of the units, then the next page
      for (int k = 0; k < mine; ++k) {
        const int tok0 = (page0 + warp + k * kWeighWarps) * kBlockTokens;
        const int p = __ldg(table + warp + k * kWeighWarps), tok = tok0 + q4 * 8 + weigh_token(g);
        const float old = tok < len ? w_row[tok] : 0.f;
        float w[4] = {0.f, 0.f, 0.f, 0.f};
        for (int hh = 0; hh < heads; ++hh) {
          cp_async_wait<S::STAGES - 1>();
          __syncwarp();
          const uint8_t* rec = ring + stage * S::REC;
          uint32_t kp[4][G];
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int gi = 0; gi < G; ++gi)
              kp[r][gi] = lds_u32(rec + S::CODES + (r * 8 + weigh_token(g)) * G * 4 + gi * 4);
          const int ub = max(u0, (h0 + hh) * tiles) - u0, ue = min(u1, (h0 + hh + 1) * tiles) - u0;
          for (int unit = ub; unit < ue; ++unit) {
            const uint2* frag = reinterpret_cast<const uint2*>(smem + S::OFF_FRAG + unit * S::FRAG) + lane;
            const uint64_t* qs2 = reinterpret_cast<const uint64_t*>(s_qs + unit * G * S::ROWS) + q4;
            uint64_t x[4][NT];
#pragma unroll
            for (int gi = 0; gi < G; ++gi) {
              uint32_t kw[4][S::BK < 4 ? 1 : S::BK / 4];
#pragma unroll
              for (int r = 0; r < 4; ++r)
                weigh_lds<S::BK>(rec + (r * 8 + weigh_token(g)) * (D / 2) + gi * (S::GS / 2) + q4 * S::BK, kw[r]);
              float acc[2][NT][4];
#pragma unroll
              for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int c = 0; c < 4; ++c) acc[mt][nt][c] = 0.f;
#pragma unroll
              for (int s = 0; s < S::GS / 16; ++s) {
                const int ks = gi * (S::GS / 16) + s;
                uint2 b[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) b[nt] = frag[(ks * NT + nt) * 32];
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                  uint32_t a[4];
#pragma unroll
                  for (int r = 0; r < 2; ++r) {
                    uint32_t v;
                    if constexpr (S::BK >= 4) v = s & 1 ? kw[2 * mt + r][s / 2] >> 8 : kw[2 * mt + r][s / 2];
                    else v = prmt(kw[2 * mt + r][0], 0u, 0x4140);
                    a[r] = v & 0x000F000Fu;
                    a[2 + r] = v & 0x00F000F0u;
                  }
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) mma_16816(acc[mt][nt], a[0], a[1], a[2], a[3], b[nt].x, b[nt].y);
                }
              }
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const float2 sz = __half22float2(u32_as_h2(kp[r][gi]));
                const float up = sz.x * 16777216.f;
                const uint64_t s2 = f2_make(up, up), z2 = f2_make(sz.y, sz.y);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                  const uint64_t q2 = qs2[(gi * S::ROWS + nt * 8) / 2];
                  const float* a = acc[r >> 1][nt] + (r & 1) * 2;
                  const uint64_t zq = gi == 0 ? f2_mul(z2, q2) : f2_fma(z2, q2, x[r][nt]);
                  x[r][nt] = f2_fma(f2_make(a[0], a[1]), s2, zq);
                }
              }
            }
            const bool tail = tok0 + kBlockTokens > len - n_new;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const int c0 = unit * S::ROWS + nt * 8 + 2 * q4;
              const float2 cq = *reinterpret_cast<const float2*>(s_cq + c0), l2 = *reinterpret_cast<const float2*>(s_l2 + c0);
              const int2 see = *reinterpret_cast<const int2*>(s_see + c0);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                float2 y = f2_split(f2_fma(x[r][nt], f2_make(cq.x, cq.y), f2_make(l2.x, l2.y)));
                if (tail) {
                  const int tok = tok0 + r * 8 + weigh_token(g);
                  if (tok >= see.x) y.x = -INFINITY;
                  if (tok >= see.y) y.y = -INFINITY;
                }
                w[r] += fast_exp2(y.x) + fast_exp2(y.y);
              }
            }
          }
          __syncwarp();
          issue(stage);
          if (++stage == S::STAGES) stage = 0;
        }
        // lane q4 keeps row q4's sum
        const bool odd = q4 & 1, high = q4 & 2;
        const float a = (odd ? w[1] : w[0]) + __shfl_xor_sync(~0u, odd ? w[0] : w[1], 1);
        const float b = (odd ? w[3] : w[2]) + __shfl_xor_sync(~0u, odd ? w[2] : w[3], 1);
        const float sum = (high ? b : a) + __shfl_xor_sync(~0u, high ? a : b, 2);
        if (tok < len && p >= 0 && p < P.c.n_pages) w_row[tok] = old + sum;
      }
    }
    pos += n_pages;
  }
}

template <int D, int G, int NT>
static int launch_few(const WeighParams& P, cudaStream_t st) {
  using S = WeighShape<D, G, NT>;
  const int smem = S::smem(P.R);
  if (!ensure_dynamic_smem<weigh_few_kernel<D, G, NT>>(smem)) return AKV_ERR_LAUNCH;
  // CTAs that an SM holds: what its registers allow, and its 228 KB of shared memory, of which each takes 1 KB
  // more than it asks for.  Shares for those that registers alone allow ran in two waves where the fragments of 16
  // columns are large, us: 16 rows x 8,192, 32 / 8 heads of 256 112, so 92; 4 x 16,384, 16 / 2 of 128 in four
  // groups 24, so 18.
  constexpr int kSmem = 228 * 1024, kSmemOfCta = 1024 + kWeighWarps * 32;
  const int fit = kSmem / (smem + kSmemOfCta), per_sm = fit < kWeighPerSm<D> ? fit : kWeighPerSm<D>;
  const int64_t pages = static_cast<int64_t>(P.R) * P.c.max_blocks;
  const int64_t most = 148 * per_sm, want = (pages + kWeighWarps - 1) / kWeighWarps;
  weigh_few_kernel<D, G, NT><<<static_cast<int>(want < most ? want : most), kWeighThreads, smem, st>>>(P);
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}

template <int D, int NT>
static int few_by_group(const WeighParams& P, cudaStream_t st) {
  switch (D / P.c.group) {
    case 1: return launch_few<D, 1, NT>(P, st);
    case 2: return launch_few<D, 2, NT>(P, st);
    default: return launch_few<D, 4, NT>(P, st);
  }
}

static int weigh_few(const WeighParams& P, cudaStream_t st) {
  const bool one = P.M * (P.Hq / P.c.kv_heads) <= 8;
  switch (P.c.head_dim) {
    case 64: return one ? few_by_group<64, 1>(P, st) : few_by_group<64, 2>(P, st);
    case 128: return one ? few_by_group<128, 1>(P, st) : few_by_group<128, 2>(P, st);
    default: return one ? few_by_group<256, 1>(P, st) : few_by_group<256, 2>(P, st);
  }
}

// Query columns (new tokens x query heads of a group) that still go to the kernel
// above; more go to the fifth-generation tensor cores, whose tiles of 64 (four
// groups) or 128 columns cost the same half empty.  Measured, us, this kernel :
// that one, for 1 row x 4,096 tokens, 32 / 8 heads | 16 x 8,192, 32 / 8 |
// 4 x 16,384, 16 / 2:
//   one group    16 columns  20 : 21 |  51 : 103 | 16 : 29
//                32          32 : 21 |  87 : 103 | 22 : 30
//                64          57 : 22 | 159 : 103 | 36 : 29
//   two groups   16          20 : 23 |  55 : 117 | 16 : 31
//                32          32 : 23 |  92 : 118 | 24 : 32
//                64          57 : 23 | 166 : 118 | 36 : 31
//   four groups  16          20 : 22 |  60 : 105 | 18 : 29
//                32          33 : 21 |  97 : 105 | 26 : 29
//                64          59 : 22 | 173 : 105 | 40 : 29
// (heads of 64 and 256 alike: one group, 32 columns 28 : 18 | 71 : 88 | 20 : 25, 42 : 25 | 146 : 168 | 32 : 37).
static int weigh_few_columns(int n_groups) { return n_groups == 1 ? 32 : 16; }

}  // namespace akv

using namespace akv;

extern "C" size_t akv_int4_weigh_workspace_bytes(int R, int M, int Hq, int kv_heads, int head_dim, int group) {
  if (R < 0 || M < 0 || Hq <= 0 || kv_heads <= 0 || Hq % kv_heads || !int4_shape_ok(head_dim, group)) return 0;
  if (R == 0 || static_cast<int64_t>(M) * (Hq / kv_heads) <= weigh_few_columns(head_dim / group)) return 16;
  if (static_cast<int64_t>(M) * Hq > INT32_MAX / 2) return 0;
  return weigh_many_workspace(R, M, Hq, kv_heads, head_dim, head_dim / group);
}

extern "C" int akv_int4_weigh(const akv_int4_weigh_args* a, void* stream) {
  if (!a) return AKV_ERR_NULL;
  const akv_int4_cache* c = a->cache;
  const int rc = int4_check(c);
  if (rc) return rc;
  if (a->dtype != AKV_FP16 && a->dtype != AKV_BF16) return AKV_ERR_UNSUPPORTED;
  if (a->R < 0 || a->M < 0 || a->Hq <= 0 || a->Hq % c->kv_heads) return AKV_ERR_SHAPE;
  if (a->w_stride < static_cast<int64_t>(c->max_blocks) * kBlockTokens) return AKV_ERR_SHAPE;
  if (a->R == 0 || a->M == 0) return AKV_OK;
  if (!a->q || !a->lse || !a->weights) return AKV_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(a->q) & 1) ||
      ((reinterpret_cast<uintptr_t>(a->lse) | reinterpret_cast<uintptr_t>(a->weights)) & 3))
    return AKV_ERR_ALIGN;
  // columns and pages of a launch are counted in 32 bits
  if (static_cast<int64_t>(a->M) * a->Hq > INT32_MAX / 2) return AKV_ERR_UNSUPPORTED;
  const bool many = a->M * (a->Hq / c->kv_heads) > weigh_few_columns(c->head_dim / c->group);
  if (many) {
    if (!a->workspace) return AKV_ERR_NULL;
    if (reinterpret_cast<uintptr_t>(a->workspace) & 15) return AKV_ERR_ALIGN;
    if (a->workspace_bytes < akv_int4_weigh_workspace_bytes(a->R, a->M, a->Hq, c->kv_heads, c->head_dim, c->group))
      return AKV_ERR_WORKSPACE;
  }
  int rows = kWeighRows;
  if (rows > INT32_MAX / c->max_blocks) rows = INT32_MAX / c->max_blocks;
  WeighParams p{};
  p.c = *c;
  p.rows = a->rows;
  p.n_new = a->n_new;
  p.M = a->M;
  p.Hq = a->Hq;
  p.q = static_cast<const uint16_t*>(a->q);
  p.q_sr = a->q_sr; p.q_sh = a->q_sh; p.q_sm = a->q_sm;
  p.lse = a->lse;
  p.scale = a->sm_scale;
  p.weights = a->weights;
  p.w_stride = a->w_stride;
  p.bf16 = a->dtype == AKV_BF16;
  p.status = a->status;
  if (many) return weigh_many(p, a->R, a->workspace, static_cast<cudaStream_t>(stream));
  for (int r = 0; r < a->R; r += rows) {
    p.row0 = r;
    p.R = a->R - r < rows ? a->R - r : rows;
    const int e = weigh_few(p, static_cast<cudaStream_t>(stream));
    if (e) return e;
  }
  return AKV_OK;
}
