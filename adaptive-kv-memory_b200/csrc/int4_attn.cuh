// Attention over the 4-bit paged cache, straight from the packed pages
// (kernel templates; one translation unit per head dim instantiates them).
//
// Mathematics.  With token t's value c*s_tg + z_tg in channel group g,
//   q.K_t = sum_g  s_tg (q_g . c_tg) + z_tg sum(q_g)
//   O     = sum_t p_t V_t
//         = sum_t (p_t s_tg)(c - m_t) + sum_t p_t (z_tg + m_t s_tg)
// so both contractions run on codes.  For K a code needs no conversion: alone
// in bits 4..7 of a half it is the fp16 subnormal c * 2^-20, one shift and one
// AND for two codes of a word.  (The MMA aligns its products by the operands'
// nominal exponents and cuts them off, so bits 0..3 would lose 4 bits more of
// the sum.)  Over the thousands of additions of P.V that cutting off is a
// drift of the growing sum; there the codes are centred, exactly, by one fp16
// operation more, and the sums stay as small as the output: m_t is 8 and 7 in
// turn, 16 tokens each, since codes lie around 7.5 (with 8 alone a CTA that
// takes 32K tokens of a row left an fp16 output 1.1 to 1.4 times as far off as
// its own rounding; with both, 1.00).  Online softmax, maximum and sums in fp32.
//
// Roundings: q is scaled per row by a power of two into fp16's middle range
// (exact unless 2^-24 of the row's largest).  p_t s_tg enters the MMA as one
// fp16 term for a bf16 output (an eighth of that output's own rounding), as
// two, the second holding the first's error, for an fp16 output (LO).  The
// zero-point sum, l and the partial results are fp32.
//
// Work.  A unit is one (row, tile of 8 or 16 query rows, KV head); the units'
// pages form one list that is cut into equal shares, one per resident CTA, from
// the lengths on the device: ragged batches balance and the host needs no
// length.  A unit cut in two or more is merged by the last of its CTAs to
// finish (or, with many query rows over a long table, by a second kernel); a
// call of short units keeps each whole.  A warp streams every fourth page of
// its share through its own ring of bulk copies and meets the others in shared
// memory at a unit's end.  Sums are taken in an order that the lengths alone
// decide, so a call repeated gives the same bits.
//
// Bound and measured (B200, 32 / 8 heads of 128, 16 x 32K tokens).  The pages
// alone stream in 95 us (6.0 TB/s).  One query token, group 128: 139 us fp16
// (4.1 TB/s).  Per page and warp some 630 instructions, 40 % of them unpacking
// (256 codes a lane); issue slots 60 %, the integer pipe 52 %, tensor cores
// 25 % busy, and fewer or more warps change nothing: instruction throughput
// bounds it.  Five tokens, groups of 32, bf16: 243 us; the same bound, the
// per-group scaling of scores above all.  What was tried and did not help: two
// pages per iteration, one CTA of 16 warps an SM, keeping warps in step, three
// or four query tiles a CTA (the registers leave too few warps), three or more
// CTAs' worth of shares.
#pragma once

#include <type_traits>

#include "int4.cuh"

namespace akv {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kAttnEntries = 1024;  // (row, row tile) pairs of one launch
constexpr int kAttnUnits = 16384;   // units of one launch
// Pages of a CTA's share, at least (two per warp): with 4 more parts are merged,
// with 16 a share takes longer (1 x 4K tokens 15.3 / 14.6 / 16.6 us, 1 x 32K
// 30.9 / 22.7 / 20.6 us with 4 / 8 / 16).
constexpr int kAttnMinPages = 8;
// Up to this many pages no unit is split, where all are so short (64 x 100-300
// tokens: 24.7 us split, 18.5 us whole; 64 x 400-1000 32.8 and 30.8).
constexpr int kAttnWhole = 32;
// The pages that such a unit's set-up counts for in its share (90 short rows of
// 12 drafted tokens: 107 us with 0, 80 with 4, 72 with 8 and 16; 64 x 100-300
// tokens 18.5, 18.6, 16.5 and 15.5).
constexpr int kAttnSetup = 16;
constexpr int kAttnFused = 1024;  // partial rows of a unit that its last CTA merges by itself
// The maximum's weight stands at 2^9, and weights may reach 2^15, fp16's last
// binade, before the maximum moves: the rescaling of the sums becomes rare.
// fp16 loses bits below 2^-14, so a weight keeps 11 of them down to 2^-23 of
// the maximum, and the 22 of two terms down to 2^-12.  (With the maximum at 2^0
// and 90 % of the weight on a token of value 0, the many small weights beside it
// left the output off by 4 to 9 times its own rounding; with 99 %, by 40 to 150.)
constexpr float kTopLog2 = 9.f, kMostLog2 = 15.f;

struct Int4AttnParams {
  akv_int4_cache c;
  const int32_t* rows;
  const int32_t* n_new;
  int row0, R;  // call rows [row0, row0 + R) of this launch
  int M, Hq, tiles;
  const uint16_t* q;
  int64_t q_sr, q_sh, q_sm;
  float scale;
  uint16_t* out;
  int64_t o_sr, o_sh, o_sm;
  float* lse;
  int bf16;
  int out4;  // output rows on 4-byte boundaries
  float* part;         // [slot][8 NT][D + 2]
  unsigned* arrived;   // per unit: CTAs that have stored their part; 0 between calls
  int2* meta;          // per unit: first and last CTA, for the combine kernel (NULL: the last CTA merges)
  int* status;
};

// resident CTAs of an SM: what the registers of 128 threads leave
constexpr int attn_occ(int D, int nt) { return D == 256 ? 2 : (nt == 1 ? 4 : 3); }

// Terms of a weight in P.V (LO): 0 one fp16 term; 1 two, the second the first's
// error, in an MMA of its own; 2 two, the second in columns 4..7, where the
// queries of columns 0..3 stand once more (at most four query rows: a grouped
// decode step's usual count leaves those columns free).
//
// A bf16 output leaves room to round each value of V to fp16 as it is unpacked,
// scale and zero applied (AttnShape::AV); the weights are then the same for
// every group.  It costs a second fp16 operation for each pair of codes, and a
// look for values past fp16's range (1 to 4 % of the time), and saves per group
// and query tile what the weights cost: it pays from four (group, tile) pairs
// on.  Against the formula a bf16 output is then 1.01 to 1.03 times as far off
// as by its own rounding.
constexpr bool attn_av(int G, int NT, int LO) { return !LO && G * NT >= 4; }

template <int D, int G, int NT, int LO>
struct AttnShape {
  static constexpr int GS = D / G;              // channels of a group
  static constexpr int BK = GS / 8;             // K bytes of a thread per token and group
  static constexpr bool AV = attn_av(G, NT, LO);
  static constexpr int GV = AV ? 1 : G;         // groups the weights differ for
  static constexpr int BV = D / GV / 16;        // V bytes of a thread per token and such group
  static constexpr int REC = int4_layout(D, G).bytes;
  static constexpr int ROWS = 8 * NT;           // query rows of a CTA
  static constexpr int STAGES = D == 64 ? 4 : (D == 128 && (NT > 1 || G == 1) ? 3 : 2);
  static constexpr int RING = kAttnWarps * STAGES * REC;
  static constexpr int PITCH = D + 4;
  static constexpr int MERGE = kAttnWarps * ROWS * PITCH * 4;
  static constexpr int BUF = RING > MERGE ? RING : MERGE;
  static constexpr int FRAG = D / 16 * NT * 32 * 8;
  // ring / merge buffer, fragments, then: group sums of q, exponent factors,
  // visible lengths, output offsets, (y, l) per warp and row and of all warps,
  // barriers; per entry: prefix sums of pages, lengths, new tokens
  static constexpr int OFF_FRAG = (BUF + 127) / 128 * 128;
  static constexpr int OFF_QS = OFF_FRAG + FRAG;
  static constexpr int OFF_CQ = OFF_QS + ROWS * G * 4;
  static constexpr int OFF_SEE = OFF_CQ + ROWS * 4;
  static constexpr int OFF_OUT = OFF_SEE + ROWS * 4;
  static constexpr int OFF_LSE = OFF_OUT + ROWS * 8;
  static constexpr int OFF_ON = OFF_LSE + ROWS * 4;
  static constexpr int OFF_ML = OFF_ON + ROWS * 4;
  static constexpr int OFF_TL = OFF_ML + kAttnWarps * ROWS * 8;
  static constexpr int OFF_BAR = OFF_TL + ROWS * 8;
  static constexpr int OFF_PREF = OFF_BAR + kAttnWarps * STAGES * 8;
  static constexpr int OCC = attn_occ(D, NT);
  static constexpr int smem(int entries) { return OFF_PREF + (3 * entries + 1) * 4; }
  static_assert(OCC * (smem(64) + 1024) <= 228 * 1024, "resident CTAs do not fit");
  static_assert(kAttnFused * 4 + ROWS * 8 <= BUF, "the merge of a unit's parts does not fit the buffer");
};

// token of tile row g: a permutation within 8 that spreads the V loads of the
// four thread columns over the banks (rows of both parities in every load)
AKV_DEV int tile_token(int g) { return g ^ ((g >> 2) & 1); }

// m_t for the tokens of each P.V step.  Codes lie around 7.5: with one of them
// the sums would grow by half a scale a token, far past the output.
AKV_DEV constexpr int code_centre(int step) { return step ? 7 : 8; }

// the codes in bits 0..3 (4..7) of both halves, as the fp16 pair c - centre
AKV_DEV uint32_t low_code(uint32_t y, int centre) {
  const uint32_t back = 0x10001u * (0xE400u + centre);  // -(1024 + centre)
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(lop_magic<0x000F000Fu>(y)), "r"(back));  // 1024 + c - ...
  return r;
}
AKV_DEV uint32_t high_code(uint32_t y, int centre) {
  const uint32_t back = 0x10001u * (0xD400u + 16 * centre);  // -(64 + centre)
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;"  // (1024 + 16 c) / 16 - ...
      : "=r"(r)
      : "r"(lop_magic<0x00F000F0u>(y)), "r"(0x2C002C00u), "r"(back));
  return r;
}

template <int BYTES>
AKV_DEV void lds_bytes(const uint8_t* p, uint32_t (&w)[BYTES < 4 ? 1 : BYTES / 4]) {
  if constexpr (BYTES >= 16) {
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 16 * i);
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else if constexpr (BYTES == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else if constexpr (BYTES == 2) {
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else {
    w[0] = *p;
  }
}

// the query row that stands in column n of a tile
template <int LO>
AKV_DEV int tile_row(int n) {
  return LO == 2 ? n & 3 : n;
}

// the (scale, zero) pairs of a token
template <int G>
AKV_DEV void lds_pairs(const uint8_t* p, uint32_t (&w)[G]) {
  if constexpr (G == 4) {
    lds_u32x4(p, w);
  } else if constexpr (G == 2) {
    const uint2 v = lds_v2(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = lds_u32(p);
  }
}

// Element offset of the output row of query token m, head hq of call row i.
AKV_DEV int64_t out_row(const Int4AttnParams& P, int i, int hq, int m) {
  return i * P.o_sr + hq * P.o_sh + m * P.o_sm;
}

// What a row's maximum (log2) and sum L make of its output: its lse, and the
// factor of the sums of p V.  L 0: a row that sees nothing.  L NaN (a query
// that is not finite, scores past fp32): both NaN.
AKV_DEV float2 row_scale(float top, float L) {
  return L == 0.f ? make_float2(-INFINITY, 0.f) : make_float2((top + log2f(L)) * 0.6931471805599453f, 1.f / L);
}

// Output channels of accumulator pair p (order of the merge buffer) of the row
// at `row`; its lse with pair 0.  scale: row_scale().
template <int D, int G>
AKV_DEV void store_pair(const Int4AttnParams& P, int64_t row, float* lse, int p, float2 v, float2 scale) {
  constexpr int GS = D / G, BV = GS / 16;
  const int j = p / 8, g = p % 8;
  const int ch = j / BV * GS + g * 2 * BV + 2 * (j % BV);
  const bool on = scale.y != 0.f;
  v.x = on ? v.x * scale.y : 0.f;
  v.y = on ? v.y * scale.y : 0.f;
  uint16_t* o = P.out + row + ch;
  const uint32_t w = P.bf16 ? pack_elems<true>(v.x, v.y) : pack_elems<false>(v.x, v.y);
  if (P.out4) {
    *reinterpret_cast<uint32_t*>(o) = w;
  } else {
    o[0] = static_cast<uint16_t>(w);
    o[1] = static_cast<uint16_t>(w >> 16);
  }
  if (lse && p == 0) *lse = scale.x;
}

// One CTA merges the parts of a unit (segs * 8 NT <= kAttnFused, so their
// weights fit the buffer w).
template <int D, int G, int NT>
AKV_DEV void merge_parts(const Int4AttnParams& P, const float* part, int segs, const int64_t* s_out, const int* s_lse,
                         int valid, float* w) {
  constexpr int ROWS = 8 * NT;
  constexpr int64_t STEP = static_cast<int64_t>(ROWS) * (D + 2);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  float2* s_tl = reinterpret_cast<float2*>(w + kAttnFused);  // per row: lse, factor
  for (int n = warp; n < valid; n += kAttnWarps) {
    const float* ml = part + n * (D + 2) + D;
    float top = -INFINITY, L = 0.f;
    const float2 none = make_float2(-INFINITY, 0.f);
    const float2 first = lane < segs ? __ldcg(reinterpret_cast<const float2*>(ml + lane * STEP)) : none;
    top = first.x;
    for (int s = lane + 32; s < segs; s += 32) top = fmaxf(top, __ldcg(ml + s * STEP));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    for (int s = lane; s < segs; s += 32) {
      const float2 yl = s < 32 ? first : __ldcg(reinterpret_cast<const float2*>(ml + s * STEP));
      const float x = yl.x == -INFINITY ? 0.f : exp2f(yl.x - top);
      w[n * segs + s] = x;
      L = fmaf(x, yl.y, L);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
    if (lane == 0) s_tl[n] = row_scale(top, L);
  }
  __syncthreads();
  constexpr int T = 4;  // output pairs of a thread at a time
  for (int k0 = t; k0 < valid * (D / 2); k0 += T * kAttnThreads) {
    const float* at[T];
    const float* wn[T];
    float2 acc[T];
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const int k = min(k0 + j * kAttnThreads, valid * (D / 2) - 1);
      at[j] = part + k / (D / 2) * (D + 2) + 2 * (k % (D / 2));
      wn[j] = w + k / (D / 2) * segs;
      acc[j] = make_float2(0.f, 0.f);
    }
#pragma unroll 8
    for (int s = 0; s < segs; ++s)
#pragma unroll
      for (int j = 0; j < T; ++j) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(at[j] + s * STEP));
        acc[j].x = fmaf(wn[j][s], v.x, acc[j].x);
        acc[j].y = fmaf(wn[j][s], v.y, acc[j].y);
      }
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const int k = k0 + j * kAttnThreads;
      if (k >= valid * (D / 2)) break;
      const int n = k / (D / 2);
      store_pair<D, G>(P, s_out[n], P.lse ? P.lse + s_lse[n] : nullptr, k % (D / 2), acc[j], s_tl[n]);
    }
  }
}

template <int D, int G, int NT, int LO>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<D, G, NT, LO>::OCC) int4_attn_kernel(const Int4AttnParams P) {
  using S = AttnShape<D, G, NT, LO>;
  constexpr int KS = D / 16;  // MMA steps of q.K
  extern __shared__ __align__(128) uint8_t smem[];
  float* s_qs = reinterpret_cast<float*>(smem + S::OFF_QS);
  float* s_cq = reinterpret_cast<float*>(smem + S::OFF_CQ);
  int* s_see = reinterpret_cast<int*>(smem + S::OFF_SEE);
  float* s_on = reinterpret_cast<float*>(smem + S::OFF_ON);  // 1; 0 past n_new; NaN for a query that is not finite
  int* s_lse = reinterpret_cast<int*>(smem + S::OFF_LSE);
  int64_t* s_out = reinterpret_cast<int64_t*>(smem + S::OFF_OUT);
  float2* s_ml = reinterpret_cast<float2*>(smem + S::OFF_ML);
  float2* s_tl = reinterpret_cast<float2*>(smem + S::OFF_TL);
  uint64_t* s_bar = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  int* s_pref = reinterpret_cast<int*>(smem + S::OFF_PREF);
  __shared__ int s_scan[kAttnWarps], s_max[kAttnWarps], s_last;

  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int g = lane >> 2, q4 = lane & 3;
  const int H = P.c.kv_heads, rep = P.Hq / H;
  const int entries = P.R * P.tiles;
  int* s_len = s_pref + entries + 1;
  int* s_new = s_len + entries;

  if (lane < S::STAGES) mbar_init(s_bar + warp * S::STAGES + lane, 1);
  fence_mbar_init();

  // Pages of every entry (row, row tile); all heads of a row alike.
  for (int e = t; e < entries; e += kAttnThreads) {
    const Int4Row r = int4_row(P.c, P.rows, P.n_new, P.row0 + e / P.tiles, P.M, P.status);
    s_len[e] = r.len;
    s_new[e] = r.n_new;
  }
  auto pages_of = [&](int e) -> int {
    const int tile = e % P.tiles, n_new = s_new[e];
    const int first = tile * S::ROWS / rep;  // its first query token
    const int last = min((tile * S::ROWS + S::ROWS - 1) / rep, n_new - 1);
    const int see = s_len[e] - n_new + last + 1;
    return first <= last && see > 0 ? (see + kBlockTokens - 1) / kBlockTokens : 0;
  };
  // Prefix sums of (pages + extra) over the entries that have any; whether some
  // have none, and the longest.
  bool empty = false;
  int longest = 0;
  auto scan = [&](int extra) {
    int base = 0, most = 0;
    for (int e0 = 0; e0 < entries; e0 += kAttnThreads) {
      __syncthreads();
      const int e = e0 + t;
      const int n = e < entries ? pages_of(e) : 0;
      empty |= e < entries && n == 0;
      most = max(most, n);
      int x = n ? n + extra : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_scan[warp] = x;
      __syncthreads();
      int before = base, sum = base;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        if (w < warp) before += s_scan[w];
        sum += s_scan[w];
      }
      if (e < entries) s_pref[e + 1] = before + x;
      base = sum;
    }
    most = __reduce_max_sync(~0u, most);
    if (lane == 0) s_max[warp] = most;
    if (t == 0) s_pref[0] = 0;
    empty = __syncthreads_or(empty);
    longest = max(max(s_max[0], s_max[1]), max(s_max[2], s_max[3]));
  };
  scan(0);
  // Where every unit is short, none is split (below), and a unit's cost is more
  // its set-up than its pages: it counts as so many pages more.
  const int extra = longest <= kAttnWhole ? kAttnSetup : 0;
  if (extra) scan(extra);

  // rows without any visible token: zero output
  for (int u = empty ? blockIdx.x : entries * H; u < entries * H; u += gridDim.x) {
    const int e = u / H, h = u % H;
    if (s_pref[e + 1] != s_pref[e]) continue;
    const int i = P.row0 + e / P.tiles;
    if (t == 0 && P.meta) P.meta[u] = make_int2(0, 0);
    for (int n = warp; n < S::ROWS; n += kAttnWarps) {
      const int rr = e % P.tiles * S::ROWS + n, m = rr / rep;
      if (m >= P.M) break;
      const int hq = h * rep + rr - m * rep;
      uint16_t* o = P.out + out_row(P, i, hq, m);
      for (int c = lane; c < D / 2; c += 32) {
        if (P.out4) {
          reinterpret_cast<uint32_t*>(o)[c] = 0u;
        } else {
          o[2 * c] = 0;
          o[2 * c + 1] = 0;
        }
      }
      if (P.lse && lane == 0) P.lse[(i * P.Hq + hq) * P.M + m] = -INFINITY;
    }
  }

  // This CTA's share of all pages, a contiguous run over (row, tile, head, page);
  // their number fits 31 bits (the caller sees to it).  Where every unit (row,
  // tile, head) is short, a share's ends move up to the next unit's start:
  // no unit is split, so none has parts to merge.
  const int total = s_pref[entries] * H;
  int share = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  const bool keep = extra > 0;
  if (!keep && share < kAttnMinPages) share = kAttnMinPages;
  if (static_cast<int64_t>(share) * blockIdx.x >= total) return;
  int begin = share * blockIdx.x;
  int end = total - begin > share ? begin + share : total;
  auto entry_at = [&](int pos) -> int {  // the last entry that starts at or before pos
    int lo = 0, hi = entries;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (s_pref[mid] * H <= pos) lo = mid; else hi = mid;
    }
    return lo;
  };
  if (keep) {
    auto next_unit = [&](int pos) -> int {
      if (pos >= total) return total;
      const int x = entry_at(pos), start = s_pref[x] * H, pages = s_pref[x + 1] - s_pref[x];
      return start + (pos - start + pages - 1) / pages * pages;
    };
    begin = next_unit(begin);
    end = next_unit(end);
    if (begin >= end) return;
  }
  int pos = begin;
  int e = entry_at(begin);
  uint32_t stage = 0, phase = 0;
  bool alive = true;
  uint8_t* ring = smem + warp * S::STAGES * S::REC;
  uint64_t* bars = s_bar + warp * S::STAGES;

  while (pos < end) {
    while (s_pref[e + 1] == s_pref[e]) ++e;
    const int e_start = s_pref[e] * H;
    const int weight = s_pref[e + 1] - s_pref[e], pages = weight - extra;
    const int h = (pos - e_start) / weight;
    const int u_start = e_start + h * weight;
    const int page0 = pos - u_start;
    int n_pages = pages - page0;
    if (n_pages > end - pos) n_pages = end - pos;
    const int unit = e * H + h;
    const bool whole = u_start >= begin && u_start + weight <= end;
    const int i = P.row0 + e / P.tiles, tile = e % P.tiles;
    const int len = s_len[e], n_new = s_new[e];
    const int seq = P.rows ? __ldg(P.rows + i) : i;  // in range: its pages are not 0
    const int32_t* table = P.c.table + seq * P.c.table_stride + page0;
    const uint8_t* pool = P.c.pool + h * P.c.head_stride;
    const int mine = (n_pages - warp + kAttnWarps - 1) / kAttnWarps;  // pages warp, warp + 4, ...

    // page numbers of this warp's next 32 pages, one per lane
    auto page_ids = [&](int k0) -> int {
      const int k = k0 + lane;
      int p = 0;
      if (k < mine) {
        p = __ldg(table + warp + k * kAttnWarps);
        if (p < 0 || p >= P.c.n_pages) {
          set_status(P.status, AKV_ERR_SHAPE);
          p = 0;
        }
      }
      return p;
    };
    auto issue = [&](int p, uint32_t st) {
      if (lane == 0) {
        mbar_arrive_expect_tx(bars + st, S::REC);
        tma_load_1d(ring + st * S::REC, pool + p * P.c.page_stride, S::REC, bars + st);
      }
    };
    int ids = page_ids(0);
    // the query rows this warp prepares, on their way with the page numbers
    constexpr int PER = D / 32;
    constexpr int RW = S::ROWS / kAttnWarps;  // rows of a warp, all loads in flight at once
    uint16_t raw[RW][PER];
#pragma unroll
    for (int k2 = 0; k2 < RW; ++k2) {
      const int rr = tile * S::ROWS + tile_row<LO>(k2 * kAttnWarps + warp), m = rr / rep;
      const uint16_t* src = P.q + i * P.q_sr + (h * rep + rr % rep) * P.q_sh + m * P.q_sm + lane * PER;
#pragma unroll
      for (int k = 0; k < PER; ++k) raw[k2][k] = m < n_new ? src[k] : 0;
    }
#pragma unroll
    for (int k = 0; k < S::STAGES; ++k) {
      const int p = __shfl_sync(~0u, ids, k);
      if (k < mine && alive) issue(p, (stage + k) % S::STAGES);
    }

    // Queries of the tile: scaled to fp16, placed as MMA operands; sums per group.
    {
      uint16_t* frag = reinterpret_cast<uint16_t*>(smem + S::OFF_FRAG);
#pragma unroll
      for (int k2 = 0; k2 < RW; ++k2) {
        const int n = k2 * kAttnWarps + warp;
        const int nr = tile_row<LO>(n), m = (tile * S::ROWS + nr) / rep;
        float x[PER];
        uint32_t top = 0u;  // bits of the largest magnitude: infinity, then NaN, above all others
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          x[k] = P.bf16 ? elem_to_float<true>(raw[k2][k]) : elem_to_float<false>(raw[k2][k]);
          top = max(top, __float_as_uint(x[k]) & 0x7FFFFFFFu);
        }
        top = __reduce_max_sync(~0u, top);
        const bool bad = top >= 0x7F800000u;  // no softmax: computed as zeros, NaN at the end
        int ex = 0;  // 2^ex brings the largest into [2^9, 2^10)
        if (top && !bad) ex = 9 - (static_cast<int>(top >> 23) - 127);
        ex = ex > 120 ? 120 : (ex < -120 ? -120 : ex);
        const float up = exp2f(static_cast<float>(ex)) * (P.scale < 0.f ? -1.f : 1.f);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int c = lane * PER + k;
          const __half hv = __float2half_rn(bad ? 0.f : x[k] * up);
          sum += __half2float(hv);
          const int gi = c / S::GS, r = c % S::GS, col = r / (S::GS / 4), r2 = r % (S::GS / 4);
          int ks, reg, half;
          if constexpr (S::BK >= 4) {
            ks = gi * (S::GS / 16) + (r2 / 8) * 2 + ((r2 >> 1) & 1);
            half = (r2 >> 2) & 1;
          } else {
            ks = gi;
            half = r2 >> 1;
          }
          reg = c & 1 ? 0 : 1;
          frag[(((ks * NT + n / 8) * 32 + (n % 8) * 4 + col) * 2 + reg) * 2 + half] = __half_as_ushort(hv);
        }
        constexpr int GL = 32 / G;  // lanes of a group
#pragma unroll
        for (int o = 1; o < GL; o <<= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (lane % GL == 0) s_qs[lane / GL * S::ROWS + n] = sum * 9.5367431640625e-7f;  // 2^-20, the codes' unit
        if (lane == 0) {
          // log2 e * scale in units of the MMA result; never 0, so that -inf stays -inf
          s_cq[n] = fmaxf(ldexpf(fabsf(P.scale) * 1.4426950408889634f, 20 - ex), 1e-37f);
          const int see = len - n_new + (m < n_new ? m : n_new - 1) + 1;
          s_see[n] = see;
          s_on[n] = m < n_new ? (bad && see > 0 ? NAN : 1.f) : 0.f;
          if (m < P.M) {
            const int hq = h * rep + (tile * S::ROWS + nr) - m * rep;
            s_out[n] = out_row(P, i, hq, m);
            s_lse[n] = (i * P.Hq + hq) * P.M + m;
          }
        }
      }
    }
    __syncthreads();

    uint2 qf[NT == 1 ? KS : 1];
    const uint2* frag2 = reinterpret_cast<const uint2*>(smem + S::OFF_FRAG) + lane;
    if constexpr (NT == 1) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = frag2[ks * 32];
    }
    // Per pair of queries (columns 2 q4, 2 q4 + 1), as packed fp32 pairs: group
    // sums of q (in registers where they are few), exponent factors, minus the
    // exponent of the maximum (0 before any token), sums of weights and of
    // weights times zeros; and the score from which the maximum moves.
    constexpr bool QS_REG = NT * G <= 2;
    const uint64_t* s_qs2 = reinterpret_cast<const uint64_t*>(s_qs) + q4;
    uint64_t qs[QS_REG ? NT : 1][QS_REG ? G : 1], cq[NT], nm[NT], l[NT], zs[NT][S::AV ? 1 : G];
    float lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      cq[nt] = f2_make(s_cq[nt * 8 + q4 * 2], s_cq[nt * 8 + q4 * 2 + 1]);
      nm[nt] = l[nt] = 0;
      lim[nt][0] = lim[nt][1] = -INFINITY;
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        if constexpr (QS_REG) qs[nt][gi] = s_qs2[(gi * S::ROWS + nt * 8) / 2];
        if constexpr (!S::AV) zs[nt][gi] = 0;
      }
      if constexpr (S::AV) zs[nt][0] = 0;
    }
    const int see_min = s_see[0];
    float O[NT][D / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) O[nt][j][k] = 0.f;
    float vref = 0.f, vinv = 0.f;  // power of two above the V scales seen so far, its inverse

    for (int k = 0; k < mine; ++k) {
      if (!alive || !__all_sync(~0u, mbar_wait(bars + stage, phase, P.status))) {
        // a copy never came: take no more, but see the ones in flight land
        if (alive)
          for (int r = 1; r < S::STAGES && k + r < mine; ++r) {
            const uint32_t st = stage + r;
            mbar_wait(bars + st % S::STAGES, st >= S::STAGES ? phase ^ 1 : phase, P.status);
          }
        alive = false;
        break;
      }
      const uint8_t* rec = ring + stage * S::REC;
      const int tok0 = (page0 + warp + k * kAttnWarps) * kBlockTokens;

      // ---- scores: tokens are the MMA's rows, queries its columns; x holds the
      // pairs of a token row (mt, half) as (2 q4, 2 q4 + 1)
      uint64_t x[4][NT];
      uint32_t kp[4][G];
#pragma unroll
      for (int r = 0; r < 4; ++r) lds_pairs<G>(rec + int4_layout(D, G).kp + (r * 8 + tile_token(g)) * G * 4, kp[r]);
#pragma unroll
      for (int gi = 0; gi < G; ++gi) {
        uint32_t kw[4][S::BK < 4 ? 1 : S::BK / 4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          lds_bytes<S::BK>(rec + (r * 8 + tile_token(g)) * (D / 2) + gi * (S::GS / 2) + q4 * S::BK, kw[r]);
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
          for (int nt = 0; nt < NT; ++nt) b[nt] = NT == 1 ? qf[NT == 1 ? ks : 0] : frag2[(ks * NT + nt) * 32];
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            // codes of the step's two channel pairs, at bits 4..7 of each half
            uint32_t a[4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              uint32_t w;
              if constexpr (S::BK >= 4) w = s & 1 ? kw[2 * mt + r][s / 2] >> 8 : kw[2 * mt + r][s / 2];
              else w = prmt(kw[2 * mt + r][0], 0u, 0x4140);
              a[r] = (w * 16u) & 0x00F000F0u;  // a product: the shifts' pipe is the busy one
              a[2 + r] = w & 0x00F000F0u;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816(acc[mt][nt], a[0], a[1], a[2], a[3], b[nt].x, b[nt].y);
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 sz = __half22float2(u32_as_h2(kp[r][gi]));
          const uint64_t s2 = f2_make(sz.x, sz.x), z2 = f2_make(sz.y, sz.y);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint64_t q2 = QS_REG ? qs[QS_REG ? nt : 0][QS_REG ? gi : 0] : s_qs2[(gi * S::ROWS + nt * 8) / 2];
            const float* a = acc[r >> 1][nt] + (r & 1) * 2;
            const uint64_t zq = gi == 0 ? f2_mul(z2, q2) : f2_fma(z2, q2, x[r][nt]);
            x[r][nt] = f2_fma(f2_make(a[0], a[1]), s2, zq);
          }
        }
      }
      const bool tail = tok0 + kBlockTokens > see_min;
      if (tail) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int see0 = s_see[nt * 8 + q4 * 2] - tok0, see1 = s_see[nt * 8 + q4 * 2 + 1] - tok0;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float2 v = f2_split(x[r][nt]);
            if (r * 8 + tile_token(g) >= see0) v.x = -INFINITY;
            if (r * 8 + tile_token(g) >= see1) v.y = -INFINITY;
            x[r][nt] = f2_make(v.x, v.y);
          }
        }
      }
      // ---- V scales and zeros of this thread's tokens (slots past the row's end
      // hold anything: nothing of them may reach a sum)
      uint32_t vp[4][G];
      if constexpr (!S::AV) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lds_pairs<G>(rec + int4_layout(D, G).vp + (r * 8 + tile_token(g)) * G * 4, vp[r]);
#pragma unroll
          for (int gi = 0; gi < G; ++gi)
            if (tail && tok0 + r * 8 + tile_token(g) >= len) vp[r][gi] = 0u;
        }
      }
      // ---- running maximum and V unit move together, rarely
      bool move = false;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float2 v = f2_split(x[r][nt]);
          top[nt][0] = fmaxf(top[nt][0], v.x);
          top[nt][1] = fmaxf(top[nt][1], v.y);
        }
        move |= top[nt][0] > lim[nt][0];
        move |= top[nt][1] > lim[nt][1];
      }
      float vtop = 0.f;
      if constexpr (!S::AV) {
        __half2 vtop2 = u32_as_h2(0u);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int gi = 0; gi < G; ++gi) vtop2 = __hmax2(vtop2, __habs2(u32_as_h2(vp[r][gi])));
        vtop = __low2float(vtop2);
        move |= vtop > vref;
      }
      if (__any_sync(~0u, move)) {
        float fv = 1.f;
        if constexpr (!S::AV) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) vtop = fmaxf(vtop, __shfl_xor_sync(~0u, vtop, o));
          if (vtop > vref) {
            // the power of two above vtop (scales are finite fp16 values)
            const float ref = __uint_as_float((__float_as_uint(vtop) & 0x7F800000u) + 0x00800000u);
            fv = vref > 0.f ? vref / ref : 1.f;
            vref = ref;
            vinv = 1.f / ref;
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 c2 = f2_split(cq[nt]);
          float2 n2 = f2_split(nm[nt]);
          float f[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float m = top[nt][c];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
            const float cqc = c ? c2.y : c2.x, old = -(c ? n2.y : n2.x);
            const bool any = lim[nt][c] != -INFINITY;
            float y = m == -INFINITY ? 0.f : fmaf(m, cqc, -kTopLog2);
            if (any) y = fmaxf(y, old);
            f[c] = any ? exp2f(old - y) : 0.f;
            if (any || m != -INFINITY) lim[nt][c] = (y + kMostLog2) / cqc;
            (c ? n2.y : n2.x) = -y;
          }
          nm[nt] = f2_make(n2.x, n2.y);
          const uint64_t f2 = f2_make(f[0], f[1]);
          l[nt] = f2_mul(l[nt], f2);
#pragma unroll
          for (int gi = 0; gi < S::GV; ++gi) zs[nt][gi] = f2_mul(zs[nt][gi], f2);
#pragma unroll
          for (int j = 0; j < D / 16; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) O[nt][j][c] *= f[c & 1] * fv;
        }
      }
      // ---- weights
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 v = f2_split(f2_fma(x[r][nt], cq[nt], nm[nt]));
          x[r][nt] = f2_make(fast_exp2(v.x), fast_exp2(v.y));
          l[nt] = f2_add(l[nt], x[r][nt]);
        }
        if constexpr (!S::AV) {
#pragma unroll
          for (int gi = 0; gi < G; ++gi) {
            const float2 sz = __half22float2(u32_as_h2(vp[r][gi]));
            const float mid = fmaf(static_cast<float>(code_centre(r / 2)), sz.x, sz.y);
            const uint64_t z2 = f2_make(mid, mid);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) zs[nt][gi] = f2_fma(x[r][nt], z2, zs[nt][gi]);
          }
        }
      }
      // ---- values: channels are the MMA's rows, tokens its depth
#pragma unroll
      for (int gi = 0; gi < S::GV; ++gi) {
        uint32_t pb[4][NT], pl[LO == 1 ? 4 : 1][LO == 1 ? NT : 1];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint64_t sn2 = 0;
          if constexpr (!S::AV) {
            const float sn = __low2float(u32_as_h2(vp[r][gi])) * vinv;
            sn2 = f2_make(sn, sn);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float2 w = f2_split(S::AV ? x[r][nt] : f2_mul(x[r][nt], sn2));
            uint32_t hi = pack_h2(w.x, w.y);
            if constexpr (LO) {
              const float2 back = __half22float2(u32_as_h2(hi));
              const uint32_t lo = pack_h2(w.x - back.x, w.y - back.y);
              if constexpr (LO == 1) pl[r][nt] = movmatrix_trans(lo);
              else hi = q4 < 2 ? hi : lo;
            }
            pb[r][nt] = movmatrix_trans(hi);
          }
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          constexpr int NW = S::BV < 4 ? 1 : S::BV / 4;
          const int mid = S::AV ? 8 : code_centre(kk);
          uint32_t va[2][NW], vb[2][NW];  // the two tokens of each 8-token tile
          uint32_t vs2[2], vz2[2];        // AV: their scales, zeros + 8 scales
          uint32_t far = 0u;              // AV: the furthest that a code may lie from 0
#pragma unroll
          for (int T = 0; T < 2; ++T) {
            const int t0 = (2 * kk + T) * 8 + tile_token(2 * q4), t1 = (2 * kk + T) * 8 + tile_token(2 * q4 + 1);
            const uint8_t* vr = rec + int4_layout(D, G).vc + gi * (S::GS / 2) + g * S::BV;
            lds_bytes<S::BV>(vr + t0 * (D / 2), va[T]);
            lds_bytes<S::BV>(vr + t1 * (D / 2), vb[T]);
            if constexpr (S::AV) {
              const uint8_t* pr = rec + int4_layout(D, G).vp + g * (D / 8) / S::GS * 4;
              uint32_t w0 = lds_u32(pr + t0 * G * 4), w1 = lds_u32(pr + t1 * G * 4);
              if (tail) {
                if (tok0 + t0 >= len) w0 = 0u;
                if (tok0 + t1 >= len) w1 = 0u;
              }
              vs2[T] = prmt(w0, w1, 0x5410);
              vz2[T] = h2_as_u32(__hfma2(u32_as_h2(vs2[T]), u32_as_h2(0x48004800u), u32_as_h2(prmt(w0, w1, 0x7632))));
              const __half2 reach = __hfma2(u32_as_h2(vs2[T]), u32_as_h2(0x48004800u), __habs2(u32_as_h2(vz2[T])));
              far = h2_as_u32(__hmax2(u32_as_h2(far), reach));
            }
          }
          auto products = [&](auto held) {
            auto value = [&](uint32_t c, int T) -> uint32_t {
              if constexpr (!S::AV) return c;
              __half2 v = __hfma2(u32_as_h2(c), u32_as_h2(vs2[T]), u32_as_h2(vz2[T]));
              if constexpr (decltype(held)::value) v = __hmax2(__hmin2(v, u32_as_h2(0x7BFF7BFFu)), u32_as_h2(0xFBFFFBFFu));
              return h2_as_u32(v);
            };
            // two channels' bytes at a time: the two terms of a sum stand apart
#pragma unroll
            for (int b0 = 0; b0 < S::BV; b0 += 2) {
              constexpr int BB = S::BV < 2 ? 1 : 2;
              uint32_t a[BB][4];
#pragma unroll
              for (int b2 = 0; b2 < BB; ++b2) {
                const int b = b0 + b2;
                // bytes b of both tokens, the first in the low half
                const uint32_t y0 = prmt(va[0][b / 4], vb[0][b / 4], (b & 2) ? 0x7632 : 0x5410) >> (8 * (b & 1));
                const uint32_t y1 = prmt(va[1][b / 4], vb[1][b / 4], (b & 2) ? 0x7632 : 0x5410) >> (8 * (b & 1));
                a[b2][0] = value(low_code(y0, mid), 0), a[b2][1] = value(high_code(y0, mid), 0);
                a[b2][2] = value(low_code(y1, mid), 1), a[b2][3] = value(high_code(y1, mid), 1);
              }
#pragma unroll
              for (int term = 0; term < (LO == 1 ? 2 : 1); ++term)
#pragma unroll
                for (int b2 = 0; b2 < BB; ++b2)
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma_16816(O[nt][gi * S::BV + b0 + b2], a[b2][0], a[b2][1], a[b2][2], a[b2][3],
                              term ? pl[LO == 1 ? 2 * kk : 0][LO == 1 ? nt : 0] : pb[2 * kk][nt],
                              term ? pl[LO == 1 ? 2 * kk + 1 : 0][LO == 1 ? nt : 0] : pb[2 * kk + 1][nt]);
            }
          };
          // Codes 0 and 15 of a group that append held to +-65504 can round to
          // infinity, and a token that a query does not see has weight 0 times
          // that.  Where the sum 8 s + |z + 8 s| is infinite (no code's value is
          // otherwise) the warp takes the values with a clamp.
          if constexpr (S::AV) {
            if (__any_sync(~0u, max(far & 0x7FFFu, far >> 16) >= 0x7C00u)) products(std::true_type{});
            else products(std::false_type{});
          } else {
            products(std::false_type{});
          }
        }
      }
      // ---- the stage is free: the page STAGES ahead
      __syncwarp();
      const int next = k + S::STAGES;
      if (next < mine) {
        if ((next & 31) == 0) ids = page_ids(next);
        const int p = __shfl_sync(~0u, ids, next & 31);
        issue(p, stage);
      }
      if (++stage == S::STAGES) stage = 0, phase ^= 1;
    }

    // ---- the warps' results meet
    float2 zf[NT][S::GV];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float2 lf = f2_split(l[nt]), nf = f2_split(nm[nt]);
#pragma unroll
      for (int gi = 0; gi < S::GV; ++gi) zf[nt][gi] = f2_split(zs[nt][gi]);
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        lf.x += __shfl_xor_sync(~0u, lf.x, o);
        lf.y += __shfl_xor_sync(~0u, lf.y, o);
        if constexpr (!S::AV) {
#pragma unroll
          for (int gi = 0; gi < G; ++gi) {
            zf[nt][gi].x += __shfl_xor_sync(~0u, zf[nt][gi].x, o);
            zf[nt][gi].y += __shfl_xor_sync(~0u, zf[nt][gi].y, o);
          }
        }
      }
      if (g == 0) {
        float2* ml = s_ml + warp * S::ROWS + nt * 8 + q4 * 2;
        ml[0] = make_float2(lim[nt][0] == -INFINITY ? -INFINITY : -nf.x, lf.x);
        ml[1] = make_float2(lim[nt][1] == -INFINITY ? -INFINITY : -nf.y, lf.y);
      }
    }
    __syncthreads();  // every warp is done with its ring
    if (t < S::ROWS) {  // maximum and sum of a row over the warps
      float top = -INFINITY, L = 0.f;
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, s_ml[w * S::ROWS + t].x);
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float2 a = s_ml[w * S::ROWS + t];
        if (a.x != -INFINITY) L = fmaf(a.y, exp2f(a.x - top), L);
      }
      if (s_on[t] != 1.f) L = s_on[t];
      s_tl[t] = whole ? row_scale(top, L) : make_float2(top, L);
    }
    float* merge = reinterpret_cast<float*>(smem);
    float f[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float2 nf = f2_split(nm[nt]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int n = nt * 8 + q4 * 2 + c;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) m = fmaxf(m, s_ml[w * S::ROWS + n].x);
        f[nt][c] = lim[nt][c] == -INFINITY ? 0.f : exp2f(-(c ? nf.y : nf.x) - m);
      }
    }
    // each warp's share, scaled to the common maximum; within a row the
    // channels stand in the accumulators' order, 16 (j, g, parity) at a time
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int gi = 0; gi < S::GV; ++gi)
#pragma unroll
        for (int b = 0; b < S::BV; ++b) {
          const int j = gi * S::BV + b;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float2 v;  // even channel (high nibble), odd channel
            const float z = S::AV || (LO == 2 && q4 >= 2) ? 0.f : (c ? zf[nt][gi].y : zf[nt][gi].x), unit = S::AV ? 1.f : vref;
            v.x = f[nt][c] * fmaf(O[nt][j][2 + c], unit, z);
            v.y = f[nt][c] * fmaf(O[nt][j][c], unit, z);
            *reinterpret_cast<float2*>(merge + (warp * S::ROWS + nt * 8 + q4 * 2 + c) * S::PITCH + j * 16 + g * 2) = v;
          }
        }
    __syncthreads();
    const int valid = min(S::ROWS, P.M * rep - tile * S::ROWS);  // query rows of this tile
    constexpr int64_t STEP = static_cast<int64_t>(S::ROWS) * (D + 2);
    float* part = P.part + (static_cast<int64_t>(blockIdx.x) + unit) * STEP;
#pragma unroll 2
    for (int k = t; k < valid * (D / 2); k += kAttnThreads) {
      const int n = k / (D / 2), p = k % (D / 2);
      float2 v = make_float2(0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float2 o = *reinterpret_cast<const float2*>(merge + (w * S::ROWS + n) * S::PITCH + 2 * p);
        v.x += o.x, v.y += o.y;
        if constexpr (LO == 2) {
          const float2 o2 = *reinterpret_cast<const float2*>(merge + (w * S::ROWS + n + 4) * S::PITCH + 2 * p);
          v.x += o2.x, v.y += o2.y;
        }
      }
      const float2 tl = s_tl[n];
      if (whole) {
        store_pair<D, S::GV>(P, s_out[n], P.lse ? P.lse + s_lse[n] : nullptr, p, v, tl);
      } else {
        *reinterpret_cast<float2*>(part + n * (D + 2) + 2 * p) = v;
        if (p == 0) *reinterpret_cast<float2*>(part + n * (D + 2) + D) = tl;
      }
    }
    if (whole) {
      if (t == 0 && P.meta) P.meta[unit] = make_int2(0, 0);
    } else {
      const int cta0 = u_start / share, cta1 = (u_start + pages - 1) / share;
      if (P.meta) {
        if (t == 0 && page0 == 0) P.meta[unit] = make_int2(cta0, cta1);
      } else {
        // the last of the unit's CTAs to arrive merges their parts
        __threadfence();
        __syncthreads();
        if (t == 0) {
          const unsigned segs = cta1 - cta0 + 1;
          s_last = atomicInc(P.arrived + unit, segs - 1) == segs - 1;  // wraps to 0 for the next call
        }
        __syncthreads();
        if (s_last) {
          __threadfence();
          merge_parts<D, S::GV, NT>(P, P.part + (static_cast<int64_t>(cta0) + unit) * STEP, cta1 - cta0 + 1, s_out, s_lse, valid,
                                reinterpret_cast<float*>(smem));
        }
      }
    }
    // the merge buffer goes back to the copies
    fence_proxy_async_shared();
    __syncthreads();
    pos += n_pages + extra;
    if (pos - e_start >= weight * H) ++e;
  }
}

// Partial results of the units that several CTAs shared, one query row per CTA.
template <int D, int G, int NT>
__global__ void __launch_bounds__(128) int4_combine_kernel(const Int4AttnParams P) {
  constexpr int ROWS = 8 * NT;
  constexpr int64_t STEP = static_cast<int64_t>(ROWS) * (D + 2);
  __shared__ float s_w[128], s_red[8];
  __shared__ float2 s_acc[128];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int unit = blockIdx.x, n = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int2 cta = P.meta[unit];
  const int segs = cta.y - cta.x + 1;
  if (segs <= 1) return;
  const int H = P.c.kv_heads, rep = P.Hq / H;
  const int e = unit / H, h = unit % H, i = P.row0 + e / P.tiles;
  const int rr = e % P.tiles * ROWS + n;
  if (rr / rep >= P.M) return;
  const float* part = P.part + (static_cast<int64_t>(cta.x) + unit) * STEP + n * (D + 2);
  float top = -INFINITY;
  for (int s = t; s < segs; s += 128) top = fmaxf(top, part[s * STEP + D]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if (lane == 0) s_red[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
  // channel pairs across, the rest of the threads take every other part
  constexpr int PAIRS = D / 2, WAYS = 128 / PAIRS;
  const int p = t % PAIRS, way = t / PAIRS;
  float L = 0.f;
  float2 acc = make_float2(0.f, 0.f);
  for (int s0 = 0; s0 < segs; s0 += 128) {
    __syncthreads();
    if (s0 + t < segs) {
      const float2 yl = *reinterpret_cast<const float2*>(part + (s0 + t) * STEP + D);
      const float w = yl.x == -INFINITY ? 0.f : exp2f(yl.x - top);
      s_w[t] = w;
      L += w * yl.y;
    }
    __syncthreads();
    const int cnt = segs - s0 < 128 ? segs - s0 : 128;
#pragma unroll 8
    for (int s = way; s < cnt; s += WAYS) {
      const float2 v = *reinterpret_cast<const float2*>(part + (s0 + s) * STEP + 2 * p);
      acc.x = fmaf(s_w[s], v.x, acc.x);
      acc.y = fmaf(s_w[s], v.y, acc.y);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) L += __shfl_xor_sync(~0u, L, o);
  if (lane == 0) s_red[4 + warp] = L;
  if (way) s_acc[(way - 1) * PAIRS + p] = acc;
  __syncthreads();
  if (way) return;
  L = s_red[4] + s_red[5] + s_red[6] + s_red[7];
#pragma unroll
  for (int w = 1; w < WAYS; ++w) {
    acc.x += s_acc[(w - 1) * PAIRS + p].x;
    acc.y += s_acc[(w - 1) * PAIRS + p].y;
  }
  const int m = rr / rep, hq = h * rep + rr % rep;
  store_pair<D, G>(P, out_row(P, i, hq, m), P.lse ? P.lse + (i * P.Hq + hq) * P.M + m : nullptr, p, acc,
                   row_scale(top, L));
}

// ---------------------------------------------------------------- host
constexpr int kSMs = 148;

// column tiles of 8 query rows for `rows` rows of a (sequence, KV head)
inline int attn_nt(int rows) {
  return rows <= 8 ? 1 : 2;
}

template <int D, int G, int NT, int LO>
int attn_launch(const Int4AttnParams& p, cudaStream_t st) {
  using S = AttnShape<D, G, NT, LO>;
  const int entries = p.R * p.tiles;
  const int smem = S::smem(entries);
  if (!ensure_dynamic_smem<int4_attn_kernel<D, G, NT, LO>>(S::smem(kAttnEntries))) return AKV_ERR_LAUNCH;
  const int grid = kSMs * S::OCC;
  int4_attn_kernel<D, G, NT, LO><<<grid, kAttnThreads, smem, st>>>(p);
  if (cudaGetLastError() != cudaSuccess) return AKV_ERR_LAUNCH;
  if (!p.meta) return AKV_OK;
  cudaLaunchConfig_t cfg{};
  const int q_rows = p.M * (p.Hq / p.c.kv_heads);
  cfg.gridDim = dim3(entries * p.c.kv_heads, q_rows < S::ROWS ? q_rows : S::ROWS);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, int4_combine_kernel<D, S::GV, NT>, p) == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}

template <int D, int G, int NT>
int attn_dispatch_lo(const Int4AttnParams& p, cudaStream_t st) {
  if (p.bf16) return attn_launch<D, G, NT, 0>(p, st);
  if constexpr (NT == 1)
    if (p.M * (p.Hq / p.c.kv_heads) <= 4) return attn_launch<D, G, NT, 2>(p, st);
  return attn_launch<D, G, NT, 1>(p, st);
}

template <int D, int G>
int attn_dispatch_nt(const Int4AttnParams& p, int nt, cudaStream_t st) {
  return nt == 1 ? attn_dispatch_lo<D, G, 1>(p, st) : attn_dispatch_lo<D, G, 2>(p, st);
}

template <int D>
int attn_dispatch(const Int4AttnParams& p, int nt, cudaStream_t st) {
  const int G = D / p.c.group;
  if (G == 1) return attn_dispatch_nt<D, 1>(p, nt, st);
  if (G == 2) return attn_dispatch_nt<D, 2>(p, nt, st);
  return attn_dispatch_nt<D, 4>(p, nt, st);
}

int int4_attn_64(const Int4AttnParams& p, int nt, cudaStream_t st);
int int4_attn_128(const Int4AttnParams& p, int nt, cudaStream_t st);
int int4_attn_256(const Int4AttnParams& p, int nt, cudaStream_t st);

}  // namespace akv
