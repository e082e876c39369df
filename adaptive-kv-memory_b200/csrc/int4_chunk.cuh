// Attention of a chunk of new tokens over the 4-bit paged cache, on the fifth-
// generation tensor cores (kernel templates; one translation unit per head dim
// instantiates them).
//
//   S = Q K^T   softmax over the tokens a query sees   O = P V
// with K, V values c*s + z unpacked from the pages, a tile of TK tokens at a
// time, into shared memory, where all query heads of the KV head read them.
//
// Work.  A unit is one (call row, KV head, tile of NQ x 128 query rows), a row
// being one (token, query head of the group), tokens outer.  The units' token
// tiles form one list that is cut into equal shares, one per CTA (one CTA an
// SM), from the lengths on the device; a unit's set-up counts kChunkSetup tiles
// more.  A unit cut in two or more leaves unnormalised parts that a second
// kernel joins in order.
//
// Roles of a CTA's warps, which meet at mbarriers only:
//   softmax  one warpgroup per 128 query rows, thread = row = TMEM lane: query
//            rows into shared memory, online softmax, P into tensor memory over
//            S, O out
//   pages    one warp: a tile's records as they are, by bulk copies
//   values   two warpgroups: K and V of the tile out of them, into their rings
//   MMA      a warp per 128 query rows: S = Q K^T from shared memory, O += P V with P from
//            tensor memory
// While one tile's softmax runs, the other's MMAs do.
//
// Roundings.  Queries are scaled per row by a power of two into fp16's middle
// range (bf16; exact unless 2^-24 of the row's largest) or taken as they are
// (fp16).  For a bf16 output K, V and the weights enter the MMAs as one fp16
// term each, every one an eighth of the output's own rounding.  For an fp16
// output (LO) K and the weights are two terms, the second the first's error,
// and V one: its rounding and the output's are alike.  The accumulators, the
// maximum (its weight stands at 2^9, so that small weights keep their bits) and
// the sums are fp32.
//
// Shared-memory operands have the 128-byte swizzle: 64 channels of a row in 128
// bytes, rows 128 B apart, the 16-byte pieces of row r permuted by r % 8 (XOR),
// the next 64 channels of all rows behind.  So a value thread's stores (its row,
// piece after piece) meet no bank twice, and one layout serves as the K-major
// operand (Q, K) and the MN-major one (V: tokens = K, channels = N).
// Within a block of 8 channels they stand as the codes come out of a word,
// 0 4 1 5 2 6 3 7, in Q and K alike; V's order is undone when O is stored.
#pragma once

#include <type_traits>

#include "int4.cuh"
#include "umma.cuh"

namespace akv {

constexpr int kChunkSMs = 148;      // CTAs: one an SM
constexpr int kChunkEntries = 1536; // (row, tile) pairs of one launch
constexpr int kChunkRowsMax = 384;  // call rows of one launch
constexpr int kChunkRep = 4096;     // query heads of a group, at most (the division below)
constexpr int kChunkSetup = 2;      // token tiles that a unit's set-up counts for
// When a row's unit is set its maximum stands at 2^9, and a thread's weights of a
// tile sum up to 2^15 at most before it moves, so that fp16 holds them down to
// 2^-23 of the maximum with all their bits.  The sum says so without the tile's
// maximum, which is formed only where a unit moves.
constexpr float kChunkTop = 9.f, kChunkMost = 32768.f;

// Pairs of weights, of four, whose exponentials run on the FMA pipes where the
// special-function units bound the softmax (bf16, two query tiles).
constexpr int kChunkPoly = 0;

struct ChunkParams {
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
  int q16, o16;   // query, output rows on 16-byte boundaries
  uint32_t rep_inv;  // 2^32 / (query heads of a group), rounded up; 0 for one head
  int4* meta;     // per CTA: (entry, head, last CTA, 1) of the unit whose first part it holds
  float* part;    // [2 * CTA + (first part ? 1 : 0)][D / 4][rows][4]
  float2* ml;     // [slot][rows]: log2 of the maximum's unit, sum
  int* status;
};

template <int D, int G, int LO>
struct ChunkShape {
  static constexpr int NQ = D == 256 ? 1 : 2;
  static constexpr int TK = 64;                     // tokens of a tile
  static constexpr int ROWS = 128 * NQ;
  static constexpr int QB = 128 * D * 2;            // a query tile
  static constexpr int VB = TK * D * 2;             // a tile of V
  static constexpr int KB = VB * (LO ? 2 : 1);      // of K: one or two terms
  static constexpr int KS = D == 256 ? 1 : (LO ? 2 : 3);          // ring slots
  static constexpr int VS = D == 256 ? (LO ? 1 : 2) : (LO ? 2 : 3);
  static constexpr int RS = D == 256 ? (LO ? 3 : 2) : 4;          // of the raw tiles
  static constexpr int SOFT = 4 * NQ;               // softmax warps
  static constexpr int THREADS = SOFT * 32 + 256 + 128;
  // registers of a softmax / value / other thread: 640 threads are launched with 96 each
  static constexpr bool SPLIT = THREADS == 640;
  static constexpr int R_SOFT = 136, R_VAL = 72, R_MMA = 64;
  static_assert(2 * R_SOFT + 2 * R_VAL + R_MMA == 5 * 96, "register shares");
  static constexpr int PARTS = 128 / TK;            // value threads of a token
  static constexpr int CH = D / PARTS;              // channels of a value thread
  static constexpr int PIECES = CH / 32;            // its 16-byte pieces of codes
  static constexpr int PAGES = TK / kBlockTokens;
  // a tile's codes and pairs as they stand in the pages, K or V
  static constexpr int RAW_CODES = TK * D / 2, RAW = RAW_CODES + TK * G * 4;
  // pairs of weights, of four, whose exponentials run on the FMA pipes
  static constexpr int POLY = NQ == 2 && !LO ? kChunkPoly : 0;
  static constexpr int OFF_K = NQ * QB;
  static constexpr int OFF_V = OFF_K + KS * KB;
  static constexpr int OFF_RAW = OFF_V + VS * VB;   // K's slots, then V's
  static constexpr int OFF_EX = OFF_RAW + 2 * RS * RAW;    // per row: exponent, or a mark for a query that is not finite
  static constexpr int OFF_BAR = OFF_EX + ROWS * 4;
  static constexpr int OFF_ROWS = OFF_BAR + 352;    // lengths, new tokens, prefix sums
  static constexpr int smem(int rows, int entries) { return 1024 + OFF_ROWS + (2 * rows + entries + 1) * 4; }
  // tensor memory: two tiles of S (and P) of each query tile, then O
  static constexpr int T_S = 0, T_O = NQ * 2 * TK;
  static_assert(NQ * (2 * TK + D) <= 512, "tensor memory");
  static_assert(smem(kChunkRowsMax, kChunkEntries) <= 227 * 1024, "shared memory");
};

// The part of a unit that a CTA takes: tiles [t0, t1) of `tiles`.
struct ChunkPart {
  int e, h, i, len, n_new, row;  // row: first query row of the tile
  int t0, t1, tiles, unit_end;   // unit_end: where the unit ends in the list
};

// What the walk over the CTA's share needs, in shared memory: a role keeps its
// position only.
struct ChunkList {
  const int *len, *n_new, *pref;  // per call row; per entry
  int share, end;
};
struct ChunkPos {
  int pos, e, h;   // the entry and head that pos stands in
  int r, tile;     // the entry's call row and its tile
};

// query row rr of a (row, head): its token, exact for rr * heads < 2^32
AKV_DEV int chunk_token(const ChunkParams& P, int rr) {
  return P.rep_inv ? static_cast<int>(__umulhi(static_cast<uint32_t>(rr), P.rep_inv)) : rr;
}

template <int TK, int ROWS>
AKV_DEV int chunk_tiles(int len, int n_new, int rep, int tile) {
  const int first = tile * ROWS / rep;  // its first query token
  const int last = min((tile * ROWS + ROWS - 1) / rep, n_new - 1);
  const int see = len - n_new + last + 1;
  return first <= last && see > 0 ? (see + TK - 1) / TK : 0;
}

// where the list's position pos stands
AKV_DEV ChunkPos chunk_at(const ChunkParams& P, const ChunkList& L, int pos) {
  const int H = P.c.kv_heads, entries = P.R * P.tiles;
  int lo = 0, hi = entries;  // the last entry that starts at or before pos
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (L.pref[mid] * H <= pos) lo = mid; else hi = mid;
  }
  const int weight = L.pref[lo + 1] - L.pref[lo];
  return ChunkPos{pos, lo, weight ? (pos - L.pref[lo] * H) / weight : 0, lo / P.tiles, lo % P.tiles};
}

// The part at w, which moves past it; false at the share's end.
template <int ROWS>
AKV_DEV bool chunk_next(const ChunkParams& P, const ChunkList& L, ChunkPos& w, ChunkPart& u) {
  const int H = P.c.kv_heads;
  while (w.pos < L.end) {
    const int first = L.pref[w.e], weight = L.pref[w.e + 1] - first;
    if (weight == 0 || w.h == H) {
      w.h = 0;
      ++w.e;
      if (++w.tile == P.tiles) w.tile = 0, ++w.r;
      continue;
    }
    const int unit = first * H + w.h * weight, off = w.pos - unit, stop = min(unit + weight, L.end);
    u.h = w.h;
    u.e = w.e;
    u.i = P.row0 + w.r;
    u.len = L.len[w.r];
    u.n_new = L.n_new[w.r];
    u.row = w.tile * ROWS;
    u.tiles = weight - kChunkSetup;
    u.t0 = max(0, off - kChunkSetup);
    u.t1 = stop - unit - kChunkSetup;
    u.unit_end = unit + weight;
    w.pos = stop;
    if (stop == u.unit_end) ++w.h;
    if (u.t1 > u.t0) return true;
  }
  return false;
}

// ------------------------------------------------------------------ values
// c = the codes of a word, as fp16 pairs of channels (0, 4) (1, 5) (2, 6) (3, 7)
AKV_DEV void codes_of_word(uint32_t w, __half2 (&c)[4]) {
  const uint32_t v = w >> 8;
  const __half2 back = u32_as_h2(0xE400E400u), back16 = u32_as_h2(0xD400D400u), sixteenth = u32_as_h2(0x2C002C00u);
  c[0] = __hfma2(u32_as_h2(lop_magic<0x00F000F0u>(w)), sixteenth, back16);
  c[1] = __hadd2(u32_as_h2(lop_magic<0x000F000Fu>(w)), back);
  c[2] = __hfma2(u32_as_h2(lop_magic<0x00F000F0u>(v)), sixteenth, back16);
  c[3] = __hadd2(u32_as_h2(lop_magic<0x000F000Fu>(v)), back);
}

AKV_DEV __half2 hold(__half2 x) {  // past fp16's range: its ends
  const __half2 top = u32_as_h2(0x7BFF7BFFu);
  return __hmax2(__hmin2(x, top), __hneg2(top));
}

// 32 channels (a 16-byte piece of codes) of one or two terms: c*s + z rounded to
// fp16, or (TWO) a coarser first term and what it leaves.  dst: the row's 64
// channels; blk, x: the piece's first block of 8 and the row's permutation, both
// times 16; second: from the first term to the second.
//
// Two terms: with 2^E above the group's magnitudes, M = 1.5 * 2^(E + 1) and z =
// z1 + z2, z1 = (z + M) - M, both exact, the first term hi = fma(c, s, z1 + M) - M
// is a multiple of 2^(E - 9), as z1 is, so that z1 - hi is exact, and the second
// is fma(c, s, z1 - hi) + z2: together 2^(E - 20) or better.  Groups that reach
// 2^13 (FAR) take the exact difference in halves instead.
template <bool TWO, bool FAR, int W0, int W1>
AKV_DEV void store_words(uint4 code, uint32_t sz, unsigned char* dst, int blk, int x, int second) {
  const uint32_t w[4] = {code.x, code.y, code.z, code.w};
  const __half2 s = u32_as_h2(prmt(sz, sz, 0x1010)), z = u32_as_h2(prmt(sz, sz, 0x3232));
  __half2 big = z, z1 = z, z1m = z, z2 = z, sh = s, zh = z;
  if constexpr (TWO && !FAR) {
    const float2 f = __half22float2(u32_as_h2(sz));
    const float most = fmaxf(fabsf(f.y), fabsf(fmaf(15.f, f.x, f.y)));
    // 2^(E + 1) with 2^(E - 1) <= most < 2^E, 2^-13 at least
    const int e = max((static_cast<int>(__float_as_uint(most)) >> 23) - 127 + 2, -13);
    big = __float2half2_rn(__int_as_float((127 + e) << 23) * 1.5f);
    z1m = __hadd2(z, big);
    z1 = __hsub2(z1m, big);
    z2 = __hsub2(z, z1);
  }
  if constexpr (TWO && FAR) {
    const __half2 half = u32_as_h2(0x38003800u);
    sh = __hmul2(s, half), zh = __hmul2(z, half);
  }
#pragma unroll
  for (int i = W0; i < W1; ++i) {
    __half2 c[4], v[4], r[4];
    codes_of_word(w[i], c);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (!TWO) {
        v[k] = __hfma2(c[k], s, z);
        if constexpr (FAR) v[k] = hold(v[k]);
      } else if constexpr (!FAR) {
        v[k] = __hsub2(__hfma2(c[k], s, z1m), big);
        r[k] = __hadd2(__hfma2(c[k], s, __hsub2(z1, v[k])), z2);
      } else {
        // z - v = d + e exactly, both halved; c*s + d is what v left out, but for e
        v[k] = hold(__hfma2(c[k], s, z));
        const __half2 vh = __hmul2_rn(v[k], u32_as_h2(0x38003800u)), d = __hsub2(zh, vh), b = __hsub2(d, zh);
        const __half2 e = __hsub2(__hsub2(zh, __hsub2(d, b)), __hadd2(vh, b));
        const __half2 h = __hadd2(__hfma2(c[k], sh, d), e);
        r[k] = __hadd2(h, h);
      }
    }
    unsigned char* at = dst + ((blk + 16 * i) ^ x);
    *reinterpret_cast<uint4*>(at) = make_uint4(h2_as_u32(v[0]), h2_as_u32(v[1]), h2_as_u32(v[2]), h2_as_u32(v[3]));
    if constexpr (TWO)
      *reinterpret_cast<uint4*>(at + second) =
          make_uint4(h2_as_u32(r[0]), h2_as_u32(r[1]), h2_as_u32(r[2]), h2_as_u32(r[3]));
  }
}

template <bool TWO, bool FAR>
AKV_DEV void store_piece(uint4 code, uint32_t sz, unsigned char* dst, int blk, int x, int second) {
  store_words<TWO, FAR, 0, 4>(code, sz, dst, blk, x, second);
}
// the same with a pair for each 16 channels
template <bool TWO, bool FAR>
AKV_DEV void store_halves(uint4 code, uint32_t s0, uint32_t s1, unsigned char* dst, int blk, int x, int second) {
  store_words<TWO, FAR, 0, 2>(code, s0, dst, blk, x, second);
  store_words<TWO, FAR, 2, 4>(code, s1, dst, blk, x, second);
}

// whether a value of the group reaches `most` in magnitude
AKV_DEV bool far_values(uint32_t pair, float most) {
  const float2 sz = __half22float2(u32_as_h2(pair));
  return !(fmaxf(fabsf(sz.y), fabsf(fmaf(15.f, sz.x, sz.y))) < most);
}

// 2^y of two values, y held to -126 and more, by a Chebyshev fit of degree 4 of
// 2^f on [-1/2, 1/2] (2.7e-6 of the value) and its exponent added to the bits.
AKV_DEV uint64_t exp2_fma(uint64_t y2) {
  const float2 y = f2_split(y2);
  const uint64_t v = f2_make(fmaxf(y.x, -126.f), fmaxf(y.y, -126.f));
  const uint64_t t = f2_add(v, f2_make(12582912.f, 12582912.f));  // 1.5 * 2^23: the whole part in the low bits
  const uint64_t f = f2_add(v, f2_fma(t, f2_make(-1.f, -1.f), f2_make(12582912.f, 12582912.f)));
  uint64_t p = f2_make(0.009570102207362652f, 0.009570102207362652f);
  p = f2_fma(p, f, f2_make(0.05591785907745361f, 0.05591785907745361f));
  p = f2_fma(p, f, f2_make(0.240247443318367f, 0.240247443318367f));
  p = f2_fma(p, f, f2_make(0.6931217908859253f, 0.6931217908859253f));
  p = f2_fma(p, f, f2_make(0.9999992847442627f, 0.9999992847442627f));
  const float2 a = f2_split(p), n = f2_split(t);
  return f2_make(__int_as_float(__float_as_int(a.x) + (__float_as_int(n.x) << 23)),
                 __int_as_float(__float_as_int(a.y) + (__float_as_int(n.y) << 23)));
}

// Lane i of four holds piece k of its row in w[k]: afterwards piece i of row k.
AKV_DEV void transpose4(uint4 (&w)[4]) {
  const int lane = threadIdx.x & 31;
  auto swap = [&](int a, int b, int bit) {
    const bool up = lane & bit;
    const uint4 give = up ? w[a] : w[b];
    const uint4 got = make_uint4(__shfl_xor_sync(~0u, give.x, bit), __shfl_xor_sync(~0u, give.y, bit),
                                 __shfl_xor_sync(~0u, give.z, bit), __shfl_xor_sync(~0u, give.w, bit));
    (up ? w[a] : w[b]) = got;
  };
  swap(0, 1, 1), swap(2, 3, 1), swap(0, 2, 2), swap(1, 3, 2);
}

// ------------------------------------------------------------------ the kernel
template <int D, int G, int LO>
__global__ void __launch_bounds__(ChunkShape<D, G, LO>::THREADS, 1) int4_chunk_kernel(const ChunkParams P) {
  using S = ChunkShape<D, G, LO>;
  constexpr int NQ = S::NQ, TK = S::TK, ROWS = S::ROWS;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  // the swizzle goes by the address: tiles start on 1 KB
  unsigned char* smem = smem_raw + (1024 - (smem_u32(smem_raw) & 1023)) % 1024;
  int* s_ex = reinterpret_cast<int*>(smem + S::OFF_EX);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
  // per query tile: queries there; [buffer] scores, weights there; P V done.  Rings: [slot] filled, free
  uint64_t *q_ready = bars, *pv_done = bars + 2, *s_full = bars + 4, *p_ready = bars + 8;
  uint64_t *k_full = bars + 12, *k_free = bars + 15, *v_full = bars + 18, *v_free = bars + 21;
  uint64_t *raw_full = bars + 24, *raw_free = bars + 32, *drained = bars + 40, *o_full = bars + 41;  // raw: K's slots, V's slots
  int* s_len = reinterpret_cast<int*>(smem + S::OFF_ROWS);
  int* s_new = s_len + P.R;
  int* s_pref = s_new + P.R;
  __shared__ uint32_t s_tmem;
  __shared__ int s_scan[S::THREADS / 32];
  __shared__ ChunkList s_list;
  __shared__ ChunkPos s_begin;

  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int H = P.c.kv_heads, rep = P.Hq / H, entries = P.R * P.tiles;

  if (t == 0) {
    for (int k = 0; k < 2; ++k) {
      mbar_init(q_ready + k, 128);
      mbar_init(pv_done + k, 1);
      mbar_init(o_full + k, 1);
    }
    for (int k = 0; k < 3; ++k) {
      mbar_init(v_full + k, 128);
      mbar_init(v_free + k, NQ);
      mbar_init(k_full + k, 128);
      mbar_init(k_free + k, NQ);
    }
    for (int k = 0; k < 4; ++k) {
      mbar_init(s_full + k, 1);
      mbar_init(p_ready + k, 128);
    }
    for (int k = 0; k < 8; ++k) {
      mbar_init(raw_full + k, 1);
      mbar_init(raw_free + k, 128);
    }
    mbar_init(drained, 1);
    mbar_init(drained + 3, 1);
    fence_mbar_init();
    P.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  // ---- lengths; prefix sums of the entries' weights (tiles and set-up)
  for (int r = t; r < P.R; r += S::THREADS) {
    const Int4Row row = int4_row(P.c, P.rows, P.n_new, P.row0 + r, P.M, P.status);
    s_len[r] = row.len;
    s_new[r] = row.n_new;
  }
  __syncthreads();
  {
    int base = 0;
    for (int e0 = 0; e0 < entries; e0 += S::THREADS) {
      const int e = e0 + t;
      int x = 0;
      if (e < entries) {
        x = chunk_tiles<TK, ROWS>(s_len[e / P.tiles], s_new[e / P.tiles], rep, e % P.tiles);
        if (x) x += kChunkSetup;
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(~0u, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) s_scan[warp] = x;
      __syncthreads();
      int before = base;
#pragma unroll
      for (int w = 0; w < S::THREADS / 32; ++w) {
        if (w < warp) before += s_scan[w];
        base += s_scan[w];
      }
      if (e < entries) s_pref[e + 1] = before + x;
      __syncthreads();
    }
    if (t == 0) {
      s_pref[0] = 0;
      const int total = base * H;
      int share = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
      if (share < 2 + kChunkSetup) share = 2 + kChunkSetup;
      const int begin = static_cast<int>(min(static_cast<int64_t>(share) * blockIdx.x, static_cast<int64_t>(total)));
      s_list = ChunkList{s_len, s_new, s_pref, share, total - begin > share ? begin + share : total};
      s_begin = chunk_at(P, s_list, begin);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;

  // ---- entries without any visible token: zero output
  for (int u = blockIdx.x; u < entries * H; u += gridDim.x) {
    const int e = u / H, h = u % H, i = P.row0 + e / P.tiles;
    if (s_pref[e + 1] != s_pref[e]) continue;
    for (int n = warp; n < ROWS; n += S::THREADS / 32) {
      const int rr = e % P.tiles * ROWS + n, m = rr / rep, hq = h * rep + rr - m * rep;
      if (m >= P.M) break;
      uint16_t* o = P.out + i * P.o_sr + hq * P.o_sh + m * P.o_sm;
      for (int c = lane; c < D; c += 32) o[c] = 0;
      if (P.lse && lane == 0) P.lse[(static_cast<int64_t>(i) * P.Hq + hq) * P.M + m] = -INFINITY;
    }
  }

  ChunkPos walk = s_begin;
  auto next = [&](ChunkPart& x) { return chunk_next<ROWS>(P, s_list, walk, x); };
  bool ok = true;  // no bounded wait of this warp has run out
  auto wait = [&](uint64_t* bar, uint32_t phase) {  // by whole warps
    if (ok) ok = __all_sync(~0u, mbar_wait(bar, phase, P.status));
    return ok;
  };

  if (warp < S::SOFT) {
    // ================================================================ softmax
    if constexpr (S::SPLIT) regs_up<S::R_SOFT>();
    
    const int qt = warp >> 2, r = t & 127;        // query tile, row = TMEM lane
    unsigned char* q_tile = smem + qt * S::QB;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lanes + S::T_O + qt * D;

    // The warp's 32 query rows into shared memory, as fp16; their exponents for
    // later.  A load takes 64 bytes of 8 rows, a store 8 rows of a column block.
    auto load_q = [&](const ChunkPart& x) {
      constexpr int IT = D / 32;             // loads of a row
      const int piece = lane >> 3;
      constexpr int GR = IT < 4 ? 4 : 16 / IT;  // groups of 8 rows in flight
#pragma unroll 1
      for (int g0 = 0; g0 < 4; g0 += GR) {
        uint4 va[GR][IT];
#pragma unroll
        for (int g = 0; g < GR; ++g) {
          const int rr = x.row + qt * 128 + (warp & 3) * 32 + (g0 + g) * 8 + (lane & 7);
          const int m = chunk_token(P, rr), hq = x.h * rep + rr - m * rep;
          const uint16_t* src = P.q + x.i * P.q_sr + hq * P.q_sh + m * P.q_sm + piece * 8;
          if (m >= x.n_new || g0 + g > 3) {
#pragma unroll
            for (int k = 0; k < IT; ++k) va[g][k] = make_uint4(0u, 0u, 0u, 0u);
          } else if (P.q16) {
#pragma unroll
            for (int k = 0; k < IT; ++k) va[g][k] = *reinterpret_cast<const uint4*>(src + 32 * k);
          } else {
#pragma unroll
            for (int k = 0; k < IT; ++k) {
              uint32_t w[4];
#pragma unroll
              for (int c = 0; c < 4; ++c)
                w[c] = src[32 * k + 2 * c] | static_cast<uint32_t>(src[32 * k + 2 * c + 1]) << 16;
              va[g][k] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
#pragma unroll
        for (int g = 0; g < GR; ++g) {
        if (g0 + g > 3) break;
        const int row = (warp & 3) * 32 + (g0 + g) * 8 + (lane & 7);
        const uint4(&v)[IT] = va[g];
        uint32_t top = 0u;  // largest magnitude of the row, as the 15 bits of the type
#pragma unroll
        for (int k = 0; k < IT; ++k)
          top = __vmaxu2(__vmaxu2(top, v[k].x & 0x7FFF7FFFu),
                         __vmaxu2(v[k].y & 0x7FFF7FFFu, __vmaxu2(v[k].z & 0x7FFF7FFFu, v[k].w & 0x7FFF7FFFu)));
        top = max(top & 0xFFFFu, top >> 16);
        top = max(top, __shfl_xor_sync(~0u, top, 8));
        top = max(top, __shfl_xor_sync(~0u, top, 16));
        const bool bad = top >= (LO ? 0x7C00u : 0x7F80u);  // no softmax: computed as zeros, NaN at the end
        int ex = 0;  // bf16: 2^ex brings the largest into [2^9, 2^10)
        if (!LO && top && !bad) ex = 9 - (static_cast<int>(top >> 7) - 127);
        ex = ex > 120 ? 120 : (ex < -120 ? -120 : ex);
        const float up = __int_as_float((127 + ex) << 23) * (P.scale < 0.f ? -1.f : 1.f);
        const uint32_t flip = P.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int k = 0; k < IT; ++k) {
          uint32_t w[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if constexpr (!LO)
              w[c] = pack_h2(__uint_as_float(w[c] << 16) * up, __uint_as_float(w[c] & 0xFFFF0000u) * up);
            else
              w[c] ^= flip;
            if (bad) w[c] = 0u;
          }
          *reinterpret_cast<uint4*>(q_tile + (k >> 1) * (128 * 128) + row * 128 + (((4 * (k & 1) + piece) ^ (lane & 7)) * 16)) =
              make_uint4(prmt(w[0], w[2], 0x5410), prmt(w[0], w[2], 0x7632), prmt(w[1], w[3], 0x5410),
                         prmt(w[1], w[3], 0x7632));
        }
        if (piece == 0) s_ex[qt * 128 + row] = bad ? INT32_MAX : ex;
        }
      }
      fence_proxy_async_shared();
      __syncwarp();
      mbar_arrive(q_ready + qt);
    };

    uint32_t ph_s = 0, ph_o = 0, pv = 0;  // the buffers' phases; P V's so far
    ChunkPos here = walk;  // where the part at hand is decoded from: its fields are not kept over the tiles
    bool more;
    {
      ChunkPart u;
      more = next(u);
      if (more) load_q(u);
    }
    while (more && ok) {
      int see, tiles;  // tokens that the row sees, from the part's first; tiles
      bool any;        // it sees one
      {
        ChunkPart u;
        ChunkPos w = here;
        chunk_next<ROWS>(P, s_list, w, u);
        const int m = chunk_token(P, u.row + qt * 128 + r);
        see = (m < u.n_new ? u.len - u.n_new + m + 1 : 0);
        tiles = u.t1 - u.t0;
        see -= u.t0 * TK;  // from the part's first token
        any = m < u.n_new && u.len - u.n_new + m + 1 > 0;
      }
      const int ex = s_ex[qt * 128 + r];
      const bool bad = ex == INT32_MAX;
      // log2 e * scale in units of S; never 0, so that -inf stays -inf
      const float sl2 = fmaxf(ldexpf(fabsf(P.scale) * 1.4426950408889634f, bad ? 0 : -ex), 1e-37f);
      float unit = 0.f, l = 0.f;  // weights are 2^(S sl2 - unit), l their sum
      bool fresh = true;          // no token seen: the unit is not set
      for (int j = 0; j < tiles; ++j) {
        const int buf = j & 1;
        const uint32_t tS = tmem + lanes + S::T_S + (2 * qt + buf) * TK;
        if (!wait(s_full + 2 * qt + buf, ph_s >> buf & 1)) break;
        ph_s ^= 1u << buf;
        tc_fence_after();
        const int n = see - j * TK;  // tokens of the tile that the row sees
        const bool full = __all_sync(~0u, n >= TK);
        uint32_t hi[TK / 32][16], lo[LO ? TK / 32 : 1][16];
        float part;
        for (bool moved = false;; moved = true) {
          const uint64_t sl22 = f2_make(sl2, sl2), un2 = f2_make(-unit, -unit);
          uint64_t sum = 0;
#pragma unroll
          for (int c = 0; c < TK / 32; ++c) {
            float x[32];
            tmem_ld32(tS + c * 32, x);
            tmem_wait_ld();
            if (!full) {
#pragma unroll
              for (int k = 0; k < 32; ++k) x[k] = c * 32 + k < n ? x[k] : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              uint64_t y2 = f2_fma(f2_make(x[2 * k], x[2 * k + 1]), sl22, un2);
              float2 y = f2_split(y2);
              if (k % 4 < S::POLY) {
                y2 = exp2_fma(y2);
                y = f2_split(y2);
              } else {
                y.x = fast_exp2(y.x);
                y.y = fast_exp2(y.y);
                y2 = f2_make(y.x, y.y);
              }
              sum = f2_add(sum, y2);
              hi[c][k] = pack_h2(y.x, y.y);
              if constexpr (LO) {
                const float2 b = __half22float2(u32_as_h2(hi[c][k]));
                lo[c][k] = pack_h2(y.x - b.x, y.y - b.y);
              }
            }
          }
          const float2 s2 = f2_split(sum);
          part = s2.x + s2.y;
          if (moved || __all_sync(~0u, part <= kChunkMost && !(fresh && n > 0))) break;
          // ---- the unit moves
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < TK / 16; ++c) {
            float x[16];
            tmem_ld16(tS + c * 16, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) mx = fmaxf(mx, c * 16 + k < n ? x[k] : -INFINITY);
          }
          const float to = fmaf(mx, sl2, -kChunkTop);
          float f = 1.f;
          if (mx > -INFINITY && (fresh || to > unit)) {
            f = fresh ? 0.f : exp2f(unit - to);
            unit = to;
            l *= f;
            fresh = false;
          }
          if (j > 0) {
            wait(pv_done + qt, (pv + j - 1) & 1);  // the last tile's P V may still run; those before are done
            tc_fence_after();
#pragma unroll 1
            for (int k = 0; k < D / 16; ++k) {
              float o[16];
              tmem_ld16(tO + k * 16, o);
              tmem_wait_ld();
              uint32_t w[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(o[i] * f);
              tmem_st16u(tO + k * 16, w);
            }
          }
        }
        l += part;
#pragma unroll
        for (int c = 0; c < TK / 32; ++c) {
          if constexpr (LO) {
            tmem_st16u(tS + c * 32, hi[c]);
            tmem_st16u(tS + c * 32 + 16, lo[c]);
          } else {
            tmem_st16u(tS + c * 16, hi[c]);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(p_ready + 2 * qt + buf);
      }
      if (fresh) l = 0.f;
      pv += tiles;
      ChunkPart u;
      chunk_next<ROWS>(P, s_list, here, u);
      here = walk;
      {
        ChunkPart nx;
        more = next(nx);
        if (more && ok) load_q(nx);  // every S of this part is out: its queries are done with
      }
      const int rr = u.row + qt * 128 + r, m = chunk_token(P, rr), hq = u.h * rep + rr - m * rep;
      if (!wait(o_full + qt, ph_o)) break;
      ph_o ^= 1;
      tc_fence_after();
      const bool whole = u.t0 == 0 && u.t1 == u.tiles;
      const bool in = m < P.M;
      const int64_t row = static_cast<int64_t>(u.i) * P.o_sr + static_cast<int64_t>(hq) * P.o_sh + m * P.o_sm;
      const float nan = bad && any ? NAN : 0.f;
      const float inv = 1.f / l;
      const bool dead = l == 0.f;  // sees nothing
      const int slot = 2 * blockIdx.x + (u.t0 == 0 ? 1 : 0);
      float* part = P.part + static_cast<int64_t>(slot) * ROWS * D + (qt * 128 + r) * 4;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
        if (whole) {
          uint4 w[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = dead ? 0.f : o[8 * b + (k & 3) * 2 + (k >> 2)] * inv + nan;
            w[b] = make_uint4(pack_elems<!LO>(v[0], v[1]), pack_elems<!LO>(v[2], v[3]), pack_elems<!LO>(v[4], v[5]),
                              pack_elems<!LO>(v[6], v[7]));
          }
          if (P.o16) {
            // four lanes exchange, so that a store takes 64 bytes of 8 rows
            transpose4(w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int64_t at = __shfl_sync(~0u, in ? row : -1, (lane & 28) + k);  // lane k's row
              if (at >= 0) *reinterpret_cast<uint4*>(P.out + at + c * 32 + (lane & 3) * 8) = w[k];
            }
          } else if (in) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const uint32_t x[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
              for (int k = 0; k < 8; ++k) P.out[row + c * 32 + b * 8 + k] = static_cast<uint16_t>(x[k / 2] >> (16 * (k & 1)));
            }
          }
        } else {
#pragma unroll
          for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
              *reinterpret_cast<float4*>(part + static_cast<int64_t>((c * 4 + b) * 2 + hf) * ROWS * 4) =
                  make_float4(o[8 * b + hf] + nan, o[8 * b + 2 + hf] + nan, o[8 * b + 4 + hf] + nan, o[8 * b + 6 + hf] + nan);
        }
      }
      if (whole) {
        if (in && P.lse)
          P.lse[(static_cast<int64_t>(u.i) * P.Hq + hq) * P.M + m] =
              dead ? -INFINITY : (unit + log2f(l)) * 0.6931471805599453f + nan;
      } else {
        P.ml[static_cast<int64_t>(slot) * ROWS + qt * 128 + r] = make_float2(fresh ? -INFINITY : unit, l + nan);
        if (t == 0 && u.t0 == 0) P.meta[blockIdx.x] = make_int4(u.e, u.h, (u.unit_end - 1) / s_list.share, 1);
      }
      tc_fence_before();
    }
  } else if (warp < S::SOFT + 8) {
    // ================================================================ values
    if constexpr (S::SPLIT) regs_down<S::R_VAL>();
    const int r = (t & 127) % TK, part = (t & 127) / TK;  // token of the tile, channels part * CH on
    const int page = r / kBlockTokens, slot = r % kBlockTokens;
    constexpr int NEXT = TK * 128;  // from 64 channels to the next
    const int x = (r & 7) * 16;
    // a tile of K or V: raw codes and pairs -> rows of fp16
    auto unpack = [&](const unsigned char* raw, unsigned char* dst, bool there, auto two) {
      constexpr bool TWO = decltype(two)::value;
      const unsigned char* code = raw + page * (kBlockTokens * D / 2) + slot * (D / 2) + part * (S::CH / 2);
      const uint32_t* pair = reinterpret_cast<const uint32_t*>(raw + S::RAW_CODES) + r * G;
      dst += r * 128;
      // the lanes start on different pieces, so that neither their loads nor their stores meet
#pragma unroll 1
      for (int k = 0; k < S::PIECES; ++k) {
        const int p = (k + (r >> 1)) % S::PIECES, ch = part * S::CH + p * 32;
        const uint4 w = there ? lds_v4(code + p * 16) : make_uint4(0u, 0u, 0u, 0u);
        unsigned char* at = dst + (ch >> 6) * NEXT;
        const int blk = (ch & 32) * 2;
        if constexpr (D / G >= 32) {
          const uint32_t sz = there ? pair[ch / (D / G)] : 0u;
          if (__any_sync(~0u, far_values(sz, TWO ? 8192.f : 65000.f))) store_piece<TWO, true>(w, sz, at, blk, x, S::VB);
          else store_piece<TWO, false>(w, sz, at, blk, x, S::VB);
        } else {  // two groups of 16 channels
          const uint32_t s0 = there ? pair[ch / 16] : 0u, s1 = there ? pair[ch / 16 + 1] : 0u;
          if (__any_sync(~0u, far_values(s0, TWO ? 8192.f : 65000.f) || far_values(s1, TWO ? 8192.f : 65000.f)))
            store_halves<TWO, true>(w, s0, s1, at, blk, x, S::VB);
          else
            store_halves<TWO, false>(w, s0, s1, at, blk, x, S::VB);
        }
      }
    };
    const int kv = (warp - S::SOFT) >> 2;  // 0: K, 1: V
    const int slots = kv ? S::VS : S::KS;
    uint64_t *full = kv ? v_full : k_full, *freed = kv ? v_free : k_free;
    int at = 0, rs = 0;
    uint32_t ph_raw = 0, ph = 1;  // a fresh barrier passes a wait for the phase before its first
    ChunkPart u;
    while (ok && next(u)) {
      for (int j = u.t0; j < u.t1; ++j) {
        const bool there = j * TK + r < u.len;
        const int slot_raw = kv * S::RS + rs;
        const unsigned char* raw = smem + S::OFF_RAW + slot_raw * S::RAW;
        if (!wait(raw_full + slot_raw, ph_raw) || !wait(freed + at, ph)) break;
        if (kv) unpack(raw, smem + S::OFF_V + at * S::VB, there, std::false_type());
        else unpack(raw, smem + S::OFF_K + at * S::KB, there, std::bool_constant<LO != 0>());
        mbar_arrive(raw_free + slot_raw);
        fence_proxy_async_shared();
        mbar_arrive(full + at);
        if (++at == slots) at = 0, ph ^= 1;
        if (++rs == S::RS) rs = 0, ph_raw ^= 1;
      }
    }
  } else {
    // ================================================================ MMA
    if constexpr (S::SPLIT) regs_down<S::R_MMA>();
    if (warp < S::SOFT + 8 + NQ) {
    // a warp for each query tile
    const int q = warp - S::SOFT - 8;
    const uint32_t lead = elect_one();
    constexpr uint32_t NEXT = TK * 128;  // from 64 channels to the next
    constexpr uint32_t HI = desc_hi_sw128(1024);
    constexpr uint32_t IDESC_S = instr_desc(128, TK, 0);  // S = Q K^T: B (= K) K-major
    constexpr uint32_t IDESC_O = instr_desc(128, D, 1);   // O = P V: B (= V) MN-major
    const uint32_t base = smem_u32(smem);
    int ks = 0, vs = 0;
    uint32_t kph = 0, vph = 0, ph_p = 0, ph_q = 0;
    const uint32_t q_tile = desc_lo(base + q * S::QB, 16);
    const uint32_t tO = tmem + S::T_O + q * D;
    // S of the next tile into its buffer
    auto qk = [&](int buf) {
      const uint32_t b = desc_lo(base + S::OFF_K + ks * S::KB, 16);
      const uint32_t d = tmem + S::T_S + (2 * q + buf) * TK;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t ak = q_tile + ((k >> 2) * (128 * 128) + (k & 3) * 32) / 16, bk = b + ((k >> 2) * NEXT + (k & 3) * 32) / 16;
        umma_ss<HI, HI, IDESC_S>(d, ak, bk, k > 0 ? 1u : 0u, lead);
        if constexpr (LO) umma_ss<HI, HI, IDESC_S>(d, ak, bk + S::VB / 16, 1u, lead);
      }
      umma_commit(s_full + 2 * q + buf, lead);
      umma_commit(k_free + ks, lead);
      if (++ks == S::KS) ks = 0, kph ^= 1;
    };
    ChunkPart u;
    while (ok && next(u)) {
      wait(q_ready + q, ph_q);
      ph_q ^= 1;
      const int tiles = u.t1 - u.t0;
      for (int j = 0; j < 2 && j < tiles; ++j) {
        if (!wait(k_full + ks, kph)) break;
        tc_fence_after();
        qk(j);
      }
      for (int j = 0; j < tiles; ++j) {
        const int buf = j & 1;
        const bool again = j + 2 < tiles;
        // what is there early first: the weights are what takes its time
        if (!wait(v_full + vs, vph) || (again && S::KS > 1 && !wait(k_full + ks, kph)) ||
            !wait(p_ready + 2 * q + buf, ph_p >> buf & 1))
          break;
        ph_p ^= 1u << buf;
        tc_fence_after();
        const uint32_t v = desc_lo(base + S::OFF_V + vs * S::VB, NEXT);
        const uint32_t tP = tmem + S::T_S + (2 * q + buf) * TK;
#pragma unroll
        for (int k = 0; k < TK / 16; ++k) {
          const uint32_t on = j > 0 || k > 0 ? 1u : 0u;
          if constexpr (LO) {
            const uint32_t p = tP + 32 * (k >> 1) + 8 * (k & 1);
            umma_ts<HI, IDESC_O>(tO, p, v + k * 128, on, lead);
            umma_ts<HI, IDESC_O>(tO, p + 16, v + k * 128, 1u, lead);
          } else {
            umma_ts<HI, IDESC_O>(tO, tP + 8 * k, v + k * 128, on, lead);
          }
        }
        umma_commit(pv_done + q, lead);
        umma_commit(v_free + vs, lead);
        if (j + 1 == tiles) umma_commit(o_full + q, lead);
        if (++vs == S::VS) vs = 0, vph ^= 1;
        if (again) {  // P is read before this overwrites it: a thread's MMAs run in order
          if (S::KS == 1) {
            if (!wait(k_full + ks, kph)) break;
            tc_fence_after();
          }
          qk(buf);
        }
      }
    }
    if (!ok) {  // a wait ran out: see what was issued end before the tensor memory goes
      umma_commit(drained + 3 * q, lead);
      mbar_wait(drained + 3 * q, 0, P.status);
    }
    } else if (warp == S::SOFT + 8 + NQ) {
      // ============================================================== pages
      constexpr Int4Layout L = int4_layout(D, G);
      constexpr int CODES = kBlockTokens * D / 2, PAIRS = kBlockTokens * G * 4;
      uint32_t ph = 1;  // a fresh barrier passes a wait for the phase before its first
      int rs = 0;
      bool flying = false;
      ChunkPart u;
      while (ok && next(u)) {
        const int seq = P.rows ? __ldg(P.rows + u.i) : u.i;  // in range: it has tiles
        const int32_t* table = P.c.table + seq * P.c.table_stride;
        const int pages = (u.len + kBlockTokens - 1) / kBlockTokens;
        auto page_of = [&](int tile) -> int {  // a page for each of the first lanes; -1: none
          const int b = tile * S::PAGES + lane;
          return lane < S::PAGES && b < pages ? __ldg(table + b) : -1;
        };
        int p = page_of(u.t0);
        for (int j = u.t0; j < u.t1; ++j) {
          const int b = j * S::PAGES + lane;
          const bool on = lane < S::PAGES && b < pages;
          if (on && (p < 0 || p >= P.c.n_pages)) {
            set_status(P.status, AKV_ERR_SHAPE);
            p = 0;
          }
          const uint8_t* rec = P.c.pool + p * P.c.page_stride + u.h * P.c.head_stride;
          const uint32_t bytes = __popc(__ballot_sync(~0u, on)) * (CODES + PAIRS);
          const int ahead = j + 1 < u.t1 ? page_of(j + 1) : 0;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int at = v * S::RS + rs;
            if (!wait(raw_free + at, ph)) break;
            unsigned char* raw = smem + S::OFF_RAW + at * S::RAW;
            if (lane == 0) mbar_arrive_expect_tx(raw_full + at, bytes);
            __syncwarp();
            if (on) {
              tma_load_1d(raw + lane * CODES, rec + (v ? L.vc : L.kc), CODES, raw_full + at);
              tma_load_1d(raw + S::RAW_CODES + lane * PAIRS, rec + (v ? L.vp : L.kp), PAIRS, raw_full + at);
            }
            flying = true;
          }
          if (!ok) break;
          if (++rs == S::RS) rs = 0, ph ^= 1;
          p = ahead;
        }
      }
      if (!ok && flying)  // a wait ran out: see the copies in flight land
        for (int v = 0; v < 2 * S::RS; ++v) {
          mbar_wait(raw_full + v, ph, P.status);
          mbar_wait(raw_full + v, ph ^ 1, P.status);
        }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// ------------------------------------------------------------------ joining parts
// Block (c, k): 32 query rows of the unit whose first part CTA c holds; its
// parts lie in the slots 2c + 1, 2 (c + 1), ..., 2 last.
template <int D, int ROWS>
__global__ void __launch_bounds__(128) int4_chunk_join_kernel(const ChunkParams P) {
  const int4 meta = P.meta[blockIdx.x];
  if (!meta.w) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int H = P.c.kv_heads, rep = P.Hq / H;
  const int n = blockIdx.y * 32 + lane;  // query row of the tile
  const int e = meta.x, i = P.row0 + e / P.tiles;
  const int rr = e % P.tiles * ROWS + n, m = rr / rep, hq = meta.y * rep + rr - m * rep;
  const int c0 = blockIdx.x, parts = meta.z - c0 + 1;
  auto slot = [&](int s) -> int64_t { return s == 0 ? 2 * c0 + 1 : 2 * (c0 + s); };
  float top = -INFINITY;
  for (int s = 0; s < parts; ++s) top = fmaxf(top, __ldcg(&P.ml[slot(s) * ROWS + n].x));
  float L = 0.f;
  for (int s = 0; s < parts; ++s) {
    const float2 x = __ldcg(&P.ml[slot(s) * ROWS + n]);
    L += x.x == -INFINITY ? x.y : exp2f(x.x - top) * x.y;
  }
  const bool dead = L == 0.f, in = m < P.M;
  const float inv = 1.f / L;
  for (int b = warp; b < D / 8; b += 4) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < parts; ++s) {
      const float x = __ldcg(&P.ml[slot(s) * ROWS + n].x);
      const float f = x == -INFINITY ? 0.f : exp2f(x - top);
      const float4* at = reinterpret_cast<const float4*>(P.part) + slot(s) * ROWS * (D / 4) + n;
      const float4 a = __ldcg(at + static_cast<int64_t>(2 * b) * ROWS), c = __ldcg(at + static_cast<int64_t>(2 * b + 1) * ROWS);
      // channels 0..3 and 4..7 of the block
      v[0] = fmaf(f, a.x, v[0]), v[1] = fmaf(f, a.y, v[1]), v[2] = fmaf(f, a.z, v[2]), v[3] = fmaf(f, a.w, v[3]);
      v[4] = fmaf(f, c.x, v[4]), v[5] = fmaf(f, c.y, v[5]), v[6] = fmaf(f, c.z, v[6]), v[7] = fmaf(f, c.w, v[7]);
    }
    if (!in) continue;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = dead ? 0.f : v[2 * k] * inv, c = dead ? 0.f : v[2 * k + 1] * inv;
      w[k] = P.bf16 ? pack_elems<true>(a, c) : pack_elems<false>(a, c);
    }
    uint16_t* dst = P.out + i * P.o_sr + hq * P.o_sh + m * P.o_sm + b * 8;
    if (P.o16) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) dst[k] = static_cast<uint16_t>(w[k / 2] >> (16 * (k & 1)));
    }
  }
  if (in && P.lse && warp == 0)
    P.lse[(static_cast<int64_t>(i) * P.Hq + hq) * P.M + m] = dead ? -INFINITY : (top + log2f(L)) * 0.6931471805599453f;
}

template <int D, int G, int LO>
static int chunk_launch(const ChunkParams& P, cudaStream_t st) {
  using S = ChunkShape<D, G, LO>;
  const int smem = S::smem(P.R, P.R * P.tiles);
  if (!ensure_dynamic_smem<int4_chunk_kernel<D, G, LO>>(smem)) return AKV_ERR_LAUNCH;
  int4_chunk_kernel<D, G, LO><<<kChunkSMs, S::THREADS, smem, st>>>(P);
  int4_chunk_join_kernel<D, S::ROWS><<<dim3(kChunkSMs, S::ROWS / 32), 128, 0, st>>>(P);
  return cudaGetLastError() == cudaSuccess ? AKV_OK : AKV_ERR_LAUNCH;
}

template <int D>
static int chunk_dispatch(const ChunkParams& P, cudaStream_t st) {
  switch (D / P.c.group) {
    case 1: return P.bf16 ? chunk_launch<D, 1, 0>(P, st) : chunk_launch<D, 1, 1>(P, st);
    case 2: return P.bf16 ? chunk_launch<D, 2, 0>(P, st) : chunk_launch<D, 2, 1>(P, st);
    default: return P.bf16 ? chunk_launch<D, 4, 0>(P, st) : chunk_launch<D, 4, 1>(P, st);
  }
}

int int4_chunk_64(const ChunkParams& P, cudaStream_t st);
int int4_chunk_128(const ChunkParams& P, cudaStream_t st);
int int4_chunk_256(const ChunkParams& P, cudaStream_t st);

}  // namespace akv
